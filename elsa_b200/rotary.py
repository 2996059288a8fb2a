"""Rotary positions for the q and k of a decoder layer: the angles of each token's position, applied by one launch
(csrc/rotary.cu) in front of `twopass_attention`, `shared_prefix_attention` or `differential_attention`.

The reference has no position encoding of this kind; names and checks follow this package's attention operators.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Literal, NamedTuple, Optional, Union

import torch

from . import _lib
from .attention import _DeviceScope, _empty_like_layout

_MAX_ROTARY_DIM = 256
_MAX_HEAD_DIM = 1024
_MAX_SIZE = (1 << 30) - 1


def _check_sizes(*tensors):
    """No axis longer than the kernels' 32-bit indices count."""
    for t in tensors:
        if any(n > _MAX_SIZE for n in t.shape):
            raise ValueError(f"an axis of more than {_MAX_SIZE} elements is not supported by the current kernels")


def rotary_frequencies(
    rotary_dim: int,
    *,
    base: float = 10000.0,
    scaling: Literal["none", "linear", "ntk", "yarn"] = "none",
    factor: float = 1.0,
    original_positions: Optional[int] = None,
    beta_fast: float = 32.0,
    beta_slow: float = 1.0,
    device: Optional[torch.device] = None,
) -> tuple[torch.Tensor, float]:
    """The rotary_dim / 2 frequencies base^(-2i / rotary_dim) in 64 bits, and the magnitude that goes with them.

    `scaling` stretches them for contexts `factor` times as long as the trained one:
      linear  every frequency divided by `factor` (positions interpolated);
      ntk     the base multiplied by factor^(R / (R - 2)): the fastest pair keeps its frequency, the slowest is divided by
              `factor`;
      yarn    pairs that turn more than `beta_fast` times within `original_positions` keep their frequency, those that turn
              less than `beta_slow` times are divided by `factor`, linearly blended in between (over the pair's index); the
              magnitude is 0.1 ln(factor) + 1.
    Both go to `rotary_embedding`; a program makes them once."""
    rotary_dim = int(rotary_dim)
    if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > _MAX_ROTARY_DIM:
        raise ValueError(f"rotary_dim must be even and between 2 and {_MAX_ROTARY_DIM}")
    if not (math.isfinite(base) and base > 0.0):
        raise ValueError("base must be positive")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError("scaling must be 'none', 'linear', 'ntk', or 'yarn'")
    if not (math.isfinite(factor) and factor >= 1.0):
        raise ValueError("factor must be at least 1")
    index = torch.arange(rotary_dim // 2, dtype=torch.float64)
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("scaling='ntk' needs a rotary_dim of at least 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    frequencies = base ** (-2.0 * index / rotary_dim)
    magnitude = 1.0
    if scaling == "linear":
        frequencies = frequencies / factor
    elif scaling == "yarn":
        if original_positions is None or int(original_positions) <= 0:
            raise ValueError("scaling='yarn' needs original_positions")
        if not beta_fast > beta_slow > 0.0 or base == 1.0:
            raise ValueError("scaling='yarn' needs beta_fast > beta_slow > 0 and a base other than 1")

        def pair_of(turns):     # the (fractional) pair that turns so many times within original_positions
            return rotary_dim * math.log(original_positions / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        low = max(math.floor(pair_of(beta_fast)), 0)
        high = min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        kept = 1.0 - ((index - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        frequencies = frequencies / factor * (1.0 - kept) + frequencies * kept
        magnitude = 0.1 * math.log(factor) + 1.0
    return frequencies.to(device) if device is not None else frequencies, magnitude


def _refuse_transforms(who: str, *tensors):
    """An operator without an autograd function of its own is neither recorded by torch.jit.trace (the trace would hold its memory, not
    its work) nor given a tangent by forward-mode differentiation: it says so."""
    if torch.jit.is_tracing():
        raise RuntimeError(f"{who} cannot be recorded by torch.jit.trace")
    if any(torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{who} has no forward-mode derivative")


def _row_strides(t: torch.Tensor):
    """(batch, head, row) element strides, or None where the D axis is not contiguous."""
    b, h, n, d = t.shape
    s0, s1, s2, s3 = t.stride()
    if d > 1 and s3 != 1:
        return None
    # (an axis of one has no stride that matters: 0 keeps it out of the alignment rule)
    return (s0 if b > 1 else 0, s1 if h > 1 else 0, s2 if n > 1 else 0)


def _overlaps(t: torch.Tensor) -> bool:
    """Whether two rows of a [B, H, N, D] view share memory, as far as its strides tell: axes from the smallest stride up, each
    must step over all that lies below it."""
    reach = int(t.shape[3])
    for stride, size in sorted((int(st), int(sz)) for st, sz in zip(t.stride()[:3], t.shape[:3]) if sz > 1):
        if stride < reach:
            return True
        reach = stride * (size - 1) + reach
    return False


def _meet(q: torch.Tensor, k: torch.Tensor) -> bool:
    """Whether an element of q and one of k share memory, for two [B, H, N, D] views without overlaps of their own (`_overlaps`).  Views
    of one buffer with the same strides, as of a packed projection, are told apart exactly; others count as meeting where the
    ranges of their addresses do."""
    size = q.element_size()
    extent = lambda t: (sum((n - 1) * st for n, st in zip(t.shape[:3], t.stride()[:3])) + int(t.shape[3])) * size
    offset = k.data_ptr() - q.data_ptr()
    if offset >= extent(q) or -offset >= extent(k):
        return False
    axes = [(1, 1 - int(k.shape[3]), int(q.shape[3]) - 1)]               # (stride, least and most that an index of q is ahead of k's)
    for sq, sk, nq, nk in zip(q.stride()[:3], k.stride()[:3], q.shape[:3], k.shape[:3]):
        if nq > 1 and nk > 1 and sq != sk:
            return True
        if nq > 1 or nk > 1:
            axes.append((sq if nq > 1 else sk, 1 - nk, nq - 1))
    axes.sort(reverse=True)

    def reaches(rest, axes):
        if not axes:
            return rest == 0
        (stride, low, high), below = axes[0], axes[1:]
        least, most = (sum(x[0] * x[i] for x in below) for i in (1, 2))
        first, last = max(low, -((most - rest) // stride)), min(high, (rest - least) // stride)
        return any(reaches(rest - e * stride, below) for e in range(first, last + 1))

    return offset % size != 0 or reaches(offset // size, axes)


def _launch(q, k, q_out, k_out, frequencies, positions, magnitude, interleaved, inverse):
    b, h, n, d = q.shape
    args_k = (None, None, None, 0)
    if k is not None:
        args_k = (k.data_ptr(), k_out.data_ptr(), (ctypes.c_int64 * 6)(*_row_strides(k), *_row_strides(k_out)), int(k.shape[1]))
    args_p = (None, 0, 0, 0)
    if positions is not None:
        args_p = (positions.data_ptr(), positions.element_size(), int(positions.stride(0)) if positions.dim() == 2 and positions.shape[0] > 1 else 0,
                  int(positions.stride(-1)))
    with _DeviceScope(q.device):
        rc = _lib.load().elsa_rotary(
            q.data_ptr(), q_out.data_ptr(), (ctypes.c_int64 * 6)(*_row_strides(q), *_row_strides(q_out)), h, *args_k,
            frequencies.data_ptr(), *args_p, magnitude, _lib.dtype_code(q.dtype), b, n, d, 2 * int(frequencies.shape[0]),
            int(interleaved), int(inverse), _lib.raw_stream(q.device))
    _lib.check(rc, "elsa_rotary")


def _rotate(q, k, frequencies, positions, magnitude, interleaved, inverse=False, inplace=False):
    if q.numel() == 0:          # (then k has no rows either, or only q has no heads: nothing that could be turned together)
        if k is None or k.numel() == 0:
            return (q, k) if inplace else (torch.empty_like(q), None if k is None else torch.empty_like(k))
        turned, _ = _rotate(k, None, frequencies, positions, magnitude, interleaved, inverse, inplace)
        return (q if inplace else torch.empty_like(q)), turned
    if k is not None and k.numel() == 0:
        turned, _ = _rotate(q, None, frequencies, positions, magnitude, interleaved, inverse, inplace)
        return turned, (k if inplace else torch.empty_like(k))
    if inplace:
        q_out, k_out = q, k
    else:
        q = q if _row_strides(q) is not None else q.contiguous()
        q_out = _empty_like_layout(q, q.stride())
        k_out = None
        if k is not None:
            k = k if _row_strides(k) is not None else k.contiguous()
            k_out = _empty_like_layout(k, k.stride())
    _launch(q, k, q_out, k_out, frequencies, positions, magnitude, interleaved, inverse)
    return q_out, k_out


def _check_saved(t, like_shape, dtype, device):
    """Saved-tensor hooks may return the values in another memory layout, but nothing else."""
    if tuple(t.shape) != tuple(like_shape) or t.dtype != dtype or t.device != device:
        raise RuntimeError("a saved tensor came back from its unpack hook with another shape, dtype or device")
    return t


def _once_differentiable(backward):
    """A backward whose results have no gradients of their own, and say so when one is asked for."""

    @functools.wraps(backward)
    def wrapper(ctx, *grads):
        record = torch.is_grad_enabled()
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not record:
            return out
        error = torch._C._functions.DelayedError(b"this gradient is not differentiable twice", len(out))
        return error(*(None if t is None else t.detach().requires_grad_() for t in out))

    return wrapper


class _RotaryAutograd(torch.autograd.Function):
    """The gradient of a rotation is the rotation back: nothing but positions and frequencies is kept."""

    @staticmethod
    def forward(ctx, q, k, frequencies, positions, magnitude, interleaved):
        ctx.save_for_backward(frequencies, *(() if positions is None else (positions,)))
        ctx.kept = [(t.shape, t.dtype, t.device) for t in (frequencies, *(() if positions is None else (positions,)))]
        ctx.magnitude, ctx.interleaved = magnitude, interleaved
        ctx.set_materialize_grads(False)
        q_out, k_out = _rotate(q, k, frequencies, positions, magnitude, interleaved)
        return q_out if k is None else (q_out, k_out)

    @staticmethod
    @_once_differentiable
    def backward(ctx, dq, dk=None):
        frequencies, *rest = (_check_saved(t, *kept) for t, kept in zip(ctx.saved_tensors, ctx.kept))
        frequencies, positions = frequencies.contiguous(), rest[0] if rest else None
        back = (frequencies, positions, ctx.magnitude, ctx.interleaved, True)
        if not ctx.needs_input_grad[0]:
            dq = None
        if not ctx.needs_input_grad[1]:
            dk = None
        if dq is not None and dk is not None:
            dq, dk = _rotate(dq, dk, *back)
        elif dq is not None:
            dq, _ = _rotate(dq, None, *back)
        elif dk is not None:
            dk, _ = _rotate(dk, None, *back)
        return dq, dk, None, None, None, None


def rotary_embedding(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    frequencies: torch.Tensor,
    *,
    positions: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    magnitude: float = 1.0,
    inplace: bool = False,
) -> Union[torch.Tensor, tuple[torch.Tensor, torch.Tensor]]:
    """q and k with the first R = 2 * len(frequencies) dimensions of every head turned by their token's position.

    q: [B, H, N, D], k: [B, Hkv, N, D] (its own number of heads) or None; fp16, bf16 or fp32, any strides (rows of D contiguous
    elements are read in place: views of a packed projection need no copy).  frequencies: [R / 2], fp64, from
    `rotary_frequencies`, with its `magnitude`.  positions: int32 or int64, [N] or [B, N], any values; None: 0 .. N-1.
    Dimension i is paired with i + R/2, or, with `interleaved`, 2i with 2i + 1; dimensions from R on stay as they are.
    Differentiable in q and k (not in frequencies).  `inplace` writes over q and k instead (no gradients then).  Returns q', or (q', k')."""
    if not inplace and isinstance(q, torch.Tensor) and q.is_cuda:
        host = _lib.host()
        if host is not None:
            out = host.rotary(q, k, frequencies, positions, interleaved, magnitude)
            if out is not None:
                return out
    # the general path: what the native one does not cover, and the errors
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("q, k must have shape [B,H,N,D]")
    if k is not None and (k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:]):
        raise ValueError("q and k must agree in batch, tokens, and head_dim")
    _check_sizes(q, *(() if k is None else (k,)))
    if q.device.type != "cuda":
        raise ValueError("rotary_embedding currently requires CUDA tensors")
    if q.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise ValueError("supported dtypes are fp16, bf16, and fp32")
    if k is not None and (k.dtype != q.dtype or k.device != q.device):
        raise ValueError("q, k must share one dtype and one device")
    if frequencies.dim() != 1 or frequencies.dtype != torch.float64 or frequencies.device != q.device:
        raise ValueError("frequencies must be a float64 vector on the device of q")
    rotary_dim = 2 * int(frequencies.shape[0])
    if not 2 <= rotary_dim <= min(int(q.shape[3]), _MAX_ROTARY_DIM):
        raise ValueError(f"2 * len(frequencies) must be between 2 and head_dim, and at most {_MAX_ROTARY_DIM}")
    if int(q.shape[3]) > _MAX_HEAD_DIM:
        raise ValueError(f"head_dim > {_MAX_HEAD_DIM} is not supported by the current kernels")
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device:
            raise ValueError("positions must be int32 or int64 on the device of q")
        if positions.dim() not in (1, 2) or positions.shape[-1] != q.shape[2] or (positions.dim() == 2 and positions.shape[0] not in (1, q.shape[0])):
            raise ValueError("positions must have shape [N] or [B,N]")
    if torch.is_grad_enabled() and frequencies.requires_grad:
        raise ValueError("frequencies have no gradient: detach them")
    if not frequencies.is_contiguous():
        frequencies = frequencies.contiguous()
    magnitude = float(magnitude)
    if inplace:
        _refuse_transforms("rotary_embedding(inplace=True)", q, *(() if k is None else (k,)))
        if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
            raise ValueError("inplace=True has no gradients: use it under torch.no_grad()")
        for t in (q,) if k is None else (q, k):
            if _row_strides(t) is None or _overlaps(t):
                raise ValueError("inplace=True needs rows of contiguous elements that do not overlap")
        if k is not None and q.numel() > 0 and k.numel() > 0 and _meet(q, k):
            raise ValueError("inplace=True needs q and k in different memory")
        _rotate(q, k, frequencies, positions, magnitude, interleaved, inplace=True)
        torch.autograd.graph.increment_version((q,) if k is None else (q, k))     # (what a graph had saved is gone)
        return q if k is None else (q, k)
    return _RotaryAutograd.apply(q, k, frequencies, positions, magnitude, bool(interleaved))


class Rotary(NamedTuple):
    """Rotary positions as one value, for calls that apply them on the way: `twopass_attention_qkvpacked(..., rotary=Rotary(...))` and the
    ViT hooks (`patch_timm_attention(model, elsa_kwargs={"rotary": Rotary(...)})`).  The fields are `rotary_embedding`'s arguments; its
    tensors are no part of a model and do not move with it (frequencies would lose their 64 bits to `model.half()`): make them on the
    device that the model runs on."""

    frequencies: torch.Tensor
    positions: Optional[torch.Tensor] = None
    interleaved: bool = False
    magnitude: float = 1.0

    def apply(self, q: torch.Tensor, k: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return rotary_embedding(q, k, self.frequencies, positions=self.positions, interleaved=self.interleaved, magnitude=self.magnitude)

"""Differential attention: the difference of two softmax maps with a learned weight, over one set of values -- forward, backward, and the
form for single tokens over a key cache (csrc/pair_tc.cu, csrc/diff_bwd_tc.cu, csrc/diff_any.cu, csrc/decode.cu).

The reference has no counterpart; names and checks follow `twopass_attention` and `twopass_attention_train`.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Union

import torch

from . import _lib
from .attention import _DeviceScope, _aligned, _cached_bytes, _in_place_or_copy
from .rotary import _MAX_SIZE, _check_saved, _check_sizes, _once_differentiable, _refuse_transforms
from .shared_prefix import _check_lengths, _positive_scale, _readable, _strides


def differential_lambda(lambda_q1: torch.Tensor, lambda_k1: torch.Tensor, lambda_q2: torch.Tensor, lambda_k2: torch.Tensor,
                        lambda_init: float) -> torch.Tensor:
    """The weight of the second map from its learned vectors (the last axis of each):
    exp(lambda_q1 . lambda_k1) - exp(lambda_q2 . lambda_k2) + lambda_init, in fp32; differentiable."""
    first = torch.exp((lambda_q1.float() * lambda_k1.float()).sum(-1))
    second = torch.exp((lambda_q2.float() * lambda_k2.float()).sum(-1))
    return first - second + lambda_init


def _check(q, k, v, lam, who: str):
    """(batch, heads, kv_heads, nq, nk, dim, v_dim)"""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k, v must have shape [B,H,N,D]")
    batch, heads2, nq, dim = map(int, q.shape)
    if heads2 % 2 or k.shape[1] % 2:
        raise ValueError("q and k must have two heads for each head of the output and of v")
    heads, kv_heads = heads2 // 2, int(k.shape[1]) // 2
    if k.shape[0] != batch or v.shape[0] != batch or k.shape[3] != dim or v.shape[1] != kv_heads or v.shape[2] != k.shape[2]:
        raise ValueError("q, k, v must agree in batch and head_dim, k and v in heads and keys")
    if kv_heads == 0 or heads % kv_heads:
        raise ValueError("the number of output heads must be a multiple of the number of value heads")
    _check_sizes(q, k, v)
    if q.device.type != "cuda":
        raise ValueError(f"{who} currently requires CUDA tensors")
    if q.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise ValueError("supported dtypes are fp16, bf16, and fp32")
    if k.dtype != q.dtype or v.dtype != q.dtype or k.device != q.device or v.device != q.device:
        raise ValueError("q, k, v must share one dtype and one device")
    if dim > 128 or v.shape[3] > 128:
        raise ValueError("head dims > 128 are not supported by the current kernels")
    if isinstance(lam, torch.Tensor):
        if lam.dtype not in (torch.float16, torch.bfloat16, torch.float32) or lam.device != q.device or tuple(lam.shape) not in ((), (1,), (heads,)):
            raise ValueError("lam must be a number, or a float tensor of one value or of one for each output head, on the device of q")
    elif not isinstance(lam, (int, float)):
        raise ValueError("lam must be a number or a tensor")
    return batch, heads, kv_heads, nq, int(k.shape[2]), dim, int(v.shape[3])


def _lam_args(lam, heads, like):
    """(tensor to keep, pointer, dtype code, stride in elements)"""
    if not isinstance(lam, torch.Tensor):
        lam = torch.full((), float(lam), device=like.device, dtype=torch.float32)
    lam = lam.detach()
    if lam.dim() == 1 and lam.stride(0) > _MAX_SIZE:
        lam = lam.contiguous()
    stride = int(lam.stride(0)) if lam.dim() == 1 and lam.shape[0] > 1 else 0
    return lam, lam.data_ptr(), _lib.dtype_code(lam.dtype), stride


def _forward(q, k, v, lam, sizes, is_causal, scale, lengths, want_state):
    """(out, out2, lse, q, k, v): the last three as they were read."""
    batch, heads, kv_heads, nq, nk, dim, v_dim = sizes
    (q, qs), (k, ks), (v, vs) = _readable(q), _readable(k), _readable(v)
    if qs[1] and qs[2] and qs[1] < qs[2]:                # q as [B, N, H, D] in memory: out too
        out = torch.empty((batch, nq, heads, v_dim), device=q.device, dtype=q.dtype).transpose(1, 2)
    else:
        out = torch.empty((batch, heads, nq, v_dim), device=q.device, dtype=q.dtype)
    out2 = lse = None
    if want_state:
        out2 = torch.empty((batch, heads, nq, v_dim), device=q.device, dtype=q.dtype)
        lse = torch.empty((2, batch, heads, nq), device=q.device, dtype=torch.float32)
    lam, lam_ptr, lam_dtype, lam_stride = _lam_args(lam, heads, q)
    dt = _lib.dtype_code(q.dtype)
    flat = (ctypes.c_int64 * 12)(*qs, *ks, *vs, *_strides(out))
    n = None if lengths is None else lengths.data_ptr()
    with _DeviceScope(q.device):
        need = int(_lib.load().elsa_differential_workspace_bytes_for(q.data_ptr(), k.data_ptr(), v.data_ptr(), n, out.data_ptr(), flat, dt, *sizes))
        if need < 0:
            raise ValueError("elsa_b200: unsupported problem size for differential_attention")
        ws = torch.empty((need,), device=q.device, dtype=torch.uint8)      # (the tiles need none)
        rc = _lib.load().elsa_differential_forward(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), lam_ptr, lam_dtype, lam_stride, n, out.data_ptr(), flat,
            None if out2 is None else out2.data_ptr(), None if lse is None else lse.data_ptr(), ws.data_ptr(), need, dt, *sizes,
            int(bool(is_causal)), scale, _lib.raw_stream(q.device))
    _lib.check(rc, "elsa_differential_forward")
    return out, out2, lse, q, k, v


def differential_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    lam: Union[torch.Tensor, float],
    *,
    is_causal: bool = False,
    scale: Optional[float] = None,
    lengths: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """(softmax(q1 k1^T scale) - lam softmax(q2 k2^T scale)) v for every output head.

    q: [B, 2H, Nq, D], heads 2h and 2h + 1 the two maps of output head h; k: [B, 2Hkv, Nk, D] alike; v: [B, Hkv, Nk, Dv], usually
    Dv = 2D; H is a multiple of Hkv, consecutive output heads share a key head.  lam: a number, or a float tensor with one value or
    one for each output head (`differential_lambda`).  is_causal: the queries are the last Nq tokens, query i sees the first
    Nk - Nq + i + 1 keys.  lengths: int32 [B] on the device: sequence b has lengths[b] keys instead of Nk (a cache with room to grow;
    nothing behind them is read).  A query without any key gives zeros.  D, Dv <= 128; fp16, bf16 or fp32; rows of contiguous
    elements are read in place.  16-bit inputs run on the tensor cores' 16-bit instructions with D <= 64, D and Dv multiples of 8 and
    rows on 16-byte boundaries; all others, and fp32, on fp32 arithmetic that is several times slower.  Of the former, calls without
    `lengths` and with more than 64 rows for a key head need no scratch memory, all others at most 1 GiB.  scale: 1 / sqrt(D) by default.
    Forward only: the result has no gradients, whatever the inputs ask for; see `differential_attention_train`.
    Returns [B, H, Nq, Dv]."""
    if isinstance(q, torch.Tensor) and q.is_cuda:
        host = _lib.host()
        if host is not None:
            out = host.differential(q, k, v, lam, is_causal, scale, lengths, False) if isinstance(lam, torch.Tensor) else None
            if out is not None:
                return out
    # the general path: what the native one does not cover, and the errors
    sizes = _check(q, k, v, lam, "differential_attention")
    _check_lengths(lengths, sizes[0], q.device)
    scale = _positive_scale(scale, sizes[5])
    _refuse_transforms("differential_attention", q, k, v, *((lam,) if isinstance(lam, torch.Tensor) else ()))
    if sizes[0] * sizes[1] * sizes[3] * sizes[6] == 0:
        return torch.empty((sizes[0], sizes[1], sizes[3], sizes[6]), device=q.device, dtype=q.dtype)
    return _forward(q, k, v, lam, sizes, is_causal, scale, lengths, False)[0]


def _for_tiles(t):
    """Rows on 16-byte boundaries, in place or copied; other head dims as they are."""
    return _in_place_or_copy(t)[0] if t.shape[-1] % 8 == 0 and t.numel() else t


class _DifferentialAutograd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, sizes, is_causal, scale):
        out, out2, lse, q, k, v = _forward(_for_tiles(q), _for_tiles(k), _for_tiles(v), lam, sizes, is_causal, scale, None, True)
        ctx.lam = None if isinstance(lam, torch.Tensor) else lam
        kept = (q, k, v, out, out2, lse, *((lam,) if isinstance(lam, torch.Tensor) else ()))
        ctx.save_for_backward(*kept)
        ctx.kept = [(t.shape, t.dtype, t.device) for t in kept]
        ctx.sizes, ctx.is_causal, ctx.scale = sizes, is_causal, scale
        return out

    @staticmethod
    @_once_differentiable
    def backward(ctx, dout):
        q, k, v, out, out2, lse, *rest = (_check_saved(t, *kept) for t, kept in zip(ctx.saved_tensors, ctx.kept))
        (q, _), (k, _), (v, _), (out, _) = (_readable(_for_tiles(t)) for t in (q, k, v, out))
        out2, lse = _aligned(out2), _aligned(lse)
        lam = rest[0] if rest else ctx.lam
        batch, heads, kv_heads, nq, nk, dim, v_dim = ctx.sizes
        dout, gs = _readable(_for_tiles(dout.to(q.dtype)))
        dq, dk, dv = (torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v))
        dlam = torch.empty_like(lam, memory_format=torch.contiguous_format) if rest and ctx.needs_input_grad[3] else None
        keep, lam_ptr, lam_dtype, lam_stride = _lam_args(lam, heads, q)
        wide = lam_stride == 0 and dlam is not None and dlam.numel() > 1    # an expanded value: one sum, shared out by autograd
        if wide:
            keep = keep.contiguous()
            lam_ptr, lam_stride = keep.data_ptr(), 1
        dt = _lib.dtype_code(q.dtype)
        need = _cached_bytes("elsa_differential_backward_workspace_bytes", q.device, dt, *ctx.sizes)
        flat = (ctypes.c_int64 * 24)(*_strides(q), *_strides(k), *_strides(v), *_strides(out), *gs, *_strides(dq), *_strides(dk), *_strides(dv))
        with _DeviceScope(q.device):
            ws = torch.empty((max(need, 256),), device=q.device, dtype=torch.uint8)
            rc = _lib.load().elsa_differential_backward(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), lam_ptr, lam_dtype, lam_stride, out.data_ptr(), out2.data_ptr(), lse.data_ptr(),
                dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), None if dlam is None else dlam.data_ptr(), flat,
                ws.data_ptr(), ws.numel(), dt, *ctx.sizes, int(ctx.is_causal), ctx.scale, _lib.raw_stream(q.device))
        _lib.check(rc, "elsa_differential_backward")
        return dq, dk, dv, dlam, None, None, None


def differential_attention_train(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    lam: Union[torch.Tensor, float],
    *,
    is_causal: bool = False,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """Differentiable `differential_attention` (without lengths), in q, k, v and, where it is a tensor, lam: the forward keeps P2 v and each
    row's log sum, the backward recomputes the maps.  Gradients repeat bit for bit; those of shared key heads and of a shared lam are
    summed.  Rows that the tensor cores' 16-bit instructions would take but for their addresses or strides are copied first."""
    if isinstance(q, torch.Tensor) and q.is_cuda:
        host = _lib.host()
        if host is not None:
            out = host.differential(q, k, v, lam, is_causal, scale, None, True) if isinstance(lam, torch.Tensor) else None
            if out is not None:
                return out
    # the general path: what the native one does not cover, and the errors
    sizes = _check(q, k, v, lam, "differential_attention_train")
    scale = _positive_scale(scale, sizes[5])
    if any(x == 0 for x in (sizes[0], sizes[1], sizes[3], sizes[4], sizes[6])):
        # nothing to attend to: zeros that depend on nothing but shapes (and have zero gradients)
        # (sums of no elements: a sum of all of q may be infinite, or NaN)
        zero = sum(t.flatten()[:0].sum() for t in (q, k, v) + ((lam.to(q.dtype),) if isinstance(lam, torch.Tensor) else ()))
        return torch.zeros((sizes[0], sizes[1], sizes[3], sizes[6]), device=q.device, dtype=q.dtype) + zero
    return _DifferentialAutograd.apply(q, k, v, lam, sizes, bool(is_causal), scale)

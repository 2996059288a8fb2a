"""Attention of a batch whose sequences share a long prefix (a system prompt, a document, the samples of one prompt): the serving
form of the two-pass scheme, in which the prefix and each sequence's own cache give (m, z, s) summaries that one merge joins
(csrc/pair_tc.cu, csrc/decode.cu).

The reference has no counterpart; names and checks follow `twopass_attention`.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .attention import _DeviceScope, _cached_bytes, _empty_like_layout
from .rotary import _check_sizes, _refuse_transforms


def _strides(t: torch.Tensor):
    """Element strides of all axes but the last (0 for an axis of one), or None where the last is not contiguous."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        return None
    return tuple(st if size > 1 else 0 for st, size in zip(t.stride()[:-1], t.shape[:-1]))


def _readable(t: torch.Tensor):
    """(tensor, strides): itself, or a contiguous copy where its rows are not contiguous."""
    st = _strides(t)
    if st is None:
        t = t.contiguous()
        st = _strides(t)
    return t, st


def _check_lengths(lengths, batch, device):
    if lengths is None:
        return
    if lengths.dtype != torch.int32 or lengths.device != device or tuple(lengths.shape) != (batch,) or not lengths.is_contiguous():
        raise ValueError("lengths must be a contiguous int32 vector [B] on the device of q")


def _positive_scale(scale, dim):
    scale = max(1, int(dim)) ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -126 <= scale <= 2.0 ** 127:           # (the kernels hold scale log2 e in fp32)
        raise ValueError("scale must be positive and finite in fp32")
    return scale


def shared_prefix_attention(
    q: torch.Tensor,
    k_prefix: torch.Tensor,
    v_prefix: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    lengths: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """softmax(q [k_prefix; k_b]^T scale) [v_prefix; v_b] for every sequence b of the batch, the prefix read once for all.

    q: [B, H, Nq, D], the Nq newest tokens of each sequence (1 in plain decoding); k_prefix, v_prefix: [Hkv, P, D]; k, v: each
    sequence's own cache, [B, Hkv, S, D], of which the first lengths[b] keys count (int32 on the device; None: all S) and nothing
    behind them is read.  The queries are the last Nq of those tokens: query i sees the prefix and the first
    lengths[b] - Nq + i + 1 own keys (the prefix alone where that is not positive).  H is a multiple of Hkv; consecutive query
    heads share a key head.  P or S may be 0; a query without any key gives zeros.  D <= 128; fp16, bf16 or fp32; rows of D
    contiguous elements are read in place, whatever the other strides.  scale: 1 / sqrt(D) by default.  Forward only: the result has no
    gradients, whatever the inputs ask for.  Scratch memory: the summaries of a chunk of the queries, 1 GiB at most.
    Returns [B, H, Nq, D]."""
    if isinstance(q, torch.Tensor) and q.is_cuda:
        host = _lib.host()
        if host is not None:
            out = host.shared_prefix(q, k_prefix, v_prefix, k, v, lengths, scale)
            if out is not None:
                return out
    # the general path: what the native one does not cover, and the errors
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k, v must have shape [B,H,N,D]")
    if k_prefix.dim() != 3 or v_prefix.dim() != 3:
        raise ValueError("k_prefix, v_prefix must have shape [H,N,D]")
    if k.shape != v.shape or k_prefix.shape != v_prefix.shape:
        raise ValueError("k and v must have identical shapes, k_prefix and v_prefix too")
    batch, heads, nq, dim = q.shape
    kv_heads = int(k.shape[1])
    if k.shape[0] != batch or k.shape[3] != dim or k_prefix.shape[0] != kv_heads or k_prefix.shape[2] != dim:
        raise ValueError("q, k, k_prefix must agree in batch, key heads, and head_dim")
    if kv_heads == 0 or heads % kv_heads:
        raise ValueError("the number of query heads must be a multiple of the number of key heads")
    _check_sizes(q, k_prefix, k)
    if q.device.type != "cuda":
        raise ValueError("shared_prefix_attention currently requires CUDA tensors")
    if q.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise ValueError("supported dtypes are fp16, bf16, and fp32")
    for t in (k_prefix, v_prefix, k, v):
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError("q, k_prefix, v_prefix, k, v must share one dtype and one device")
    if dim > 128:
        raise ValueError("head_dim > 128 is not supported by the current kernels")
    _check_lengths(lengths, batch, q.device)
    scale = _positive_scale(scale, dim)
    _refuse_transforms("shared_prefix_attention", q, k_prefix, v_prefix, k, v)
    if q.numel() == 0:
        return torch.empty_like(q)
    n_prefix, n_own = int(k_prefix.shape[1]), int(k.shape[2])
    q, qs = _readable(q)
    (k_prefix, kps), (v_prefix, vps), (k, ks), (v, vs) = (_readable(t) for t in (k_prefix, v_prefix, k, v))
    out = _empty_like_layout(q, q.stride())
    dt = _lib.dtype_code(q.dtype)
    need = _cached_bytes("elsa_shared_prefix_workspace_bytes", q.device, dt, batch, heads, kv_heads, nq, dim, n_prefix, n_own)
    if need < 0:
        raise ValueError("elsa_b200: unsupported problem size for shared_prefix_attention")
    flat = (ctypes.c_int64 * 16)(*qs, *kps, *vps, *ks, *vs, *_strides(out))
    with _DeviceScope(q.device):
        ws = torch.empty((max(need, 256),), device=q.device, dtype=torch.uint8)
        rc = _lib.load().elsa_shared_prefix_attention(
            q.data_ptr(), k_prefix.data_ptr(), v_prefix.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), flat,
            None if lengths is None else lengths.data_ptr(), ws.data_ptr(), ws.numel(), dt, batch, heads, kv_heads, nq, dim,
            n_prefix, n_own, scale, _lib.raw_stream(q.device))
    _lib.check(rc, "elsa_shared_prefix_attention")
    return out

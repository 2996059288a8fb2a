"""Differential attention against the definition in 64 bits: forward, state, gradients, single tokens; head layouts, odd sizes, masks
that leave rows empty, strides, what stands behind a sequence's last key."""
import pytest
import torch

import elsa_b200 as E
from elsa_b200 import _lib

pytestmark = pytest.mark.gpu


def _normal(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def _inputs(b, h, hkv, nq, nk, d, dv, dtype, seed=0, scale=1.0):
    lam = (0.2 + 0.6 * torch.rand(h, generator=torch.Generator().manual_seed(seed + 3))).cuda()
    return _normal((b, 2 * h, nq, d), dtype, seed, scale), _normal((b, 2 * hkv, nk, d), dtype, seed + 1, scale), _normal((b, hkv, nk, dv), dtype, seed + 2), lam


class _Map:
    """One softmax map of the definition: P, its sums' size and how far the arithmetic may move a weight.
      scores   (D + 8) roundings of 2^-24 of the sum of |q_i k_i| scale, and 2^-19 for the exponential and its argument; a weight and
               the sum of weights each carry that: twice"""

    def __init__(self, q, k, seen, scale):
        d = q.shape[-1]
        score = (q.double() @ k.double().transpose(-1, -2)) * scale
        size = (q.double().abs() @ k.double().abs().transpose(-1, -2)) * scale
        score, size = score.masked_fill(~seen, float("-inf")), size.masked_fill(~seen, 0.0)
        w = torch.softmax(score, -1)
        self.p = torch.where(seen.any(-1, keepdim=True), w, torch.zeros_like(w))
        self.lse2 = torch.logsumexp(score, -1) / torch.log(torch.tensor(2.0, dtype=torch.float64))
        self.e = 2 * ((d + 8) * 2.0 ** -24 * (size.amax(-1, keepdim=True) if size.shape[-1] else 0.0) + 2.0 ** -19)


def _maps(q, k, lam, causal, lengths, scale, i, h, hkv):
    nq, nk, d = q.shape[2], k.shape[2], q.shape[3]
    scale = d ** -0.5 if scale is None else scale
    n = nk if lengths is None else max(0, min(nk, int(lengths[i])))
    last = n - nq + torch.arange(nq, device=q.device) if causal else torch.full((nq,), n - 1, device=q.device)
    seen = (torch.arange(nk, device=q.device) <= last[:, None]) & (torch.arange(nk, device=q.device) < n)
    g = h // (q.shape[1] // 2 // hkv)
    return [_Map(q[i, 2 * h + m], k[i, 2 * g + m], seen, scale) for m in (0, 1)], g, n


SUMS = 1088 * 2.0 ** -24        # at most 1024 + 64 roundings in a row (a split's keys, then the merge; less in a tile's accumulators)


def _check_forward(got, q, k, v, lam, causal=False, lengths=None, scale=None):
    """16-bit: a weight is rounded to the type before the second product (eps / 2 of it); both maps' sums, then one rounding"""
    b, h, hkv = q.shape[0], q.shape[1] // 2, v.shape[1]
    eps = torch.finfo(q.dtype).eps / 2
    assert got.shape == (b, h, q.shape[2], v.shape[3]) and got.dtype == q.dtype
    for i in range(b):
        for j in range(h):
            (one, two), g, n = _maps(q, k, lam, causal, lengths, scale, i, j, hkv)
            value = torch.where((torch.arange(v.shape[2], device=q.device) < n)[:, None], v[i, g].double(), torch.zeros((), device=q.device, dtype=torch.float64))
            w = float(lam[j]) if isinstance(lam, torch.Tensor) and lam.numel() > 1 else float(lam)
            want = one.p @ value - w * (two.p @ value)
            half = eps if q.dtype != torch.float32 else 0.0
            limit = (one.e + SUMS + half) * (one.p @ value.abs()) + abs(w) * (two.e + SUMS + half + 2.0 ** -23) * (two.p @ value.abs())
            limit = limit + eps * want.abs() * 1.01 + 2.0 ** -25
            err = (got[i, j].double() - want).abs()
            assert bool((err <= limit).all()), f"batch {i}, head {j}: {float((err / limit).max())} of the limit"
    assert _lib.load().elsa_device_status(0) == 0


FORWARD = [
    # b, h, hkv, nq, nk, d, dv
    (1, 1, 1, 1, 1, 64, 128), (2, 2, 1, 1, 100, 64, 128), (3, 4, 2, 5, 77, 32, 64), (1, 2, 2, 65, 65, 64, 128), (2, 4, 4, 128, 128, 64, 128),
    (2, 4, 1, 129, 300, 64, 128), (1, 2, 2, 257, 257, 32, 64), (1, 3, 3, 200, 1000, 48, 96), (2, 2, 2, 300, 90, 64, 128), (1, 1, 1, 513, 640, 8, 16),
    (1, 2, 1, 70, 513, 64, 64), (1, 2, 2, 100, 260, 64, 72), (1, 2, 2, 33, 70, 128, 128), (2, 2, 1, 90, 33, 20, 12), (1, 1, 1, 66, 40, 7, 5),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", FORWARD, ids=str)
def test_forward(case, dtype, causal):
    args = _inputs(*case, dtype)
    _check_forward(E.differential_attention(*args, is_causal=causal), *args, causal=causal)


@pytest.mark.parametrize("case", [(2, 2, 1, 200, 600, 64, 128), (1, 2, 2, 3, 600, 64, 128)], ids=str)
def test_long_range_of_scores(case):
    """Scores of several hundred, growing along the keys: the reference maximum moves again and again."""
    q, k, v, lam = _inputs(*case, torch.float16, scale=6.0)
    k = (k.float() * torch.linspace(0.1, 1.5, k.shape[2], device="cuda")[:, None]).half()
    _check_forward(E.differential_attention(q, k, v, lam, scale=0.9), q, k, v, lam, scale=0.9)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_lam_of_every_form(dtype):
    q, k, v, lam = _inputs(1, 4, 2, 70, 70, 64, 128, dtype)
    for lam in (0.3, 1, -0.7, 0.0, torch.tensor(0.4, device="cuda"), torch.tensor([0.4], device="cuda", dtype=torch.bfloat16), lam.half(),
                torch.stack((lam, lam)).t()[:, 1], lam[:1].expand(4)):
        _check_forward(E.differential_attention(q, k, v, lam), q, k, v, lam)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq", [1, 4, 80])
def test_lengths_of_a_cache(dtype, nq, causal):
    q, k, v, lam = _inputs(4, 4, 2, nq, 230, 64, 128, dtype)
    lengths = torch.tensor([0, 1, 129, 230], dtype=torch.int32)
    want = E.differential_attention(q, k, v, lam, is_causal=causal, lengths=lengths.cuda())
    _check_forward(want, q, k, v, lam, causal=causal, lengths=lengths)
    assert not bool(want[0].any())
    for i, n in enumerate(lengths.tolist()):
        k[i, :, n:], v[i, :, n:] = float("nan"), float("inf")
    got = E.differential_attention(q, k, v, lam, is_causal=causal, lengths=lengths.cuda())
    assert torch.equal(got, want)


@pytest.mark.parametrize("nq", [2, 150])
def test_nan_is_answered_and_masked_keys_are_not_seen(nq):
    q, k, v, lam = _inputs(1, 2, 2, nq, 150, 64, 128, torch.float16)
    clean = E.differential_attention(q, k, v, lam, is_causal=True)
    k[0, 0, 149, 3] = float("inf")          # the last key: of head 0's first map, seen by the last query alone
    got = E.differential_attention(q, k, v, lam, is_causal=True)
    assert torch.equal(got[:, :, :-1], clean[:, :, :-1]) and torch.equal(got[:, 1], clean[:, 1])
    k[0, 0, 149, 3] = float("nan")
    got = E.differential_attention(q, k, v, lam, is_causal=True)
    assert torch.equal(got[:, :, :-1], clean[:, :, :-1]) and bool(torch.isnan(got[0, 0, -1]).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("nq", [3, 100])
@pytest.mark.parametrize("layout", ["bnhd", "odd_offset", "odd_stride", "strided_d", "expanded", "capacity"])
def test_strided_inputs(layout, nq, dtype):
    q, k, v, lam = _inputs(2, 4, 2, nq, 140, 64, 128, dtype)
    if layout == "bnhd":
        move = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "odd_offset":
        move = lambda t: torch.cat((t.new_zeros(1), t.flatten()))[1:].view(t.shape)
    elif layout == "odd_stride":
        move = lambda t: torch.cat((t, t[..., :1]), -1)[..., : t.shape[-1]]
    elif layout == "strided_d":
        move = lambda t: t.repeat_interleave(2, -1)[..., ::2]
    elif layout == "capacity":
        move = lambda t: torch.cat((t, torch.full_like(t, float("nan"))), -2)[..., : t.shape[-2], :]
    else:
        k, v = k[:1].expand_as(k), v[:, :1].expand_as(v)
        move = lambda t: t
    q, k, v = move(q), move(k), move(v)
    keep = [t.clone() for t in (q, k, v)]
    got = E.differential_attention(q, k, v, lam, is_causal=True)
    _check_forward(got, q, k, v, lam, causal=True)
    assert all(torch.equal(x, y) for x, y in zip((q, k, v), keep))
    if layout == "bnhd":
        assert got.transpose(1, 2).is_contiguous()


def test_no_keys_and_empty_calls():
    q, k, v, lam = _inputs(2, 2, 2, 3, 0, 64, 128, torch.float16)
    assert not bool(E.differential_attention(q, k, v, lam).any())
    q, k, v, lam = _inputs(2, 2, 2, 100, 0, 64, 128, torch.float16)
    assert not bool(E.differential_attention(q, k, v, lam, is_causal=True).any())
    q, k, v, lam = _inputs(2, 2, 2, 0, 9, 64, 128, torch.float16)
    assert E.differential_attention(q, k, v, lam).shape == (2, 2, 0, 128)


@pytest.mark.parametrize("nq", [1, 200])
def test_another_stream_and_captured_graphs(nq):
    args, other = _inputs(2, 4, 2, nq, 300, 64, 128, torch.bfloat16), _inputs(2, 4, 2, nq, 300, 64, 128, torch.bfloat16, seed=9)
    want, want2 = E.differential_attention(*args, is_causal=True), E.differential_attention(*other, is_causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = E.differential_attention(*args, is_causal=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        a = E.differential_attention(*args, is_causal=True)
    with torch.cuda.graph(two):
        c = E.differential_attention(*other, is_causal=True)
    for _ in range(2):
        one.replay()
        two.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(c, want2)


def test_refusals():
    q, k, v, lam = _inputs(2, 4, 2, 3, 9, 64, 128, torch.float16)
    n = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    for args, kw, match in (
            ((q[0], k, v, lam), {}, "shape"), ((q[:, :7], k, v, lam), {}, "two heads"), ((q, k[:, :3], v, lam), {}, "two heads"),
            ((q, k, v[:, :1], lam), {}, "agree"), ((q, k, v[:, :, :8], lam), {}, "agree"), ((q[:1], k, v, lam), {}, "agree"),
            ((q[..., :32], k, v, lam), {}, "agree"), ((q[:, :6], k, v, lam), {}, "multiple"), ((q.float(), k, v, lam), {}, "dtype"),
            ((q, k.cpu(), v, lam), {}, "device"), ((q, k, v, lam[:3]), {}, "lam"), ((q, k, v, lam.cpu()), {}, "lam"),
            ((q, k, v, lam.double()), {}, "lam"), ((q, k, v, None), {}, "lam"), ((q, k, v, lam), dict(lengths=n.long()), "lengths"),
            ((q, k, v, lam), dict(scale=0.0), "scale"), ((q, k, v, lam), dict(scale=-1.0), "scale"), ((q, k, v, lam), dict(scale=float("nan")), "scale")):
        with pytest.raises(ValueError, match=match):
            E.differential_attention(*args, **kw)
    wide = _inputs(1, 1, 1, 3, 9, 64, 136, torch.float16)
    with pytest.raises(ValueError, match="128"):
        E.differential_attention(*wide)

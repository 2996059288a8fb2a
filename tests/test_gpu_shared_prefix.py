"""Attention over a shared prefix against the definition in 64 bits: head layouts, odd sizes, lengths from none to all, strides,
what stands behind a sequence's last key."""
import pytest
import torch

import elsa_b200 as E
from elsa_b200 import _lib

pytestmark = pytest.mark.gpu


def _normal(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def _inputs(b, h, hkv, nq, d, p, s, dtype, seed=0, scale=1.0):
    return (_normal((b, h, nq, d), dtype, seed, scale), _normal((hkv, p, d), dtype, seed + 1, scale), _normal((hkv, p, d), dtype, seed + 2),
            _normal((b, hkv, s, d), dtype, seed + 3, scale), _normal((b, hkv, s, d), dtype, seed + 4))


def _check(got, q, kp, vp, k, v, lengths=None, scale=None):
    """The definition, row by row of the batch, with the error that the arithmetic may have:
      scores      (D + 8) roundings of 2^-24 of the sum of |q_i k_i| scale, and 2^-19 for the exponential and its argument; a
                  weight and the sum of weights each carry that: twice
      sums        at most 1024 + 64 roundings in a row (a split's keys, then the merge) of 2^-24
      16-bit      a weight is rounded to the type before the second product: eps / 2
    all relative to sum_j w_j |v_j|; and one rounding of the result, eps / 2 of it."""
    b, h, nq, d = q.shape
    hkv, p, s = k.shape[1], kp.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    eps = torch.finfo(q.dtype).eps / 2
    assert got.shape == q.shape and got.dtype == q.dtype
    for i in range(b):
        n = s if lengths is None else max(0, min(s, int(lengths[i])))
        keys, values = torch.cat((kp, k[i, :, :n]), 1).double(), torch.cat((vp, v[i, :, :n]), 1).double()
        keys, values = (x.repeat_interleave(h // hkv, 0) for x in (keys, values))
        score = q[i].double() @ keys.transpose(1, 2) * scale
        size = q[i].double().abs() @ keys.abs().transpose(1, 2) * scale
        last = p + n - nq + torch.arange(nq, device=q.device)
        seen = (torch.arange(p + n, device=q.device) <= torch.maximum(last, torch.tensor(p - 1, device=q.device))[:, None])
        score = score.masked_fill(~seen, float("-inf"))
        w = torch.softmax(score, -1) if p + n else score
        w = torch.where(seen.any(-1)[:, None], w, torch.zeros_like(w))
        want, mass = w @ values, w @ values.abs()
        e = 2 * ((d + 8) * 2.0 ** -24 * torch.where(seen, size, torch.zeros_like(size)).amax(-1, keepdim=True) + 2.0 ** -19) if p + n else 0.0
        limit = (e + 1088 * 2.0 ** -24 + (eps if q.dtype != torch.float32 else 0.0)) * mass + eps * want.abs() * 1.01 + 2.0 ** -25
        err = (got[i].double() - want).abs()
        assert bool((err <= limit).all()), f"sequence {i}: {float((err / limit).max())} of the limit"
    assert _lib.load().elsa_device_status(0) == 0


CASES = [
    # b, h, hkv, nq, d, p, s
    (1, 1, 1, 1, 64, 1, 1), (1, 1, 1, 1, 128, 16, 3), (3, 4, 2, 1, 64, 100, 70), (2, 8, 8, 1, 128, 65, 17), (5, 8, 1, 1, 96, 129, 33),
    (4, 6, 2, 3, 80, 64, 50), (2, 16, 2, 5, 64, 300, 90), (9, 8, 2, 1, 128, 1025, 200), (33, 2, 2, 1, 64, 128, 40), (40, 4, 1, 2, 128, 520, 65),
    (70, 4, 2, 1, 72, 257, 31), (2, 4, 4, 40, 64, 129, 130), (3, 2, 1, 7, 8, 40, 20), (130, 8, 2, 1, 40, 700, 9),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_values(case, dtype):
    b, h, hkv, nq, d, p, s = case
    args = _inputs(*case, dtype)
    _check(E.shared_prefix_attention(*args), *args)
    lengths = torch.randint(0, s + 1, (b,), generator=torch.Generator().manual_seed(9), dtype=torch.int32)
    lengths[0] = 0
    lengths[-1] = s
    got = E.shared_prefix_attention(*args, lengths=lengths.cuda())
    _check(got, *args, lengths=lengths)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("d", [1, 7, 20, 66])
def test_head_dims_that_no_tile_likes(dtype, d):
    args = _inputs(3, 4, 2, 2, d, 37, 21, dtype)
    _check(E.shared_prefix_attention(*args), *args)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_no_prefix_no_own_keys_or_neither(dtype):
    q, kp, vp, k, v = _inputs(3, 4, 2, 2, 64, 0, 33, dtype)
    lengths = torch.tensor([0, 1, 33], dtype=torch.int32)
    got = E.shared_prefix_attention(q, kp, vp, k, v, lengths=lengths.cuda())
    _check(got, q, kp, vp, k, v, lengths=lengths)
    assert not bool(got[0].any()) and not bool(got[1, :, 0].any())      # rows whose mask leaves nothing
    args = _inputs(3, 4, 2, 2, 64, 50, 0, dtype)
    _check(E.shared_prefix_attention(*args), *args)
    args = _inputs(3, 4, 2, 2, 64, 0, 0, dtype)
    assert not bool(E.shared_prefix_attention(*args).any())
    for shape in ((0, 4, 2, 64), (3, 4, 0, 64)):
        q = torch.empty(shape, device="cuda", dtype=dtype)
        k = torch.empty((shape[0], 2, 5, 64), device="cuda", dtype=dtype)
        assert E.shared_prefix_attention(q, kp[:, :0], vp[:, :0], k, k).shape == shape


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nothing_behind_a_sequences_last_key_is_read(dtype):
    """A cache is allocated longer than what it holds: whatever stands there, infinities and NaN among it."""
    q, kp, vp, k, v = _inputs(4, 8, 2, 2, 64, 90, 150, dtype)
    lengths = torch.tensor([2, 64, 77, 149], dtype=torch.int32)
    want = E.shared_prefix_attention(q, kp, vp, k, v, lengths=lengths.cuda())
    for i, n in enumerate(lengths.tolist()):
        k[i, :, n:], v[i, :, n:] = float("nan"), float("inf")
    got = E.shared_prefix_attention(q, kp, vp, k, v, lengths=lengths.cuda())
    assert torch.equal(got, want) and bool(torch.isfinite(got).all())
    over = torch.tensor([-3, 64, 77, 400], dtype=torch.int32)              # clamped to 0 .. S
    k[3, :, 149], v[3, :, 149] = 0.5, 0.5
    got = E.shared_prefix_attention(q, kp, vp, k, v, lengths=over.cuda())
    assert torch.equal(got[1:3], want[1:3])
    _check(got, q, kp, vp, torch.nan_to_num(k), torch.nan_to_num(v, posinf=0.0), lengths=over)


def test_a_nan_that_is_seen_is_answered():
    q, kp, vp, k, v = _inputs(2, 4, 2, 1, 64, 90, 20, torch.float16)
    kp[1, 7, 3] = float("nan")
    got = E.shared_prefix_attention(q, kp, vp, k, v)
    assert bool(torch.isnan(got[:, 2:]).all()) and bool(torch.isfinite(got[:, :2]).all())


@pytest.mark.parametrize("rows", [2, 40])
def test_large_scores(rows):
    """Scores of several hundred: the running maximum carries the whole range."""
    args = _inputs(rows, 2, 2, 1, 64, 300, 40, torch.float16, scale=8.0)
    got = E.shared_prefix_attention(*args, scale=1.0)
    _check(got, *args, scale=1.0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["bnhd", "odd_offset", "odd_stride", "strided_d", "expanded", "capacity"])
@pytest.mark.parametrize("b", [3, 24])
def test_strided_inputs(layout, dtype, b):
    h, hkv, nq, d, p, s = 4, 2, 1, 64, 200, 30
    q, kp, vp, k, v = _inputs(b, h, hkv, nq, d, p, s, dtype)
    if layout == "bnhd":
        move = lambda t: t.transpose(-3, -2).contiguous().transpose(-3, -2)
    elif layout == "odd_offset":
        move = lambda t: torch.cat((t.new_zeros(1), t.flatten()))[1:].view(t.shape)
    elif layout == "odd_stride":
        move = lambda t: torch.cat((t, t[..., :1]), -1)[..., :d]
    elif layout == "strided_d":
        move = lambda t: t.repeat_interleave(2, -1)[..., ::2]
    elif layout == "capacity":
        move = lambda t: torch.cat((t, torch.full_like(t, float("nan"))), -2)[..., : t.shape[-2], :]
    else:
        kp, vp, k, v = kp[:1].expand(hkv, p, d), vp[:1].expand(hkv, p, d), k[:1].expand(b, hkv, s, d), v[:, :1].expand(b, hkv, s, d)
        move = lambda t: t
    args = [move(t) for t in (q, kp, vp, k, v)]
    keep = [t.clone() for t in args]
    got = E.shared_prefix_attention(*args)
    _check(got, *args)
    assert all(torch.equal(a, b) for a, b in zip(args, keep))
    if layout == "bnhd":
        assert got.transpose(1, 2).is_contiguous()


def test_long_cache_offsets_pass_32_bits():
    """A key cache of more than 2^31 elements: the last sequence's keys are the right ones."""
    b, hkv, s, d = 3, 16, 4096 * 88, 128
    k = torch.zeros((b, hkv, s, d), device="cuda", dtype=torch.float16)
    assert k.numel() > 1 << 31
    v = torch.zeros_like(k)
    tail = _normal((b, hkv, 50, d), torch.float16, 5), _normal((b, hkv, 50, d), torch.float16, 6)
    k[:, :, -50:], v[:, :, -50:] = tail
    q, kp, vp = _normal((b, hkv, 1, d), torch.float16, 7), _normal((hkv, 64, d), torch.float16, 8), _normal((hkv, 64, d), torch.float16, 9)
    # zero keys score 0 and have zero values: their weights are all that they add
    got = E.shared_prefix_attention(q, kp, vp, k, v).double()
    keys = torch.cat((kp.expand(b, hkv, 64, d), tail[0]), 2).double()
    values = torch.cat((vp.expand(b, hkv, 64, d), tail[1]), 2).double()
    score = (q.double() @ keys.transpose(2, 3)) * d ** -0.5
    e = torch.exp(score)
    want = (e @ values) / (e.sum(-1, keepdim=True) + (s - 50))
    mass = (e @ values.abs()) / (e.sum(-1, keepdim=True) + (s - 50))
    # as in _check, with the merge of 344 splits on top of a split's own sums (together below 2048 roundings), fp16 subnormals
    assert bool(((got - want).abs() <= (2.0 ** -11 + 2.0 ** -12) * mass + 2.0 ** -11 * want.abs() + 2.0 ** -25).all())


def test_refusals():
    q, kp, vp, k, v = _inputs(2, 4, 2, 1, 64, 10, 8, torch.float16)
    n = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    for args, kw, match in (
            ((q[0], kp, vp, k, v), {}, "shape"), ((q, kp[0], vp, k, v), {}, "shape"), ((q, kp, vp[:, :9], k, v), {}, "identical"),
            ((q, kp, vp, k, v[:, :, :7]), {}, "identical"), ((q[:1], kp, vp, k, v), {}, "agree"), ((q, kp[:1], vp[:1], k, v), {}, "agree"),
            ((q[..., :32], kp, vp, k, v), {}, "agree"), ((q[:, :3], kp, vp, k, v), {}, "multiple"), ((q.float(), kp, vp, k, v), {}, "dtype"),
            ((q.double(),) * 5, {}, "shape"), ((q, kp, vp, k.cpu(), v), {}, "device"), ((q, kp, vp, k, v), dict(lengths=n.long()), "lengths"),
            ((q, kp, vp, k, v), dict(lengths=n[:1]), "lengths"), ((q, kp, vp, k, v), dict(lengths=n.cpu()), "lengths")):
        with pytest.raises(ValueError, match=match):
            E.shared_prefix_attention(*args, **kw)
    wide = _inputs(2, 4, 2, 1, 136, 10, 8, torch.float16)
    with pytest.raises(ValueError, match="128"):
        E.shared_prefix_attention(*wide)


@pytest.mark.parametrize("b", [2, 40])
def test_another_stream_and_two_captured_graphs(b):
    args = _inputs(b, 4, 2, 1, 64, 300, 80, torch.float16)
    other = _inputs(b, 4, 2, 1, 64, 300, 80, torch.float16, seed=50)
    lengths = torch.full((b,), 33, dtype=torch.int32, device="cuda")
    want, want2 = E.shared_prefix_attention(*args, lengths=lengths), E.shared_prefix_attention(*other, lengths=lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = E.shared_prefix_attention(*args, lengths=lengths)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        a = E.shared_prefix_attention(*args, lengths=lengths)
    with torch.cuda.graph(two):
        c = E.shared_prefix_attention(*other, lengths=lengths)
    for _ in range(2):
        one.replay()
        two.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(c, want2)
    lengths.fill_(80)                                        # the next token's step: lengths live on the device
    one.replay()
    assert torch.equal(a, E.shared_prefix_attention(*args, lengths=lengths))


@pytest.mark.parametrize("scale", [1e-46, 1e39, float("inf"), float("nan"), 0.0])
def test_a_scale_that_fp32_does_not_hold_is_refused(scale):
    """(one that is zero there would turn masked scores into NaN)"""
    with pytest.raises(ValueError, match="scale"):
        E.shared_prefix_attention(*_inputs(2, 4, 2, 2, 64, 90, 20, torch.float16), scale=scale)


@pytest.mark.parametrize("shape", [(40, 8, 2, 1, 64, 700, 300), (3, 8, 2, 1, 64, 700, 300), (24, 12, 3, 5, 96, 1000, 333)], ids=str)
def test_calls_in_a_row_and_side_by_side_do_not_meet(shape):
    """The kernels of a call overlap one another; those of the next call, or of one on another stream, must find nothing of theirs."""
    calls = [_inputs(*shape, torch.float16) for _ in range(4)]
    for i, args in enumerate(calls):
        args[0].mul_(1 + i)
        args[4].add_(i)
    want = [E.shared_prefix_attention(*args) for args in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        row = [E.shared_prefix_attention(*args) for args in calls]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(row, want))
        beside = []
        for i, args in enumerate(calls):
            with torch.cuda.stream(streams[i % 2]):
                beside.append(E.shared_prefix_attention(*args) * 1)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(beside, want))



@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("nq,p", [(4096, 2000), (8000, 2000), (8000, 0)])
def test_queries_in_chunks(nq, p, aligned):
    """Summaries of more than 1 GiB (9 parts or 8 of 32 heads): tokens of a sequence, or whole sequences, in turn.  Rows on either side of
    the chunks' borders, behind caches that are empty, shorter than a chunk's first query's, full."""
    b, h, hkv, d, s = 4, 32, 8, 128, 8192
    q, kp, vp, k, v = (torch.randn(shape, device="cuda", generator=torch.Generator("cuda").manual_seed(i)).half()
                       for i, shape in enumerate(((b, h, nq, d), (hkv, p, d), (hkv, p, d), (b, hkv, s, d), (b, hkv, s, d))))
    if not aligned:                                          # (a layout that the tile kernel does not take)
        kp, vp = (torch.cat((t.new_zeros(1), t.flatten()))[1:].view(t.shape) for t in (kp, vp))
    lengths = torch.tensor([0, 300, 5001, s], dtype=torch.int32)
    for i, n in enumerate(lengths.tolist()):
        k[i, :, n:], v[i, :, n:] = float("nan"), float("inf")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = E.shared_prefix_attention(q, kp, vp, k, v, lengths=lengths.cuda())
    assert torch.cuda.max_memory_allocated() - before <= 2 ** 30 + got.numel() * 2 + 2 ** 22
    for i, n in enumerate(lengths.tolist()):
        one = slice(i, i + 1)
        # (7168 and 8064 tokens go at a time; the first own key is seen by query nq - n)
        for t0, t1 in ((0, 2), (7166, 7170), (8062, 8066), (nq - n - 1, nq - n + 2), (nq - 3, nq)):
            if 0 <= t0 < t1 <= nq:
                last = n - nq + t1                           # own keys that the last of these rows sees
                part = max(0, last)
                rows = q[one, :, t0:t1]
                if last <= 0:                                # none of them sees one
                    _check(got[one, :, t0:t1], rows, kp, vp, k[one, :, :0], v[one, :, :0])
                else:
                    _check(got[one, :, t0:t1], rows, kp, vp, k[one, :, :part], v[one, :, :part])


def _planned_parts(dtype, b, h, hkv, nq, d, p, s):
    """(parts of the prefix, parts of the own caches), from the bytes of their summaries (calls of one chunk)."""
    size = _lib.load().elsa_shared_prefix_workspace_bytes
    code, row = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype], b * h * nq * (d + 2) * 4
    own = size(code, b, h, hkv, nq, d, 0, s) // row if s else 0
    return size(code, b, h, hkv, nq, d, p, s) // row - own, own


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", [(256, 32, 8, 1, 128, 6001, 1100), (256, 32, 8, 1, 64, 6001, 1100), (200, 16, 8, 3, 96, 5000, 1025), (300, 8, 8, 2, 40, 7777, 40)], ids=str)
def test_many_tiles_of_one_part(case, dtype, aligned):
    """Enough rows that a part of the prefix has twenty or more 64-key tiles: the ring of stages goes round, both P buffers are used again,
    and the maximum of growing keys moves after O holds sums; beside it caches with about a thousand keys in a split.  Not aligned: the
    same wide parts on the split kernel."""
    b, h, hkv, nq, d, p, s = case
    q, kp, vp, k, v = _inputs(b, h, hkv, nq, d, p, s, dtype, scale=1.5)
    kp = (kp.float() * torch.linspace(0.05, 1.6, p, device="cuda")[:, None]).to(dtype)
    k = (k.float() * torch.linspace(0.5, 2.0, s, device="cuda")[:, None]).to(dtype)
    if not aligned:
        kp, vp = (torch.cat((t.new_zeros(1), t.flatten()))[1:].view(t.shape) for t in (kp, vp))
    prefix_parts, own_parts = _planned_parts(dtype, *case)
    assert p / prefix_parts >= 20 * 64 and own_parts == -(-s // 1024)
    lengths = torch.randint(0, s + 1, (b,), generator=torch.Generator().manual_seed(4), dtype=torch.int32)
    lengths[:5] = torch.tensor([s, s - 1, min(s, 1024), 17, 0])
    for i, n in enumerate(lengths.tolist()):
        k[i, :, n:], v[i, :, n:] = float("nan"), float("inf")
    got = E.shared_prefix_attention(q, kp, vp, k, v, lengths=lengths.cuda())
    for rows in (slice(0, 6), slice(62, 66), slice(b - 3, b)):
        _check(got[rows], q[rows], kp, vp, k[rows], v[rows], lengths=lengths[rows])
    assert torch.equal(got, E.shared_prefix_attention(q, kp, vp, k, v, lengths=lengths.cuda()))


def test_many_tiles_of_one_split_fp32():
    case = (200, 8, 8, 1, 64, 3001, 1100)
    q, kp, vp, k, v = _inputs(*case, torch.float32, scale=1.5)
    kp *= torch.linspace(0.05, 1.6, 3001, device="cuda")[:, None]
    prefix_parts, own_parts = _planned_parts(torch.float32, *case)
    assert 3001 / prefix_parts >= 128 and own_parts <= 2
    got = E.shared_prefix_attention(q, kp, vp, k, v)
    for rows in (slice(0, 4), slice(197, 200)):
        _check(got[rows], q[rows], kp, vp, k[rows], v[rows])

"""Rotary positions against the definition in 64 bits: layouts, strides, positions, types, both directions, in place."""
import pytest
import torch

import elsa_b200 as E

pytestmark = pytest.mark.gpu


def _inputs(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype).cuda()


def _reference(x, frequencies, positions, interleaved, magnitude=1.0, inverse=False):
    """(y, size of the summands of each element) in 64 bits"""
    r = 2 * frequencies.shape[0]
    angle = positions.double()[..., None] * frequencies * (-1 if inverse else 1)
    if angle.dim() == 2:
        angle = angle[None]
    cos, sin = torch.cos(angle)[:, None] * magnitude, torch.sin(angle)[:, None] * magnitude
    y = x.double().clone()
    size = torch.zeros_like(y)
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    xa, xb = x[..., a].double(), x[..., b].double()
    y[..., a], y[..., b] = xa * cos - xb * sin, xb * cos + xa * sin
    size[..., a] = size[..., b] = (xa.abs() + xb.abs()) * magnitude
    return y, size


def _check(got, x, frequencies, positions, interleaved, **kw):
    y, size = _reference(x, frequencies, positions, interleaved, **kw)
    # one rounding to the type (half a step, or half the smallest fp16 step); in fp32: cosine and sine to 2 * 2^-24 each (their own
    # rounding and the magnitude's), two products and a sum: 5 roundings of 2^-24 of the summands, taken as 8
    limit = torch.finfo(x.dtype).eps / 2 * y.abs() * 1.01 + 8 * 2.0 ** -24 * size
    if x.dtype == torch.float16:
        limit = limit + 2.0 ** -25
    bad = (got.double() - y).abs() > limit
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} elements, worst {(got.double() - y).abs().max().item()}"


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,h,hkv,n,d,r", [(1, 1, 1, 1, 64, 64), (3, 4, 2, 37, 64, 64), (2, 8, 8, 129, 128, 128), (2, 3, 1, 65, 80, 40),
                                           (1, 5, 5, 7, 96, 96), (1, 2, 2, 33, 10, 6), (64, 8, 2, 1, 128, 64), (1, 2, 1, 300, 256, 256),
                                           (1, 2, 1, 9, 2, 2)])
def test_values(interleaved, dtype, b, h, hkv, n, d, r):
    q, k = _inputs((b, h, n, d), dtype, 1), _inputs((b, hkv, n, d), dtype, 2)
    f = E.rotary_frequencies(r, device="cuda")[0]
    pos = torch.randint(0, 1 << 20, (b, n), generator=torch.Generator().manual_seed(3)).cuda()
    q2, k2 = E.rotary_embedding(q, k, f, positions=pos, interleaved=interleaved)
    _check(q2, q, f, pos, interleaved)
    _check(k2, k, f, pos, interleaved)


def test_positions_of_every_form():
    q = _inputs((3, 2, 50, 64), torch.float32, 4)
    f, g = E.rotary_frequencies(64, scaling="yarn", factor=8.0, original_positions=512, device="cuda")
    ar = torch.arange(50, device="cuda")
    for pos in (None, ar, ar.int(), (ar * 3 - 40)[None], torch.stack((ar, ar + 7, -ar)).int(), torch.stack((ar, ar + 2 ** 33, ar * 1000))[:, :],
                torch.arange(100, device="cuda")[::2], torch.arange(300, device="cuda").view(50, 6).t()[:3]):
        out = E.rotary_embedding(q, None, f, positions=pos, magnitude=g)
        _check(out, q, f, ar if pos is None else pos, False, magnitude=g)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["packed", "bnhd", "odd_offset", "odd_stride", "strided_d", "expanded"])
def test_strided_inputs_are_read_as_they_are(layout, interleaved):
    dtype, b, h, n, d = torch.bfloat16, 2, 4, 21, 64
    if layout == "packed":
        q, k, _ = _inputs((b, n, 3, h, d), dtype, 5).permute(2, 0, 3, 1, 4).unbind(0)
    elif layout == "bnhd":
        q, k = _inputs((b, n, h, d), dtype, 5).transpose(1, 2), _inputs((b, n, h, d), dtype, 6).transpose(1, 2)
    elif layout == "odd_offset":
        q, k = _inputs((b, h, n, d + 3), dtype, 5)[..., 3:], _inputs((b * h * n * d + 1,), dtype, 6)[1:].view(b, h, n, d)
    elif layout == "odd_stride":
        q, k = _inputs((b, h, n, d + 1), dtype, 5)[..., :d], _inputs((b, h, 2 * n, d), dtype, 6)[:, :, ::2]
    elif layout == "strided_d":
        q, k = _inputs((b, h, n, 2 * d), dtype, 5)[..., ::2], _inputs((b, h, d, n), dtype, 6).transpose(2, 3)
    else:
        q, k = _inputs((1, h, n, d), dtype, 5).expand(b, h, n, d), _inputs((b, 1, n, d), dtype, 6).expand(b, h, n, d)
    f = E.rotary_frequencies(32, device="cuda")[0]
    pos = torch.arange(n, device="cuda") + 1000
    q0, k0 = q.clone(), k.clone()
    q2, k2 = E.rotary_embedding(q, k, f, positions=pos, interleaved=interleaved)
    assert torch.equal(q, q0) and torch.equal(k, k0)
    _check(q2, q, f, pos, interleaved)
    _check(k2, k, f, pos, interleaved)
    if layout == "bnhd":
        assert q2.transpose(1, 2).is_contiguous()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r", [(64, 64), (64, 24), (10, 4)])
def test_in_place(interleaved, d, r):
    qkv = _inputs((2, 19, 3, 4, d), torch.float16, 7)
    keep = qkv.clone()
    q, k, v = qkv.permute(2, 0, 3, 1, 4).unbind(0)
    f = E.rotary_frequencies(r, device="cuda")[0]
    pos = torch.arange(19, device="cuda")
    q1, k1 = E.rotary_embedding(q, k, f, positions=pos, interleaved=interleaved)
    version = qkv._version
    q2, k2 = E.rotary_embedding(q, k, f, positions=pos, interleaved=interleaved, inplace=True)
    assert q2 is q and k2 is k and qkv._version > version
    assert torch.equal(q, q1) and torch.equal(k, k1) and torch.equal(v, keep.permute(2, 0, 3, 1, 4)[2])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_gradients(interleaved, dtype):
    q = _inputs((2, 4, 33, 64), dtype, 8).requires_grad_(True)
    k = _inputs((2, 1, 33, 64), dtype, 9).requires_grad_(True)
    f, g = E.rotary_frequencies(48, device="cuda")[0], 1.25
    pos = torch.arange(33, device="cuda") * 17
    dq, dk = _inputs((2, 33, 4, 64), dtype, 10).transpose(1, 2), _inputs((2, 1, 33, 64), dtype, 11)
    q2, k2 = E.rotary_embedding(q, k, f, positions=pos, interleaved=interleaved, magnitude=g)
    gq, gk = torch.autograd.grad((q2, k2), (q, k), (dq, dk), retain_graph=True)
    _check(gq, dq, f, pos, interleaved, magnitude=g, inverse=True)
    _check(gk, dk, f, pos, interleaved, magnitude=g, inverse=True)
    # one gradient alone, and an expanded one (a sum's)
    assert torch.equal(torch.autograd.grad(q2, q, dq, retain_graph=True)[0], gq)
    assert torch.equal(torch.autograd.grad(k2, k, dk, retain_graph=True)[0], gk)
    ones = torch.autograd.grad(q2.sum(), q)[0]
    _check(ones, torch.ones_like(q), f, pos, interleaved, magnitude=g, inverse=True)


def test_gradient_against_differences():
    """A linear map: the difference over any step is the derivative, up to the roundings of two fp32 results."""
    q = _inputs((1, 2, 5, 16), torch.float32, 12).requires_grad_(True)
    f = E.rotary_frequencies(16, device="cuda")[0]
    weights = _inputs((1, 2, 5, 16), torch.float32, 13)
    out = E.rotary_embedding(q, None, f)
    grad, = torch.autograd.grad(out, q, weights)
    base = (out.detach().double() * weights.double()).sum()
    for at in ((0, 0, 0, 0), (0, 1, 3, 9), (0, 0, 4, 15), (0, 1, 1, 7)):
        moved = q.detach().clone()
        moved[at] += 4.0
        diff = ((E.rotary_embedding(moved, None, f).double() * weights.double()).sum() - base) / 4.0
        # two outputs change, each by an amount known to 8 * 2^-24 of summands of at most ~10
        assert abs(diff.item() - grad[at].item()) < 2 * 8 * 2.0 ** -24 * 10 * float(weights.abs().max())


def test_special_values_stay_in_their_pair():
    q = _inputs((1, 1, 3, 16), torch.float32, 14)
    q[0, 0, 1, 2] = float("inf")
    f = E.rotary_frequencies(16, device="cuda")[0]
    out = E.rotary_embedding(q, None, f)
    clean = q.clone()
    clean[0, 0, 1, 2] = 0.0
    ref = E.rotary_embedding(clean, None, f)
    same = torch.ones(16, dtype=torch.bool)
    same[[2, 10]] = False
    assert torch.equal(out[..., same], ref[..., same]) and not bool(torch.isfinite(out[0, 0, 1, [2, 10]]).any())


def test_empty_and_refused_calls():
    f = E.rotary_frequencies(16, device="cuda")[0]
    q = _inputs((2, 2, 4, 16), torch.float16, 15)
    for shape in ((0, 2, 4, 16), (2, 2, 0, 16), (2, 0, 4, 16)):
        e = torch.empty(shape, device="cuda", dtype=torch.float16)
        assert E.rotary_embedding(e, None, f).shape == e.shape
    q2, k2 = E.rotary_embedding(q, q[:, :0], f)
    assert k2.shape == (2, 0, 4, 16) and torch.equal(q2, E.rotary_embedding(q, None, f))
    for args, kw, match in (((q.double(), None, f), {}, "dtypes"), ((q, q.float(), f), {}, "dtype"), ((q, None, f.float()), {}, "float64"),
                            ((q, None, f.cpu()), {}, "float64"), ((q, None, torch.ones(9, device="cuda", dtype=torch.float64)), {}, "head_dim"),
                            ((q, None, f), dict(positions=torch.zeros(4, device="cuda")), "int32"),
                            ((q, None, f), dict(positions=torch.zeros(4, dtype=torch.int64)), "int32"),
                            ((q, None, f), dict(positions=torch.zeros(5, dtype=torch.int64, device="cuda")), "positions"),
                            ((q, None, f), dict(positions=torch.zeros((3, 4), dtype=torch.int64, device="cuda")), "positions"),
                            ((q[:1].expand(2, 2, 4, 16), None, f), dict(inplace=True), "overlap"), ((q, q, f), dict(inplace=True), "different"),
                            ((q.transpose(2, 3)[:, :, :, :4].contiguous().transpose(2, 3), None, f), dict(inplace=True), "contiguous"),
                            ((q.float().requires_grad_(True), None, f), dict(inplace=True), "gradients")):
        with pytest.raises(ValueError, match=match):
            E.rotary_embedding(*args, **kw)


def test_another_stream_and_a_captured_call():
    q, k = _inputs((2, 4, 64, 64), torch.float16, 16), _inputs((2, 4, 64, 64), torch.float16, 17)
    f, pos = E.rotary_frequencies(64, device="cuda")[0], torch.arange(64, device="cuda")
    want = E.rotary_embedding(q, k, f, positions=pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = E.rotary_embedding(q, k, f, positions=pos)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = E.rotary_embedding(q, k, f, positions=pos)
    q.copy_(q.flip(2).clone())
    pos.add_(100)
    graph.replay()
    again = E.rotary_embedding(q, k, f, positions=pos)
    assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])


def test_in_place_refuses_q_and_k_that_share_elements():
    f = E.rotary_frequencies(16, device="cuda")[0]
    pool = _inputs((2, 19, 6, 16), torch.float16, 31)
    keep = pool.clone()
    heads = pool.transpose(1, 2)
    for q, k in ((heads[:, :4], heads[:, 3:]), (heads, heads), (heads[:, :4, :10], heads[:, 2:, 9:])):
        q, k = q[:, :, :k.shape[2]], k[:, :, :q.shape[2]]
        with pytest.raises(ValueError, match="different memory"):
            E.rotary_embedding(q, k, f, inplace=True)
    assert torch.equal(pool, keep)
    want = E.rotary_embedding(heads[:, :4], heads[:, 4:], f)
    E.rotary_embedding(heads[:, :4], heads[:, 4:], f, inplace=True)
    assert torch.equal(heads, torch.cat(want, 1))


def test_frequencies_that_ask_for_a_gradient_are_refused():
    """They would get none: a call must not drop it in silence."""
    q = _inputs((1, 2, 5, 16), torch.float32, 32)
    f = E.rotary_frequencies(16, device="cuda")[0].requires_grad_(True)
    with pytest.raises(ValueError, match="no gradient"):
        E.rotary_embedding(q, None, f)
    with torch.no_grad():
        want = E.rotary_embedding(q, None, f)
    assert torch.equal(E.rotary_embedding(q, None, f.detach()), want)

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


# ---- gradients ---------------------------------------------------------------------------------------------------------
def _gradients(q, k, v, lam, dout, causal, scale=None):
    """(gradients, limits) in 64 bits, from the formulas.  The limits, with h the half step of the type (2^-24 for fp32), per map m:
      P        the weight's own error e (as in the forward)
      D        g . (P V): the saved output's rounding h, of sum_d |g_d| mass_d (mass = P |V|), and SUMS for P V and the dot
      G        64 or 128 products: (Dv + 8) 2^-24 of sum |g||v|
      dS       P (G - D): P e |G - D| + P (err G + err D), then one rounding h of it (16-bit: the second product's operand)
      products sums of at most `terms` roundings of 2^-24 (a tile's accumulators; the FMA kernels add key after key), each operand's error
               times the other operand's size; then one rounding h of the result"""
    b, h, hkv, nq, nk, d = q.shape[0], q.shape[1] // 2, v.shape[1], q.shape[2], k.shape[2], q.shape[3]
    scale = d ** -0.5 if scale is None else scale
    u, half = 2.0 ** -24, torch.finfo(q.dtype).eps / 2
    op = half if q.dtype != torch.float32 else 0.0           # operands of the second products are rounded to 16-bit types only
    grads = [torch.zeros(t.shape, device=q.device, dtype=torch.float64) for t in (q, k, v)] + [torch.zeros(h, device=q.device, dtype=torch.float64)]
    limits = [torch.zeros_like(t) for t in grads]
    terms = (max(nq, nk) + 64) * u
    for i in range(b):
        for j in range(h):
            maps, g, _ = _maps(q, k, lam, causal, None, scale, i, j, hkv)
            w = float(lam[j]) if isinstance(lam, torch.Tensor) and lam.numel() > 1 else float(lam)
            go, val = dout[i, j].double(), v[i, g].double()
            gv, gv_size = go @ val.T, go.abs() @ val.abs().T
            e_gv = (v.shape[3] + 8) * u * gv_size
            outs = [m.p @ val for m in maps]
            mass = [m.p @ val.abs() for m in maps]
            out_size = mass[0] + abs(w) * mass[1]
            dd = [(go * o).sum(-1, keepdim=True) for o in outs]
            # D2 from the saved P2 V; D1 = g . out + lam D2 with the saved out
            e_o = [(m.e + SUMS + op) * s for m, s in zip(maps, mass)]
            e_d2 = (go.abs() * (e_o[1] + half * outs[1].abs() * 1.01 + 2.0 ** -25)).sum(-1, keepdim=True) + 140 * u * (go.abs() * mass[1]).sum(-1, keepdim=True)
            e_out = e_o[0] + abs(w) * e_o[1] + half * (outs[0] - w * outs[1]).abs() * 1.01 + 2.0 ** -25
            e_d1 = (go.abs() * e_out).sum(-1, keepdim=True) + abs(w) * e_d2 + 280 * u * (go.abs() * out_size).sum(-1, keepdim=True)
            sign = (1.0, -w)
            ds, e_ds = [], []
            for m, mp, dm, e_dm in zip((0, 1), maps, dd, (e_d1, e_d2)):
                x = mp.p * (gv - dm)
                ex = mp.p * (e_gv + e_dm + 4 * u * (gv.abs() + dm.abs())) + mp.e * x.abs()
                ds.append(sign[m] * x)
                e_ds.append(abs(sign[m]) * (ex + op * (x.abs() + ex) + 2.0 ** -26 * (op > 0)))     # (2^-26: fp16 below its normal range)
            pc = maps[0].p - w * maps[1].p
            e_pc = maps[0].p * maps[0].e + abs(w) * maps[1].p * maps[1].e
            e_pc = e_pc + op * (pc.abs() + e_pc) + 4 * u * (maps[0].p + abs(w) * maps[1].p) + 2.0 ** -26 * (op > 0)
            for m in (0, 1):
                qm, km = q[i, 2 * j + m].double(), k[i, 2 * g + m].double()
                grads[0][i, 2 * j + m] += scale * ds[m] @ km
                limits[0][i, 2 * j + m] += scale * (e_ds[m] + terms * ds[m].abs()) @ km.abs()
                grads[1][i, 2 * g + m] += scale * ds[m].T @ qm
                limits[1][i, 2 * g + m] += scale * (e_ds[m] + (h // hkv) * terms * ds[m].abs()).T @ qm.abs()
            grads[2][i, g] += pc.T @ go
            limits[2][i, g] += (e_pc + (h // hkv) * terms * pc.abs()).T @ go.abs()
            grads[3][j] -= dd[1].sum()
            # dlam is summed from P2 and G in fp32, not from the rounded outputs: the weight's error, G's, and the additions
            limits[3][j] += (maps[1].p * (maps[1].e * gv.abs() + e_gv)).sum() + (nk + 600) * u * (maps[1].p * gv.abs()).sum()
    for t, lim in zip(grads, limits):
        lim += half * t.abs() * 1.01 + 2.0 ** -25
    return grads, limits


def _run_train(q, k, v, lam, dout, **kw):
    leaves = [t.detach().clone().requires_grad_(True) if isinstance(t, torch.Tensor) else t for t in (q, k, v, lam)]
    out = E.differential_attention_train(*leaves, **kw)
    return out.detach(), torch.autograd.grad(out, [t for t in leaves if isinstance(t, torch.Tensor)], dout)


def _check_gradients(got, q, k, v, lam, dout, causal=False, scale=None):
    grads, limits = _gradients(q, k, v, lam, dout, causal, scale)
    names = ("dq", "dk", "dv", "dlam")
    if len(got) == 4 and got[3].numel() == 1 and grads[3].numel() > 1:
        grads[3], limits[3] = grads[3].sum().view(got[3].shape), limits[3].sum().view(got[3].shape)
        if got[3].dtype != q.dtype:
            limits[3] = limits[3] + torch.finfo(got[3].dtype).eps * grads[3].abs()
    for name, a, b, lim in zip(names, got, grads, limits):
        if name == "dlam":
            lim = lim + torch.finfo(a.dtype).eps / 2 * b.abs() * 1.01
        err = (a.double() - b.view(a.shape)).abs()
        assert bool((err <= lim.view(a.shape)).all()), f"{name}: {float((err / lim.view(a.shape)).max())} of the limit"
    assert _lib.load().elsa_device_status(0) == 0


TRAIN = [
    # b, h, hkv, nq, nk, d, dv
    (1, 1, 1, 1, 1, 64, 128), (2, 2, 1, 5, 9, 32, 64), (1, 2, 2, 65, 65, 64, 128), (2, 4, 4, 128, 128, 64, 128), (1, 4, 1, 129, 300, 64, 128),
    (1, 2, 2, 257, 257, 32, 64), (1, 3, 3, 200, 500, 48, 96), (2, 2, 2, 300, 90, 64, 128), (1, 1, 1, 320, 640, 8, 16), (1, 2, 1, 70, 513, 64, 64),
    (1, 2, 2, 100, 260, 64, 72), (1, 2, 2, 33, 70, 128, 128), (2, 2, 1, 90, 33, 20, 12), (1, 1, 1, 66, 40, 7, 5),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", TRAIN, ids=str)
def test_gradients(case, dtype, causal):
    q, k, v, lam = _inputs(*case, dtype)
    dout = _normal((case[0], case[1], case[3], case[6]), dtype, 20)
    out, got = _run_train(q, k, v, lam, dout, is_causal=causal)
    _check_forward(out, q, k, v, lam, causal=causal)
    _check_gradients(got, q, k, v, lam, dout, causal)
    again = _run_train(q, k, v, lam, dout, is_causal=causal)[1]
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_of_lam_in_its_own_type_and_shape(dtype):
    q, k, v, lam = _inputs(2, 4, 2, 100, 100, 64, 128, dtype)
    dout = _normal((2, 4, 100, 128), dtype, 21)
    for lam in (lam, lam.bfloat16(), torch.tensor(0.4, device="cuda"), torch.tensor([0.4], device="cuda", dtype=torch.float16)):
        out, got = _run_train(q, k, v, lam, dout)
        assert got[3].shape == lam.shape and got[3].dtype == lam.dtype
        _check_gradients(got, q, k, v, lam, dout)
    out, got = _run_train(q, k, v, 0.4, dout)
    assert len(got) == 3
    _check_gradients(got, q, k, v, 0.4, dout)
    # one value expanded over the heads: its gradient is the sum
    one = torch.tensor([0.4], device="cuda", requires_grad=True)
    E.differential_attention_train(q, k, v, one.expand(4)).backward(dout)
    single = _run_train(q, k, v, one, dout)[1][3]
    assert abs(float(one.grad) - float(single)) <= 2.0 ** -20 * float(_gradients(q, k, v, one.detach(), dout, False)[0][3].abs().sum()) + 4 * 2.0 ** -24


def test_gradients_against_differences():
    """fp32, along random directions: (f(x + e u) - f(x - e u)) / 2e with e = 2^-6 is off by e^2 / 6 times a third derivative and by the
    roundings of the two sums, 2^-24 times the 768 summands' size over e."""
    q, k, v, lam = _inputs(1, 2, 1, 12, 12, 16, 32, torch.float32)
    dout = _normal((1, 2, 12, 32), torch.float32, 22)
    got = _run_train(q, k, v, lam, dout, is_causal=True)[1]
    leaves = [q, k, v, lam]
    e = 2.0 ** -6

    def f(args):
        return float((E.differential_attention(*args, is_causal=True).double() * dout.double()).sum())

    def exact(args):                 # the same function in 64 bits, to know the third-order term
        total = 0.0
        for j in range(2):
            maps, g, _ = _maps(args[0], args[1], args[3], True, None, None, 0, j, 1)
            total += float((dout[0, j].double() * ((maps[0].p - float(args[3][j]) * maps[1].p) @ args[2][0, g].double())).sum())
        return total

    for n in range(4):
        u = _normal(leaves[n].shape, torch.float32, 30 + n)
        step = lambda s: [x + s * u if i == n else x for i, x in enumerate(leaves)]
        diff = (f(step(e)) - f(step(-e))) / (2 * e)
        third = abs((exact(step(2 * e)) - exact(step(-2 * e))) / (4 * e) - (exact(step(e)) - exact(step(-e))) / (2 * e))   # = e^2 / 2 f'''
        rounding = 2 * 2.0 ** -20 * float(dout.abs().sum()) / e / 16
        assert abs(diff - float((got[n].double() * u.double()).sum())) <= third + rounding


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["bnhd", "odd_offset", "strided_d", "expanded_dout", "expanded_kv"])
def test_strided_training(layout, dtype):
    q, k, v, lam = _inputs(2, 4, 2, 90, 90, 64, 128, dtype)
    dout = _normal((2, 4, 90, 128), dtype, 23)
    if layout == "bnhd":
        q, k, v, dout = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, dout))
    elif layout == "odd_offset":
        q, k, v, dout = (torch.cat((t.new_zeros(1), t.flatten()))[1:].view(t.shape) for t in (q, k, v, dout))
    elif layout == "strided_d":
        q, k, v, dout = (t.repeat_interleave(2, -1)[..., ::2] for t in (q, k, v, dout))
    elif layout == "expanded_dout":
        dout = torch.ones((), device="cuda", dtype=dtype).expand(2, 4, 90, 128)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
    args = list(leaves)
    if layout == "expanded_kv":
        leaves[1] = k[:1].detach().clone().requires_grad_(True)
        args[1] = leaves[1].expand_as(k)
    out = E.differential_attention_train(*args, is_causal=True)
    got = list(torch.autograd.grad(out, args, dout))
    _check_gradients(got, *(t.detach() for t in args), dout, causal=True)


def test_some_inputs_without_gradients_and_no_keys():
    q, k, v, lam = _inputs(1, 2, 2, 70, 70, 64, 128, torch.float16)
    k.requires_grad_(True)
    out = E.differential_attention_train(q, k, v, lam)
    out.sum().backward()
    assert k.grad is not None and q.grad is None and lam.grad is None
    e = torch.empty((1, 4, 0, 64), device="cuda", dtype=torch.float16, requires_grad=True)
    q.requires_grad_(True)
    out = E.differential_attention_train(q, e, v[:, :, :0], lam)
    out.sum().backward()
    assert not bool(out.any()) and not bool(q.grad.any()) and e.grad.shape == e.shape


def test_a_changed_input_is_noticed():
    q, k, v, lam = _inputs(1, 1, 1, 70, 70, 64, 128, torch.float16)
    q.requires_grad_(True)
    out = E.differential_attention_train(q, k, v, lam)
    k.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_training_step_on_another_stream_and_captured(dtype):
    q, k, v, lam = (t.requires_grad_(True) for t in _inputs(1, 4, 2, 200, 200, 64, 128, dtype))
    dout = _normal((1, 4, 200, 128), dtype, 24)

    def step():
        out = E.differential_attention_train(q, k, v, lam, is_causal=True)
        return (out,) + torch.autograd.grad(out, (q, k, v, lam), dout)

    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        q.copy_(q.flip(2).clone())
    graph.replay()
    torch.cuda.synchronize()
    fresh = step()
    assert all(torch.equal(a, b) for a, b in zip(held, fresh))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_training_without_keys_is_zeros_whatever_q_holds(dtype):
    q, k, v, lam = _inputs(2, 2, 1, 300, 0, 64, 128, dtype)
    q.fill_(100.0)                                     # (the sum of q is infinite in fp16)
    q[1, 0, 7, 3] = float("nan")
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
    out = E.differential_attention_train(*leaves)
    assert out.shape == (2, 2, 300, 128) and out.dtype == dtype and not bool(out.any())
    grads = torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert all(g.shape == t.shape and not bool(g.any()) for g, t in zip(grads, leaves))


@pytest.mark.parametrize("scale", [1e-46, 1e39, float("inf"), float("nan"), 0.0])
def test_a_scale_that_fp32_does_not_hold_is_refused(scale):
    """(one that is zero there would turn masked scores into NaN)"""
    q, k, v, lam = _inputs(1, 2, 2, 150, 150, 64, 128, torch.float16)
    for call in (E.differential_attention, E.differential_attention_train):
        with pytest.raises(ValueError, match="scale"):
            call(q, k, v, lam, is_causal=True, scale=scale)


def test_training_with_more_sequences_than_the_tile_kernels_grid():
    q, k, v, lam = _inputs(33000, 1, 1, 1, 2, 8, 8, torch.float16)
    dout = _normal((33000, 1, 1, 8), torch.float16, 9)
    out, got = _run_train(q, k, v, lam, dout)
    for rows in (slice(0, 20), slice(32980, 33000)):
        _check_forward(out[rows], q[rows], k[rows], v[rows], lam)
        _check_gradients([g[rows] for g in got[:3]], q[rows], k[rows], v[rows], lam, dout[rows])


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b", [20, 40])
def test_gradients_with_tiles_of_one_two_and_four_blocks(b, causal):
    """Blocks of the fp32 kernels share a tile while there are few tiles: 640 or 320 of queries, 400 or 200 of keys."""
    q, k, v, lam = _inputs(b, 4, 2, 128, 150, 64, 128, torch.float32)
    dout = _normal((b, 4, 128, 128), torch.float32, 20)
    out, got = _run_train(q, k, v, lam, dout, is_causal=causal)
    _check_forward(out, q, k, v, lam, causal=causal)
    _check_gradients(got, q, k, v, lam, dout, causal)
    assert all(torch.equal(x, y) for x, y in zip(got, _run_train(q, k, v, lam, dout, is_causal=causal)[1]))



def test_tiles_ask_for_no_workspace():
    from tests.test_decoder_cpu import _differential_bytes
    lib = _lib.load()
    for batch, heads, kv, n in ((2, 4, 2, 300), (2, 8, 8, 8192), (1, 16, 16, 32768), (1, 32, 8, 65536), (1, 16, 16, 131072)):
        assert _differential_bytes(lib, batch, heads, kv, n, n) == 0
        assert _differential_bytes(lib, batch, heads, kv, n, n, out=4104) == lib.elsa_differential_workspace_bytes(2, batch, heads, kv, n, n, 64, 128) > 0


def _peak(call):
    """(result, bytes that the call had allocated at its fullest, what it returned among them)"""
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    result = call()
    torch.cuda.synchronize()
    return result, torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("native", [True, False])
def test_a_long_prompt_allocates_what_it_returns(native, monkeypatch):
    """16 heads of 32768 tokens: the result, for a training step its state, and no scratch that grows with queries times keys."""
    if not native:
        monkeypatch.setattr(_lib, "host", lambda: None)
    n, h, d, dv = 32768, 16, 64, 128
    q, k, v = (torch.randn((1, heads, n, width), device="cuda", dtype=torch.bfloat16) for heads, width in ((2 * h, d), (2 * h, d), (h, dv)))
    lam = torch.full((h,), 0.5, device="cuda")
    out_bytes, state_bytes = h * n * dv * 2, 2 * h * n * 4
    out, peak = _peak(lambda: E.differential_attention(q, k, v, lam, is_causal=True))
    assert peak <= out_bytes + 2 ** 22
    _check_forward(out[:, :1, -3:].contiguous(), q[:, :2, -3:], k[:, :2], v[:, :1], lam[:1], causal=True)
    q.requires_grad_(True)
    out2, peak = _peak(lambda: E.differential_attention_train(q, k, v, lam, is_causal=True))
    assert torch.equal(out2, out) and peak <= 2 * out_bytes + state_bytes + 2 ** 22


def _rows(q, k, t0, t1):
    """What queries t0 .. t1 of a causal call are to a call of their own: themselves and the keys up to the last one's."""
    return q[:, :, t0:t1], k[:, :, : k.shape[2] - q.shape[2] + t1]


@pytest.mark.parametrize("case", [(1, 2, 1, 9000, 65536, 64, 128), (9, 16, 16, 1001, 16001, 32, 64)], ids=str)
def test_queries_in_chunks(case):
    """Summaries of more than 1 GiB: the split kernels take tokens of a sequence, or whole sequences, in turn.  Rows on either side of the
    chunks' borders (8064 tokens; 7 sequences), their saved P2 v and sums among them."""
    b, h, hkv, nq, nk, d, dv = case
    q, k, v, lam = _inputs(*case, torch.float32)
    (out, out2, lse, *_), peak = _peak(lambda: E.differential._forward(q, k, v, lam, (b, h, hkv, nq, nk, d, dv), True, d ** -0.5, None, True))
    assert peak <= 2 ** 30 + sum(t.numel() * 4 for t in (out, out2, lse)) + 2 ** 22
    for i in {0, 6, 7, b - 1} & set(range(b)):
        one = slice(i, i + 1)
        for t0, t1 in ((0, 3), (nq // 2, nq // 2 + 2), (min(8062, nq - 4), min(8066, nq)), (nq - 3, nq)):
            qs, ks = _rows(q[one], k[one], t0, t1)
            vs = v[one, :, : ks.shape[2]]
            _check_forward(out[one, :, t0:t1], qs, ks, vs, lam, causal=True)
            for j in {0, h - 1}:
                maps, g, _ = _maps(qs, ks, lam, True, None, None, 0, j, hkv)
                want = maps[1].p @ vs[0, g].double()
                limit = (maps[1].e + SUMS) * (maps[1].p @ vs[0, g].double().abs()) + 2.0 ** -24 * want.abs() * 1.01 + 2.0 ** -25
                assert bool(((out2[i, j, t0:t1].double() - want).abs() <= limit).all())
                # (a sum of weights is off by e and SUMS of itself, its log2 by that / ln 2; one rounding of the result, of the maximum and of the sum)
                for m in (0, 1):
                    off = (lse[m, i, j, t0:t1].double() - maps[m].lse2).abs()
                    assert bool((off <= 1.5 * (maps[m].e[:, 0] + SUMS) + 3 * 2.0 ** -24 * (maps[m].lse2.abs() + 32)).all())


@pytest.mark.parametrize("causal", [False, True])
def test_queries_of_caches_with_lengths_in_chunks(causal):
    """As above, bf16, behind caches of different lengths: shorter than a chunk's first query's, empty, full."""
    b, h, hkv, nq, nk, d, dv = 4, 4, 1, 9000, 32768, 64, 128
    q, k, v, lam = _inputs(b, h, hkv, nq, nk, d, dv, torch.bfloat16)
    lengths = torch.tensor([0, 700, 20001, nk], dtype=torch.int32)
    for i, n in enumerate(lengths.tolist()):
        k[i, :, n:], v[i, :, n:] = float("nan"), float("inf")
    got = E.differential_attention(q, k, v, lam, is_causal=causal, lengths=lengths.cuda())
    assert not bool(got[0].any())
    for i, n in enumerate(lengths.tolist()):
        for t0, t1 in ((0, 2), (8062, 8066), (nq - n - 1, nq - n + 2), (nq - 3, nq)):
            if 0 <= t0 < t1 <= nq:
                last = n - nq + t1 if causal else n             # keys that the last of these rows sees
                if last <= 0:
                    assert not bool(got[i, :, t0:t1].any())
                    continue
                _check_forward(got[i:i + 1, :, t0:t1], q[i:i + 1, :, t0:t1], k[i:i + 1, :, :last], v[i:i + 1, :, :last], lam, causal=causal)


def _planned_parts(dtype, b, h, hkv, nq, nk, d, dv):
    """Parts of the keys that the split kernels take (from the bytes of their summaries; calls of one chunk)."""
    every = _lib.load().elsa_differential_workspace_bytes({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype], b, h, hkv, nq, nk, d, dv)
    return every // (2 * b * h * nq * (dv + 2) * 4)          # (padding: less than a part's)


@pytest.mark.parametrize("growing", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", [(64, 8, 8, 1, 2000, 64, 128), (64, 32, 8, 3, 1500, 64, 128), (70, 8, 8, 2, 1025, 32, 64), (48, 16, 8, 9, 1300, 48, 96)], ids=str)
def test_many_keys_of_one_split(case, dtype, growing):
    """Enough caches that a split has about a thousand keys: a warp's ring of stages goes round many times, its sources move on, and sums
    gather over its chunks -- up to 8 rows of a key head and more, caches that end anywhere in a split.  Growing keys: the maximum
    moves again and again after there are sums."""
    b, h, hkv, nq, nk, d, dv = case
    q, k, v, lam = _inputs(*case, dtype, scale=2.0 if growing else 1.0)
    if growing:
        k = (k.float() * torch.linspace(0.05, 2.0, nk, device="cuda")[:, None]).to(dtype)
    parts = _planned_parts(dtype, *case)
    assert parts == -(-nk // 1024)                           # 16 chunks of 16 keys for each warp
    lengths = torch.randint(0, nk + 1, (b,), generator=torch.Generator().manual_seed(4), dtype=torch.int32)
    lengths[:6] = torch.tensor([nk, nk - 1, 1024, 1023, 65, 0])
    for i, n in enumerate(lengths.tolist()):
        k[i, :, n:], v[i, :, n:] = float("nan"), float("inf")
    got = E.differential_attention(q, k, v, lam, is_causal=True, lengths=lengths.cuda())
    for rows in (slice(0, 8), slice(b - 3, b)):
        # (what stands behind the last key: NaN would reach the definition's products)
        _check_forward(got[rows], q[rows], torch.nan_to_num(k[rows]), torch.nan_to_num(v[rows], posinf=0.0), lam, causal=True, lengths=lengths[rows])
    assert torch.equal(got, E.differential_attention(q, k, v, lam, is_causal=True, lengths=lengths.cuda()))


@pytest.mark.parametrize("causal", [False, True])
def test_many_keys_of_one_split_fp32(causal):
    """As above for the kernel of any type: a block's 32-key tiles, the running maximum, sums over them."""
    case = (40, 8, 8, 5, 2100, 64, 128)
    q, k, v, lam = _inputs(*case, torch.float32, scale=2.0)
    k *= torch.linspace(0.05, 2.0, 2100, device="cuda")[:, None]
    assert _planned_parts(torch.float32, *case) <= 6         # at least ten tiles each
    _check_forward(E.differential_attention(q, k, v, lam, is_causal=causal)[-4:], q[-4:], k[-4:], v[-4:], lam, causal=causal)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
def test_growing_scores_over_many_tiles(causal, dtype):
    """The tile kernel, 33 key tiles: the maximum moves again and again after O holds sums."""
    case = (1, 2, 1, 150, 2083, 64, 128)
    q, k, v, lam = _inputs(*case, dtype, scale=2.0)
    k = (k.float() * torch.linspace(0.05, 2.0, 2083, device="cuda")[:, None]).to(dtype)
    _check_forward(E.differential_attention(q, k, v, lam, is_causal=causal), q, k, v, lam, causal=causal)
    q = q * 0.25                                             # (gradients: weights of more than one key)
    dout = _normal((1, 2, 150, 128), dtype, 21)
    out, got = _run_train(q, k, v, lam, dout, is_causal=causal)
    _check_gradients(got, q, k, v, lam, dout, causal)

"""CPU checks of the decoder-side operators: what they refuse, in Python and at the C ABI, and the host-side formulas."""
import math

import pytest
import torch

import elsa_b200 as E


@pytest.fixture(scope="module")
def lib():
    from elsa_b200 import _lib, build
    build.build()
    return _lib.load()


# ---- rotary -----------------------------------------------------------------------------------------------------
def test_rotary_frequencies_plain_and_scaled():
    plain, one = E.rotary_frequencies(8, base=10000.0)
    assert plain.dtype == torch.float64 and one == 1.0
    assert plain.tolist() == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-14)
    linear, _ = E.rotary_frequencies(8, scaling="linear", factor=4.0)
    assert torch.allclose(linear, plain / 4, rtol=1e-15)
    ntk, _ = E.rotary_frequencies(8, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and float(ntk[-1]) == pytest.approx(float(plain[-1]) / 4, rel=1e-12)


def test_rotary_yarn_keeps_fast_pairs_and_divides_slow_ones():
    r, original, factor = 128, 4096, 16.0
    plain, _ = E.rotary_frequencies(r)
    yarn, magnitude = E.rotary_frequencies(r, scaling="yarn", factor=factor, original_positions=original)
    assert magnitude == pytest.approx(0.1 * math.log(factor) + 1.0)
    turns = plain * original / (2 * math.pi)
    index = torch.arange(r // 2)
    fast, slow = index[turns > 32.0][:-1], index[turns < 1.0][1:]     # (the borders round outward by at most one pair)
    assert len(fast) > 5 and len(slow) > 5
    assert torch.equal(yarn[fast], plain[fast])
    assert torch.allclose(yarn[slow], plain[slow] / factor, rtol=1e-14)
    ratio = (yarn / plain)
    assert bool((ratio[1:] <= ratio[:-1] + 1e-15).all()) and float(ratio.min()) >= 1 / factor - 1e-15


@pytest.mark.parametrize("kwargs,match", [
    (dict(rotary_dim=7), "rotary_dim"), (dict(rotary_dim=0), "rotary_dim"), (dict(rotary_dim=258), "rotary_dim"),
    (dict(rotary_dim=8, base=0.0), "base"), (dict(rotary_dim=8, base=math.inf), "base"),
    (dict(rotary_dim=8, scaling="cubic"), "scaling"), (dict(rotary_dim=8, scaling="linear", factor=0.5), "factor"),
    (dict(rotary_dim=2, scaling="ntk", factor=2.0), "rotary_dim"), (dict(rotary_dim=8, scaling="yarn", factor=2.0), "original"),
    (dict(rotary_dim=8, scaling="yarn", factor=2.0, original_positions=64, beta_fast=1.0, beta_slow=2.0), "beta_fast"),
])
def test_rotary_frequencies_refusals(kwargs, match):
    with pytest.raises(ValueError, match=match):
        E.rotary_frequencies(**kwargs)


def test_rotary_embedding_refuses_cpu_tensors_and_wrong_shapes():
    q, f = torch.randn(1, 2, 8, 4), torch.ones(2, dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA"):
        E.rotary_embedding(q, None, f)
    with pytest.raises(ValueError, match="shape"):
        E.rotary_embedding(q[0], None, f)
    with pytest.raises(ValueError, match="agree"):
        E.rotary_embedding(q, q[:, :, :4], f)


def test_rotary_overlap_check():
    from elsa_b200.rotary import _overlaps
    base = torch.zeros(2, 3, 5, 8)
    assert not _overlaps(base) and not _overlaps(base.transpose(1, 2)) and not _overlaps(base[:, :, ::2])
    assert _overlaps(base[:1].expand(4, 3, 5, 8)) and _overlaps(base.as_strided((2, 3, 5, 8), (120, 40, 4, 1)))
    assert not _overlaps(base[:1, :1, :1])


def _elements(t):
    at = t.storage_offset()
    return {at + b * t.stride(0) + h * t.stride(1) + n * t.stride(2) + d for b in range(t.shape[0]) for h in range(t.shape[1])
            for n in range(t.shape[2]) for d in range(t.shape[3])}


@pytest.mark.parametrize("seed", range(8))
def test_rotary_in_place_tells_views_that_share_elements(seed):
    from elsa_b200 import rotary
    gen = torch.Generator().manual_seed(seed)
    pick = lambda n: int(torch.randint(n, (), generator=gen))
    found = {False: 0, True: 0}
    for _ in range(200):
        b, n, width, d = 1 + pick(3), 1 + pick(4), 4 + pick(3), 2 * (1 + pick(3))
        pool = torch.zeros(b * n * width * d + 16)
        x = pool[:b * n * width * d].view(b, n, width * d)
        if pick(4) == 0:                    # heads in front of tokens
            x = pool[:b * n * width * d].view(b, width, n * d)
            views = [x.view(b, width, n, d)] * 2
        else:
            shift = pick(2) * pick(d)       # half of a head's columns, or whole ones
            views = [x[:, :, :(width - 1) * d].view(b, n, width - 1, d).transpose(1, 2),
                     x[:, :, shift:shift + (width - 1) * d].unflatten(2, (width - 1, d)).transpose(1, 2)]
        total = views[0].shape[1]
        q, k = (v[:, (at := pick(total)):at + 1 + pick(total - at)] for v in views)
        want = bool(_elements(q) & _elements(k))
        found[want] += 1
        assert rotary._meet(q, k) == want
        assert rotary._meet(k, q) == want
    assert min(found.values()) > 20
    q = torch.zeros(1, 2, 4, 8)
    assert rotary._meet(q, q.transpose(1, 2)) and not rotary._meet(q, torch.zeros(1, 2, 4, 8))


def test_rotary_abi_refuses_before_any_launch(lib):
    import ctypes
    st = (ctypes.c_int64 * 6)(512, 256, 64, 512, 256, 64)
    other = (ctypes.c_int64 * 6)(512, 256, 64, 512, 64, 256)

    def call(q=64, q_out=128, strides=st, heads=2, k=None, k_out=None, ks=None, kh=0, freq=64, pos=None, pos_bytes=0, dtype=1, batch=1,
             n=4, d=64, r=64):
        return lib.elsa_rotary(q, q_out, strides, heads, k, k_out, ks, kh, freq, pos, pos_bytes, 0, 1, 1.0, dtype, batch, n, d, r, 0, 0, None)

    assert call(q=None) == 1 and call(q_out=None) == 1 and call(strides=None) == 1 and call(freq=None) == 1
    assert call(heads=0) == 1 and call(n=0) == 1 and call(batch=0) == 1 and call(dtype=9) == 1
    assert call(k=64) == 1 and call(k=64, k_out=64, ks=st, kh=0) == 1
    assert call(r=65) == 2 and call(r=0) == 2 and call(d=64, r=128) == 2 and call(d=2048) == 2 and call(d=512, r=512) == 2
    assert call(pos=64, pos_bytes=0) == 1 and call(pos=None, pos_bytes=8) == 1 and call(pos=64, pos_bytes=2) == 1
    assert call(q=64, q_out=64, strides=other) == 1


# ---- attention over a shared prefix --------------------------------------------------------------------------------
def test_shared_prefix_refuses_before_any_launch(lib):
    import ctypes
    q, kp, k = torch.zeros(2, 4, 1, 16), torch.zeros(2, 5, 16), torch.zeros(2, 2, 3, 16)
    with pytest.raises(ValueError, match="CUDA"):
        E.shared_prefix_attention(q, kp, kp, k, k)
    with pytest.raises(ValueError, match="multiple"):
        E.shared_prefix_attention(q[:, :3], kp, kp, k, k)
    size = lib.elsa_shared_prefix_workspace_bytes
    assert size(1, 2, 4, 2, 1, 64, 100, 50) > 0 and size(1, 2, 4, 2, 1, 64, 0, 0) == 0
    for bad in ((9, 2, 4, 2, 1, 64, 100, 50), (1, 0, 4, 2, 1, 64, 100, 50), (1, 2, 4, 3, 1, 64, 100, 50), (1, 2, 4, 2, 0, 64, 100, 50),
                (1, 2, 4, 2, 1, 129, 100, 50), (1, 2, 4, 2, 1, 64, -1, 50), (1, 1 << 28, 4, 2, 1, 64, 100, 50)):
        assert size(*bad) == -1
    st = (ctypes.c_int64 * 16)(*([64] * 16))

    def call(q=256, kp=256, k=256, out=256, strides=st, ws=256, nbytes=1 << 40, dtype=1, batch=2, heads=4, kv=2):
        return lib.elsa_shared_prefix_attention(q, kp, kp, k, k, out, strides, None, ws, nbytes, dtype, batch, heads, kv, 1, 64, 100, 50, 0.125, None)

    assert call(q=None) == 1 and call(kp=None) == 1 and call(k=None) == 1 and call(out=None) == 1 and call(strides=None) == 1
    assert call(dtype=5) == 1 and call(kv=3) == 1 and call(batch=-1) == 1
    assert call(ws=None) == 4 and call(ws=128) == 4 and call(nbytes=1000) == 4


def test_shared_prefix_splits_cover_every_key(lib):
    """Summaries for every part, whatever the sizes (the workspace holds m, z and D sums of each row and part)."""
    for batch, heads, kv, nq, d, p, s in ((1, 1, 1, 1, 64, 1, 1), (256, 32, 8, 1, 128, 32768, 2048), (8, 8, 8, 1, 64, 512, 128), (24, 12, 3, 5, 96, 4097, 333)):
        rows = batch * heads // kv * nq
        least = 2 * kv * rows * (d + 2) * 4
        assert lib.elsa_shared_prefix_workspace_bytes(2, batch, heads, kv, nq, d, p, s) >= least


# ---- differential attention -----------------------------------------------------------------------------------------
def test_differential_lambda():
    a = [torch.randn(3, 8, generator=torch.Generator().manual_seed(i)) for i in range(4)]
    got = E.differential_lambda(*a, 0.3)
    want = torch.exp((a[0] * a[1]).sum(-1)) - torch.exp((a[2] * a[3]).sum(-1)) + 0.3
    assert torch.allclose(got, want) and got.dtype == torch.float32
    assert E.differential_lambda(*(x.bfloat16() for x in a), 0.3).dtype == torch.float32


def test_differential_refuses_before_any_launch(lib):
    import ctypes
    q, k, v = torch.zeros(1, 4, 3, 16), torch.zeros(1, 4, 5, 16), torch.zeros(1, 2, 5, 32)
    with pytest.raises(ValueError, match="CUDA"):
        E.differential_attention(q, k, v, 0.5)
    with pytest.raises(ValueError, match="two heads"):
        E.differential_attention(q[:, :3], k, v, 0.5)
    size = lib.elsa_differential_workspace_bytes
    assert size(1, 1, 4, 2, 3, 100, 64, 128) > 0 and size(1, 1, 4, 2, 3, 0, 64, 128) == 0
    for bad in ((9, 1, 4, 2, 3, 100, 64, 128), (1, 1, 4, 3, 3, 100, 64, 128), (1, 1, 4, 2, 0, 100, 64, 128), (1, 1, 4, 2, 3, 100, 129, 128),
                (1, 1, 4, 2, 3, 100, 64, 129), (1, 1, 4, 2, 3, -1, 64, 128), (1, 70000, 4, 2, 3, 100, 64, 128)):
        assert size(*bad) == -1
    st = (ctypes.c_int64 * 12)(*([64] * 12))

    def call(q=256, k=256, v=256, lam=256, lam_dtype=0, out=256, strides=st, ws=256, nbytes=1 << 40, dtype=1, heads=4, kv=2, scale=0.125):
        return lib.elsa_differential_forward(q, k, v, lam, lam_dtype, 0, None, out, strides, None, None, ws, nbytes, dtype, 1, heads, kv, 3, 100,
                                             64, 128, 0, scale, None)

    for name in ("q", "k", "v", "lam", "out", "strides"):
        assert call(**{name: None}) == 1
    assert call(lam_dtype=7) == 1 and call(dtype=7) == 1 and call(kv=3) == 1 and call(scale=0.0) == 1 and call(scale=float("nan")) == 1
    assert call(scale=1e-46) == 1 and call(scale=float("inf")) == 1 and call(scale=3e38) == 1
    assert call(ws=None) == 4 and call(ws=100) == 4 and call(nbytes=100) == 4


def test_differential_backward_refuses_before_any_launch(lib):
    import ctypes
    q, k, v = torch.zeros(1, 4, 3, 16), torch.zeros(1, 4, 5, 16), torch.zeros(1, 2, 5, 32)
    with pytest.raises(ValueError, match="CUDA"):
        E.differential_attention_train(q, k, v, 0.5)
    size = lib.elsa_differential_backward_workspace_bytes
    assert size(1, 2, 4, 2, 3, 100, 64, 128) >= 2 * 4 * (4 * 128 + 1) * 4 and size(1, 2, 4, 2, 3, 100, 64, 130) == -1
    st = (ctypes.c_int64 * 24)(*([64] * 24))

    def call(strides=st, ws=256, nbytes=1 << 40, dtype=1, lam_dtype=0, scale=0.125, **null):
        ptr = [None if name in null else 256 for name in ("q", "k", "v", "lam")]
        more = [None if name in null else 256 for name in ("out", "out2", "lse", "dout", "dq", "dk", "dv", "dlam")]
        return lib.elsa_differential_backward(*ptr, lam_dtype, 1, *more, strides, ws, nbytes, dtype, 2, 4, 2, 3, 100, 64, 128, 0, scale, None)

    for name in ("q", "k", "v", "lam", "out", "out2", "lse", "dout", "dq", "dk", "dv"):
        assert call(**{name: 0}) == 1
    assert call(strides=None) == 1 and call(dtype=8) == 1 and call(lam_dtype=8) == 1 and call(scale=-1.0) == 1
    assert call(ws=None) == 4 and call(ws=64) == 4 and call(nbytes=64) == 4


def test_axes_that_32_bits_do_not_count_are_refused():
    """(expanded: no memory behind them)"""
    long = lambda *shape: torch.zeros((1,) * len(shape)).expand(shape)
    n = 2 ** 32 + 1
    with pytest.raises(ValueError, match="an axis of more than"):
        E.rotary_embedding(long(1, 1, n, 2), None, torch.ones(1, dtype=torch.float64))
    with pytest.raises(ValueError, match="an axis of more than"):
        E.shared_prefix_attention(long(1, 1, 1, 8), long(1, n, 8), long(1, n, 8), long(1, 1, 4, 8), long(1, 1, 4, 8))
    for call in (E.differential_attention, E.differential_attention_train):
        with pytest.raises(ValueError, match="an axis of more than"):
            call(long(1, 2, 1, 8), long(1, 2, n, 8), long(1, 1, n, 8), 0.5)



# ---- what the calls ask for ------------------------------------------------------------------------------------------
def _differential_bytes(lib, batch, heads, kv, nq, nk, d=64, dv=128, dtype=2, q=4096, out=4096, lengths=None):
    """Of contiguous operands (nothing is read through the addresses)."""
    import ctypes
    st = (ctypes.c_int64 * 12)(2 * heads * nq * d, nq * d, d, 2 * kv * nk * d, nk * d, d, kv * nk * dv, nk * dv, dv, heads * nq * dv, nq * dv, dv)
    return lib.elsa_differential_workspace_bytes_for(q, 4096, 4096, lengths, out, st, dtype, batch, heads, kv, nq, nk, d, dv)


def test_differential_workspace_of_a_layout(lib):
    """What the tiles do not take goes through the split kernels, with their summaries (what they take: test_gpu_differential.py)."""
    sizes = (2, 4, 2, 100, 300)
    every = lib.elsa_differential_workspace_bytes(2, *sizes, 64, 128)
    assert every > 0 and _differential_bytes(lib, *sizes, lengths=4096) == every
    assert _differential_bytes(lib, *sizes, q=4098) == every and _differential_bytes(lib, *sizes, out=4104) == every
    assert _differential_bytes(lib, *sizes, dtype=0) == lib.elsa_differential_workspace_bytes(0, *sizes, 64, 128)
    assert _differential_bytes(lib, 2, 4, 2, 1, 300) == lib.elsa_differential_workspace_bytes(2, 2, 4, 2, 1, 300, 64, 128)
    assert _differential_bytes(lib, 1, 4, 3, 100, 300) == -1 and _differential_bytes(lib, *sizes, d=136) == -1
    assert lib.elsa_differential_workspace_bytes_for(4096, 4096, 4096, None, 4096, None, 2, *sizes, 64, 128) == -1


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_differential_summaries_are_bounded(lib, dtype):
    """The split kernels' summaries, queries times parts of the keys: no call asks for more than 1 GiB of them."""
    size = lib.elsa_differential_workspace_bytes
    for batch, heads, kv, nq, nk in ((2, 8, 8, 8192, 8192), (1, 16, 16, 32768, 32768), (1, 32, 8, 65536, 65536), (1, 16, 16, 131072, 131072),
                                     (1, 128, 1, 1, 1 << 23), (1, 65535, 1, 1, 1 << 20), (4096, 32, 8, 4, 8192), (1, 1, 1, 1 << 20, 1 << 20)):
        assert 0 < size(dtype, batch, heads, kv, nq, nk, 64, 128) <= (1 << 30) + 1024
    # small calls: every summary at once, as before
    parts = -(-100 // 64)
    assert size(dtype, 2, 4, 2, 3, 100, 64, 128) == 2 * 512 + parts * 2 * 4 * 2 * 3 * 128 * 4


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_shared_prefix_summaries_are_bounded(lib, dtype):
    size = lib.elsa_shared_prefix_workspace_bytes
    for batch, heads, kv, nq, d, p, s in ((64, 32, 8, 4096, 128, 8192, 8192), (1, 32, 8, 32768, 128, 0, 32768), (3, 32, 8, 8000, 128, 2000, 8192),
                                          (1, 128, 1, 1, 128, 1 << 23, 1 << 23), (4096, 32, 8, 8, 128, 100000, 4096)):
        assert 0 < size(dtype, batch, heads, kv, nq, d, p, s) <= (1 << 30) + 1024
    # small calls: every summary at once, as before
    assert size(dtype, 2, 4, 2, 1, 64, 100, 50) == 2 * 256 + (2 + 1) * 2 * 2 * 2 * 64 * 4


@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("rotary", [True, False])
def test_packed_attention_checks_backward_hints_with_and_without_rotary(rotary, train):
    from elsa_b200.attention_bwd import twopass_attention_qkvpacked
    qkv = torch.zeros(1, 4, 3, 2, 16)
    kw = {"rotary": E.Rotary(E.rotary_frequencies(16)[0])} if rotary else {}
    with pytest.raises(ValueError, match="input_precision"):
        twopass_attention_qkvpacked(qkv, train=train, bwd_input_precision="fp4", **kw)
    with pytest.raises(ValueError, match="num_warps"):
        twopass_attention_qkvpacked(qkv, train=train, bwd_num_warps=3, **kw)
    with pytest.raises(ValueError, match="CUDA"):
        twopass_attention_qkvpacked(qkv, train=train, bwd_input_precision="tf32", bwd_num_warps=4, bwd_block_m=64, **kw)

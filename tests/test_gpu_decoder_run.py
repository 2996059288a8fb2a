"""The decoder operators as they are used together: a training step through rotary positions and differential attention, decoding over
a prefix that a batch shares, decoding with differential attention over growing caches, rotary positions in the packed path and the ViT
hooks."""
import pytest
import torch

import elsa_b200 as E
from elsa_b200.attention_bwd import twopass_attention_qkvpacked

pytestmark = pytest.mark.gpu


def _normal(shape, seed, dtype=torch.float16, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def _turn64(x, frequencies, positions):
    """The definition in 64 bits: [B, H, N, D], half layout, positions [N] or [B, N]"""
    r = 2 * frequencies.shape[0]
    angle = (positions if positions.dim() == 2 else positions[None]).double()[:, None, :, None] * frequencies
    a, b = x[..., : r // 2], x[..., r // 2: r]
    return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), x[..., r:]), -1)


def _rel(got, want):
    return float((got.double() - want).norm() / want.norm())


# Relative 2-norm of the difference.  Every fp16 rounding of an intermediate is at most 2^-11 of it: the turned q and k (their scores
# move by sqrt(2) 2^-11 of their size, of order 1), the weights, the outputs and, in a backward, dS and the gradient that is turned back:
# eight independent ones at the full half step, of which none is amplified by more than 2 (softmax's gradient): 2 sqrt(8) 2^-11.
LIMIT = 2 * 8 ** 0.5 * 2.0 ** -11


def test_a_training_step_of_a_differential_layer():
    b, n, h, hkv, d, width = 2, 150, 4, 2, 32, 96
    w = {name: _normal((cols, width), i, scale=width ** -0.5) for i, (name, cols) in enumerate((("q", 2 * h * d), ("k", 2 * hkv * d), ("v", hkv * 2 * d)))}
    lam_vectors = [_normal((d,), 10 + i, torch.float32, 0.1) for i in range(4)]
    x, dout = _normal((b, n, width), 20), _normal((b, h, n, 2 * d), 21)
    frequencies, _ = E.rotary_frequencies(d, device="cuda")
    positions = torch.arange(n, device="cuda")
    leaves = [x, *w.values(), *lam_vectors]
    for t in leaves:
        t.requires_grad_(True)

    def heads(y, count, dim):
        return y.view(b, n, count, dim).transpose(1, 2)

    q, k, v = heads(x @ w["q"].T, 2 * h, d), heads(x @ w["k"].T, 2 * hkv, d), heads(x @ w["v"].T, hkv, 2 * d)
    q, k = E.rotary_embedding(q, k, frequencies, positions=positions)
    out = E.differential_attention_train(q, k, v, E.differential_lambda(*lam_vectors, 0.2), is_causal=True)
    got = (out,) + torch.autograd.grad(out, leaves, dout)

    leaves64 = [t.detach().double().requires_grad_(True) for t in leaves]
    x64, wq, wk, wv, *l64 = leaves64
    q, k, v = heads(x64 @ wq.T, 2 * h, d), heads(x64 @ wk.T, 2 * hkv, d), heads(x64 @ wv.T, hkv, 2 * d)
    q, k = _turn64(q, frequencies, positions), _turn64(k, frequencies, positions)
    lam = torch.exp((l64[0] * l64[1]).sum()) - torch.exp((l64[2] * l64[3]).sum()) + 0.2
    k, v = (t.view(b, hkv, -1, n, t.shape[-1]).repeat_interleave(h // hkv, 1).flatten(1, 2) for t in (k, v))
    p = torch.softmax((q @ k.transpose(-1, -2) * d ** -0.5).masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), float("-inf")), -1)
    want_out = (p[:, 0::2] - lam * p[:, 1::2]) @ v
    want = (want_out,) + torch.autograd.grad(want_out, leaves64, dout.double())
    # (the projections round x W and their gradients to fp16 as well: twice the limit)
    for name, a, c in zip(("out", "x", "wq", "wk", "wv", "l1", "l2", "l3", "l4"), got, want):
        assert _rel(a, c) <= 2 * LIMIT, name


@pytest.mark.parametrize("batch", [3, 40])
def test_decoding_behind_a_shared_prefix(batch):
    """Every step: turn the new token's q and k, put k and v into each sequence's cache, attend.  Against full causal attention over each
    sequence's whole history."""
    h, hkv, d, prefix, room, steps = 8, 2, 64, 150, 24, 6
    frequencies, magnitude = E.rotary_frequencies(d, scaling="yarn", factor=4.0, original_positions=64, device="cuda")
    kp_raw, vp = _normal((1, hkv, prefix, d), 1), _normal((hkv, prefix, d), 2)
    kp = E.rotary_embedding(kp_raw, None, frequencies, magnitude=magnitude)[0]
    k_cache, v_cache = (torch.full((batch, hkv, room, d), float("nan"), device="cuda", dtype=torch.float16) for _ in range(2))
    lengths = torch.randint(0, 10, (batch,), generator=torch.Generator().manual_seed(3)).int().cuda()
    history_k, history_v = [], []
    for i, n in enumerate(lengths.tolist()):                    # what each sequence has said so far
        k_raw, v = _normal((1, hkv, n, d), 100 + i), _normal((hkv, n, d), 200 + i)
        if n:
            k_cache[i, :, :n] = E.rotary_embedding(k_raw, None, frequencies, positions=prefix + torch.arange(n, device="cuda"), magnitude=magnitude)[0]
        v_cache[i, :, :n] = v
        history_k.append(torch.cat((kp_raw[0], k_raw[0]), 1).double())
        history_v.append(torch.cat((vp, v), 1).double())
    for step in range(steps):
        q_raw, k_raw, v = _normal((batch, h, 1, d), 300 + step), _normal((batch, hkv, 1, d), 400 + step), _normal((batch, hkv, 1, d), 500 + step)
        q, k = E.rotary_embedding(q_raw, k_raw, frequencies, positions=(prefix + lengths.long())[:, None], magnitude=magnitude)
        at = lengths.long()[:, None, None, None].expand(batch, hkv, 1, d)
        k_cache.scatter_(2, at, k)
        v_cache.scatter_(2, at, v)
        lengths += 1
        out = E.shared_prefix_attention(q, kp, vp, k_cache, v_cache, lengths=lengths)
        for i in range(batch):
            history_k[i], history_v[i] = torch.cat((history_k[i], k_raw[i].double()), 1), torch.cat((history_v[i], v[i].double()), 1)
            n = history_k[i].shape[1]
            turned = _turn64(history_k[i][None], frequencies, torch.arange(n, device="cuda"))[0] * magnitude
            query = _turn64(q_raw[i].double()[None], frequencies, torch.tensor([n - 1], device="cuda"))[0] * magnitude
            w = torch.softmax(query @ turned.repeat_interleave(h // hkv, 0).transpose(1, 2) * d ** -0.5, -1)
            assert _rel(out[i], w @ history_v[i].repeat_interleave(h // hkv, 0)) <= LIMIT


@pytest.mark.parametrize("new", [1, 3])
def test_decoding_with_differential_attention_agrees_with_the_whole_sequence(new):
    b, h, hkv, n, d = 2, 4, 2, 140, 64
    q, k, v = _normal((b, 2 * h, n, d), 1), _normal((b, 2 * hkv, n, d), 2), _normal((b, hkv, n, 2 * d), 3)
    lam = torch.tensor([0.2, 0.4, 0.6, 0.8], device="cuda")
    whole = E.differential_attention(q, k, v, lam, is_causal=True)
    room_k, room_v = (torch.full((b, t.shape[1], 200, t.shape[3]), float("nan"), device="cuda", dtype=torch.float16) for t in (k, v))
    room_k[:, :, :n], room_v[:, :, :n] = k, v
    for end in (new, 64, 65, n):
        got = E.differential_attention(q[:, :, end - new:end], room_k, room_v, lam, is_causal=True, lengths=torch.full((b,), end, dtype=torch.int32, device="cuda"))
        assert _rel(got, whole[:, :, end - new:end].double()) <= LIMIT


@pytest.mark.parametrize("train", [False, True])
def test_rotary_positions_in_the_packed_path(train):
    qkv = _normal((2, 130, 3, 4, 64), 1).requires_grad_(train)
    rotary = E.Rotary(E.rotary_frequencies(32, device="cuda")[0], torch.arange(130, device="cuda") + 7, True, 1.25)
    out = twopass_attention_qkvpacked(qkv, is_causal=True, train=train, rotary=rotary)
    q, k, v = qkv.permute(2, 0, 3, 1, 4).unbind(0)
    q, k = E.rotary_embedding(q, k, rotary.frequencies, positions=rotary.positions, interleaved=True, magnitude=1.25)
    want = (E.twopass_attention_train if train else E.twopass_attention)(q, k, v, is_causal=True)
    assert torch.equal(out, want) and out.transpose(1, 2).is_contiguous()
    if train:
        dout = _normal((2, 4, 130, 64), 2)
        got, = torch.autograd.grad(out, qkv, dout)
        ref, = torch.autograd.grad(want, qkv, dout)
        # (the 16-bit backward adds dq in arrival order)
        assert _rel(got, ref.double()) <= 1e-3


@pytest.mark.parametrize("norms", [False, True])
def test_rotary_positions_in_the_vit_hooks(norms):
    from elsa_b200.vision import VitAttention
    module = VitAttention(128, 2).cuda().half().eval()
    if norms:
        module.q_norm, module.k_norm = torch.nn.LayerNorm(64).cuda().half(), torch.nn.LayerNorm(64).cuda().half()
    rotary = E.Rotary(E.rotary_frequencies(64, device="cuda")[0])
    x = _normal((2, 90, 128), 3)
    holder, plain = torch.nn.Sequential(module), module
    assert E.patch_timm_attention(holder, elsa_kwargs={"rotary": rotary}).vit_attention == 1
    with torch.no_grad():
        got = holder(x)
        q, k, v = plain.qkv(x).reshape(2, 90, 3, 2, 64).permute(2, 0, 3, 1, 4).unbind(0)
        q, k = rotary.apply(plain.q_norm(q), plain.k_norm(k))
        w = torch.softmax(q.double() @ k.double().transpose(-1, -2) * 64 ** -0.5, -1)
        want = torch.nn.functional.linear((w @ v.double()).transpose(1, 2).reshape(2, 90, 128), plain.proj.weight.double(), plain.proj.bias.double())
    assert _rel(got, want) <= LIMIT


def test_rotary_positions_are_refused_for_swin_windows():
    from tests.standins import SwinWindowAttention
    with pytest.raises(ValueError, match="rotary"):
        E.patch_timm_attention(torch.nn.Sequential(SwinWindowAttention(32, 2, (7, 7))), elsa_kwargs={"rotary": E.Rotary(E.rotary_frequencies(16)[0])})


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_whose_offsets_pass_32_bits(dtype):
    """Rows 2^23 elements apart: the last ones begin behind element 2^31."""
    n, step = 300, 2 ** 23
    pool = torch.empty(n * step, dtype=dtype, device="cuda")

    def spread(t, at):
        view = pool[at:].as_strided(t.shape, (t.shape[1] * t.shape[3], t.shape[3], step, 1))
        return view.copy_(t)

    gen = torch.Generator().manual_seed(5)
    q, k, v, dout = (torch.randn(shape, generator=gen).to(dtype).cuda() for shape in ((1, 4, n, 64), (1, 2, n, 64), (1, 1, n, 128), (1, 2, n, 128)))
    far = [spread(t, 1024 * i) for i, t in enumerate((q, k, v, dout))]
    assert far[0][0, 0, -1].data_ptr() - pool.data_ptr() > 2 ** 31 * pool.element_size()
    f, lam = E.rotary_frequencies(64, device="cuda")[0], torch.tensor([0.3, 0.6], device="cuda")
    for got, want in zip(E.rotary_embedding(far[0], far[1], f), E.rotary_embedding(q, k, f)):
        assert torch.equal(got, want)
    for nq in (1, n):                       # the decoding form and the tiles
        assert torch.equal(E.differential_attention(far[0][:, :, n - nq:], far[1], far[2], lam, is_causal=True),
                           E.differential_attention(q[:, :, n - nq:].contiguous(), k, v, lam, is_causal=True))
    grads = []
    for args, g in (((q, k, v), dout), (far[:3], far[3])):
        leaves = [t.detach().requires_grad_(True) for t in args]
        grads.append(torch.autograd.grad(E.differential_attention_train(*leaves, lam, is_causal=True), leaves, g))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    # the prefix's rows for many and for few queries, the own caches beside it
    for b in (1, 40):
        qs = torch.randn((b, 4, 1, 64), generator=gen).to(dtype).cuda()
        own = torch.randn((b, 2, 50, 64), generator=gen).to(dtype).cuda()
        assert torch.equal(E.shared_prefix_attention(qs, far[1][0], far[1][0], own, own), E.shared_prefix_attention(qs, k[0], k[0], own, own))


def test_calls_from_several_threads():
    import threading
    gen = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(shape, generator=gen).half().cuda() for shape in ((2, 4, 200, 64), (2, 2, 200, 64), (2, 1, 200, 128)))
    f, lam = E.rotary_frequencies(64, device="cuda")[0], torch.tensor([0.3, 0.6], device="cuda")
    qs, own = (torch.randn(shape, generator=gen).half().cuda() for shape in ((40, 4, 1, 64), (40, 2, 50, 64)))

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        turned = E.rotary_embedding(leaves[0], leaves[1], f)
        out = E.differential_attention_train(*turned, leaves[2], lam, is_causal=True)
        return [out.detach(), *torch.autograd.grad(out, leaves, v.repeat(1, 2, 1, 1)), E.shared_prefix_attention(qs, k[0], k[0], own, own),
                E.differential_attention(q[:, :, :1], k, v, lam)]

    want = step()
    torch.cuda.synchronize()
    failures = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = step()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    failures.append(threading.get_ident())

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


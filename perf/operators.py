"""Performance cases of the decoder-side operators: rotary positions, attention over a shared prefix, differential attention.

A case is a dict of plain values; "op" names the operator and the rest are its sizes:

  rotary        q [B, H, N, D] and k [B, Hkv, N, D] turned by position-dependent angles in their first `rot` dimensions
                (pairs (i, i + rot/2), or neighbours where `interleaved`), positions `far` apart from 0 at most;
                `train`: the gradients of q and k too
  prefix        queries q [B, H, Nq, D] of a batch over one prefix cache [Hkv, P, D] that all sequences share and a cache
                of their own [B, Hkv, S, D] with a length for each sequence
  differential  out = (softmax(q1 k1^T s) - lam softmax(q2 k2^T s)) v with q [B, 2H, Nq, D], k [B, 2Hkv, Nk, D],
                v [B, Hkv, Nk, Dv], lam [H]; `causal`, `train` (gradients of q, k, v, lam too), `ragged` (a length of the
                key cache for each sequence)
"""
from __future__ import annotations

import math

import torch

own = False         # False: the plain forms below; True: the package's operators


def _rotary(b, h, hkv, n, d, rot, dtype, *, interleaved=False, train=False, far=131072, factor=1.0, name=None):
    c = {"op": "rotary", "b": b, "h": h, "hkv": hkv, "n": n, "d": d, "rot": rot, "dtype": dtype, "interleaved": interleaved,
         "train": train, "far": far, "factor": factor}
    return c if name is None else dict(c, name=name)


def _prefix(b, h, hkv, nq, d, p, s, dtype, name=None):
    c = {"op": "prefix", "b": b, "h": h, "hkv": hkv, "nq": nq, "d": d, "p": p, "s": s, "dtype": dtype}
    return c if name is None else dict(c, name=name)


def _differential(b, h, hkv, nq, nk, d, dv, dtype, *, causal=True, train=False, ragged=False, name=None):
    c = {"op": "differential", "b": b, "h": h, "hkv": hkv, "nq": nq, "nk": nk, "d": d, "dv": dv, "dtype": dtype,
         "causal": causal, "train": train, "ragged": ragged}
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one decoding step of 64 sequences, each at a far position of its own: the smallest call, latency counts
        _rotary(64, 32, 8, 1, 128, 128, "bfloat16", name="rotary_token"),
        # a long prompt with grouped key heads, positions interpolated by a factor of 8
        _rotary(1, 32, 8, 16384, 128, 128, "bfloat16", far=16384, factor=8.0, name="rotary_prompt"),
        # a training step: half of each head turned, neighbouring pairs, an odd length
        _rotary(4, 16, 16, 4097, 64, 32, "float16", interleaved=True, train=True, far=4097, name="rotary_train"),
        # a few sequences behind a short instruction: little work, latency counts
        _prefix(8, 8, 8, 1, 64, 512, 128, "float16", name="prefix_small"),
        # 64 conversations behind one long instruction, grouped key heads
        _prefix(64, 32, 8, 1, 128, 8192, 1024, "bfloat16", name="prefix_serving"),
        # 256 samples drawn from one very long document
        _prefix(256, 32, 8, 1, 128, 32768, 2048, "bfloat16", name="prefix_samples"),
        # five drafted tokens of each sequence at once; odd sizes everywhere
        _prefix(24, 12, 3, 5, 96, 4097, 333, "float16", name="prefix_draft"),
        # a short training step without a mask, ragged tiles
        _differential(2, 4, 4, 257, 257, 32, 64, "float16", causal=False, train=True, name="diff_short_train"),
        # a causal training step at 8192 tokens: the largest case
        _differential(2, 8, 8, 8192, 8192, 64, 128, "bfloat16", train=True, name="diff_long_train"),
        # fp32 training at a thousand tokens
        _differential(1, 4, 4, 1000, 1000, 64, 128, "float32", train=True, name="diff_fp32_train"),
        # one decoding step over caches of different lengths, grouped key heads
        _differential(16, 16, 4, 1, 8192, 64, 128, "bfloat16", ragged=True, name="diff_token"),
        # a piece of a long prompt over everything before it
        _differential(1, 16, 4, 1024, 8192, 64, 128, "float16", name="diff_prompt_piece"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges; its work stays below that of the largest listed case."""
    op = rng.choice(("rotary", "prefix", "prefix", "differential", "differential"))
    half = rng.choice(("float16", "bfloat16"))
    if op == "rotary":
        dtype = rng.choice((half, half, "float32"))
        d = rng.choice((32, 64, 80, 96, 128))
        rot = rng.choice((d, d, d // 2))
        hkv, group = rng.choice((1, 4, 8, 16)), rng.choice((1, 1, 4))
        budget = (1 << 27) // (hkv * (group + 1) * d * (2 if dtype == "float32" else 1))      # tokens of the batch
        n = _log_int(rng, 1, min(32768, budget))
        b = _log_int(rng, 1, max(1, min(64, budget // n)))
        far = max(n, _log_int(rng, 1024, 1 << 20))
        return _rotary(b, hkv * group, hkv, n, d, rot, dtype, interleaved=rng.random() < 0.4, train=rng.random() < 0.5, far=far,
                       factor=rng.choice((1.0, 1.0, 4.0)))
    if op == "prefix":
        dtype = rng.choice((half, half, half, "float32"))
        most = 16 if dtype == "float32" else 256
        d = rng.choice((32, 64, 96, 128))
        hkv, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 8))
        nq = rng.choice((1, 1, 1, 2, 5))
        p = _log_int(rng, 16, 4096 if dtype == "float32" else 32768)
        s = _log_int(rng, max(1, nq), 1024)
        b = _log_int(rng, 1, max(1, min(most, 65536 // (hkv * group * nq * 2))))
        return _prefix(b, hkv * group, hkv, nq, d, p, s, dtype)
    dtype = rng.choice((half, half, half, "float32"))
    d = rng.choice((32, 48, 64, 64))
    dv = 2 * d
    hkv, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 1, 2, 4))
    h = hkv * group
    kind = rng.choice(("train", "train", "token", "piece"))
    longest = 2048 if dtype == "float32" else 8192
    if kind == "train":
        n = _log_int(rng, 64, longest)
        b = _log_int(rng, 1, max(1, min(16, (1 << 28) // (h * n * n), 8 if dtype == "float32" else 16)))
        if h * n * n > 1 << 29:
            h = hkv = 4
        return _differential(b, h, hkv, n, n, d, dv, dtype, causal=rng.random() < 0.6, train=True)
    nk = _log_int(rng, 64, longest)
    if kind == "token":
        return _differential(_log_int(rng, 1, 4 if dtype == "float32" else 32), h, hkv, rng.choice((1, 1, 2, 4)), nk, d, dv, dtype, ragged=True)
    return _differential(1, h, hkv, _log_int(rng, 16, min(nk, 2048)), nk, d, dv, dtype, causal=rng.random() < 0.8)


def _lengths(most, least, count, gen):
    """`count` lengths from least to most, evenly spread and in an order that the seed gives."""
    even = torch.tensor([least + (i * (most - least)) // max(1, count - 1) if count > 1 else most for i in range(count)])
    return even[torch.randperm(count, generator=torch.Generator().manual_seed(gen.initial_seed() % (1 << 62)))].to("cuda", torch.int32)


def prepare(case, seed):
    """q, k, v and their gradients from N(0, 1), as after the normalisation in front of a projection; positions of a batch
    start anywhere below `far`; lam between 0.2 and 0.8, where training takes it."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    state = {"case": case}
    if case["op"] == "rotary":
        b, h, hkv, n, d, rot = (case[x] for x in ("b", "h", "hkv", "n", "d", "rot"))
        # projections come as [B, N, heads, D]: the operator sees their [B, heads, N, D] views
        state["q"], state["k"] = normal(b, n, h, d).transpose(1, 2), normal(b, n, hkv, d).transpose(1, 2)
        start = torch.randint(0, case["far"] - n + 1, (b, 1), generator=gen, device="cuda")
        state["positions"] = start + torch.arange(n, device="cuda")
        exponent = torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot
        state["frequencies"] = 10000.0 ** -exponent / case["factor"]
        if case["train"]:
            state["q"].requires_grad_(True)
            state["k"].requires_grad_(True)
            state["dq"], state["dk"] = normal(b, n, h, d).transpose(1, 2), normal(b, n, hkv, d).transpose(1, 2)
    elif case["op"] == "prefix":
        b, h, hkv, nq, d, p, s = (case[x] for x in ("b", "h", "hkv", "nq", "d", "p", "s"))
        state["q"] = normal(b, nq, h, d).transpose(1, 2)
        state["kp"], state["vp"] = normal(hkv, p, d), normal(hkv, p, d)
        state["k"], state["v"] = normal(b, hkv, s, d), normal(b, hkv, s, d)
        state["lengths"] = _lengths(s, min(nq, s), b, gen)
    else:
        b, h, hkv, nq, nk, d, dv = (case[x] for x in ("b", "h", "hkv", "nq", "nk", "d", "dv"))
        state["q"], state["k"], state["v"] = normal(b, 2 * h, nq, d), normal(b, 2 * hkv, nk, d), normal(b, hkv, nk, dv)
        state["lam"] = (0.2 + 0.6 * torch.rand((h,), generator=gen, device="cuda")).to(dtype)
        state["lengths"] = _lengths(nk, max(nq, nk // 4), b, gen) if case["ragged"] else None
        if case["train"]:
            for x in ("q", "k", "v", "lam"):
                state[x].requires_grad_(True)
            state["dout"] = normal(b, h, nq, dv)
    return state


def run(state):
    return {"rotary": _run_rotary, "prefix": _run_prefix, "differential": _run_differential}[state["case"]["op"]](state)


# ---- rotary positions -------------------------------------------------------------------------------------------
def _turn(x, cos, sin, rot, interleaved):
    """x [B, H, N, D] with its first `rot` dimensions turned by the angles whose cosine and sine are [B, 1, N, rot/2]."""
    x32 = x.to(torch.float32)
    if interleaved:
        a, b = x32[..., 0:rot:2], x32[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x32[..., : rot // 2], x32[..., rot // 2: rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x32[..., rot:]), dim=-1).to(x.dtype)


def _run_rotary(state):
    case, q, k = state["case"], state["q"], state["k"]
    if own:
        from elsa_b200 import rotary_embedding
        q2, k2 = rotary_embedding(q, k, state["frequencies"], positions=state["positions"], interleaved=case["interleaved"])
        if not case["train"]:
            return q2, k2
        return (q2.detach(), k2.detach()) + torch.autograd.grad((q2, k2), (q, k), (state["dq"], state["dk"]))
    q, k = q.detach(), k.detach()
    angle = state["positions"].to(torch.float64)[:, None, :, None] * state["frequencies"]
    cos, sin = torch.cos(angle).to(torch.float32), torch.sin(angle).to(torch.float32)
    rot, inter = case["rot"], case["interleaved"]
    out = (_turn(q, cos, sin, rot, inter), _turn(k, cos, sin, rot, inter))
    if case["train"]:       # the transpose of a rotation is the rotation back
        out += (_turn(state["dq"], cos, -sin, rot, inter), _turn(state["dk"], cos, -sin, rot, inter))
    return out


# ---- attention over a shared prefix -----------------------------------------------------------------------------
def _run_prefix(state):
    case, q, kp, vp, k, v, lengths = (state[x] for x in ("case", "q", "kp", "vp", "k", "v", "lengths"))
    if own:
        from elsa_b200 import shared_prefix_attention
        return shared_prefix_attention(q, kp, vp, k, v, lengths=lengths)
    b, h, hkv, nq, d, s = (case[x] for x in ("b", "h", "hkv", "nq", "d", "s"))
    rows = q.to(torch.float32).reshape(b, hkv, h // hkv * nq, d)
    s_prefix = rows @ kp.to(torch.float32).transpose(-1, -2) / math.sqrt(d)
    s_own = rows @ k.to(torch.float32).transpose(-1, -2) / math.sqrt(d)
    last = lengths[:, None] - nq + torch.arange(nq, device=q.device)              # last own key of each query
    seen = torch.arange(s, device=q.device) <= last[:, None, :, None]
    s_own = torch.where(seen, s_own.reshape(b, h, nq, s), -math.inf).reshape(b, hkv, h // hkv * nq, s)
    top = torch.maximum(s_prefix.amax(-1, keepdim=True), s_own.amax(-1, keepdim=True))
    e_prefix, e_own = torch.exp(s_prefix - top), torch.exp(s_own - top)
    total = e_prefix.sum(-1, keepdim=True) + e_own.sum(-1, keepdim=True)
    out = (e_prefix @ vp.to(torch.float32) + e_own @ v.to(torch.float32)) / total
    return out.reshape(b, h, nq, d).to(q.dtype)


# ---- differential attention -------------------------------------------------------------------------------------
def _admissible(case, lengths, device):
    """[B or 1, 1, Nq, Nk] truth values, or None where every query sees every key."""
    nq, nk = case["nq"], case["nk"]
    if not case["causal"] and lengths is None:
        return None
    ends = torch.full((1,), nk, device=device) if lengths is None else lengths
    last = (ends[:, None] - nq + torch.arange(nq, device=device) if case["causal"] else (ends[:, None] - 1).expand(-1, nq))
    return torch.arange(nk, device=device) <= last[:, None, :, None]


def _run_differential(state):
    case, q, k, v, lam, lengths = (state[x] for x in ("case", "q", "k", "v", "lam", "lengths"))
    if own:
        from elsa_b200 import differential_attention, differential_attention_train
        if not case["train"]:
            return differential_attention(q, k, v, lam, is_causal=case["causal"], lengths=lengths)
        out = differential_attention_train(q, k, v, lam, is_causal=case["causal"])
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v, lam), state["dout"])
    b, h, hkv, nq, nk, d, dv = (case[x] for x in ("b", "h", "hkv", "nq", "nk", "d", "dv"))
    group, scale = h // hkv, 1.0 / math.sqrt(d)
    q32, k32, v32 = q.detach().to(torch.float32), k.detach().to(torch.float32), v.detach().to(torch.float32)
    lam32 = lam.detach().to(torch.float32).reshape(h, 1, 1)
    # head h of the output takes the query heads 2h, 2h+1 and the key heads 2g, 2g+1 of its group g
    q32 = q32.reshape(b, hkv, group, 2, nq, d)
    k32 = k32.reshape(b, hkv, 1, 2, nk, d)
    p = (q32 @ k32.transpose(-1, -2)).mul_(scale).reshape(b, 2 * h, nq, nk)
    seen = _admissible(case, lengths, q.device)
    if seen is not None:
        p.masked_fill_(~seen, -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    p = p.reshape(b, h, 2, nq, nk)
    mixed = (p[:, :, 0] - lam32 * p[:, :, 1]).reshape(b, hkv, group, nq, nk)
    out = (mixed @ v32[:, :, None]).reshape(b, h, nq, dv).to(q.dtype)
    if not case["train"]:
        return out
    g = state["dout"].to(torch.float32).reshape(b, hkv, group, nq, dv)
    dv32 = (mixed.transpose(-1, -2) @ g).sum(2)
    del mixed
    dp = (g @ v32[:, :, None].transpose(-1, -2)).reshape(b, h, 1, nq, nk)
    mean = (p * dp).sum(-1, keepdim=True)                                  # [B, H, 2, Nq, 1]
    dlam = -mean[:, :, 1].sum((0, 2, 3))
    ds = p.mul_(dp - mean)
    del dp
    ds[:, :, 1].mul_(-lam32)
    ds = ds.mul_(scale).reshape(b, hkv, group, 2, nq, nk)
    dq = (ds @ k32).reshape(b, 2 * h, nq, d)
    dk = (ds.transpose(-1, -2) @ q32).sum(2).reshape(b, 2 * hkv, nk, d)
    return out, dq.to(q.dtype), dk.to(k.dtype), dv32.to(v.dtype), dlam.to(lam.dtype)


def work(case):
    """Every input read once and every output written once; products over the admissible (query, key) pairs."""
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "rotary":
        elements = case["b"] * (case["h"] + case["hkv"]) * case["n"] * case["d"]
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * elements * size + case["b"] * case["n"] * 8, "flops": passes * 3 * elements * case["rot"] // case["d"]}
    if case["op"] == "prefix":
        b, h, hkv, nq, d, p, s = (case[x] for x in ("b", "h", "hkv", "nq", "d", "p", "s"))
        least = min(nq, s)
        lengths = [least + (i * (s - least)) // max(1, b - 1) if b > 1 else s for i in range(b)]
        keys = sum(lengths)
        pairs = h * (b * nq * p + sum(max(0, n - nq + i + 1) for n in lengths for i in range(nq)))
        return {"bytes": size * d * (2 * b * h * nq + 2 * hkv * (p + keys)), "flops": 4 * d * pairs}
    b, h, hkv, nq, nk, d, dv = (case[x] for x in ("b", "h", "hkv", "nq", "nk", "d", "dv"))
    least = max(nq, nk // 4)
    lengths = [least + (i * (nk - least)) // max(1, b - 1) if b > 1 else nk for i in range(b)] if case["ragged"] else [nk] * b
    pairs = h * sum(sum(max(0, n - nq + i + 1) for i in range(nq)) if case["causal"] else nq * n for n in lengths)
    keys = sum(lengths)
    q_elements, kv_elements, out_elements = 2 * b * h * nq * d, hkv * keys * (2 * d + dv), b * h * nq * dv
    if not case["train"]:
        return {"bytes": size * (q_elements + kv_elements + out_elements), "flops": pairs * (4 * d + 4 * dv)}
    return {"bytes": size * (2 * q_elements + 2 * kv_elements + 2 * out_elements), "flops": pairs * (12 * d + 8 * dv)}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    return {"rotary": _exact_rotary, "prefix": _exact_prefix, "differential": _exact_differential}[case["op"]](case, state)


def _exact_rotary(case, state):
    """Each pair as a complex number times exp(i angle)."""
    rot, inter = case["rot"], case["interleaved"]
    angle = state["positions"].double().unsqueeze(-1) * state["frequencies"]
    unit = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)

    def turned(x, unit):
        y = x.detach().double().clone()
        first, second = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
        z = torch.complex(y[..., first], y[..., second]) * unit
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = (turned(state["q"], unit), turned(state["k"], unit))
    if case["train"]:
        out += (turned(state["dq"], unit.conj()), turned(state["dk"], unit.conj()))
    return out


def _exact_prefix(case, state):
    """Sequence by sequence: softmax over the keys that it really has."""
    q, kp, vp, k, v = (state[x] for x in ("q", "kp", "vp", "k", "v"))
    group, nq = case["h"] // case["hkv"], case["nq"]
    kp, vp = kp.double(), vp.double()
    out = torch.empty(q.shape, device=q.device, dtype=torch.float64)
    for i, length in enumerate(state["lengths"].tolist()):
        keys = torch.cat((kp, k[i, :, :length].double()), 1)
        values = torch.cat((vp, v[i, :, :length].double()), 1)
        for t in range(nq):
            n = case["p"] + length - nq + t + 1
            rows = q[i, :, t].double().view(case["hkv"], group, case["d"])
            weights = torch.softmax(torch.einsum("hgd,hnd->hgn", rows, keys[:, :n]) * case["d"] ** -0.5, -1)
            out[i, :, t] = torch.einsum("hgn,hnd->hgd", weights, values[:, :n]).flatten(0, 1)
    return out


def _exact_differential(case, state):
    """Head by head, with the gradients that automatic differentiation gives."""
    train, group = case["train"], case["h"] // case["hkv"]
    q, k, v, lam = (state[x].detach().double().requires_grad_(train) for x in ("q", "k", "v", "lam"))
    seen = _admissible(case, state["lengths"], q.device)
    out = torch.empty((case["b"], case["h"], case["nq"], case["dv"]), device=q.device, dtype=torch.float64)
    grads = [torch.zeros_like(x, requires_grad=False) for x in (q, k, v, lam)] if train else []
    for i in range(case["b"]):
        mask = None if seen is None else seen[i % seen.shape[0], 0]
        for h in range(case["h"]):
            g = h // group

            def attend(which):
                score = torch.einsum("md,nd->mn", q[i, 2 * h + which], k[i, 2 * g + which]) * case["d"] ** -0.5
                return torch.softmax(score if mask is None else score.masked_fill(~mask, -math.inf), -1)

            with torch.set_grad_enabled(train):
                one = (attend(0) - lam[h] * attend(1)) @ v[i, g]
            out[i, h] = one.detach()
            if train:
                for total, part in zip(grads, torch.autograd.grad(one, (q, k, v, lam), state["dout"][i, h].double())):
                    total += part
            del one
    return (out, *grads) if train else out

"""The decoder operators beside autograd's other machinery, through the native host path and the general one: what a user's program may
put around a call.  Both paths launch the same kernels, which repeat bit for bit: results are compared as bits."""
import pytest
import torch
import torch.utils.checkpoint

import elsa_b200 as E
from elsa_b200 import _lib

pytestmark = pytest.mark.gpu

ENTRIES = ["rotary", "rotary_q", "differential", "differential_fp32"]


def _normal(shape, seed, dtype=torch.float16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _problem(entry):
    """(differentiable inputs, function of them that gives a tuple, gradients of the tuple)"""
    if entry.startswith("rotary"):
        f, g = E.rotary_frequencies(32, device="cuda")
        pos = torch.stack((torch.arange(70), torch.arange(70) + 1000)).cuda()
        inputs = [_normal((2, 4, 70, 64), 1), _normal((2, 2, 70, 64), 2)]
        if entry == "rotary_q":
            return inputs[:1], lambda q: (E.rotary_embedding(q, None, f, interleaved=True),), [_normal((2, 4, 70, 64), 3)]
        return inputs, lambda q, k: E.rotary_embedding(q, k, f, positions=pos, magnitude=1.5), [_normal((2, 4, 70, 64), 3), _normal((2, 2, 70, 64), 4)]
    dtype = torch.float32 if entry.endswith("fp32") else torch.float16
    inputs = [_normal((2, 4, 90, 64), 5, dtype), _normal((2, 2, 90, 64), 6, dtype), _normal((2, 1, 90, 128), 7, dtype), torch.tensor([0.3, 0.6], device="cuda")]
    return inputs, lambda q, k, v, lam: (E.differential_attention_train(q, k, v, lam, is_causal=True),), [_normal((2, 2, 90, 128), 8, dtype)]


def _without_host(monkeypatch):
    monkeypatch.setattr(_lib, "_host_module", None)
    monkeypatch.setattr(_lib, "_host_tried", True)


def _results(entry):
    inputs, call, grads = _problem(entry)
    leaves = [t.requires_grad_(True) for t in inputs]
    out = call(*leaves)
    return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, grads))


def _assert_equal(got, want):
    assert len(got) == len(want)
    for g, w in zip(got, want):
        assert g.shape == w.shape and g.dtype == w.dtype and torch.equal(g, w)


@pytest.fixture(params=["native", "general"])
def path(request, monkeypatch):
    if request.param == "general":
        _without_host(monkeypatch)
    else:
        assert _lib.host() is not None
    return request.param


@pytest.mark.parametrize("entry", ENTRIES)
def test_the_native_path_is_taken_and_the_general_one_agrees(entry, monkeypatch):
    want = _results(entry)
    inputs, call, _ = _problem(entry)
    node = call(*(t.requires_grad_(True) for t in inputs))[0].grad_fn.name()
    assert node == ("RotaryEmbeddingBackward" if entry.startswith("rotary") else "DifferentialAttentionBackward")
    _without_host(monkeypatch)
    _assert_equal(_results(entry), want)


def test_forward_only_operators_agree(monkeypatch):
    q, kp, k = _normal((3, 4, 2, 64), 1), _normal((2, 50, 64), 2), _normal((3, 2, 30, 64), 3)
    n = torch.tensor([2, 30, 17], dtype=torch.int32, device="cuda")
    d = [_normal((3, 4, 2, 64), 4), _normal((3, 2, 40, 64), 5), _normal((3, 1, 40, 96), 6), torch.tensor([0.3, 0.6], device="cuda")]
    calls = [lambda: E.shared_prefix_attention(q, kp, kp, k, k, lengths=n), lambda: E.shared_prefix_attention(q, kp, kp, k, k, scale=0.3),
             lambda: E.differential_attention(*d, is_causal=True, lengths=n), lambda: E.differential_attention(*d, scale=0.2),
             lambda: E.differential_attention(q.transpose(1, 2).contiguous().transpose(1, 2), *d[1:])]
    want = [c() for c in calls]
    _without_host(monkeypatch)
    got = [c() for c in calls]
    _assert_equal(got, want)
    assert [t.stride() for t in got] == [t.stride() for t in want]


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("hook", ["offload", "by_size", "off_alignment", "transposed"])
def test_saved_tensors_may_come_back_in_another_layout(entry, hook, path):
    def off_alignment(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].copy_(t.reshape(-1)).view(t.shape)

    def transposed(t):
        return t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else t.clone()

    want = _results(entry)
    if hook == "offload":
        hooks = torch.autograd.graph.save_on_cpu(pin_memory=True)
    else:
        pack = {"by_size": lambda t: torch.empty(t.size(), dtype=t.dtype, device=t.device).copy_(t), "off_alignment": off_alignment, "transposed": transposed}[hook]
        hooks = torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t)
    with hooks:
        got = _results(entry)
    _assert_equal(got, want)


@pytest.mark.parametrize("entry", ENTRIES)
def test_a_saved_tensor_of_another_kind_is_refused(entry, path):
    for unpack in (lambda t: t.to(torch.int16), lambda t: t.cpu(), lambda t: t[..., :1] if t.dim() else t[None]):
        inputs, call, grads = _problem(entry)
        leaves = [t.requires_grad_(True) for t in inputs]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            out = call(*leaves)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out, leaves, grads)


@pytest.mark.parametrize("entry", ENTRIES)
def test_checkpoint(entry, path):
    inputs, call, grads = _problem(entry)
    want = _results(entry)[len(grads):]
    leaves = [t.requires_grad_(True) for t in inputs]
    out = torch.utils.checkpoint.checkpoint(lambda *x: tuple(t * 1 for t in call(*x)), *leaves, use_reentrant=False)
    _assert_equal(torch.autograd.grad(out, leaves, grads), want)


@pytest.mark.parametrize("entry", ENTRIES)
def test_forward_mode_is_refused_not_dropped(entry, path):
    for i in range(len(_problem(entry)[0])):
        inputs, call, _ = _problem(entry)
        with torch.autograd.forward_ad.dual_level():
            inputs[i] = torch.autograd.forward_ad.make_dual(inputs[i], torch.ones_like(inputs[i]))
            with pytest.raises(NotImplementedError):
                call(*inputs)


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("grad", [False, True])
def test_a_traced_call_follows_its_inputs(entry, grad):
    inputs, call, _ = _problem(entry)
    inputs = [t.requires_grad_(grad) for t in inputs]
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(lambda *x: call(*x), tuple(inputs), check_trace=False)
        other = [(t * 0.5 + 0.1).detach() for t in inputs]
        _assert_equal(traced(*other), call(*other))


@pytest.mark.parametrize("op", ["shared_prefix", "differential", "rotary_inplace"])
def test_forward_only_operators_refuse_traces_and_tangents(op, path):
    """A trace would hold their memory and not their work, a dual number's result no tangent."""
    inputs = {"shared_prefix": [_normal((3, 4, 2, 64), 1), _normal((2, 50, 64), 2), _normal((2, 50, 64), 3), _normal((3, 2, 30, 64), 4), _normal((3, 2, 30, 64), 5)],
              "differential": [_normal((3, 4, 2, 64), 4), _normal((3, 2, 40, 64), 5), _normal((3, 1, 40, 96), 6), torch.tensor([0.3, 0.6], device="cuda")],
              "rotary_inplace": [_normal((2, 4, 70, 64), 1), _normal((2, 2, 70, 64), 2)]}[op]
    f = E.rotary_frequencies(32, device="cuda")[0]
    call = {"shared_prefix": E.shared_prefix_attention, "differential": E.differential_attention,
            "rotary_inplace": lambda q, k: E.rotary_embedding(q, k, f, inplace=True)}[op]
    with pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(call, tuple(inputs), check_trace=False)
    for i in range(len(inputs)):
        with torch.autograd.forward_ad.dual_level():
            dual = [torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(inputs)]
            with pytest.raises(NotImplementedError):
                call(*dual)


@pytest.mark.parametrize("entry", ENTRIES)
def test_a_second_derivative_is_refused_not_dropped(entry, path):
    inputs, call, grads = _problem(entry)
    leaves = [t.requires_grad_(True) for t in inputs]
    first = torch.autograd.grad(call(*leaves), leaves, grads, create_graph=True)
    _assert_equal([t.detach() for t in first], _results(entry)[len(grads):])
    with pytest.raises(RuntimeError, match="twice"):
        first[0].float().square().sum().backward()


@pytest.mark.parametrize("entry", ["differential", "differential_fp32"])
@pytest.mark.parametrize("which", [0, 1, 2, 3, "out"])
def test_a_change_before_the_backward_is_found(entry, which, path):
    inputs, call, grads = _problem(entry)
    leaves = [t.requires_grad_(True) for t in inputs]
    out = call(*leaves)
    with pytest.raises(RuntimeError):
        with torch.no_grad():
            (out[0] if which == "out" else leaves[which]).mul_(2)
        torch.autograd.grad(out, leaves, grads)


@pytest.mark.parametrize("entry", ENTRIES)
def test_backward_under_compiled_autograd(entry):
    from torch._dynamo import compiled_autograd
    want = _results(entry)
    for _ in range(2):
        inputs, call, grads = _problem(entry)
        leaves = [t.requires_grad_(True) for t in inputs]
        out = call(*leaves)
        with compiled_autograd._enable(torch.compile(backend="eager")):
            torch.autograd.backward([t * 0.5 for t in out], [g * 2 for g in grads])      # (exact: halving first would lose fp16's smallest)
        _assert_equal([t.grad for t in leaves], want[len(grads):])


@pytest.mark.parametrize("entry", ENTRIES)
def test_under_a_dispatch_mode_the_general_path_agrees(entry):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Passing(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    want = _results(entry)
    with Passing():
        got = _results(entry)
    _assert_equal(got, want)


def test_one_of_two_gradients_alone(path):
    inputs, call, grads = _problem("rotary")
    want = _results("rotary")
    for i in (0, 1):
        q, k = (t.detach().requires_grad_(j == i) for j, t in enumerate(inputs))
        out = call(q, k)
        _assert_equal(torch.autograd.grad(out[i], (q, k)[i], grads[i]), [want[2 + i]])
        q, k = (t.detach().requires_grad_(True) for t in inputs)
        _assert_equal(torch.autograd.grad(call(q, k)[i], (q, k)[i], grads[i]), [want[2 + i]])


@pytest.mark.parametrize("entry", ENTRIES)
def test_a_step_captured_while_an_eager_graph_lives(entry, path):
    """The leaves of a captured step are its own: an eager graph of other tensors may live beside it."""
    kept_inputs, call, grads = _problem(entry)
    kept = call(*(t.requires_grad_(True) for t in kept_inputs))
    want = _results(entry)
    inputs, call, grads = _problem(entry)
    leaves = [t.requires_grad_(True) for t in inputs]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = call(*leaves)
        got = list(out) + list(torch.autograd.grad(out, leaves, grads))
    graph.replay()
    torch.cuda.synchronize()
    _assert_equal([t.detach() for t in got], want)
    del kept

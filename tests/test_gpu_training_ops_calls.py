"""Calls of the operators around a training step in graphs, on several streams, in inference mode and under other transforms."""
import pytest
import torch

from q38 import ops
from q38.losses import vocabulary_cross_entropy

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def installed():
    ops.install()
    yield
    ops.check_errors()


# ---- vocabulary loss with an fp32 weight ---------------------------------------------------------------------------------------------
def master(seed, rows=200, words=3000, width=64):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(rows, width, device="cuda", generator=gen).to(BF16)
    w = torch.randn(words, width, device="cuda", generator=gen) * 0.3
    return h.requires_grad_(), w.requires_grad_(), torch.randint(0, words, (rows,), device="cuda", generator=gen)


def step(h, w, target):
    loss = vocabulary_cross_entropy(w, h, target)
    return (loss.detach(), *torch.autograd.grad(loss, [h, w]))


def from_bf16(h, w, target):
    """The same with a weight that is bf16 from the start."""
    loss, dh, dw = step(h, w.detach().to(BF16).requires_grad_(), target)
    return loss, dh, dw


def same(got, want):
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(got[2].to(BF16), want[2])                       # the fp32 gradient, rounded as the other is


@pytest.mark.parametrize("width", [64, 71])
def test_master_weight_changes_between_replays(width):
    h, w, target = master(0, width=width)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step(h, w, target)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(h, w, target)
    for change in (lambda: w.mul_(1.5), lambda: w.data.mul_(-0.5), lambda: w.data.copy_(master(1, width=width)[1])):
        with torch.no_grad():
            change()
        graph.replay()
        same(held, from_bf16(h, w, target))
    step(h, w, target)
    graph.replay()
    same(held, from_bf16(h, w, target))


def test_master_weight_on_a_second_stream():
    """The first call's rounding waits behind a long kernel on its stream; the second call, on a stream of its own, must not depend on it."""
    h, w, target = master(2)
    want = step(h, w, target)
    with torch.no_grad():
        w.add_(0)                                                     # a version that no call has seen
    torch.cuda.synchronize()
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(first):
        torch.cuda._sleep(50_000_000)
        one = step(h, w, target)
    with torch.cuda.stream(second):
        two = step(h, w, target)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for got in (one, two) for a, b in zip(got, want))


def test_master_weight_changes_outside_the_version_counter():
    h, w, target = master(3)
    step(h, w, target)
    w.data.mul_(2)
    same(step(h, w, target), from_bf16(h, w, target))
    w.data = w.data * 0.25
    same(step(h, w, target), from_bf16(h, w, target))
    assert not vars(w)


def test_master_weight_made_in_inference_mode():
    h, w, target = master(4)
    with torch.inference_mode():
        seen = w.detach().clone()
        inside = vocabulary_cross_entropy(seen, h, target)
    want = step(h, w, target)
    loss = vocabulary_cross_entropy(seen, h, target)
    assert torch.equal(inside, want[0]) and torch.equal(loss, want[0])
    assert torch.equal(torch.autograd.grad(loss, h)[0], want[1])


# ---- gradients that are no memory ------------------------------------------------------------------------------------------------------
def outputs():
    """A result of each differentiable operator and its leaf."""
    x = torch.randn(6, 64, device="cuda", requires_grad=True)
    q = torch.randn(1, 6, 2, 16, device="cuda", requires_grad=True)
    h, w, target = master(5, 6, 100)
    freq, _ = ops.rotary_frequencies(16, device="cuda")
    return [(ops.layer_norm(x), x), (ops.rotary(q, None, torch.arange(6, device="cuda"), freq)[0], q), (vocabulary_cross_entropy(w, h, target, "none"), h)]


@pytest.mark.parametrize("which", range(3))
def test_batched_gradients_are_refused(which):
    y, leaf = outputs()[which]
    with pytest.raises(ValueError, match="values in memory of its own"):
        torch.autograd.grad(y, leaf, torch.ones(3, *y.shape, device="cuda"), is_grads_batched=True)


def test_layer_norm_under_vmap():
    x = torch.randn(3, 5, 64, device="cuda")
    assert torch.equal(torch.func.vmap(ops.layer_norm)(x), ops.layer_norm(x))


# ---- views with the other sign -----------------------------------------------------------------------------------------------------------
def negated(t):
    """The same values, as the imaginary part of a conjugate is held: in memory with the other sign, a bit saying so."""
    return torch._neg_view(-t)


def test_negated_views_have_their_values():
    x, w, b, dy = (torch.randn(*s, device="cuda") for s in ((6, 64), (64,), (64,), (6, 64)))
    assert negated(x).is_neg() and torch.equal(negated(x) + 0, x)
    want, got = [], []
    for out, wrap in ((want, lambda t: t), (got, negated)):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = ops.layer_norm(*(wrap(t) for t in leaves))
        out += [y, *torch.autograd.grad(y, leaves, wrap(dy))]
        q, k = (torch.randn(2, 6, n, 16, device="cuda", generator=torch.Generator("cuda").manual_seed(n)).requires_grad_() for n in (4, 2))
        freq, _ = ops.rotary_frequencies(16, device="cuda")
        turned = ops.rotary(wrap(q), wrap(k), torch.arange(6, device="cuda"), wrap(freq))
        out += [*turned, *torch.autograd.grad(turned, [q, k], [wrap(q.detach()), wrap(k.detach())])]
        h, m, target = master(6)
        losses = vocabulary_cross_entropy(wrap(m), wrap(h), target, "none")
        out += [losses, *torch.autograd.grad(losses, [h, m], wrap(losses.detach()))]
        mean = vocabulary_cross_entropy(wrap(m.detach().to(BF16)), h, target)
        out += [mean, *torch.autograd.grad(mean, h, wrap(torch.ones_like(mean)))]
        grads = [x.clone(), w.clone()]
        out += [ops.grad_norm([wrap(g) for g in grads]), ops.clip_grad_norm([wrap(g) for g in grads], 1.0, out=(into := [torch.empty_like(g) for g in grads])), *into]
        grads = [wrap(g) for g in grads]
        out += [ops.clip_grad_norm(grads, 1.0), *(g + 0 for g in grads)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- derivatives that are not offered ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("call", [
    lambda t: ops.layer_norm(t), lambda t: ops.layer_norm(t.detach(), t[0]), lambda t: ops.layer_norm(t.detach(), None, t[0]),
    lambda t: ops.rotary(t.view(1, 6, 4, 16), None, torch.arange(6, device="cuda"), ops.rotary_frequencies(16, device="cuda")[0]),
    lambda t: ops.rotary(t.detach().view(6, 4, 16), t.view(6, 4, 16), torch.arange(6, device="cuda"), ops.rotary_frequencies(16, device="cuda")[0]),
    lambda t: ops.rotary(t.detach().view(6, 4, 16), None, torch.arange(6, device="cuda"), t[0, :8].double()),
    lambda t: vocabulary_cross_entropy(t.detach(), t, torch.arange(6, device="cuda")), lambda t: vocabulary_cross_entropy(t, t.detach(), torch.arange(6, device="cuda")),
    lambda t: ops.grad_norm([t]), lambda t: ops.clip_grad_norm([t], 1.0), lambda t: ops.clip_grad_norm([t], 1.0, out=[t.detach().clone()]),
    lambda t: ops.clip_grad_norm([t.detach().clone()], 1.0, out=[t]),
])
def test_forward_mode_is_refused(call):
    x = torch.randn(6, 64, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        t = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward mode"):
            call(t)
    with pytest.raises((RuntimeError, ValueError)):
        torch.func.jvp(call, (x,), (torch.ones_like(x),))


@pytest.mark.parametrize("which", range(3))
def test_gradients_with_a_tangent_are_refused(which):
    y, leaf = outputs()[which]
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward mode"):
            torch.autograd.grad(y, leaf, torch.autograd.forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_a_gradient_of_the_frequencies_is_refused():
    q = torch.randn(1, 6, 2, 16, device="cuda", requires_grad=True)
    freq, _ = ops.rotary_frequencies(16, device="cuda")
    learned, pos = freq.clone().requires_grad_(), torch.arange(6, device="cuda")
    for arg in (q, q.detach()):
        with pytest.raises(ValueError, match="frequencies"):
            ops.rotary(arg, None, pos, learned)
    want = ops.rotary(q, None, pos, freq)[0]
    with torch.no_grad():
        assert torch.equal(ops.rotary(q, None, pos, learned)[0], want)
    assert torch.equal(ops.rotary(q, None, pos, learned.detach())[0], want)


# ---- the kernel bench ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens,turned", [(100, 100), (5000, 4096)])
def test_kernel_bench_labels_what_ran(tokens, turned):
    from q38.utils.kernel_bench import bench_training
    rows = []
    bench_training(rows, dict(hidden=64, heads=3, kv_heads=1, rope_theta=1e6), tokens, 1, dict(tflops=1.0, hbm_gbs=1.0, source="test"))
    row, = [r for r in rows if r["kernel"].startswith("rotary")]
    assert row["kernel"] == f"rotary T={turned} heads=3+1"
    assert abs(row["gbs"] * row["us"] * 1e3 / (4 * turned * 4 * 64) - 1) < 1e-6


# ---- inference mode ------------------------------------------------------------------------------------------------------------------------
def test_gradients_enabled_inside_inference_mode_are_not_recorded():
    """As for torch's own operators: inference mode comes before `enable_grad`."""
    x = torch.randn(6, 64, device="cuda", requires_grad=True)
    q = torch.randn(1, 6, 2, 16, device="cuda", requires_grad=True)
    h, w, target = master(7, 6, 100)
    freq, pos = ops.rotary_frequencies(16, device="cuda")[0], torch.arange(6, device="cuda")
    calls = [lambda: ops.layer_norm(x), lambda: ops.rotary(q, None, pos, freq)[0], lambda: ops.rotary(q, None, pos, freq.clone().requires_grad_())[0],
             lambda: vocabulary_cross_entropy(w, h, target), lambda: vocabulary_cross_entropy(w.detach().to(BF16), h, target, "none")]
    want = [ops.layer_norm(x), *[ops.rotary(q, None, pos, freq)[0]] * 2, vocabulary_cross_entropy(w, h, target), vocabulary_cross_entropy(w, h, target, "none")]
    for call, value in zip(calls, want):
        with torch.inference_mode(), torch.enable_grad():
            got = call()
            assert not got.requires_grad and got.is_inference()
        assert torch.equal(got, value)


def test_a_first_call_is_not_captured(monkeypatch):
    h, w, target = master(8, 6, 100)
    with monkeypatch.context() as m:
        m.setattr(ops, "_error_flags", flags := {})
        m.setattr("q38.ops.vocab._error_flags", flags)
        with pytest.raises(RuntimeError, match="before it is captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                vocabulary_cross_entropy(w, h, target)
        assert not flags
        want = vocabulary_cross_entropy(w, h, target)
        assert list(flags) == [0]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = vocabulary_cross_entropy(w, h, target)
        ops.check_errors()
        graph.replay()
        assert torch.equal(held, want)
        target[2] = 100                                               # outside the vocabulary: reported by the replay, once
        graph.replay()
        with pytest.raises(RuntimeError, match="index"):
            ops.check_errors()
        ops.check_errors()

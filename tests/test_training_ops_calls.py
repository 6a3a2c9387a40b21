"""Calls of the operators around a training step that are answered, or refused, before a kernel runs."""
import pytest
import torch

from q38 import ops
from q38.ops import vocab


class Native:
    """Stands in for the compiled library: notes what the vocabulary loss is given."""

    def __init__(self):
        self.weights = []

    def check_operands(self, tensors, name):
        pass

    def vocab_loss(self, hidden, weight, weight16, target, reduction, managed, workspace, err):
        self.weights.append(weight16)
        return torch.zeros(())


@pytest.fixture
def native(monkeypatch):
    lib = Native()
    monkeypatch.setattr(vocab, "load", lambda: lib)
    monkeypatch.setattr(vocab, "error_flag", lambda device: None)
    monkeypatch.setattr(vocab, "_error_flags", {None: None})
    return lib


def _call(weight):
    vocab.vocabulary_loss(torch.zeros(3, 8, dtype=torch.bfloat16), weight, torch.zeros(3, dtype=torch.int64), "mean")


# ---- the weight's bf16 form -----------------------------------------------------------------------------------------------------------
def test_a_master_weight_is_rounded_in_every_call(native):
    """A copy that outlived the call would be missing from a captured graph, unordered on another stream and stale after a change through `.data`."""
    weight = torch.randn(5, 8)
    _call(weight)
    _call(weight)
    first, second = native.weights
    assert first.dtype == torch.bfloat16 and torch.equal(first, weight.to(torch.bfloat16)) and torch.equal(first, second)
    assert first.data_ptr() != second.data_ptr() and not vars(weight)
    weight.data.mul_(3)
    _call(weight)
    weight.data = torch.randn(5, 8)
    _call(weight)
    assert torch.equal(native.weights[-1], weight.to(torch.bfloat16)) and not torch.equal(native.weights[-2], second)


def test_a_weight_made_in_inference_mode(native):
    with torch.inference_mode():
        weight = torch.randn(5, 8)
    _call(weight)
    assert torch.equal(native.weights[0], weight.to(torch.bfloat16))


def test_a_bf16_weight_and_an_arena_shadow_go_in_as_they_are(native):
    weight = torch.randn(5, 8, dtype=torch.bfloat16)
    _call(weight)
    managed = torch.randn(5, 8)
    managed._q38_bf16 = managed.to(torch.bfloat16)
    _call(managed)
    assert [w.data_ptr() for w in native.weights] == [weight.data_ptr(), managed._q38_bf16.data_ptr()]


# ---- tensors that are no memory --------------------------------------------------------------------------------------------------------
def _normal(x):
    return ops.load().layer_norm(x, None, None, 1e-5)


def _scaled(w):
    return ops.load().layer_norm(torch.zeros(3, 8), w[0, 0], None, 1e-5)


def _shifted(b):
    return ops.load().layer_norm(torch.zeros(3, 8), None, b[0, 0], 1e-5)


def _turned(q):
    return ops.load().rotary(q[None], None, torch.zeros(4, dtype=torch.int64), torch.zeros(4, dtype=torch.float64), 1.0, False)


def _turned_key(k):
    return ops.load().rotary(torch.zeros(1, 4, 8, 8), k[None], torch.zeros(4, dtype=torch.int64), torch.zeros(4, dtype=torch.float64), 1.0, False)


def _turned_at(pos):
    return ops.load().rotary(torch.zeros(1, 4, 8, 8), None, pos.flatten()[:4].long(), torch.zeros(4, dtype=torch.float64), 1.0, False)


def _turned_by(f):
    return ops.load().rotary(torch.zeros(1, 4, 8, 8), None, torch.zeros(4, dtype=torch.int64), f.flatten()[:4].double(), 1.0, False)


def _total(g):
    return ops.load().grad_norm([torch.ones(3), g])


def _clipped(g):
    return ops.load().clip_grad_norm_([g], 1.0)


def _clipped_into(o):
    return ops.load().clip_grad_norm_out([torch.ones(4, 8, 8)], [o], 1.0)


def _losses(h):
    return vocab.vocabulary_loss(h, torch.zeros(11, 8), torch.zeros(h.shape[:-1], dtype=torch.int64), "none")


def _losses_by(w):
    return vocab.vocabulary_loss(torch.zeros(3, 8), w[0], torch.zeros(3, dtype=torch.int64), "mean")


def _losses_of(t):
    return vocab.vocabulary_loss(torch.zeros(3, 8), torch.zeros(11, 8), t.flatten()[:3].long(), "mean")


class Wrapped(torch.Tensor):
    """As sharded tensors are made: a device and sizes, and the values in another tensor."""

    @staticmethod
    def __new__(cls, inner, device):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=device)

    def __init__(self, inner, device):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        args = [a.inner if isinstance(a, cls) else a for a in args]
        return cls(func(*args, **(kwargs or {})), "cuda")


ENTRIES = [_normal, _scaled, _shifted, _turned, _turned_key, _turned_at, _turned_by, _total, _clipped, _clipped_into, _losses, _losses_by, _losses_of]


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("kind", ["fake", "wrapped", "differentiated"])
def test_tensors_without_memory_are_refused(entry, kind, monkeypatch):
    """Their address is null, or not to be had.  They are refused before the error word is made, which would be one of them."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    monkeypatch.setattr(ops, "_error_flags", flags := {})
    monkeypatch.setattr(vocab, "_error_flags", flags)
    with pytest.raises(ValueError, match="values in memory of its own"):
        if kind == "fake":
            with FakeTensorMode():
                entry(torch.zeros(4, 8, 8, device="cuda"))
        elif kind == "wrapped":
            entry(Wrapped(torch.zeros(4, 8, 8), "cuda"))
        else:
            torch.func.grad(entry)(torch.zeros(4, 8, 8))
    assert not flags


# ---- derivatives that are not offered ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("entry", [e for e in ENTRIES if e not in (_turned_at, _losses_of)])
def test_forward_mode_is_refused(entry):
    """A result without a tangent would be taken for a constant."""
    x = torch.zeros(4, 8, 8)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward mode"):
            entry(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))


def _learned(k=True, device="cpu"):
    q = torch.randn(1, 4, 2, 8, device=device, requires_grad=True)
    f = torch.rand(4, dtype=torch.float64, device=device).requires_grad_()
    return lambda: ops.rotary(q, q.detach() if k else None, torch.arange(4, device=device), f)


@pytest.mark.parametrize("k", [True, False])
def test_a_gradient_of_the_frequencies_is_refused(k):
    """Neither device offers one, so that neither leaves a learned vector without one unnoticed."""
    call = _learned(k)
    with pytest.raises(ValueError, match="frequencies"):
        call()
    with torch.no_grad():
        call()


def test_a_gradient_of_the_frequencies_is_refused_where_the_kernel_is_called():
    q, f = torch.zeros(1, 4, 2, 8), torch.zeros(4, dtype=torch.float64, requires_grad=True)
    with pytest.raises(ValueError, match="frequencies"):
        ops.load().rotary(q, None, torch.arange(4), f, 1.0, False)


# ---- vocabulary loss in host memory --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("ht,wt", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
def test_scores_of_the_vocabulary_loss_are_fp32(ht, wt):
    """Scores of tens: one rounded to bf16 is off by 2^-9 of itself, which is a few per cent of a probability."""
    from q38.losses import vocabulary_cross_entropy
    gen = torch.Generator().manual_seed(0)
    rows, words, width, u = 20, 300, 48, 2.0 ** -24
    h, w = (torch.randn(rows, width, generator=gen) * 2).to(ht).requires_grad_(), torch.randn(words, width, generator=gen).to(wt).requires_grad_()
    target = torch.randint(0, words, (rows,), generator=gen)
    hd = h.detach().double().requires_grad_()
    wd = w.detach().to(ht).double().requires_grad_()                        # a master weight is rounded as the hidden states are
    want = torch.nn.functional.cross_entropy(hd @ wd.T, target, reduction="none")
    got = vocabulary_cross_entropy(w, h, target, "none")
    # a score has `width` additions; a loss the sum over the words, its logarithm and the target's score
    score_off = (width + 2) * u * (hd.abs() @ wd.abs().T)
    tol = 2 * score_off.amax(-1) + (words + 8) * u + 4 * u * (hd @ wd.T).abs().amax(-1)
    assert got.dtype == torch.float32 and ((got - want).abs() <= tol).all()
    # gradients: probabilities to twice that (relative), sums over words and rows, and half a step of the result's type
    dz = torch.softmax(hd @ wd.T, -1) - torch.nn.functional.one_hot(target, words)
    dz_off = (2 * tol[:, None] + 8 * u) * dz.abs() + 4 * u
    dh, dw = torch.autograd.grad(got.sum(), [h, w])
    for g, e, off in ((dh, dz @ wd, dz_off @ wd.abs() + words * u * (dz.abs() @ wd.abs())), (dw, dz.T @ hd, dz_off.T @ hd.abs() + rows * u * (dz.abs().T @ hd.abs()))):
        kept = ht if g is dw and wt == torch.float32 else g.dtype           # a master weight's gradient passes through the type that it was rounded to
        assert ((g.double() - e).abs() <= off + torch.finfo(kept).eps / 2 * (e.abs() + off)).all()


# ---- the kernel bench ----------------------------------------------------------------------------------------------------------------------
def test_kernel_bench_sequences():
    from q38.utils.kernel_bench import sequences
    assert [sequences(t) for t in (1, 100, 4095, 4096, 10000, 16384)] == [(1, 1), (1, 100), (1, 4095), (1, 4096), (2, 4096), (4, 4096)]


# ---- the error word --------------------------------------------------------------------------------------------------------------------------
def test_the_error_word_is_not_made_in_a_capture(native, monkeypatch):
    """Its zeros would be written by the replays: garbage before the first, and what a replay reported lost in the next."""
    monkeypatch.setattr(vocab, "_error_flags", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before it is captured"):
        _call(torch.randn(5, 8))
    monkeypatch.setattr(vocab, "_error_flags", {None: torch.zeros(1)})
    _call(torch.randn(5, 8))
    assert len(native.weights) == 1

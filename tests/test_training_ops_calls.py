"""Calls of the operators around a training step that are answered, or refused, before a kernel runs."""
import pytest
import torch

from q38.ops import vocab


class Native:
    """Stands in for the compiled library: notes what the vocabulary loss is given."""

    def __init__(self):
        self.weights = []

    def vocab_loss(self, hidden, weight, weight16, target, reduction, managed, workspace, err):
        self.weights.append(weight16)
        return torch.zeros(())


@pytest.fixture
def native(monkeypatch):
    lib = Native()
    monkeypatch.setattr(vocab, "load", lambda: lib)
    monkeypatch.setattr(vocab, "error_flag", lambda device: None)
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

"""Layer norm, rotary positions and gradient clipping in host memory: the formulas and the refusals."""
import math

import pytest
import torch

from q38 import ops


def test_layer_norm_formula_and_gradient():
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(3, 4, 7, generator=gen, requires_grad=True)
    w, b = torch.randn(7, generator=gen, requires_grad=True), torch.randn(7, generator=gen, requires_grad=True)
    want = torch.nn.functional.layer_norm(x.double(), (7,), w.double(), b.double(), 1e-5)
    got = ops.layer_norm(x, w, b)
    # a handful of fp32 roundings of values below ten
    assert (got - want).abs().max() < 1e-5
    dy = torch.randn(3, 4, 7, generator=gen)
    for a, e in zip(torch.autograd.grad(got, [x, w, b], dy), torch.autograd.grad(want, [x, w, b], dy.double())):
        assert (a - e).abs().max() < 1e-5
    assert ops.layer_norm(x, out_dtype=torch.bfloat16).dtype == torch.bfloat16


@pytest.mark.parametrize("call", [
    lambda: ops.layer_norm(torch.tensor(1.0)), lambda: ops.layer_norm(torch.zeros(3, 0)), lambda: ops.layer_norm(torch.zeros(3, 4, dtype=torch.int32)),
    lambda: ops.layer_norm(torch.zeros(3, 4, dtype=torch.float64)), lambda: ops.layer_norm(torch.zeros(3, 4), torch.ones(3)), lambda: ops.layer_norm(torch.zeros(3, 4), torch.ones(4, 1)),
    lambda: ops.layer_norm(torch.zeros(3, 4), None, torch.ones(5)), lambda: ops.layer_norm(torch.zeros(3, 4), torch.ones(4, dtype=torch.int64)),
    lambda: ops.layer_norm(torch.zeros(3, 4), eps=-1.0), lambda: ops.layer_norm(torch.zeros(3, 4, dtype=torch.bfloat16), out_dtype=torch.float32),
])
def test_layer_norm_refuses(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_turns_pairs(interleaved):
    f, m = ops.rotary_frequencies(6, theta=100.0)
    assert m == 1.0 and torch.allclose(f, torch.tensor([1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3)], dtype=torch.float64), rtol=1e-14)
    q, k = torch.randn(2, 5, 3, 8), torch.randn(2, 5, 1, 8)
    pos = torch.tensor([[0, 1, 2, 3, 4], [7, 6, -5, 100000, 9]])
    for x, out in zip((q, k), ops.rotary(q, k, pos, f, magnitude=1.5, interleaved=interleaved)):
        for b in range(2):
            for s in range(5):
                for i in range(3):
                    at = (2 * i, 2 * i + 1) if interleaved else (i, i + 3)
                    z = complex(*x[b, s, 0, list(at)].tolist()) * 1.5 * complex(math.cos(pos[b, s] * f[i]), math.sin(pos[b, s] * f[i]))
                    assert abs(complex(*out[b, s, 0, list(at)].tolist()) - z) < 1e-5
        assert torch.equal(out[..., 6:], x[..., 6:])
    flat, none = ops.rotary(q[0], None, pos[0], f, interleaved=interleaved)              # packed tokens, queries only
    assert none is None and torch.equal(flat, ops.rotary(q[:1], None, pos[0], f, interleaved=interleaved)[0][0])


def test_rotary_frequencies_scaled():
    plain, _ = ops.rotary_frequencies(64, 1e4)
    linear, one = ops.rotary_frequencies(64, 1e4, dict(rope_type="linear", factor=4.0))
    assert one == 1.0 and torch.allclose(linear, plain / 4, rtol=1e-14)
    ntk, _ = ops.rotary_frequencies(64, 1e4, dict(rope_type="ntk", factor=4.0))
    assert ntk[0] == 1 and abs(ntk[-1] / plain[-1] * 4 - 1) < 1e-12
    yarn, m = ops.rotary_frequencies(64, 1e4, dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=4096))
    assert abs(m - (0.1 * math.log(8) + 1)) < 1e-12
    turns = 4096 * plain / (2 * math.pi)
    ratio = yarn / plain
    # kept above 32 turns and slowed eightfold below one (whole pairs outside the ramp), falling between
    first, last = (32 * math.log(4096 / (2 * math.pi * t)) / math.log(1e4) for t in (32, 1))
    pair = torch.arange(32)
    assert torch.allclose(ratio[pair <= math.floor(first)], torch.ones((), dtype=torch.float64)) and (turns[pair <= math.floor(first)] >= 32).all()
    assert torch.allclose(ratio[pair >= math.ceil(last)], torch.full((), 0.125, dtype=torch.float64)) and (turns[pair >= math.ceil(last)] <= 1).all()
    assert (ratio[1:] <= ratio[:-1] + 1e-12).all()
    same, m = ops.rotary_frequencies(64, 1e4, dict(rope_type="yarn", factor=1.0, original_max_position_embeddings=4096))
    assert m == 1.0 and torch.allclose(same, plain, rtol=1e-14)
    assert ops.rotary_frequencies(64, 1e4, dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=4096, attention_factor=1.25, truncate=False))[1] == 1.25
    assert ops.rotary_frequencies(2, 1e4, dict(rope_type="ntk", factor=4.0))[0].tolist() == [1.0]


@pytest.mark.parametrize("call", [
    lambda: ops.rotary_frequencies(7), lambda: ops.rotary_frequencies(0), lambda: ops.rotary_frequencies(8, 0.5), lambda: ops.rotary_frequencies(8, scaling=dict(rope_type="other")),
    lambda: ops.rotary_frequencies(8, scaling=dict(rope_type="linear", factor=0.5)), lambda: ops.rotary_frequencies(8, scaling=dict(rope_type="yarn", factor=2.0)),
    lambda: ops.rotary_frequencies(8, scaling=dict(rope_type="linear", factr=2.0)), lambda: ops.rotary_frequencies(8, scaling=dict(rope_type="ntk", factor=float("inf"))),
    lambda: ops.rotary_frequencies(8, scaling=dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=64, beta_fast=1.0, beta_slow=2.0)),
])
def test_rotary_frequencies_refuse(call):
    with pytest.raises(ValueError):
        call()


def _rotary(q=(2, 3, 4, 8), k=(2, 3, 1, 8), pos=(3,), f=4, qt=torch.float32, kt=torch.float32, pt=torch.int64, ft=torch.float64):
    return ops.rotary(torch.zeros(q, dtype=qt), None if k is None else torch.zeros(k, dtype=kt), torch.zeros(pos, dtype=pt), torch.zeros(f, dtype=ft))


@pytest.mark.parametrize("wrong", [dict(q=(2, 3)), dict(k=(2, 3, 8)), dict(k=(2, 4, 1, 8)), dict(k=(1, 3, 1, 8)), dict(k=(2, 3, 1, 6)), dict(kt=torch.bfloat16), dict(qt=torch.float64, k=None),
                                   dict(pos=(4,)), dict(pos=(3, 3)), dict(pos=()), dict(pt=torch.float32), dict(pt=torch.int16), dict(f=5), dict(f=(2, 2)), dict(ft=torch.float32)])
def test_rotary_refuses(wrong):
    _rotary()
    with pytest.raises(ValueError):
        _rotary(**wrong)


def test_clip_formula():
    grads = [torch.randn(3, 4), torch.randn(5).to(torch.bfloat16), None, torch.randn(0), torch.randn(4, 6).t()]
    given = [g for g in grads if g is not None]
    norm = math.sqrt(sum(g.double().square().sum().item() for g in given))
    assert abs(ops.grad_norm(grads).item() / norm - 1) < 2e-7
    out = [torch.empty_like(g) if g is not None else None for g in grads]
    assert abs(ops.clip_grad_norm(grads, 0.5, out=out).item() / norm - 1) < 2e-7
    before = [g.clone() for g in given]
    ops.clip_grad_norm(grads, 0.5)
    for o, g, b in zip([o for o in out if o is not None], given, before):
        assert torch.equal(o, g) and torch.allclose(g.double(), b.double() * 0.5 / (norm + 1e-6), rtol=torch.finfo(g.dtype).eps)
    kept = [g.clone() for g in given]
    ops.clip_grad_norm(given, 1e9)
    assert all(torch.equal(a, b) for a, b in zip(kept, given))
    assert torch.is_tensor(ops.clip_grad_norm(torch.ones(3), float("inf")))


def _pair():
    t = torch.zeros(8)
    return t[:4], t[4:]


@pytest.mark.parametrize("call", [
    lambda: ops.clip_grad_norm([], 1.0), lambda: ops.clip_grad_norm([None], 1.0), lambda: ops.grad_norm([]), lambda: ops.clip_grad_norm([torch.ones(3)], 0.0),
    lambda: ops.clip_grad_norm([torch.ones(3)], -1.0), lambda: ops.clip_grad_norm([torch.ones(3)], float("nan")), lambda: ops.clip_grad_norm([torch.ones(3, dtype=torch.float64)], 1.0),
    lambda: ops.grad_norm([torch.ones(3, dtype=torch.int64)]), lambda: ops.clip_grad_norm([torch.ones(4, 4)[:, :2]], 1.0), lambda: ops.clip_grad_norm([torch.ones(1).expand(4)], 1.0),
    lambda: (lambda t: ops.clip_grad_norm([t, t], 1.0))(torch.ones(3)), lambda: (lambda t: ops.clip_grad_norm([t, t[1:]], 1.0))(torch.ones(3)),
    lambda: ops.clip_grad_norm([torch.ones(3)], 1.0, out=[]), lambda: ops.clip_grad_norm([torch.ones(3)], 1.0, out=[torch.ones(4)]),
    lambda: ops.clip_grad_norm([torch.ones(3)], 1.0, out=[torch.ones(3, dtype=torch.bfloat16)]), lambda: ops.clip_grad_norm([torch.ones(2, 3)], 1.0, out=[torch.ones(3, 2).t()]),
    lambda: (lambda a, b: ops.clip_grad_norm([a, b], 1.0, out=[b, a]))(*_pair()), lambda: (lambda t: ops.clip_grad_norm([t[:4]], 1.0, out=[t[2:6]]))(torch.zeros(8)),
])
def test_clip_refuses(call):
    with pytest.raises(ValueError):
        call()


# ---- vocabulary loss -----------------------------------------------------------------------------------------------------------------
def test_vocabulary_loss_formula():
    from q38.losses import vocabulary_cross_entropy
    h, w = torch.randn(2, 5, 8, requires_grad=True), torch.randn(11, 8, requires_grad=True)
    target = torch.randint(0, 11, (2, 5))
    target[0, 1] = -100
    logp = torch.log_softmax(h.double() @ w.double().t(), -1)
    each = torch.where(target < 0, 0.0, -logp.gather(-1, target.clamp_min(0)[..., None])[..., 0])
    for reduction, want in (("none", each), ("sum", each.sum()), ("mean", each.sum() / 9)):
        got = vocabulary_cross_entropy(w, h, target, reduction)
        assert got.shape == want.shape and (got - want).abs().max() < 1e-5
    dh, dw = torch.autograd.grad(vocabulary_cross_entropy(w, h, target), [h, w])
    eh, ew = torch.autograd.grad(each.sum() / 9, [h, w])
    assert (dh - eh).abs().max() < 1e-6 and (dw - ew).abs().max() < 1e-6
    assert vocabulary_cross_entropy(w, h, torch.full((2, 5), -100)) == 0


def _vocab(h=(3, 8), w=(11, 8), t=(3,), ht=torch.float32, wt=torch.float32, tt=torch.int64, reduction="mean"):
    from q38.losses import vocabulary_cross_entropy
    return vocabulary_cross_entropy(torch.zeros(w, dtype=wt), torch.zeros(h, dtype=ht), torch.zeros(t, dtype=tt), reduction)


@pytest.mark.parametrize("wrong", [dict(h=(3, 7)), dict(h=()), dict(w=(11,)), dict(w=(0, 8)), dict(h=(3, 0), w=(11, 0)), dict(t=(4,)), dict(t=(3, 1)), dict(tt=torch.int32), dict(ht=torch.float16),
                                   dict(wt=torch.float64), dict(reduction="max")])
def test_vocabulary_loss_refuses(wrong):
    _vocab()
    with pytest.raises(ValueError):
        _vocab(**wrong)


def test_trainer_flag_for_the_loss_in_pieces():
    from q38.train import parse_args
    common = ["--run_dir", "runs/x", "--tokens", "100000"]
    assert parse_args(common).ce_pieces == 0 and parse_args(common + ["--ce_pieces", "1"]).ce_pieces == 1
    with pytest.raises(SystemExit):
        parse_args(common + ["--ce_pieces", "2"])

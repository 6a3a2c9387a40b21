"""Cross entropy over a large vocabulary in pieces against plain formulas in 64 bits.

Tolerances count roundings: u = 2^-24 per fp32 operation, 2u per addition in the tensor core (which may truncate), 2^-22 for an exponential, half a step
(2^-8) for what is bf16."""
import pytest
import torch

from q38 import ops
from q38.losses import vocabulary_cross_entropy
from q38.ops import vocab

pytestmark = pytest.mark.gpu
U, HALF = 2.0 ** -24, 2.0 ** -8
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def installed():
    ops.install()
    yield
    ops.check_errors()


def inputs(rows, vocab_size, hidden, seed=0, scale=2.0, ignored=0.1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(rows, hidden, device="cuda", generator=gen).to(BF16)
    w = (torch.randn(vocab_size, hidden, device="cuda", generator=gen) * scale / hidden ** 0.5).to(BF16)
    target = torch.randint(0, vocab_size, (rows,), device="cuda", generator=gen)
    target[torch.rand(rows, device="cuda", generator=gen) < ignored] = -100
    return h, w, target


def formula(h, w, target, up):
    """In 64 bits: losses, dz, dh, dw for row gradients `up`, and the tolerances of losses, dh and dw."""
    h, w, K, V, T = h.double(), w.double(), h.shape[1], w.shape[0], h.shape[0]
    valid = (target >= 0).double()
    z = h @ w.T
    logp = torch.log_softmax(z, -1)
    at = target.clamp_min(0)[:, None]
    losses = -logp.gather(1, at)[:, 0] * valid
    p = logp.exp()
    dz = p.scatter_add(1, at, torch.full_like(at, -1, dtype=torch.float64)) * (up.double() * valid)[:, None]
    # scores: K additions; their exponents: a product with log2 e (its rounding and the constant's) and the reference's; the sum: 2^-22 per term, chains of 150 additions
    size = (h.abs() @ w.abs().T)
    z_off = 2 * U * (K / 8 + 8) * size + 4 * U * z.abs()
    sum_off = z_off.amax(-1) + 2.0 ** -22 + 150 * U
    loss_off = (sum_off + z_off.gather(1, at)[:, 0] + 4 * U * (torch.logsumexp(z, -1).abs() + z.gather(1, at)[:, 0].abs())) * valid
    dz_off = HALF * dz.abs() + (up.double().abs() * valid)[:, None] * p * (z_off + sum_off[:, None] + 2.0 ** -20)
    dh, dw = dz @ w, dz.T @ h
    dh_off = dz_off @ w.abs() + 2 * U * (V / 8 + 8) * (dz.abs() @ w.abs())
    dw_off = dz_off.T @ h.abs() + 2 * U * (T / 8 + 8) * (dz.abs().T @ h.abs())
    return (losses, dz, dh, dw), (loss_off, dh_off, dw_off)


def within(got, want, tol, what):
    tol = tol + want.abs() * (HALF if got.dtype == BF16 else 2 * U) + 1e-37
    off = (got.double() - want).abs() - tol
    assert not (off > 0).any() and not got.isnan().any(), (what, off.max().item(), int((off > 0).sum()))


def check(h, w, target, reduction="mean", up=None):
    rows = h.shape[0]
    valid = target >= 0
    hl, wl = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = vocabulary_cross_entropy(wl, hl, target, reduction)
    count = max(1, int(valid.sum()))
    if up is None:
        up = torch.rand(rows, device="cuda") - 0.3 if reduction == "none" else torch.tensor(1.7, device="cuda")
    share = up if reduction == "none" else (up / (count if reduction == "mean" else 1)).expand(rows)
    (losses, dz, dh, dw), (loss_off, dh_off, dw_off) = formula(h.to(BF16), w.to(BF16), target, share)
    assert loss.dtype == FP32
    if reduction == "none":
        within(loss, losses, loss_off, "losses")
        assert not loss[~valid].any()
    else:
        n = count if reduction == "mean" else 1
        within(loss, losses.sum() / n, loss_off.sum() / n, "loss")
    gh, gw = torch.autograd.grad(loss, [hl, wl], up)
    assert gh.dtype == h.dtype and gw.dtype == w.dtype and gh.shape == h.shape and gw.shape == w.shape
    within(gh, dh, dh_off, "dh")
    within(gw, dw, dw_off, "dw")
    assert not gh[~valid].any()
    with torch.no_grad():
        assert torch.equal(vocabulary_cross_entropy(w, h, target, reduction), loss)
    return gh, gw


# one of everything; a vocabulary within a chunk; hidden sizes that no TMA row fits; the ends of tiles in rows and columns; the presets' vocabulary; the larger tokenizers'
SHAPES = [(1, 1, 8), (1, 5, 7), (2, 31, 1), (3, 300, 64), (37, 10112, 448), (128, 256, 64), (129, 257, 72), (257, 1000, 65), (1000, 5003, 200), (1500, 30080, 128), (5, 50048, 64),
          (4100, 2049, 96), (20000, 65, 40), (3, 200_003, 40)]


@pytest.mark.parametrize("rows,vocab_size,hidden", SHAPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_shapes(rows, vocab_size, hidden, reduction):
    check(*inputs(rows, vocab_size, hidden, seed=rows), reduction)


@pytest.mark.parametrize("rows,vocab_size,hidden,bytes_", [(300, 5003, 72, 1), (300, 5003, 72, 300 * 2 * 1024), (64, 3000, 264, 64 * 2 * 1300), (2000, 2048, 64, 2000 * 2 * 512), (7, 2561, 7, 1)])
def test_pieces(monkeypatch, rows, vocab_size, hidden, bytes_):
    args = inputs(rows, vocab_size, hidden, seed=3)
    whole = check(*args)
    monkeypatch.setattr(vocab, "PIECE_BYTES", bytes_)                # several pieces, the last of them narrower
    parts = check(*args)
    assert torch.equal(whole[1], parts[1])                           # a weight row has its sum within one piece


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_master_weights_and_sharp_scores(reduction):
    h, w, target = inputs(200, 3001, 136, seed=4, scale=12.0)        # scores of up to fifty
    check(h.float(), w.float(), target, reduction)
    check(h, w, target, reduction)


def test_strides_and_leading_dimensions():
    gen = torch.Generator(device="cuda").manual_seed(5)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(BF16)
    target = torch.randint(0, 500, (60,), device="cuda", generator=gen)
    wide, tall = rand(60, 200), rand(1001, 129)
    check(wide[:, 8:72], (0.2 * tall)[:500, 1:65], target)           # rows apart; off 16 bytes
    check(rand(64, 60).t(), (0.2 * rand(64, 500)).t(), target)       # columns apart
    check(wide[:, :65], (0.2 * rand(500, 136))[:, :65], target)      # rows that TMA takes, an odd number of their columns
    check(rand(1, 64).expand(60, 64), 0.2 * rand(500, 64), target)
    h, w = rand(3, 20, 64), 0.2 * rand(500, 64)
    got = vocabulary_cross_entropy(w, h, target.view(3, 20), "none")
    assert got.shape == (3, 20) and torch.equal(got.flatten(), vocabulary_cross_entropy(w, h.view(60, 64), target, "none"))
    every = torch.stack([target, target], 1)[:, 0]                   # targets apart
    assert torch.equal(vocabulary_cross_entropy(w, h.view(60, 64), every, "none"), got.flatten())


def test_rows_that_do_not_count():
    h, w, target = inputs(300, 1000, 64, seed=6)
    none = torch.full_like(target, -100)
    for reduction in ("mean", "sum"):
        gh, gw = check(h, w, none, reduction)
        assert not gh.any() and not gw.any()
    empty = vocabulary_cross_entropy(w.requires_grad_(), h[:0], target[:0])
    assert empty == 0 and not torch.autograd.grad(empty, w)[0].any()
    w.requires_grad_(False)
    assert vocabulary_cross_entropy(w, h[:0], target[:0], "none").shape == (0,)
    # an ignored row may hold anything without touching other rows
    spoilt = h.clone()
    spoilt[target < 0] = float("nan")
    leaf = spoilt.requires_grad_()
    got = vocabulary_cross_entropy(w, leaf, target)
    assert torch.equal(got, vocabulary_cross_entropy(w, h, target))
    clean = h.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(got, leaf)[0], torch.autograd.grad(vocabulary_cross_entropy(w, clean, target), clean)[0])


def test_targets_outside_the_vocabulary_are_reported():
    h, w, target = inputs(40, 500, 64, seed=7, ignored=0.0)
    want = vocabulary_cross_entropy(w, h, target, "none")
    for bad in (500, 511, 1 << 40, -1, -101):
        wrong = target.clone()
        wrong[3] = bad
        leaf = h.clone().requires_grad_()
        got = vocabulary_cross_entropy(w, leaf, wrong, "none")
        dh, = torch.autograd.grad(got, leaf, torch.ones_like(got))
        keep = torch.arange(40, device="cuda") != 3
        assert torch.equal(got[keep], want[keep]) and got[3] == 0 and not dh[3].any() and dh[keep].any()
        with pytest.raises(RuntimeError, match="index"):
            ops.check_errors()
    ops.check_errors()


def test_values_that_are_not_finite_stay_in_their_row():
    h, w, target = inputs(300, 700, 64, seed=8, ignored=0.0)
    clean = h.clone().requires_grad_()
    want = vocabulary_cross_entropy(w, clean, target, "none")
    ones = torch.ones_like(want)
    keep = torch.arange(300, device="cuda") != 150
    for bad in (float("nan"), float("inf"), float("-inf")):
        leaf = h.clone()
        leaf[150, 5] = bad
        leaf.requires_grad_()
        got = vocabulary_cross_entropy(w, leaf, target, "none")
        assert torch.equal(got[keep], want[keep]) and not got[150].isfinite()
        dh, = torch.autograd.grad(got, leaf, ones)
        assert torch.equal(dh[keep], torch.autograd.grad(want, clean, ones, retain_graph=True)[0][keep]) and dh[150].isnan().all()
    # columns that nothing can choose: a score of minus infinity
    h2, w2 = h.abs(), w.clone()
    w2[300:600] = float("-inf")
    target2 = target % 300
    kept = torch.cat([w2[:300], w2[600:]])
    a, b = vocabulary_cross_entropy(w2, h2, target2, "none"), vocabulary_cross_entropy(kept, h2, target2, "none")
    assert (a - b).abs().max() < 1e-4


def test_only_what_is_wanted_and_same_bits():
    h, w, target = inputs(1000, 4000, 128, seed=9)
    leaves = [h.clone().requires_grad_(), w.clone().requires_grad_()]
    loss = vocabulary_cross_entropy(leaves[1], leaves[0], target)
    first = torch.autograd.grad(loss, leaves, retain_graph=True)
    again = torch.autograd.grad(loss, leaves)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    assert torch.equal(torch.autograd.grad(vocabulary_cross_entropy(w, leaves[0], target), leaves[0])[0], first[0])
    assert torch.equal(torch.autograd.grad(vocabulary_cross_entropy(leaves[1], h, target), leaves[1])[0], first[1])
    each = vocabulary_cross_entropy(w, leaves[0], target, "none")
    total = torch.autograd.grad(each.sum(), leaves[0])[0]             # the upstream gradient is one number for all rows
    assert torch.equal(total, torch.autograd.grad(vocabulary_cross_entropy(w, leaves[0], target, "sum"), leaves[0])[0])


def test_gradient_by_differences():
    """A step of 2^-4 along bf16 directions leaves its square in third derivatives (under one per mille of the sum)."""
    h, w, target = inputs(64, 600, 64, seed=10, ignored=0.0)
    hl, wl = h.float().requires_grad_(), w.float().requires_grad_()
    dh, dw = torch.autograd.grad(vocabulary_cross_entropy(wl, hl, target, "sum"), [hl, wl])
    f = lambda a, b: torch.nn.functional.cross_entropy(a.double() @ b.double().T, target, reduction="sum")
    v = torch.sign(dh)
    assert abs((f(h.double() + v / 64, w) - f(h.double() - v / 64, w)) * 32 - (dh.double() * v).sum()) < 0.01 * dh.abs().sum()
    v = torch.sign(dw)
    assert abs((f(h, w.double() + v / 256) - f(h, w.double() - v / 256)) * 128 - (dw.double() * v).sum()) < 0.01 * dw.abs().sum()


def test_gradients_of_a_managed_parameter_are_added():
    h, w, target = inputs(500, 2000, 64, seed=11)
    plain = w.float().requires_grad_()
    want, = torch.autograd.grad(vocabulary_cross_entropy(plain, h, target), plain)
    managed = w.float().requires_grad_()
    managed._q38_bf16, managed.grad = w, torch.ones(2000, 64, device="cuda")
    vocabulary_cross_entropy(managed, h, target).backward()
    assert (managed.grad - (1 + want)).abs().max() <= 2.0 ** -23
    own = w.float().requires_grad_()
    own.grad = torch.zeros_like(own)                                  # any other parameter's gradient is returned, whatever its .grad holds
    assert torch.equal(torch.autograd.grad(vocabulary_cross_entropy(own, h, target), own)[0], want) and not own.grad.any()


def test_scores_are_not_kept():
    h, w, target = inputs(4096, 50048, 64, seed=12)
    leaf = h.requires_grad_()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    loss = vocabulary_cross_entropy(w, leaf, target)
    assert torch.cuda.memory_allocated() - base < 1 << 20
    loss.backward()
    assert torch.cuda.max_memory_allocated() - base < vocab.PIECE_BYTES + (32 << 20) < 4096 * 50048 * 2


def test_replay_from_a_graph_and_another_stream():
    h, w, target = inputs(200, 3000, 64, seed=13)
    leaves = [h.requires_grad_(), w.requires_grad_()]

    def step():
        loss = vocabulary_cross_entropy(leaves[1], leaves[0], target)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2):
        h2, _, t2 = inputs(200, 3000, 64, seed=seed)
        with torch.no_grad():
            leaves[0].copy_(h2)
        target.copy_(t2)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))


def test_more_rows_than_one_pass_takes():
    h, w, target = inputs(65536 + 300, 300, 16, seed=14)
    check(h, w, target, "none")


def test_training_after_inference_mode():
    h, w, target = inputs(50, 400, 64, seed=15)
    master = w.float().requires_grad_()
    with torch.inference_mode():
        seen = vocabulary_cross_entropy(master, h, target)           # leaves a bf16 copy of the weight behind
    loss = vocabulary_cross_entropy(master, h, target)
    assert torch.equal(loss, seen) and torch.autograd.grad(loss, master)[0].isfinite().all()


def test_changes_before_the_backward_are_noticed():
    for what in range(3):
        h, w, target = inputs(50, 400, 64, seed=16)
        leaf, other = h.clone().requires_grad_(), w.clone().requires_grad_()
        mid, mid_w = leaf * 1.0, other * 1.0
        loss = vocabulary_cross_entropy(mid_w, mid, target)
        with torch.no_grad():
            (mid, mid_w, target)[what].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_more_scores_than_2_31():
    h, w, target = inputs(70_000, 40_000, 16, seed=17)
    leaf = h.requires_grad_()
    loss = vocabulary_cross_entropy(w, leaf, target, "none")
    up = torch.rand_like(loss)
    dh, = torch.autograd.grad(loss, leaf, up)
    tail = slice(-70, None)
    (losses, _, want, _), (loss_off, dh_off, _) = formula(h.detach()[tail], w, target[tail], up[tail])
    within(loss[tail], losses, loss_off, "losses")
    within(dh[tail], want, dh_off, "dh")

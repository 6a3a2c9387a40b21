"""The training operators together, as a training step uses them: in a small decoder block against 64 bits, and in the framework's own trainer."""
from types import SimpleNamespace

import pytest
import torch

from q38 import ops
from q38.losses import LossModel, vocabulary_cross_entropy

pytestmark = pytest.mark.gpu

B, S, H, K, D, HID, VOCAB = 2, 96, 6, 2, 32, 192, 3001


def parameters():
    gen = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s, scale=1.0: scale * torch.randn(*s, device="cuda", generator=gen)
    return dict(embed=rand(VOCAB, HID), n1=1 + 0.1 * rand(HID), b1=0.1 * rand(HID), qkv=rand((H + 2 * K) * D, HID, scale=HID ** -0.5), out=rand(HID, H * D, scale=(H * D) ** -0.5),
                n2=1 + 0.1 * rand(HID), b2=0.1 * rand(HID), head=rand(VOCAB, HID, scale=2 * HID ** -0.5).to(torch.bfloat16))


def block(p, ids, target, frequencies, magnitude, norm, rotary, loss):
    """Norm, rotated causal attention, norm to bf16, vocabulary loss."""
    x = p["embed"][ids]
    qkv = (norm(x, p["n1"], p["b1"], None) @ p["qkv"].t()).view(B, S, H + 2 * K, D)
    q, k = rotary(qkv[:, :, :H], qkv[:, :, H:H + K], torch.arange(S, device="cuda") + 5000, frequencies, magnitude)
    q, k, v = q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(H // K, 1), qkv[:, :, H + K:].transpose(1, 2).repeat_interleave(H // K, 1)
    scores = (q @ k.transpose(-1, -2)) * D ** -0.5
    scores = scores.masked_fill(torch.ones(S, S, device="cuda", dtype=torch.bool).triu(1), float("-inf"))
    x = x + (scores.softmax(-1) @ v).transpose(1, 2).reshape(B, S, H * D) @ p["out"].t()
    return loss(p["head"], norm(x, p["n2"], p["b2"], torch.bfloat16), target)


def exact_norm(x, w, b, out_dtype):
    centred = x - x.mean(-1, keepdim=True)
    y = centred / torch.sqrt(centred.square().mean(-1, keepdim=True) + 1e-5) * w + b
    return y if out_dtype is None else y + (y.to(out_dtype).double() - y).detach()        # the products take bf16


def exact_rotary(q, k, pos, f, m):
    angle = pos.double()[:, None, None] * f
    def turn(x):
        a, b = x[..., :8], x[..., 8:16]
        return torch.cat([m * (a * angle.cos() - b * angle.sin()), m * (b * angle.cos() + a * angle.sin()), x[..., 16:]], -1)
    return turn(q), turn(k)


def exact_loss(w, h, target):
    logp = torch.log_softmax(h @ w.t(), -1)
    valid = target >= 0
    return -(logp.gather(-1, target.clamp_min(0)[..., None])[..., 0] * valid).sum() / valid.sum()


def test_operators_together_in_a_decoder_block():
    frequencies, magnitude = ops.rotary_frequencies(16, 1e4, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=2048), device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, VOCAB, (B, S), device="cuda", generator=gen)
    target = ids.roll(-1, 1)
    target[:, -1] = -100
    p = {n: t.requires_grad_() for n, t in parameters().items()}
    previous = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        loss = block(p, ids, target, frequencies, magnitude, lambda x, w, b, t: ops.layer_norm(x, w, b, out_dtype=t), ops.rotary, vocabulary_cross_entropy)
        grads = torch.autograd.grad(loss, list(p.values()))
    finally:
        torch.backends.cuda.matmul.allow_tf32 = previous
    e = {n: t.detach().double().requires_grad_() for n, t in p.items()}
    want = block(e, ids, target, frequencies, magnitude, exact_norm, exact_rotary, exact_loss)
    exact = torch.autograd.grad(want, list(e.values()))
    # a hidden state at the border of two bf16 values may be rounded the other way: 2^-8 of it, in one state of thousands
    assert abs(loss.item() - want.item()) < 1e-4
    for name, g, x in zip(p, grads, exact):
        # score gradients and the hidden gradient are rounded to bf16 (2^-8 each, relative to terms that partly cancel: twice that), the head's gradient once more
        assert (g.double() - x).norm() < 2.0 ** -6 * x.norm(), name
    limit = 0.5 * torch.stack([x.norm() for x in exact]).norm().item()
    out = [torch.empty_like(g) for g in grads]
    norm = ops.clip_grad_norm(list(grads), limit, out=out)
    assert abs(norm.item() / (2 * limit) - 1) < 2.0 ** -6
    assert abs(ops.grad_norm(out).item() / limit - 1) < 1e-3
    ops.check_errors()


SHAPE = dict(layers=4, hidden=128, heads=4, kv_heads=2, lin_k_heads=2, lin_v_heads=6, experts=8, topk=2, moe_ffn=32, shared_ffn=32, ngram_rows=1024, mhc_iters=5, qsa_blocks=2)


@pytest.mark.parametrize("vocab", [512, 30080])
def test_trainer_with_the_loss_in_pieces(vocab):
    """The framework's step with `--ce_pieces 1`, eager and captured: the loss terms of the same weights and batch with and without it."""
    from q38.presets import model_config
    from q38.train import TRAIN_DEFAULTS, Trainer
    x = torch.randint(1, vocab, (2, 256), generator=torch.Generator().manual_seed(3)).pin_memory()
    y = x.roll(-1, 1).pin_memory()
    first = {}
    for pieces in (0, 1):
        torch.manual_seed(0)
        args = SimpleNamespace(**{**TRAIN_DEFAULTS, "aux_coef": 0.001, "lr": 1e-3, "grad_sync": "collective", "cuda_graphs": pieces, "ce_pieces": pieces})
        trainer = Trainer(model_config(dict(SHAPE), vocab, 256, eos_token_id=7, pad_token_id=0), args, torch.device("cuda", 0))
        try:
            out = [trainer.train_step([(x, y)], lr=1e-3, dense=dense).tolist() for dense in (True, True, False)]
        finally:
            trainer.close()
        assert all(v == v and abs(v) < 1e4 for step in out for v in step)
        first[pieces] = out[0]
    ops.check_errors()
    # main and next-token terms: scores of a fresh model (below four) rounded to bf16 in one, 2^-9 of them each; the gradient norm: that and bf16 gradients
    assert abs(first[0][0] - first[1][0]) < 2.0 ** -7 and abs(first[0][2] - first[1][2]) < 2.0 ** -7
    assert abs(first[0][4] / first[1][4] - 1) < 2.0 ** -5


@pytest.mark.parametrize("vocab", [512, 30080])
def test_loss_model_gradients_with_the_loss_in_pieces(vocab):
    from q38.models import Q38ForCausalLM, modeling
    from q38.presets import model_config
    ops.install()
    torch.manual_seed(0)
    model = Q38ForCausalLM(model_config(dict(SHAPE), vocab, 256, eos_token_id=7, pad_token_id=0)).cuda()
    model.tie_embeddings()
    model.model.compute_dtype = torch.bfloat16
    model.model.qsa_dense = True
    ids = torch.randint(1, vocab, (2, 256), device="cuda")
    backend, grads = modeling.get_backend(), []
    try:
        for pieces in (False, True):
            backend.ce_pieces = pieces
            model.zero_grad(set_to_none=True)
            ce, aux, mtp, kl = LossModel(model)(ids, ids.roll(-1, 1))
            (ce + 0.3 * mtp).backward()
            grads.append(torch.cat([p.grad.flatten().double() for p in model.parameters() if p.grad is not None]))
    finally:
        backend.ce_pieces = False
    ops.check_errors()
    # two bf16 backward passes: roundings of 2^-8 in each of them, a few deep
    assert (grads[0] - grads[1]).norm() < 2.0 ** -5 * grads[0].norm()

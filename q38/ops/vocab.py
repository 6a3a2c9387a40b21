"""Cross entropy of a vocabulary projection in pieces of the vocabulary (`csrc/vocab_loss.cu`): the autograd node behind `q38.losses.vocabulary_cross_entropy`."""
import torch
from torch.autograd.function import once_differentiable

from . import error_flag, load
from .backend import _bf16_weight

# Bytes that the score gradients of one piece of the vocabulary may take.  A piece of 256 MB is written and read twice at the memory's rate while its three
# products take several times as long; smaller pieces only add launches and passes over the hidden gradient's sums.
PIECE_BYTES = 256 << 20
REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


class _VocabularyLoss(torch.autograd.Function):
    """Keeps the hidden states, the weight, the targets and one number per row; the backward forms the scores again, piece by piece."""

    @staticmethod
    def forward(ctx, hidden, weight, target, reduction):
        h = hidden if hidden.dtype == torch.bfloat16 else hidden.to(torch.bfloat16)
        loss, lse, count = load().vocab_loss_fwd(h, _bf16_weight(weight), target, reduction, error_flag(h.device))
        ctx.save_for_backward(h, weight, target, lse, count)
        ctx.reduction, ctx.dtype = reduction, hidden.dtype
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        h, weight, target, lse, count = ctx.saved_tensors
        want_dh, want_dw = ctx.needs_input_grad[:2]
        # a parameter of the trainer's arena has its gradient added in place; any other gets it returned
        grad = weight.grad if want_dw and getattr(weight, "_q38_bf16", None) is not None else None
        if grad is not None and (grad.dtype != torch.float32 or not grad.is_contiguous() or grad.shape[1] % 4 or grad.data_ptr() % 16):
            grad = None
        dh, dw = load().vocab_loss_bwd(g.float().contiguous(), h, _bf16_weight(weight), target, lse, count, ctx.reduction, want_dh, ctx.dtype == torch.float32, want_dw,
                                       weight.dtype == torch.float32, grad, PIECE_BYTES, error_flag(h.device))
        return dh, dw, None, None


def vocabulary_loss(hidden, weight, target, reduction):
    """hidden [rows, h], weight [vocabulary, h], target [rows] on one GPU; `reduction` a key of REDUCTIONS."""
    code = REDUCTIONS[reduction]
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _VocabularyLoss.apply(hidden, weight, target, code)
    h = hidden if hidden.dtype == torch.bfloat16 else hidden.to(torch.bfloat16)
    return load().vocab_loss_fwd(h, _bf16_weight(weight), target, code, error_flag(h.device))[0]

"""Training objective of Q38: main CE, router balancing, MTP CE and indexer KL.

`LossModel.forward(x, y)` returns the four terms ``(ce, aux, mtp, kl)``; the trainer combines them as
``ce + aux_coef * aux + mtp_coef * mtp + kl_coef * kl``.  Vocabulary logits are never materialised on
the GPU path: the (hidden, tied embedding, target) triple goes to a fused linear + cross-entropy op.
Semantics follow the reference (q38/train.py:215-264):

* main CE: mean over all ``B*S`` targets;
* MTP: the MTP trunk reads the un-normalised hidden state and the embedding of the next token ``y``,
  predicts ``y`` shifted left by one; the last position and every position whose ``y`` is EOS are
  ignored; loss = summed CE / max(valid, 1);
* KL: mean over QSA layers of the per-layer indexer KL;
* aux: balancing loss over the routers of all layers plus the MTP block, recorded only during this
  forward (activation-checkpoint recomputation does not record again).
"""
import torch
import torch.nn.functional as F

from .models import RouterStats, modeling
from .ops.vocab import vocabulary_loss


def linear_cross_entropy(weight, hidden, target, reduction="mean"):
    """CE of ``hidden @ weight.T`` against ``target`` (ignore index -100); fused on the GPU."""
    if modeling.get_backend() is not None and hidden.is_cuda:
        return modeling.get_backend().linear_cross_entropy(weight, hidden, target, reduction)
    logits = F.linear(hidden, weight.to(hidden.dtype)).float()
    return F.cross_entropy(logits, target, ignore_index=-100, reduction=reduction)


def vocabulary_cross_entropy(weight, hidden, target, reduction="mean"):
    """Softmax cross entropy of ``hidden @ weight.T`` against ``target`` for vocabularies of any size, without keeping logits.

    hidden: ``[..., h]`` bf16 or fp32 (rounded to bf16 for the products); weight: ``[vocabulary, h]`` bf16, or fp32 as a master weight (rounded to bf16 by every
    call, unless the trainer's arena keeps its bf16 form); target: int64 of
    hidden's leading shape, -100 where a row does not count (any other target outside the vocabulary counts as -100 and raises at
    `q38.ops.check_errors`; in host memory it raises at once).  ``reduction``: ``"mean"`` over the rows that count (0 where none does), ``"sum"``, or ``"none"`` (fp32 losses of
    target's shape, 0 where a row does not count).

    On a GPU the scores exist as one piece's bf16 gradients at most; scores, sums and losses are fp32, and results have the same bits in every
    run.  Where `linear_cross_entropy` keeps bf16 scores of all rows for the backward (vocabularies up to 16384), this forms them again: a third more
    products for memory that does not grow with the vocabulary.  First derivatives only, backward; capturable into a CUDA graph after a first call on the device;
    fake and wrapped tensors are refused."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"vocabulary_cross_entropy: reduction must be mean, sum or none, got {reduction!r}")
    if hidden.is_cuda:
        return vocabulary_loss(hidden, weight, target, reduction)
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1] or not weight.numel():
        raise ValueError("vocabulary_cross_entropy: hidden [..., h] and weight [vocabulary, h] required")
    if target.shape != hidden.shape[:-1] or target.dtype != torch.int64:
        raise ValueError("vocabulary_cross_entropy: int64 targets of hidden's leading shape required")
    if hidden.dtype not in (torch.bfloat16, torch.float32) or weight.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("vocabulary_cross_entropy: bf16 or fp32 hidden states and weight required")
    if weight.device != hidden.device or target.device != hidden.device:
        raise ValueError("vocabulary_cross_entropy: hidden, weight and target on one device required")
    h2, t1 = hidden.reshape(-1, hidden.shape[-1]), target.reshape(-1)
    scores = F.linear(h2.float(), weight.to(h2.dtype).float())              # not in bf16: half a step of a score of ten is 2 % of a probability
    losses = F.cross_entropy(scores, t1, ignore_index=-100, reduction="none")
    if reduction == "none":
        return losses.view(target.shape)
    return losses.sum() if reduction == "sum" else losses.sum() / (t1 != -100).sum().clamp_min(1)


class LossModel(torch.nn.Module):
    def __init__(self, lm, experts=None, topk=None, ce=None):
        super().__init__()
        self.lm = lm
        self.experts = experts or lm.config.num_experts
        self.topk = topk or lm.config.num_experts_per_tok
        # `ce(weight, hidden, target)` may be supplied (the reference tests pass a plain module).
        self.ce = ce
        self.last_stats = None

    def _ce(self, weight, hidden, target, reduction):
        if self.ce is not None and reduction == "mean":
            return self.ce(weight, hidden, target)
        return linear_cross_entropy(weight, hidden, target, reduction)

    def forward(self, x, y):
        m = self.lm
        stats = RouterStats(self.experts)
        blocks = m.moe_blocks()
        for block in blocks:
            block.stats_sink = stats
        try:
            hs, kls = m.model.trunk(x)
            mh = m.mtp_hidden(hs, y) if m.mtp is not None else None
        finally:
            for block in blocks:
                block.stats_sink = None
        dtype = m.model.compute_dtype or hs.dtype
        h = m.model.norm(hs, out_dtype=dtype)
        ce = self._ce(m.lm_head.weight, h.reshape(-1, h.size(-1)), y.reshape(-1), "mean")
        mtp_loss = ce.new_zeros(())
        if mh is not None:
            target = torch.cat([y[:, 1:], torch.full_like(y[:, :1], -100)], 1)
            target = target.masked_fill(y == m.config.eos_token_id, -100)
            valid = (target != -100).sum()
            mtp_loss = self._ce(m.lm_head.weight, mh.reshape(-1, mh.size(-1)), target.reshape(-1), "sum") / valid.clamp_min(1)
        kl = torch.stack(kls).mean() if kls else ce.new_zeros(())
        aux = stats.loss()
        if not torch.is_tensor(aux):
            aux = ce.new_zeros(())
        self.last_stats = stats
        return ce, aux, mtp_loss, kl

"""Cross entropy of a vocabulary projection in pieces of the vocabulary (`csrc/vocab_loss.cu`), behind `q38.losses.vocabulary_cross_entropy`."""
from . import error_flag, load
from .backend import _bf16_weight

# Bytes that the score gradients of one piece of the vocabulary may take.  A piece of 256 MB is written and read twice at the memory's rate while its three
# products take several times as long; smaller pieces only add launches and passes over the hidden gradient's sums.
PIECE_BYTES = 256 << 20
REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def vocabulary_loss(hidden, weight, target, reduction):
    """hidden [..., h], weight [vocabulary, h], target [...] on one GPU; `reduction` a key of REDUCTIONS.  A parameter of the trainer's arena (it carries its bf16
    shadow) has its gradient added to its buffer in place, any other gets it returned."""
    managed = getattr(weight, "_q38_bf16", None) is not None
    return load().vocab_loss(hidden, weight, _bf16_weight(weight), target, REDUCTIONS[reduction], managed, PIECE_BYTES, error_flag(hidden.device))

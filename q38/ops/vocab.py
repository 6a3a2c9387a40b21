"""Cross entropy of a vocabulary projection in pieces of the vocabulary (`csrc/vocab_loss.cu`), behind `q38.losses.vocabulary_cross_entropy`."""
import torch

from . import _error_flags, error_flag, load

# Bytes that the score gradients of one piece of the vocabulary may take (a piece has 256 words at least: more than this beyond 524288 rows).  A piece of 256 MB is written and read twice at the memory's rate while its three
# products take several times as long; smaller pieces only add launches and passes over the hidden gradient's sums.
PIECE_BYTES = 256 << 20
REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def vocabulary_loss(hidden, weight, target, reduction):
    """hidden [..., h], weight [vocabulary, h], target [...] on one GPU; `reduction` a key of REDUCTIONS.  A parameter of the trainer's arena (it carries its bf16
    shadow) has its gradient added to its buffer in place, any other gets it returned.  An fp32 weight outside the arena is rounded by every call (50048 x 1024: 2 % of
    a training pass): a copy kept on the weight would be missing from a captured graph, unordered on a second stream and stale after a change through `.data`."""
    lib = load()
    if hidden.device.index not in _error_flags:
        # the device's error word is about to be made and kept: not as a fake tensor, and not by a graph, whose replays would write its zeros
        lib.check_operands([hidden, weight, target], "vocabulary_cross_entropy")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("vocabulary_cross_entropy: call it once on this device (or q38.ops.install()) before it is captured")
    shadow = getattr(weight, "_q38_bf16", None)
    weight16 = shadow if shadow is not None else weight.detach().to(torch.bfloat16)
    return lib.vocab_loss(hidden, weight, weight16, target, REDUCTIONS[reduction], shadow is not None, PIECE_BYTES, error_flag(hidden.device))

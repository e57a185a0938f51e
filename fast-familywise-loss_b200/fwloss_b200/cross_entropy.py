"""Softmax cross entropy of an output layer without materialised logits.

    from fwloss_b200 import lm_head_cross_entropy
    loss = lm_head_cross_entropy(hidden, weight, target)      # hidden [B, D], weight [V, D]
    loss.backward()                                           # hidden.grad, weight.grad

The softmax counterpart of lm_head.fw_lm_head_loss, for bfloat16 operands as
there and for float16 ones; not for its float32 ones, which no tensor-core
product takes at full precision.
Forward keeps each row's log-sum-exp; backward forms the logit gradient again
in pieces of the vocabulary (a bounded workspace) and multiplies it on the
tensor cores.  Logits, statistics and sums are fp32, and so is the loss,
whatever the operands' type: a 16-bit loss near 10 would move in steps of
1/32.  No counterpart in the reference, which takes logits as input.
"""
from ._native import ext

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def lm_head_cross_entropy(hidden, weight, target, reduction="mean", ignore_index=-100, status=None):
    """Cross entropy of softmax(hidden @ weight^T) against int64 targets [B],
    fp32: 0-d for reduction "mean" / "sum", [B] for "none".

    hidden [B, D] and weight [V, D]: CUDA, both bfloat16 or both float16.  Rows
    whose target is ignore_index take no part, whatever hidden holds there:
    loss 0 under "none", gradient 0, and the mean is over the other rows (NaN
    if there is none).  Any other target outside [0, V) makes its row's loss
    and gradient NaN (and weight's gradient, a sum over the rows); an on-chip
    wait that gave up does so to what it was for.  `status`, if given, is an
    int32 CUDA tensor whose first word receives FWB_STATUS_* flags (target out
    of range, non-finite row, a wait that gave up)."""
    mode = _REDUCTIONS.get(reduction)
    if mode is None:
        raise ValueError(f"Invalid reduction mode: {reduction}")
    return ext().lm_head_cross_entropy(hidden, weight, target, mode, ignore_index, status)

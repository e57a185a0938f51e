"""Softmax cross entropy of an output layer without materialised logits.

    from fwloss_b200 import lm_head_cross_entropy
    loss = lm_head_cross_entropy(hidden, weight, target)      # hidden [B, D], weight [V, D]
    loss.backward()                                           # hidden.grad, weight.grad

The softmax counterpart of lm_head.fw_lm_head_loss, with the same operands.
Forward keeps each row's log-sum-exp; backward forms the logit gradient again
in pieces of the vocabulary (a bounded workspace) and multiplies it on the
tensor cores.  Logits, statistics and sums are fp32, and so is the loss,
whatever the operands' type: a 16-bit loss near 10 would move in steps of
1/32.  No counterpart in the reference, which takes logits as input.
"""
import torch
from torch.autograd.function import once_differentiable

from ._native import ext

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


class _LMHeadCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index, reduction, status):
        loss, state = ext().xent_forward(hidden, weight, target, ignore_index, reduction, status)
        ctx.save_for_backward(weight, state)
        ctx.rows, ctx.reduction, ctx.status = hidden.shape[0], reduction, status
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        weight, state = ctx.saved_tensors
        want_h, want_w = ctx.needs_input_grad[:2]
        dh, dw = ext().xent_backward(weight, ctx.rows, g, ctx.reduction, state, want_h, want_w, ctx.status)
        return dh if want_h else None, dw if want_w else None, None, None, None, None


def lm_head_cross_entropy(hidden, weight, target, reduction="mean", ignore_index=-100, status=None):
    """Cross entropy of softmax(hidden @ weight^T) against int64 targets [B],
    fp32: 0-d for reduction "mean" / "sum", [B] for "none".

    hidden [B, D] and weight [V, D]: CUDA, both bfloat16 or both float16.  Rows
    whose target is ignore_index take no part, whatever hidden holds there:
    loss 0 under "none", gradient 0, and the mean is over the other rows (NaN
    if there is none).  Any other target outside [0, V) makes its row's loss
    and gradient NaN.  `status`, if given, is an int32 CUDA tensor whose first
    word receives FWB_STATUS_* flags (target out of range, non-finite row, a
    wait that gave up)."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"Invalid reduction mode: {reduction}")
    if not (isinstance(hidden, torch.Tensor) and isinstance(weight, torch.Tensor) and hidden.is_cuda and weight.is_cuda):
        raise TypeError("lm_head_cross_entropy: hidden and weight must be CUDA tensors (this build has no CPU path)")
    if hidden.dim() != 2 or weight.dim() != 2 or 0 in weight.shape:
        raise TypeError("lm_head_cross_entropy: hidden [B, D] and weight [V, D] must be matrices")
    if hidden.dtype != weight.dtype or hidden.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("lm_head_cross_entropy: hidden and weight must both be bfloat16 or both float16")
    if hidden.shape[1] != weight.shape[1]:
        raise ValueError("lm_head_cross_entropy: hidden and weight disagree on D")
    if target.dtype != torch.int64:
        raise TypeError("lm_head_cross_entropy: target must be int64")
    if target.dim() != 1 or target.shape[0] != hidden.shape[0]:
        raise ValueError("lm_head_cross_entropy: target must have shape [B]")
    if weight.device != hidden.device or target.device != hidden.device:
        raise ValueError("lm_head_cross_entropy: hidden, weight and target must be on one device")
    mode = _REDUCTIONS[reduction]
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _LMHeadCrossEntropy.apply(hidden, weight, target, int(ignore_index), mode, status)
    return ext().xent_forward(hidden.detach(), weight.detach(), target, int(ignore_index), mode, status)[0]

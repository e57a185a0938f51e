"""Rows of an embedding table, scaled, and the table's gradient.

    from fwloss_b200 import embed_tokens
    x = embed_tokens(tokens, weight, scale=D ** 0.5)     # tokens [...] int64, weight [V, D]

The gradient of the table is summed from the tokens sorted by id: no atomics,
so the same inputs give the same gradient bit for bit, in fp32 whatever the
table's type.  No counterpart in the reference, which takes logits as input.
"""
import torch
from torch.autograd.function import once_differentiable

from ._native import ext

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding_idx, status):
        ctx.save_for_backward(tokens)
        ctx.rows, ctx.scale, ctx.padding_idx, ctx.status = weight.shape[0], scale, padding_idx, status
        return ext().embed_rows(tokens, weight, scale, status)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (tokens,) = ctx.saved_tensors
        return None, ext().embed_grad(tokens, g, ctx.rows, ctx.scale, ctx.padding_idx, ctx.status), None, None, None


def embed_tokens(tokens, weight, scale=1.0, padding_idx=None, status=None):
    """scale * weight[tokens], shape tokens.shape + [D], in weight's dtype.

    tokens: int64, any shape, on weight's device; weight [V, D] float32,
    bfloat16 or float16.  `padding_idx` names a row whose gradient is zero (its
    tokens are looked up like any other).  A token outside [0, V) gives a row
    of NaN, adds nothing to the gradient, and sets FWB_STATUS_LABEL_RANGE in
    `status`, if given (an int32 CUDA tensor)."""
    if not (isinstance(weight, torch.Tensor) and weight.is_cuda):
        raise TypeError("embed_tokens: weight must be a CUDA tensor (this build has no CPU path)")
    if weight.dim() != 2 or weight.dtype not in _FLOATS or 0 in weight.shape:
        raise TypeError("embed_tokens: weight must be a non-empty 2-D float32, bfloat16 or float16 tensor [V, D]")
    if not isinstance(tokens, torch.Tensor) or tokens.dtype != torch.int64:
        raise TypeError("embed_tokens: tokens must be an int64 tensor")
    if tokens.device != weight.device:
        raise ValueError("embed_tokens: tokens must be on weight's device")
    if padding_idx is None:
        padding_idx = -1
    elif not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f"embed_tokens: padding_idx {padding_idx} is outside the table")
    if torch.is_grad_enabled() and weight.requires_grad:
        return _EmbedTokens.apply(tokens, weight, float(scale), int(padding_idx), status)
    return ext().embed_rows(tokens, weight.detach(), float(scale), status)

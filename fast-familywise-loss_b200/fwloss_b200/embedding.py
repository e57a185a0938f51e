"""Rows of an embedding table, scaled, and the table's gradient.

    from fwloss_b200 import embed_tokens
    x = embed_tokens(tokens, weight, scale=D ** 0.5)     # tokens [...] int64, weight [V, D]

The gradient of the table is summed from the tokens sorted by id: no atomics,
so the same inputs give the same gradient bit for bit, in fp32 whatever the
table's type.  No counterpart in the reference, which takes logits as input.
"""
from ._native import ext


def embed_tokens(tokens, weight, scale=1.0, padding_idx=None, status=None):
    """scale * weight[tokens], shape tokens.shape + [D], in weight's dtype.

    tokens: int64, any shape, on weight's device; weight [V, D] float32,
    bfloat16 or float16.  `padding_idx` names a row whose gradient is zero (its
    tokens are looked up like any other).  A token outside [0, V) gives a row
    of NaN, adds nothing to the gradient, and sets FWB_STATUS_LABEL_RANGE in
    `status`, if given (an int32 CUDA tensor)."""
    return ext().embed_tokens(tokens, weight, scale, padding_idx, status)

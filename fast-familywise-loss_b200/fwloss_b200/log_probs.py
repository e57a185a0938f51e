"""Log probabilities of given tokens, with the entropy of their rows and the
likeliest alternatives.

    from fwloss_b200 import lm_head_log_probs, token_log_probs
    logp, entropy = token_log_probs(logits, tokens)                     # logits [..., V]
    logp, entropy, top_logp, top_ids = token_log_probs(logits, tokens, top_k=5)
    logp, entropy = lm_head_log_probs(hidden, weight, tokens)           # hidden [B, D], weight [V, D]

For scoring what a model answered (serving, evaluation), and for training on
it: a policy gradient takes the log probabilities' gradient, an entropy bonus
the entropies', both in one pass over the logits, or over the operands of the
output layer they come from, whose logits are then never stored (as in
lm_head_cross_entropy).  Results and arithmetic are fp32 whatever the operands'
type.  No counterpart in the reference.
"""
from ._native import ext


def token_log_probs(logits, tokens, top_k=0, temperature=1.0, ignore_index=-100, status=None):
    """(logp, entropy) of softmax(logits / temperature) over the last
    dimension, both fp32 in tokens' shape; with top_k, (logp, entropy,
    top_logp, top_ids), the last two [..., top_k].

    logits [..., V] float32, bfloat16 or float16, CUDA; tokens [...] int64 on
    the same device.  logp is the log probability of the row's token, entropy
    the row's, in nats; top_ids (int64) are the likeliest columns and top_logp
    their log probabilities, the likeliest first, equal logits by the lowest
    column; top_k is at most 32.  A column of -inf has probability 0.

    Rows whose token is ignore_index take no part, whatever the logits hold
    there: 0, top_ids -1, gradient 0.  Any other token outside [0, V), and a
    row whose largest logit is not finite, give NaN (top_ids -1) and a gradient
    of NaN in that row, and set FWB_STATUS_LABEL_RANGE or FWB_STATUS_NONFINITE
    in `status`, if given (an int32 CUDA tensor).

    Differentiable in logits through logp and entropy (top_logp is not): the
    backward pass reads the logits again, so they must not change before it."""
    return ext().token_log_probs(logits, tokens, top_k, temperature, ignore_index, status)


def lm_head_log_probs(hidden, weight, tokens, temperature=1.0, ignore_index=-100, status=None):
    """(logp, entropy) of softmax(hidden @ weight^T / temperature) against
    int64 tokens [B], both fp32 [B].

    hidden [B, D] and weight [V, D]: CUDA, both bfloat16 or both float16.  Rows
    whose token is ignore_index take no part, whatever hidden holds there: 0,
    gradient 0.  Any other token outside [0, V), and a row whose largest logit
    is not finite, give NaN in that row, a gradient of NaN there and, as it is a
    sum over the rows, in all of weight's; an on-chip wait that gave up does so
    to what it was for.  `status`, if given, is an int32 CUDA tensor whose first
    word receives FWB_STATUS_* flags.

    Differentiable in hidden and weight through both results.  The backward pass
    forms the logit gradient in pieces of the vocabulary (a bounded workspace)
    and rounds it, upstream factors included, to the operands' type; what that
    takes from the entry of a row's token is added to both gradients.  float16
    holds the entries relative to the largest factor m of the call: each is off
    by up to 2^-37 m / temperature, so that in a row whose own factor is 2^-20 m,
    probabilities under 2^-17 may be lost (its token's entry is not).  bfloat16
    has the range of float32.  An upstream gradient that is not finite makes its
    row of hidden's gradient, and all of weight's, NaN."""
    return ext().lm_head_log_probs(hidden, weight, tokens, temperature, ignore_index, status)

"""Log probabilities of given tokens, with the entropy of their rows and the
likeliest alternatives.

    from fwloss_b200 import token_log_probs
    logp, entropy = token_log_probs(logits, tokens)                     # logits [..., V]
    logp, entropy, top_logp, top_ids = token_log_probs(logits, tokens, top_k=5)

For scoring what a model answered (serving, evaluation), and for training on
it: a policy gradient takes the log probabilities' gradient, an entropy bonus
the entropies', both in one pass over the logits.  Results and arithmetic are
fp32 whatever the logits' type.  No counterpart in the reference.
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

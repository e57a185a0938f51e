"""Output layer in 8-bit integers, for serving.

    from fwloss_b200 import int8_linear, quantize_rows_int8
    wq, w_scale = quantize_rows_int8(weight)                   # once, weight [V, D]
    logits = int8_linear(q, q_scale, wq, w_scale)              # q, q_scale from rms_norm_int8

out[t, n] = (sum_k q[t, k] wq[n, k]) * q_scale[t] * w_scale[n]: the sum is an
exact 32-bit integer, the result is rounded once.  Any number of tokens from
one up; few tokens are read against the weight at memory speed.  No
counterpart in the reference, which takes logits as input.
"""
import torch

from ._native import ext


def quantize_rows_int8(x):
    """(q int8 [R, D], scale fp32 [R]) with x[r] = q[r] * scale[r] to within
    half a step (and fp32's rounding), scale = max|x[r]| / 127.  q's rows start on 16-byte
    boundaries (its row stride is D rounded up to 16)."""
    return ext().quantize_rows_int8(x)


def int8_linear(q, q_scale, weight, weight_scale, out_dtype=torch.bfloat16, status=None):
    """Logits [..., N] in out_dtype from q [..., K] int8 with q_scale [...] and
    weight [N, K] int8 with weight_scale [N] (scales fp32); K at most 131071.

    Rows of q and weight that do not start on 16-byte boundaries are copied
    first, at every call: lay a weight out with quantize_rows_int8.  Where an
    on-chip wait gave up, the logits it was for are NaN; `status`, if given,
    receives FWB_STATUS_TIMEOUT."""
    return ext().int8_linear(q, q_scale, weight, weight_scale, out_dtype, status)

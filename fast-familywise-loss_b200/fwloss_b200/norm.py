"""Root-mean-square norm of a residual stream.

    from fwloss_b200 import rms_norm, rms_norm_int8
    y = rms_norm(x, weight)                                   # y = x / rms(x) * weight
    y, stream = rms_norm(x, weight, residual=stream)          # stream + x, and its norm
    q, scale, stream = rms_norm_int8(x, weight, residual=stream)   # 8-bit rows for int8_linear

The sum is rounded once to the stream's dtype and the norm is that of the
stored sum, forward and backward alike; everything else is fp32 with one
rounding at the end.  No counterpart in the reference, which takes logits as
input.
"""
from ._native import ext


def rms_norm(x, weight, eps=1e-6, residual=None):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension; with
    `residual`, (the norm of x + residual, x + residual).

    x [..., D] float32, bfloat16 or float16; weight [D] in x's dtype or
    float32; results in x's dtype.  Differentiable in x, residual and weight
    (the weight's gradient is added in a fixed order)."""
    return ext().rms_norm(x, weight, eps, residual)


def rms_norm_int8(x, weight, eps=1e-6, residual=None):
    """The norm in 8-bit integers with a scale per row, the input of
    int8_linear: (q int8 [..., D], scale fp32 [...]) with norm = q * scale, and
    x + residual as a third result where `residual` is given.

    scale = max|norm| / 127 of the row, q = norm / scale to the nearest (by the
    fp32 reciprocal: within 2^-17 of the middle between two steps, either).  A row of zeros has scale 0; a row that is not finite has that scale
    and q = 0, so that what is computed from it is NaN.  For serving: not
    differentiable."""
    return ext().rms_norm_int8(x, weight, eps, residual)

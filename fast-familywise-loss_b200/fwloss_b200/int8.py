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

MAX_K = 131071  # 127 * 128 * K stays below 2^31
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def quantize_rows_int8(x):
    """(q int8 [R, D], scale fp32 [R]) with x[r] = q[r] * scale[r] to within
    half a step, scale = max|x[r]| / 127.  q's rows start on 16-byte
    boundaries (its row stride is D rounded up to 16)."""
    if not (isinstance(x, torch.Tensor) and x.is_cuda):
        raise TypeError("quantize_rows_int8: x must be a CUDA tensor (this build has no CPU path)")
    if x.dim() != 2 or x.dtype not in _FLOATS or x.shape[1] < 1:
        raise TypeError("quantize_rows_int8: x must be a 2-D float32, bfloat16 or float16 tensor [R, D]")
    return tuple(ext().quantize_rows_int8(x.detach()))


def int8_linear(q, q_scale, weight, weight_scale, out_dtype=torch.bfloat16, status=None):
    """Logits [..., N] in out_dtype from q [..., K] int8 with q_scale [...] and
    weight [N, K] int8 with weight_scale [N] (scales fp32).

    Rows of q and weight that do not start on 16-byte boundaries are copied
    first, at every call: lay a weight out with quantize_rows_int8.  `status`,
    if given, receives FWB_STATUS_TIMEOUT if an on-chip wait gave up."""
    for name, t, dt in (("q", q, torch.int8), ("weight", weight, torch.int8), ("q_scale", q_scale, torch.float32),
                        ("weight_scale", weight_scale, torch.float32)):
        if not (isinstance(t, torch.Tensor) and t.is_cuda) or t.dtype != dt:
            raise TypeError(f"int8_linear: {name} must be a CUDA tensor of {dt}")
        if t.device != q.device:
            raise ValueError("int8_linear: all inputs must be on one device")
    if out_dtype not in _FLOATS:
        raise TypeError("int8_linear: out_dtype must be float32, bfloat16 or float16")
    if weight.dim() != 2 or q.dim() < 1 or q.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError("int8_linear: q [..., K] and weight [N, K] disagree")
    if q_scale.shape != q.shape[:-1] or weight_scale.shape != weight.shape[:1]:
        raise ValueError("int8_linear: q_scale must have q's leading shape and weight_scale the shape [N]")
    if weight.shape[1] > MAX_K:
        raise ValueError(f"int8_linear: K must be at most {MAX_K}")
    if q.dim() == 2:
        return ext().int8_linear(q, q_scale, weight, weight_scale, out_dtype, status)
    out = ext().int8_linear(q.reshape(-1, q.shape[-1]), q_scale.reshape(-1), weight, weight_scale, out_dtype, status)
    return out.view(*q.shape[:-1], weight.shape[0])

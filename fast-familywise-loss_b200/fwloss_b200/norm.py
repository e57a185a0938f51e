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
import torch
from torch.autograd.function import once_differentiable

from ._native import ext

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        D = x.shape[-1]
        out = ext().rms_norm(x.reshape(-1, D), None if residual is None else residual.reshape(-1, D), weight, eps)
        ctx.save_for_backward(out[2] if residual is not None else x, weight, out[1])
        ctx.set_materialize_grads(False)
        y = out[0].view(x.shape)
        return y if residual is None else (y, out[2].view(x.shape))

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum=None):
        total, weight, rstd = ctx.saved_tensors
        want_x, want_r, want_w = ctx.needs_input_grad[:3]
        if dy is None:  # only the sum was used
            return dsum if want_x else None, dsum if want_r else None, None, None
        D = dy.shape[-1]
        grads = ext().rms_norm_grad(dy.reshape(-1, D), total.reshape(-1, D),
                                    None if dsum is None else dsum.reshape(-1, D), weight, rstd, want_w)
        dx = grads[0].view(dy.shape)
        return dx if want_x else None, dx if want_r else None, grads[1] if want_w else None, None


def _check(name, x, weight, eps, residual):
    if not (isinstance(x, torch.Tensor) and x.is_cuda):
        raise TypeError(f"{name}: x must be a CUDA tensor (this build has no CPU path)")
    if x.dim() < 1 or x.dtype not in _FLOATS or x.shape[-1] < 1:
        raise TypeError(f"{name}: x must be a float32, bfloat16 or float16 tensor [..., D]")
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"{name}: weight must have x's dtype or float32")
    if weight.dim() != 1 or weight.shape[0] != x.shape[-1] or weight.device != x.device:
        raise ValueError(f"{name}: weight must have shape [D] on x's device")
    if not eps >= 0.0:
        raise ValueError(f"{name}: eps must not be negative")
    if residual is not None:
        if residual.dtype != x.dtype:
            raise TypeError(f"{name}: residual must have x's dtype")
        if residual.shape != x.shape or residual.device != x.device:
            raise ValueError(f"{name}: residual must have x's shape and device")


def rms_norm(x, weight, eps=1e-6, residual=None):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension; with
    `residual`, (the norm of x + residual, x + residual).

    x [..., D] float32, bfloat16 or float16; weight [D] in x's dtype or
    float32; results in x's dtype.  Differentiable in x, residual and weight
    (the weight's gradient is added in a fixed order)."""
    _check("rms_norm", x, weight, eps, residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (residual is not None and residual.requires_grad)):
        return _RMSNorm.apply(x, residual, weight, float(eps))
    D = x.shape[-1]
    out = ext().rms_norm(x.detach().reshape(-1, D), None if residual is None else residual.detach().reshape(-1, D),
                         weight.detach(), float(eps))
    y = out[0].view(x.shape)
    return y if residual is None else (y, out[2].view(x.shape))


def rms_norm_int8(x, weight, eps=1e-6, residual=None):
    """The norm in 8-bit integers with a scale per row, the input of
    int8_linear: (q int8 [..., D], scale fp32 [...]) with norm = q * scale, and
    x + residual as a third result where `residual` is given.

    scale = max|norm| / 127 of the row, q rounded to the nearest (ties to
    even).  A row of zeros has scale 0; a row that is not finite has that scale
    and q = 0, so that what is computed from it is NaN.  For serving: not
    differentiable."""
    _check("rms_norm_int8", x, weight, eps, residual)
    D = x.shape[-1]
    out = ext().rms_norm_int8(x.detach().reshape(-1, D),
                              None if residual is None else residual.detach().reshape(-1, D), weight.detach(),
                              float(eps))
    if x.dim() != 2:
        out = [out[0].unflatten(0, x.shape[:-1]) if x.dim() > 1 else out[0][0], out[1].view(x.shape[:-1])] + \
            [t.view(x.shape) for t in out[2:]]
    return tuple(out)

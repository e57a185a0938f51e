"""Global norm of many gradients, and clipping to it.

    from fwloss_b200 import clip_grad_norm_, grad_norm
    norm = clip_grad_norm_([p.grad for p in parameters], 1.0)         # in place
    norm = clip_grad_norm_(grads, 1.0, out=master_grads)              # e.g. bfloat16 into float32

The norm stays on the device (nothing synchronises), and so does the decision
whether to clip: in a step captured into a CUDA graph, too.  Sums are fp32
over 32 elements and fp64 beyond, in a fixed order.  Two launches for up to
512 tensors.

Gradients sharded over ranks (vocab_parallel's weight shard, next to
replicated ones): sum the squares over the ranks, and clip to that norm.

    total = grad_norm(sharded).square()
    torch.distributed.all_reduce(total)
    norm = (total + grad_norm(replicated).square()).sqrt()
    clip_grad_norm_(sharded + replicated, 1.0, norm=norm)

No counterpart in the reference.
"""
import torch

from ._native import ext


def _tensors(grads):
    return [grads] if isinstance(grads, torch.Tensor) else list(grads)


def grad_norm(grads, status=None):
    """sqrt of the sum of the squares of all elements, a 0-d float32 tensor.

    grads: a tensor or an iterable of them, any shapes; float32, bfloat16 and
    float16 may be mixed; on one CUDA device.  Entries of None (parameters
    without a gradient) are skipped.  Tensors whose memory has gaps are copied
    first.  `status`, if given, receives FWB_STATUS_NONFINITE where the norm is
    not finite (an int32 CUDA tensor)."""
    return ext().grad_norm([g for g in _tensors(grads) if g is not None], status)


def clip_grad_norm_(grads, max_norm, out=None, norm=None, status=None):
    """Multiplies the gradients by min(1, max_norm / their global norm) and
    returns that norm (before clipping), a 0-d float32 tensor.

    grads as for grad_norm; they are changed in place, or left as they are
    where `out` has a tensor for each of them (same shapes, any of the three
    types), which then holds the products, rounded once.  Tensors that are
    written must not overlap others, nor require grad (with `out`, gradients that
    do are refused in grad mode): pass p.grad, not p.
    `norm`, a float32 CUDA tensor of one value outside the tensors that are
    written, is taken for the global norm instead of the tensors' own, and
    returned.  A norm that is not finite gives what the formula gives: infinity
    scales by 0 (NaN where an element is infinite; under a max_norm of infinity
    nothing is scaled), NaN makes everything NaN; `status` receives
    FWB_STATUS_NONFINITE when the norm is computed here.

    Unlike torch.nn.utils.clip_grad_norm_ it takes gradients, not parameters,
    adds nothing to the norm in the divisor (there 1e-6), and raises ValueError
    where no gradient is given (there a norm of 0): there is no device to put
    the norm on, so a step without gradients of its own has to skip the call."""
    grads = _tensors(grads)
    if out is not None:
        out = _tensors(out)
        if len(out) != len(grads):
            raise ValueError("clip_grad_norm_: out must have a tensor for every gradient")
        out = [o for o, g in zip(out, grads) if g is not None]
    return ext().clip_grad_norm_([g for g in grads if g is not None], max_norm, out, norm, status)

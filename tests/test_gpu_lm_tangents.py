"""Forward-mode differentiation, which the operators do not have, is refused
whether or not the operand also records for the reverse mode."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import fwloss_b200 as fw
import lm_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("record", [False, True])
@pytest.mark.parametrize("grad_mode", [False, True])
def test_tangents_are_refused(record, grad_mode):
    g = R.gen(1)
    ids = torch.randint(0, 40, (30,), generator=g, device="cuda")

    def operand(*shape):
        return R.normal(shape, torch.bfloat16, g).requires_grad_(record)

    h, w, gain = operand(30, 64), operand(40, 64), operand(64)
    dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
    with fwd.dual_level(), torch.set_grad_enabled(grad_mode):
        for call in (lambda: fw.embed_tokens(ids, dual(w)), lambda: fw.rms_norm(dual(h), gain), lambda: fw.rms_norm(h, dual(gain)),
                     lambda: fw.rms_norm(h, gain, residual=dual(h)), lambda: fw.lm_head_cross_entropy(dual(h), w, ids),
                     lambda: fw.lm_head_cross_entropy(h, dual(w), ids)):
            with pytest.raises(RuntimeError, match="forward"):
                call()
        assert fw.rms_norm(h, gain).isfinite().all()  # no tangent inside the level

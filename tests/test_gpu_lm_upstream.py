"""lm_head_cross_entropy under factors per row that are not finite."""
import pytest
import torch

import lm_ref as R
from fwloss_b200 import capi, lm_head_cross_entropy

pytestmark = pytest.mark.gpu


def operands(dtype, B=150, D=72, V=400, seed=3):
    g = R.gen(seed)
    return (R.normal((B, D), dtype, g), R.normal((V, D), dtype, g, 2.0 / D ** 0.5),
            torch.randint(0, V, (B,), generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda") + 0.5)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("what", [float("inf"), -float("inf"), float("nan")])
def test_a_factor_that_is_not_finite_stays_in_its_row(dtype, what):
    """The other rows of dhidden are those of a run without it; dweight, a sum over all rows, is not finite."""
    h, w, y, go = operands(dtype)
    a, b = h.requires_grad_(True), w.requires_grad_(True)
    loss = lm_head_cross_entropy(a, b, y, reduction="none")
    clean, hit = go.clone(), go.clone()
    clean[40], hit[40] = 0.0, what
    want, _ = torch.autograd.grad(loss, (a, b), clean, retain_graph=True)
    dh, dw = torch.autograd.grad(loss, (a, b), hit)
    others = torch.arange(len(go), device="cuda") != 40
    assert want.isfinite().all()
    assert torch.equal(dh[others], want[others])
    assert not dh[40].isfinite().any() and not dw.isfinite().any()


@pytest.mark.parametrize("what", [float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_sign_of_an_infinite_factor(dtype, what):
    """Two equal logits: the logit gradients 1/2 and -1/2 times weights of opposite signs point the same way,
    so dhidden is the factor's own infinity."""
    h = torch.zeros(1, 8, dtype=dtype, device="cuda", requires_grad=True)
    w = torch.tensor([[1.0], [-1.0]], device="cuda").expand(2, 8).to(dtype).requires_grad_(True)
    loss = lm_head_cross_entropy(h, w, torch.tensor([1], device="cuda"), reduction="none")
    (dh,) = torch.autograd.grad(loss, h, torch.tensor([what], device="cuda"))
    assert torch.equal(dh, torch.full_like(dh, what))  # 0.5 * 1 - 0.5 * -1 = 1 times the factor

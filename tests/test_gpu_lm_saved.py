"""Saved operands that come back with other strides, and forward-mode tangents."""
import pytest
import torch

import lm_ref as R
from fwloss_b200 import lm_head_cross_entropy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,ld", [(65, 72), (64, 65), (65, 65), (64, 72)])
@pytest.mark.parametrize("move", [lambda t: t.contiguous().clone(), lambda t: torch.nn.functional.pad(t, (0, 7))[..., : t.shape[-1]]],
                         ids=["contiguous", "padded"])
def test_cross_entropy_weight_restored_with_another_stride(D, ld, move):
    """Rows saved on 16-byte boundaries and restored off them, and the other way round."""
    g = R.gen(D)
    h = R.normal((90, D), torch.bfloat16, g).requires_grad_(True)
    w = R.normal((300, ld), torch.bfloat16, g, 0.2)[:, :D].requires_grad_(True)
    y = torch.randint(0, 300, (90,), generator=g, device="cuda")
    want = torch.autograd.grad(lm_head_cross_entropy(h, w, y), (h, w))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: move(t) if t.dim() == 2 else t):
        loss = lm_head_cross_entropy(h, w, y)
    for got, ref in zip(torch.autograd.grad(loss, (h, w)), want):
        assert torch.equal(got, ref)

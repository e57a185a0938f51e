"""What the extension's gradient of the embedding refuses: operands whose
memory the kernels would otherwise read as something else, or past its end."""
import pytest
import torch

from fwloss_b200._native import ext

pytestmark = pytest.mark.gpu


def test_embed_grad_refuses():
    ids, g = torch.zeros(30, dtype=torch.int64, device="cuda"), torch.zeros(30, 8, device="cuda")
    f = ext().embed_grad
    assert f(ids, g, 4, 1.0, -1, None).shape == (4, 8)
    assert f(ids.view(5, 6), g.view(5, 6, 8), 4, 1.0, 3, None).shape == (4, 8)
    for bad in ((ids.int(), g), (ids, g.double()), (ids, g.cpu()), (ids, g.long())):
        with pytest.raises(TypeError):
            f(*bad, 4, 1.0, -1, None)
    for bad in ((ids.cpu(), g), (ids, g[:29]), (ids[:29], g), (ids.view(5, 6), g)):
        with pytest.raises(ValueError):
            f(*bad, 4, 1.0, -1, None)
    for rows, padding in ((0, -1), (4, 4), (4, -2)):
        with pytest.raises(ValueError):
            f(ids, g, rows, 1.0, padding, None)

"""Operators one after the other on one stream, each reading what the one
before it has just written, against the same chain with a wait after every
call; buffers are reused from pass to pass, so that an early read would show."""
import pytest
import torch

import fwloss_b200 as fw
import lm_ref as R
from fwloss_b200._native import ext

pytestmark = pytest.mark.gpu


def norm_into_loss(x, w, gain, y, wait):
    h = fw.rms_norm(x, gain)
    wait()
    return [h, fw.lm_head_cross_entropy(h, w, y, reduction="none")]


def norm_gradient_into_table(x, w, gain, y, wait):
    a = x.detach().requires_grad_(True)
    out = fw.rms_norm(a, gain)
    wait()
    (dx,) = torch.autograd.grad(out, a, x.flip(0).contiguous())
    wait()
    return [dx, ext().embed_grad(y, dx, w.shape[0], 1.0, -1, None)]


def table_into_norm_into_8_bits(x, w, gain, y, wait):
    e = fw.embed_tokens(y, w)
    wait()
    out, total = fw.rms_norm(e, gain, residual=x)
    wait()
    q, s, total = fw.rms_norm_int8(out, gain, residual=total)
    wait()
    return [out, total, q, s]


@pytest.mark.parametrize("chain", [norm_into_loss, norm_gradient_into_table, table_into_norm_into_8_bits])
@pytest.mark.parametrize("rows,D,V", [(200, 1000, 700), (250, 1001, 3000), (5000, 264, 500)])
def test_chains(chain, rows, D, V):
    g = R.gen(D)
    w, gain = R.normal((V, D), torch.bfloat16, g, 0.2), R.normal((D,), torch.bfloat16, g)
    xs = [R.normal((rows, D), torch.bfloat16, g) for _ in range(6)]
    ys = [torch.randint(0, V, (rows,), generator=g, device="cuda") for _ in range(6)]
    want = [[t.clone() for t in chain(x, w, gain, y, torch.cuda.synchronize)] for x, y in zip(xs, ys)]
    for _ in range(5):
        for x, y, ref in zip(xs, ys, want):
            got = chain(x, w, gain, y, lambda: None)
            assert all(torch.equal(a, b) for a, b in zip(got, ref))
            del got

"""Waits inside the tensor-core kernels that give up: with the limit at 0 the
matrix issuers do at once and everybody else when nothing comes; the kernels
report it, and nothing of theirs is left behind for the launches after them."""
import contextlib

import pytest
import torch

import lm_ref as R
from fwloss_b200 import capi, int8_linear, lm_head_cross_entropy
from fwloss_b200.lm_head import chunk_summaries, tile_col_start

pytestmark = pytest.mark.gpu

TIMEOUT = 4


@contextlib.contextmanager
def giving_up():
    before = capi.load().fw_tc_wait_limit(0)
    try:
        yield
    finally:
        capi.load().fw_tc_wait_limit(before)


def new_status():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def test_the_limit_is_set_and_returned():
    f = capi.load().fw_tc_wait_limit
    before = f(-1)
    assert before == 2_000_000_000 and f(12345) == before and f(-7) == 12345 and f(before) == 12345 and f(-1) == before


# tokens as columns of 16 and 64; tiles of one CTA; of a pair
@pytest.mark.parametrize("T,N,K", [(1, 5000, 2000), (50, 19000, 700), (300, 1000, 1500), (700, 9000, 600)])
def test_int8_product(T, N, K):
    g = R.gen(T)
    q = torch.randint(-127, 128, (T, (K + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8)[:, :K]
    w = torch.randint(-127, 128, (N, (K + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8)[:, :K]
    qs, ws = torch.rand(T, generator=g, device="cuda"), torch.rand(N, generator=g, device="cuda")
    want = int8_linear(q, qs, w, ws)
    status = new_status()
    with giving_up():
        int8_linear(q, qs, w, ws, status=status)
    assert int(status) == TIMEOUT
    status.zero_()
    for _ in range(3):
        assert torch.equal(int8_linear(q, qs, w, ws, status=status), want)
    assert int(status) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_cross_entropy(dtype, reduction):
    g = R.gen(4)
    h, w = R.normal((600, 520), dtype, g).requires_grad_(True), R.normal((3000, 520), dtype, g, 0.1).requires_grad_(True)
    y = torch.randint(0, 3000, (600,), generator=g, device="cuda")
    status = new_status()
    loss = lm_head_cross_entropy(h, w, y, reduction=reduction, status=status)
    up = torch.ones_like(loss)
    want = torch.autograd.grad(loss, (h, w), up, retain_graph=True)
    assert int(status) == 0
    with giving_up():
        lost = lm_head_cross_entropy(h, w, y, reduction=reduction, status=status)
        assert int(status) & TIMEOUT and lost.isnan().all()
    status.zero_()
    with giving_up():
        torch.autograd.grad(loss, (h, w), up, retain_graph=True)
        assert int(status) == TIMEOUT
    status.zero_()
    again = lm_head_cross_entropy(h, w, y, reduction=reduction, status=status)
    assert torch.equal(again, loss)
    for got, ref in zip(torch.autograd.grad(again, (h, w), up), want):
        assert torch.equal(got, ref)
    assert int(status) == 0


def test_fused_lm_head_scan():
    g = R.gen(5)
    h, w = R.normal((300, 512), torch.bfloat16, g), R.normal((2000, 512), torch.bfloat16, g, 0.1)
    y = torch.randint(0, 2000, (300,), generator=g, device="cuda")
    starts = tile_col_start(2000, 4)
    want = chunk_summaries(h, w, y, starts, 32, True)
    assert int(want[3]) == 0
    with giving_up():
        assert int(chunk_summaries(h, w, y, starts, 32, True)[3]) == TIMEOUT
    got = chunk_summaries(h, w, y, starts, 32, True)
    used = torch.arange(32, device="cuda") < want[0][..., 1:2].clamp(max=32)  # the entries that a record's count names
    assert torch.equal(got[0][..., :4], want[0][..., :4]) and torch.equal(got[2], want[2]) and int(got[3]) == 0
    assert torch.equal(got[0][..., 4:][used], want[0][..., 4:][used]) and torch.equal(got[1][used], want[1][used])

"""lm_head_cross_entropy against its 64-bit definition: loss and gradients,
ragged sizes, ignored rows and what they hold, labels out of range, pieces."""
import pytest
import torch

import lm_ref as R
from fwloss_b200 import capi, lm_head_cross_entropy

pytestmark = pytest.mark.gpu

SHAPES = [(1, 8, 1), (1, 64, 300), (3, 1, 2), (127, 72, 255), (128, 64, 256), (129, 200, 257), (300, 513, 1001),
          (257, 1000, 5003), (700, 128, 9000), (64, 2048, 2000)]


def data(B, D, V, dtype, seed, ignored=0.0):
    g = R.gen(seed)
    h = R.normal((B, D), dtype, g)
    w = R.normal((V, D), dtype, g, 2.0 / D ** 0.5)
    y = torch.randint(0, V, (B,), generator=g, device="cuda")
    if ignored:
        y[torch.rand(B, generator=g, device="cuda") < ignored] = -100
    return h, w, y


def check(h, w, y, reduction="mean", go=None, ignore=-100):
    a, b = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = lm_head_cross_entropy(a, b, y, reduction=reduction, ignore_index=ignore)
    assert loss.dtype == torch.float32
    ref = R.xent(h, w, y, reduction, ignore, go)
    R.within(loss, ref["loss"], ref["e_loss"].nan_to_num(), "loss")
    dh, dw = torch.autograd.grad(loss, (a, b), go if go is not None else torch.ones_like(loss))
    R.within(dh, ref["dh"], ref["e_dh"].nan_to_num(), "dhidden")
    R.within(dw, ref["dw"], ref["e_dw"].nan_to_num(), "dweight")
    with torch.no_grad():
        assert torch.equal(loss.nan_to_num(), lm_head_cross_entropy(h, w, y, reduction, ignore).nan_to_num())
    return loss, dh, dw


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,D,V", SHAPES)
def test_loss_and_gradients(B, D, V, dtype):
    h, w, y = data(B, D, V, dtype, B + D + V)
    check(h, w, y, ("mean", "sum")[B % 2])


@pytest.mark.parametrize("B,D,V", [(20000, 1024, 2048), (9000, 2048, 2048), (1300, 1024, 4096), (600, 512, 9000),
                                   (64, 512, 20000)])
def test_gradient_of_hidden_whole_and_in_splits(B, D, V):
    """From rows whose products over V are far shorter than what else a
    launch holds, to rows whose products are nearly all of it."""
    h, w, y = data(B, D, V, torch.bfloat16, B + V, ignored=0.1)
    check(h, w, y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_reductions_ignored_rows_and_upstream(dtype, reduction):
    h, w, y = data(333, 136, 1500, dtype, 5, ignored=0.4)
    g = R.gen(1)
    go = torch.rand(333, generator=g, device="cuda") * 1e-3 if reduction == "none" else torch.tensor(0.37, device="cuda")
    if reduction == "none":
        go[5] = 0.0
        go[6] = 2.0
    check(h, w, y, reduction, go)


def test_what_ignored_rows_hold_does_not_matter():
    h, w, y = data(200, 96, 700, torch.bfloat16, 7, ignored=0.3)
    want = check(h, w, y)
    dirty = h.clone()
    dirty[y == -100] = float("nan")
    dirty[(y == -100).nonzero()[0]] = float("inf")
    a, b = dirty.requires_grad_(True), w.clone().requires_grad_(True)
    loss = lm_head_cross_entropy(a, b, y)
    dh, dw = torch.autograd.grad(loss, (a, b))
    for got, ref in zip((loss, dh, dw), want):
        assert torch.equal(got, ref)
    assert not dh[y == -100].any()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_every_row_ignored(reduction):
    h, w, y = data(150, 64, 300, torch.float16, 8)
    y.fill_(-100)
    a, b = h.requires_grad_(True), w.requires_grad_(True)
    loss = lm_head_cross_entropy(a, b, y, reduction=reduction)
    assert loss.isnan() if reduction == "mean" else not loss.any()
    dh, dw = torch.autograd.grad(loss, (a, b), torch.ones_like(loss))
    assert not dh.any() and not dw.any()


def test_other_ignore_index_and_labels_out_of_range():
    h, w, y = data(140, 64, 500, torch.bfloat16, 9)
    check(h, w, y, "mean", ignore=int(y[3]))
    y[10], y[20] = 500, -7
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    loss = lm_head_cross_entropy(h, w, y, reduction="none", status=status)
    assert int(status) == 1 and loss.isnan().nonzero()[:, 0].tolist() == [10, 20]
    assert lm_head_cross_entropy(h, w, y).isnan()
    a = h.clone().requires_grad_(True)
    (dh,) = torch.autograd.grad(lm_head_cross_entropy(a, w, y, reduction="none").nan_to_num().sum(), a)
    ok = torch.ones(140, dtype=torch.bool, device="cuda")
    ok[10] = ok[20] = False
    ref = R.xent(h, w, y, "none")
    R.within(dh[ok], ref["dh"][ok], ref["e_dh"][ok])


def test_confident_and_large_logits():
    """Rows whose softmax is one class, logits in the hundreds, equal logits."""
    h, w, y = data(160, 128, 900, torch.bfloat16, 10)
    h[:40] *= 30
    h[40:60] = 0
    y[:10] = (h[:10].float() @ w.float().t()).argmax(1)
    check(h, w, y, "sum")


def test_rows_that_are_not_finite():
    h, w, y = data(130, 64, 700, torch.bfloat16, 11)
    h[4, 3], h[9, 0] = float("nan"), float("inf")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    loss = lm_head_cross_entropy(h, w, y, reduction="none", status=status)
    assert loss.isnan().nonzero()[:, 0].tolist() == [4, 9] and int(status) == 2


@pytest.mark.parametrize("start", [0, 1, 8])
def test_strided_and_misaligned_operands(start):
    g = R.gen(start)
    h = R.normal((100, 200), torch.float16, g)[:, start:start + 96]
    w = R.normal((400, 300), torch.float16, g, 0.2)[:, start:start + 96]
    y = torch.randint(0, 400, (200,), generator=g, device="cuda")[::2]
    check(h, w, y)
    check(h[::2], w[::3], y[::2] % 134)
    check(h.t().contiguous().t(), w.t().contiguous().t(), y)


def test_only_one_gradient_and_twice():
    h, w, y = data(90, 64, 333, torch.bfloat16, 12)
    ref = check(h, w, y)
    a = h.clone().requires_grad_(True)
    loss = lm_head_cross_entropy(a, w, y)
    for _ in range(2):
        (dh,) = torch.autograd.grad(loss, a, retain_graph=True)
        assert torch.equal(dh, ref[1])
    b = w.clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(lm_head_cross_entropy(h, b, y), b)
    assert torch.equal(dw, ref[2])


def test_no_rows():
    h = torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    w = torch.zeros(50, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert lm_head_cross_entropy(h, w, y).isnan() and float(lm_head_cross_entropy(h, w, y, "sum").detach()) == 0.0
    loss = lm_head_cross_entropy(h, w, y, "none")
    dh, dw = torch.autograd.grad(loss, (h, w), torch.zeros_like(loss))
    assert loss.shape == (0,) and dh.shape == (0, 64) and not dw.any()


def test_several_pieces_of_the_vocabulary():
    """Rows enough that the logit gradient does not fit one workspace piece."""
    B, D, V = 33000, 64, 10007
    h, w, y = data(B, D, V, torch.bfloat16, 13, ignored=0.02)
    assert capi.load().fw_xent_workspace(B, D, V, 1) < 2 * B * V
    a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = lm_head_cross_entropy(a, b, y)
    dh, dw = torch.autograd.grad(loss, (a, b))
    ref = R.xent(h, w, y, "mean")
    R.within(loss, ref["loss"], ref["e_loss"])
    R.within(dh, ref["dh"], ref["e_dh"])
    R.within(dw, ref["dw"], ref["e_dw"])


def test_results_do_not_vary():
    h, w, y = data(500, 256, 4000, torch.bfloat16, 14, ignored=0.1)
    first = check(h, w, y)
    for got, ref in zip(check(h, w, y), first):
        assert torch.equal(got, ref)


def test_gradient_against_differences():
    h, w, y = data(60, 48, 200, torch.float16, 15, ignored=0.1)
    _, dh, dw = check(h, w, y, "sum")
    ref = R.xent(h, w, y, "sum")
    g = torch.Generator(device="cuda").manual_seed(2)
    u = torch.randn(h.shape, generator=g, device="cuda", dtype=torch.float64)
    v = torch.randn(w.shape, generator=g, device="cuda", dtype=torch.float64) * 0.1

    def f(t):
        z = (h.double() + t * u) @ (w.double() + t * v).t()
        return torch.nn.functional.cross_entropy(z, y, reduction="sum")

    slope = (f(1e-5) - f(-1e-5)) / 2e-5
    lim = (ref["e_dh"] * u.abs()).sum() + (ref["e_dw"] * v.abs()).sum() + 1e-5
    assert abs((dh.double() * u).sum() + (dw.double() * v).sum() - slope) <= lim


def test_other_stream():
    h, w, y = data(260, 128, 2000, torch.bfloat16, 16)
    want = check(h, w, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = lm_head_cross_entropy(a, b, y)
        got = [loss, *torch.autograd.grad(loss, (a, b))]
    torch.cuda.current_stream().wait_stream(side)
    for x, ref in zip(got, want):
        assert torch.equal(x, ref)


def test_refusals():
    h, w = torch.zeros(4, 8, dtype=torch.bfloat16, device="cuda"), torch.zeros(6, 8, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad in ((h.cpu(), w, y), (h.float(), w.float(), y), (h, w.half(), y), (h[0], w, y), (h, w[:0], y), (h, w, y.int())):
        with pytest.raises(TypeError):
            lm_head_cross_entropy(*bad)
    for bad in ((h, w[:, :7], y), (h, w, y[:3]), (h, w, y.cpu())):
        with pytest.raises(ValueError):
            lm_head_cross_entropy(*bad)
    with pytest.raises(ValueError):
        lm_head_cross_entropy(h, w, y, reduction="avg")

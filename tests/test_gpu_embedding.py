"""embed_tokens against its 64-bit definition: lookups, the sorted-token
gradient, odd sizes and strides, skewed and empty inputs, streams."""
import pytest
import torch

import lm_ref as R
from fwloss_b200 import embed_tokens
from fwloss_b200._native import ext

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1, 1), (5, 7, 3), (33, 1000, 127), (300, 11, 64), (2048, 4099, 100), (2049, 70001, 17), (5000, 523, 1000),
          (130, 300, 4104), (70000, 50, 9)]


def data(T, V, D, dtype, seed, skew=False):
    g = R.gen(seed)
    if skew:
        ids = ((V + 1.0) ** torch.rand(T, generator=g, device="cuda", dtype=torch.float64) - 1).long().clamp_(0, V - 1)
    else:
        ids = torch.randint(0, V, (T,), generator=g, device="cuda")
    return ids, R.normal((V, D), dtype, g), R.normal((T, D), dtype, g)


def check(ids, weight, grad, scale=1.0, padding=None):
    w = weight.detach().requires_grad_(True)
    out = embed_tokens(ids, w, scale=scale, padding_idx=padding)
    want = R.embed(ids, weight, scale)
    R.within(out, want, want.nan_to_num().abs() * R.E32 + R.rounded(want.nan_to_num(), weight.dtype), "rows")
    (dw,) = torch.autograd.grad(out, w, grad)
    assert dw.dtype == weight.dtype
    ref, total, most = R.embed_grad(ids, grad, weight.shape[0], scale, padding)
    R.within(dw, ref, total * (most + 2) * R.E32 + R.rounded(ref, weight.dtype), "gradient")
    return dw


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("T,V,D", SHAPES)
def test_rows_and_gradient(T, V, D, dtype):
    ids, w, g = data(T, V, D, dtype, T + V + D)
    check(ids, w, g)


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("T", [1, 31, 32, 33, 256, 257])
def test_few_tokens_of_a_large_table(T, dtype):
    ids, w, g = data(T, 117001, 72, dtype, T, skew=T % 2 == 0)
    check(ids, w, g)


@pytest.mark.parametrize("V,D", [(8192, 1024), (8192, 1025), (131072, 64), (131073, 64)])
def test_tables_around_the_size_that_is_sorted_for(V, D):
    ids, w, g = data(200, V, D, torch.float16, V + D)
    check(ids, w, g, scale=3.0, padding=int(ids[7]))


@pytest.mark.parametrize("T", [600, 1100, 9000, 33000])
def test_runs_of_many_parts(T):
    """A third of the tokens one row, a third another: parts joined by a warp, and by a CTA."""
    ids, w, g = data(T, 301, 520, torch.bfloat16, T)
    ids[torch.randperm(T, generator=R.gen(1), device="cuda")[: T // 3]] = 300
    ids[torch.randperm(T, generator=R.gen(2), device="cuda")[: T // 3]] = 17
    check(ids, w, g)


@pytest.mark.parametrize("T", [31, 32, 33, 64, 65, 3000, 40000])
def test_skewed_tokens(T):
    """Runs that end at, before and after a chunk boundary of the sorted order."""
    ids, w, g = data(T, 5003, 72, torch.bfloat16, T, skew=True)
    check(ids, w, g, scale=45.25)


@pytest.mark.parametrize("T", [1, 32, 33, 2048, 9001])
def test_every_position_the_same_token(T):
    ids, w, g = data(T, 77, 40, torch.float32, 3)
    check(torch.full_like(ids, 76), w, g)
    check(torch.zeros_like(ids), w, g)


def test_no_tokens_and_shapes():
    w = R.normal((10, 6), torch.float16, R.gen(1)).requires_grad_(True)
    empty = torch.zeros((0,), dtype=torch.int64, device="cuda")
    out = embed_tokens(empty, w)
    assert out.shape == (0, 6)
    (dw,) = torch.autograd.grad(out, w, torch.empty_like(out))
    assert torch.equal(dw, torch.zeros_like(w))
    ids = torch.randint(0, 10, (2, 3, 4), device="cuda")
    out = embed_tokens(ids, w)
    assert torch.equal(out, w[ids])
    (dw,) = torch.autograd.grad(out, w, torch.ones_like(out))
    assert torch.equal(dw[:, 0].long(), torch.bincount(ids.reshape(-1), minlength=10))


def test_padding_row_and_tokens_outside_the_table():
    ids, w, g = data(500, 20, 33, torch.float32, 9)
    g[ids == 4] = float("nan")  # what padding positions hold must not matter
    dw = check(ids, w, g, padding=4)
    assert torch.equal(dw[4], torch.zeros_like(dw[4]))
    g = torch.nan_to_num(g)
    ids[7], ids[300] = -3, 20
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    wr = w.clone().requires_grad_(True)
    out = embed_tokens(ids, wr, status=status)
    assert int(status) == 1
    assert out[7].isnan().all() and out[300].isnan().all() and int(out.isnan().any(1).sum()) == 2
    check(ids, w, g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("start", [0, 1, 3])
def test_strided_and_misaligned_operands(dtype, start):
    g = R.gen(4)
    store = R.normal((50, 61), dtype, g)
    w = store[:, start:start + 37]
    up = R.normal((90, 80), dtype, g)[:, start:start + 37]
    ids = torch.randint(0, 50, (90,), generator=g, device="cuda")
    check(ids, w, up)
    check(ids, store.t()[:37].t()[:, :37], up)
    check(ids[::2], w, up[::2])


def test_gradient_does_not_vary():
    ids, w, g = data(20000, 900, 130, torch.float32, 8, skew=True)
    first = ext().embed_grad(ids, g, 900, 1.5, -1, None)
    for _ in range(3):
        assert torch.equal(first, ext().embed_grad(ids, g, 900, 1.5, -1, None))


def test_gradient_against_differences():
    """The operator is linear: <gradient, d> is the change of <out, g> along d."""
    ids, w, g = data(700, 90, 31, torch.float32, 12)
    dw = check(ids, w, g, scale=3.0).double()
    d = torch.randn_like(w).double()
    f = lambda x: (R.embed(ids, x, 3.0) * g.double()).sum()  # noqa: E731
    slope = (f(w.double() + d) - f(w.double() - d)) / 2
    _, total, most = R.embed_grad(ids, g, 90, 3.0)
    assert abs((dw * d).sum() - slope) <= (total * (most + 3) * R.E32 * d.abs()).sum() + 1e-9


def test_other_stream():
    ids, w, g = data(3000, 200, 64, torch.bfloat16, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dw = ext().embed_grad(ids, g, 200, 1.0, -1, None)
    torch.cuda.current_stream().wait_stream(side)
    ref, total, most = R.embed_grad(ids, g, 200, 1.0)
    R.within(dw, ref, total * (most + 2) * R.E32 + R.rounded(ref, torch.bfloat16))


def test_refusals():
    w = torch.zeros(4, 4, device="cuda")
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (w.cpu(), w.double(), w[0], torch.zeros(0, 4, device="cuda")):
        with pytest.raises(TypeError):
            embed_tokens(ids, bad)
    with pytest.raises(TypeError):
        embed_tokens(ids.int(), w)
    with pytest.raises(ValueError):
        embed_tokens(ids.cpu(), w)
    for pad in (-1, 4):
        with pytest.raises(ValueError):
            embed_tokens(ids, w, padding_idx=pad)

"""int8_linear against the 64-bit product: the integer sum is exact, so only
three fp32 roundings and the output's stand between the two."""
import pytest
import torch

import lm_ref as R
from fwloss_b200 import int8_linear, quantize_rows_int8, rms_norm_int8

pytestmark = pytest.mark.gpu


def rows16(rows, cols, g, low=-128):
    store = torch.randint(low, 128, (rows, (cols + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8)
    return store[:, :cols]


def check(q, qs, w, ws, dtype):
    out = int8_linear(q, qs, w, ws, out_dtype=dtype)
    assert out.dtype == dtype
    want = (q.double() @ w.double().t()) * qs.double()[..., None] * ws.double()
    over = want.to(dtype).isinf()  # past the type's range: its infinity
    assert torch.equal(out[over].double(), want[over].to(dtype).double())
    R.within(out[~over], want[~over], (want.abs() * 3 * R.E32 + R.rounded(want, dtype))[~over])
    return out


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 32, 33, 64, 65, 100, 128, 129, 257, 700])
@pytest.mark.parametrize("N,K", [(1, 1), (127, 16), (128, 128), (300, 1000), (1025, 517), (5000, 2048)])
def test_product(T, N, K):
    g = R.gen(T * 31 + N + K)
    dtype = R.FLOATS[T % 3]
    check(rows16(T, K, g), torch.rand(T, generator=g, device="cuda"), rows16(N, K, g),
          torch.rand(N, generator=g, device="cuda"), dtype)


@pytest.mark.parametrize("T", [1, 16, 17, 32, 33, 64, 65, 127, 128, 129])
@pytest.mark.parametrize("N", [18943, 19000, 60001])
def test_many_columns(T, N):
    """Whole rounds of weight tiles, and what is left behind them."""
    g = R.gen(T + N)
    check(rows16(T, 300, g), torch.rand(T, generator=g, device="cuda"), rows16(N, 300, g),
          torch.rand(N, generator=g, device="cuda"), R.FLOATS[N % 3])


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("T", [3, 300])
def test_output_types_and_extreme_values(T, dtype):
    """-128 everywhere is the largest sum; K up to where it still fits 32 bits."""
    K = 131071 if T == 3 else 3000
    q = torch.full((T, (K + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")[:, :K]
    w = torch.full((130, (K + 15) // 16 * 16), -128, dtype=torch.int8, device="cuda")[:, :K]
    w[1] = 127
    ones = torch.full((T,), 2.0 ** -12, device="cuda"), torch.full((130,), 2.0 ** -8, device="cuda")
    check(q, ones[0], w, ones[1], dtype)


def test_rows_off_the_boundary_and_padding_bytes():
    """Strides that are not multiples of 16, offset views, and whatever lies past K."""
    g = R.gen(5)
    wide_q, wide_w = rows16(40, 333, g), rows16(200, 333, g)
    qs, ws = torch.rand(40, generator=g, device="cuda"), torch.rand(200, generator=g, device="cuda")
    for a, b in ((0, 333), (1, 300), (16, 301), (32, 97)):
        check(wide_q[:, a:b], qs, wide_w[:, a:b], ws, torch.float32)
    check(wide_q.contiguous(), qs, wide_w.contiguous(), ws, torch.float32)
    check(wide_q.t().contiguous().t(), qs, wide_w, ws, torch.float32)
    check(wide_q[::3], qs[::3], wide_w[::2], ws[::2], torch.float32)


def test_ranks_and_no_tokens():
    g = R.gen(6)
    w, ws = rows16(50, 64, g), torch.rand(50, generator=g, device="cuda")
    q, qs = rows16(6, 64, g), torch.rand(6, generator=g, device="cuda")
    flat = check(q, qs, w, ws, torch.float16)
    assert torch.equal(int8_linear(q.view(2, 3, 64), qs.view(2, 3), w, ws, torch.float16).view(6, 50), flat)
    assert torch.equal(int8_linear(q[0], qs[0], w, ws, torch.float16), flat[0])
    assert int8_linear(q[:0], qs[:0], w, ws).shape == (0, 50)


def test_scales_that_are_not_finite_stay_in_their_row_and_column():
    g = R.gen(7)
    q, w = rows16(20, 100, g), rows16(300, 100, g)
    qs, ws = torch.rand(20, generator=g, device="cuda"), torch.rand(300, generator=g, device="cuda")
    clean = int8_linear(q, qs, w, ws, torch.float32)
    qs[3], ws[200] = float("nan"), float("nan")
    out = int8_linear(q, qs, w, ws, torch.float32)
    hit = out.isnan()
    assert hit[3].all() and hit[:, 200].all() and int(hit.sum()) == 20 + 300 - 1
    assert torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("T,D,V", [(1, 512, 4000), (40, 1000, 3001), (500, 264, 2000)])
def test_norm_and_output_layer_together(T, D, V):
    """The 8-bit path against the float product: the two quantisations' own steps."""
    g = R.gen(T + D)
    x, res, gain = R.normal((T, D), torch.bfloat16, g), R.normal((T, D), torch.bfloat16, g), R.normal((D,), torch.bfloat16, g)
    weight = R.normal((V, D), torch.bfloat16, g)
    wq, ws = quantize_rows_int8(weight)
    q, qs, _ = rms_norm_int8(x, gain, residual=res)
    out = int8_linear(q, qs, wq, ws, torch.float32)
    _, _, y = R.norm(x, gain, 1e-6, res)
    step_y, step_w = qs.double()[:, None] * 0.51, ws.double()[:, None] * 0.51
    bound = step_y * weight.double().abs().sum(1) + y.abs().sum(1, keepdim=True) * step_w.t() + D * step_y * step_w.t()
    want = y @ weight.double().t()
    R.within(out, want, bound + want.abs() * 1e-5)


def test_other_stream():
    g = R.gen(8)
    q, w = rows16(300, 1000, g), rows16(3000, 1000, g)
    qs, ws = torch.rand(300, generator=g, device="cuda"), torch.rand(3000, generator=g, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = int8_linear(q, qs, w, ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, int8_linear(q, qs, w, ws))


def test_refusals():
    q, w = torch.zeros(4, 32, dtype=torch.int8, device="cuda"), torch.zeros(8, 32, dtype=torch.int8, device="cuda")
    qs, ws = torch.ones(4, device="cuda"), torch.ones(8, device="cuda")
    for bad in ((q.cpu(), qs, w, ws), (q.int(), qs, w, ws), (q, qs.half(), w, ws), (q, qs, w.float(), ws)):
        with pytest.raises(TypeError):
            int8_linear(*bad)
    with pytest.raises(TypeError):
        int8_linear(q, qs, w, ws, torch.float64)
    for bad in ((q[:, :31], qs, w, ws), (q, qs[:3], w, ws), (q, qs, w, ws[:7]), (q, qs, w[0], ws)):
        with pytest.raises(ValueError):
            int8_linear(*bad)
    long = torch.zeros(1, 131072, dtype=torch.int8, device="cuda")
    with pytest.raises(ValueError):
        int8_linear(long, qs[:1], long, ws[:1])

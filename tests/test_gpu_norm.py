"""rms_norm, its gradient and its 8-bit form against their 64-bit definitions."""
import pytest
import torch

import lm_ref as R
from fwloss_b200 import quantize_rows_int8, rms_norm, rms_norm_int8

pytestmark = pytest.mark.gpu

# a warp per row, CTAs of each size, the longest held in registers and one beyond, odd sizes
DIMS = [1, 3, 16, 127, 256, 511, 1000, 1025, 2049, 4096, 5001, 8190, 16400, 33001]


def tol_y(y, D, dtype):
    return y.abs() * (D + 16) * R.E32 + R.rounded(y, dtype)


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("residual", [False, True])
def test_norm_and_gradient(D, dtype, residual):
    g = R.gen(D)
    rows = 37 if D > 300 else 1501
    x, w = R.normal((rows, D), dtype, g), (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dtype)
    r = R.normal((rows, D), dtype, g, 3.0) if residual else None
    dy, ds = R.normal((rows, D), dtype, g), R.normal((rows, D), dtype, g)
    check(x, w, r, dy, ds, 1e-5)


def check(x, w, r, dy, ds, eps):
    D, dtype = x.shape[-1], x.dtype
    leaves = [t.detach().requires_grad_(True) for t in ((x, w) if r is None else (x, w, r))]
    s, rstd, y = R.norm(x, w, eps, r)
    if r is None:
        got = rms_norm(leaves[0], leaves[1], eps=eps)
        grads = torch.autograd.grad(got, leaves, dy)
        ds = None
    else:
        got, total = rms_norm(leaves[0], leaves[1], eps=eps, residual=leaves[2])
        assert torch.equal(total.double(), s)
        grads = torch.autograd.grad((got, total), leaves, (dy, ds))
        assert torch.equal(grads[0], grads[2])
    R.within(got, y, tol_y(y, D, dtype), "y")
    want, dw, e_ds, e_dw = R.norm_grad(dy, s, rstd, w, ds)
    R.within(grads[0], want, e_ds + R.rounded(want, dtype), "dx")
    R.within(grads[1], dw, e_dw + R.rounded(dw, w.dtype), "dweight")


@pytest.mark.parametrize("rows", [1, 2, 7, 9, 1185, 20011])
def test_row_counts(rows):
    g = R.gen(rows)
    x, r, dy, ds = (R.normal((rows, 201), torch.bfloat16, g) for _ in range(4))
    check(x, R.normal((201,), torch.bfloat16, g), r, dy, ds, 1e-6)


def test_float32_gains_with_a_16_bit_stream():
    g = R.gen(2)
    x, r, dy, ds = (R.normal((300, 1000), torch.float16, g) for _ in range(4))
    check(x, torch.rand(1000, generator=g, device="cuda") + 0.5, r, dy, ds, 1e-6)


@pytest.mark.parametrize("start", [0, 1, 2, 5])
def test_strided_and_misaligned_rows(start):
    g = R.gen(start)
    wide = [R.normal((65, 700), torch.bfloat16, g) for _ in range(4)]
    x, r, dy, ds = (t[:, start:start + 555] for t in wide)
    w = R.normal((700,), torch.bfloat16, g)[start:start + 555]
    check(x, w, r, dy, ds, 1e-6)
    check(x, w, wide[1][:, 3:558], dy[:, :], ds, 1e-6)  # residual at another distance from a boundary
    check(x[::2], w, r[::2], dy[::2], ds[::2], 1e-6)


def test_shapes_without_rows_and_of_any_rank():
    w = torch.ones(12, device="cuda", requires_grad=True)
    x = torch.zeros(0, 12, device="cuda", requires_grad=True)
    y = rms_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert dx.shape == (0, 12) and torch.equal(dw, torch.zeros_like(w))
    x = torch.randn(2, 3, 5, 12, device="cuda")
    y, s = rms_norm(x, w, residual=x)
    assert y.shape == s.shape == x.shape and torch.equal(s, x + x)
    q, scale, s = rms_norm_int8(x, w, residual=x)
    assert q.shape == x.shape and scale.shape == x.shape[:-1] and s.shape == x.shape
    one = rms_norm(x[0, 0, 0], w)
    assert torch.equal(one, rms_norm(x[0, 0, 0][None], w)[0])
    q1, s1 = rms_norm_int8(x[0, 0, 0], w)
    q2, s2 = rms_norm_int8(x[0, 0, :1], w)
    assert torch.equal(q1, q2[0]) and s1.shape == () and float(s1) == float(s2[0])


def test_only_one_output_used():
    g = R.gen(3)
    x, r, dy = (R.normal((20, 64), torch.float32, g).requires_grad_(True) for _ in range(3))
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, s = rms_norm(x, w, residual=r)
    gx, gw = torch.autograd.grad(s, (x, w), dy.detach(), allow_unused=True, retain_graph=True)
    assert torch.equal(gx, dy) and gw is None
    (gx,) = torch.autograd.grad(y, x, dy.detach())
    s64, rstd, _ = R.norm(x.detach(), w.detach(), 1e-6, r.detach())
    want, _, e, _ = R.norm_grad(dy.detach(), s64, rstd, w.detach())
    R.within(gx, want, e + R.rounded(want, torch.float32))


def test_not_finite_and_zero_rows_stay_in_their_row():
    g = R.gen(6)
    x = R.normal((9, 300), torch.float32, g)
    clean = x.clone()
    x[2, 5], x[4, 7], x[6] = float("nan"), float("inf"), 0.0
    w = R.normal((300,), torch.float32, g)
    y, ref = rms_norm(x, w), rms_norm(clean, w)
    keep = [0, 1, 3, 5, 7, 8]
    assert torch.equal(y[keep], ref[keep]) and y[2].isnan().all() and y[4, 7].isnan() and not y[6].any()
    q, scale = rms_norm_int8(x, w)
    assert scale[2].isnan() and not q[2].any() and scale[4].isnan() and scale[6] == 0 and not q[6].any()
    assert torch.equal(q[keep], rms_norm_int8(clean, w)[0][keep])


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("D", DIMS)
def test_int8_rows(D, dtype):
    g = R.gen(D + 1)
    rows = 21 if D > 300 else 403
    x, r = R.normal((rows, D), dtype, g), R.normal((rows, D), dtype, g)
    w = R.normal((D,), dtype, g)
    q, scale, total = rms_norm_int8(x, w, eps=1e-5, residual=r)
    s, _, y = R.norm(x, w, 1e-5, r)
    assert torch.equal(total.double(), s)
    check_int8(q, scale, y, D)
    q, scale = quantize_rows_int8(x)
    check_int8(q, scale, x.double(), 0)


def check_int8(q, scale, y, D):
    want = y.abs().amax(1) / 127
    e = (D + 20) * R.E32
    R.within(scale, want, want * e + 1e-45, "scale")
    assert q.dtype == torch.int8 and q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0
    live = want > 0
    steps = torch.where(live[:, None], y / want[:, None], torch.zeros_like(y))
    R.within(q, steps, 0.5 + 127 * 2 * e, "q")
    pad = torch.as_strided(q, (q.shape[0], q.stride(0)), (q.stride(0), 1))[:, q.shape[1]:] if q.shape[0] > 1 else q[:, :0]
    assert not pad.any()


@pytest.mark.parametrize("D", [40, 4100, 20000])
def test_int8_rows_of_the_smallest_values(D):
    """1 / scale is past fp32's range from scales of 2^-128 down.  Half a step,
    the fp32 roundings of 127 steps (three of 2^-24), and of the scale itself,
    which under 2^-126 is a multiple of 2^-149."""
    g = R.gen(D)
    x = R.normal((5, D), torch.float32, g)
    x /= x.abs().amax(-1, keepdim=True)
    top = torch.tensor([1e-30, 1e-36, 3e-38, 1e-39, 1e-40], device="cuda")
    x *= top[:, None]
    q, scale = quantize_rows_int8(x)
    step = scale.double()[:, None]
    error = (q.double() * step - x.double()).abs()
    assert bool((error <= step * (0.5 + 127 * 4 * 2.0 ** -24) + 127 * 2.0 ** -150).all())
    assert bool((q.abs().amax(-1) == 127).all())


def test_gradient_against_differences():
    g = R.gen(11)
    x, r, dy, ds = (R.normal((13, 96), torch.float32, g) for _ in range(4))
    w = R.normal((96,), torch.float32, g)
    leaves = [t.clone().requires_grad_(True) for t in (x, w)]
    y, s = rms_norm(leaves[0], leaves[1], eps=1e-3, residual=r)
    gx, gw = torch.autograd.grad((y, s), leaves, (dy, ds))

    def f(x64, w64):  # without the rounding of the sum, which has no slope
        t = x64 + r.double()
        n = t * (t.square().mean(-1, keepdim=True) + 1e-3).rsqrt() * w64
        return (n * dy.double() + t * ds.double()).sum()

    dx, dw = torch.randn_like(x).double(), torch.randn_like(w).double()
    h = 1e-5
    slope = (f(x.double() + h * dx, w.double() + h * dw) - f(x.double() - h * dx, w.double() - h * dw)) / (2 * h)
    s64, rstd, _ = R.norm(x, w, 1e-3, r)
    ref, refw, e, ew = R.norm_grad(dy, s64, rstd, w, ds)
    lim = ((e + R.rounded(ref, torch.float32)) * dx.abs()).sum() + ((ew + R.rounded(refw, torch.float32)) * dw.abs()).sum()
    # the stored sum is off by E32 of itself (slope of the slope at most 3 rstd |dy w|), and h^2 / 6 of a third derivative
    lim = lim + (3 * R.E32 * s64.abs() * rstd ** 2 * (dy * w).double().abs().amax(1, keepdim=True) * dx.abs()).sum() + 1e-6
    assert abs((gx.double() * dx).sum() + (gw.double() * dw).sum() - slope) <= lim


def test_other_stream():
    g = R.gen(8)
    x, w = R.normal((4000, 640), torch.bfloat16, g), R.normal((640,), torch.bfloat16, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = rms_norm(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, rms_norm(x, w))


def test_refusals():
    x, w = torch.zeros(4, 8, device="cuda"), torch.ones(8, device="cuda")
    for call in (rms_norm, rms_norm_int8):
        with pytest.raises(TypeError):
            call(x.cpu(), w.cpu())
        with pytest.raises(TypeError):
            call(x.double(), w.double())
        with pytest.raises(TypeError):
            call(x, w.half())
        with pytest.raises(TypeError):
            call(x, w, residual=x.half())
        with pytest.raises(ValueError):
            call(x, w[:7])
        with pytest.raises(ValueError):
            call(x, w, residual=x[:3])
        with pytest.raises(ValueError):
            call(x, w, eps=-1.0)
        with pytest.raises(ValueError):
            call(x, w.cpu())
    with pytest.raises(TypeError):
        quantize_rows_int8(x[0])

"""Rows that start anywhere: whole 16-byte slots of elements at every distance
from a 16-byte boundary, through Python and through the C entry points, with
what lies around the rows checked.  Bounds as in the operators' own tests."""
import pytest
import torch

import lm_ref as R
from fwloss_b200 import capi, quantize_rows_int8, rms_norm_int8

pytestmark = pytest.mark.gpu

# widths whose slots fill a warp or a CTA exactly (16-bit: 32, 128, 256, 512, 1024, 2048 slots; fp32: twice as many)
WIDTHS = [128, 256, 512, 1024, 2048, 4096, 8192, 16384]
NAN = float("nan")


def starts(dtype):
    return range(16 // dtype.itemsize)


def view(rows, D, ld, start, dtype, g, scale=1.0, fill=NAN):
    """(rows [rows, D] that start `start` elements past a boundary in a store of `fill`, the store)"""
    store = torch.full((rows * ld + 32,), fill, dtype=dtype, device="cuda")
    v = store[start:].as_strided((rows, D), (ld, 1))
    v.copy_(R.normal((rows, D), dtype, g, scale))
    return v, store


def strides(D, dtype):
    """Row strides that keep the distance, and one that changes it from row to row."""
    return [D + 16, D + 17] if dtype != torch.float32 else [D + 16, D + 19]


def check_q(q, scale, y, D):
    want = y.abs().amax(1) / 127
    e = (D + 20) * R.E32
    R.within(scale, want, want * e + 1e-45, "scale")
    R.within(q, y / want[:, None], 0.5 + 127 * 2 * e, "q")


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("D", WIDTHS)
def test_int8_rows_at_every_distance(D, dtype):
    g = R.gen(D)
    w = R.normal((D,), dtype, g)
    for start in starts(dtype):
        for ld in strides(D, dtype):
            x, _ = view(11, D, ld, start, dtype, g)
            x[:, -1] = 5.0  # the row's largest value, in its last place
            q, scale = quantize_rows_int8(x)
            check_q(q, scale, x.double(), 0)
            q, scale = rms_norm_int8(x, w, eps=1e-5)
            check_q(q, scale, R.norm(x, w, 1e-5)[2], D)


def test_a_column_slice_and_a_weight_inside_a_flat_buffer():
    g = R.gen(1)
    x = R.normal((300, 4097), torch.bfloat16, g)
    for v in (x[:, 1:], x[:, :4096]):
        q, scale = quantize_rows_int8(v)
        check_q(q, scale, v.double(), 0)
    flat = R.normal((3 + 50 * 1024,), torch.float32, g)
    v = flat[3:].view(50, 1024)
    q, scale = quantize_rows_int8(v)
    check_q(q, scale, v.double(), 0)


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("D", WIDTHS)
def test_norm_entry_points_with_all_operands_shifted_alike(D, dtype):
    lib, code, eps = capi.load(), capi.DTYPE_CODES[dtype], 1e-5
    rows, g = 11, R.gen(D + 1)
    w = R.normal((D,), dtype, g)
    rstd = torch.empty(rows, device="cuda")
    nparts = lib.fw_rms_norm_grad_parts(rows)
    parts, dw = torch.empty(nparts, D, device="cuda"), torch.empty(D, dtype=dtype, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    for start in starts(dtype):
        for ld in strides(D, dtype):
            x, r, dy, ds = (view(rows, D, ld, start, dtype, g)[0] for _ in range(4))
            (s, s_all), (y, y_all), (dx, dx_all) = (view(rows, D, ld, start, dtype, g) for _ in range(3))
            for t in (s, y, dx):
                t.fill_(NAN)
            dw.fill_(NAN)
            rc = lib.fw_rms_norm(code, code, x.data_ptr(), ld, r.data_ptr(), ld, w.data_ptr(), rows, D, eps, s.data_ptr(),
                                 ld, y.data_ptr(), ld, rstd.data_ptr(), st)
            assert rc == 0
            rc = lib.fw_rms_norm_grad(code, code, dy.data_ptr(), ld, s.data_ptr(), ld, ds.data_ptr(), ld, w.data_ptr(),
                                      rstd.data_ptr(), rows, D, dx.data_ptr(), ld, parts.data_ptr(), nparts,
                                      dw.data_ptr(), st)
            assert rc == 0
            s64, rstd64, y64 = R.norm(x, w, eps, r)
            assert torch.equal(s.double(), s64)
            R.within(y, y64, y64.abs() * (D + 16) * R.E32 + R.rounded(y64, dtype), "y")
            want, wantw, e, ew = R.norm_grad(dy, s64, rstd64, w, ds)
            R.within(dx, want, e + R.rounded(want, dtype), "dx")
            R.within(dw, wantw, ew + R.rounded(wantw, dtype), "dweight")
            for store in (s_all, y_all, dx_all):  # nothing written around the rows
                assert int(store.isnan().sum()) == store.numel() - rows * D

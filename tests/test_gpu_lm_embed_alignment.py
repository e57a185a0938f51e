"""The embedding's C entry points with outputs that start anywhere, in every
form of the gradient, with what lies around the outputs checked."""
import pytest
import torch

import lm_ref as R
from fwloss_b200 import capi

pytestmark = pytest.mark.gpu

NAN = float("nan")


def stream():
    return torch.cuda.current_stream().cuda_stream


def out_view(rows, D, ld, start, dtype):
    store = torch.full((rows * ld + 32,), NAN, dtype=dtype, device="cuda")
    return store[start:].as_strided((rows, D), (ld, 1)), store


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("D", [128, 250, 256, 1024])
def test_rows_into_an_output_at_every_distance(D, dtype):
    lib, code, T, V = capi.load(), capi.DTYPE_CODES[dtype], 37, 20
    g = R.gen(D)
    w, ids = R.normal((V, D), dtype, g), torch.randint(0, V, (T,), generator=g, device="cuda")
    for start in range(16 // dtype.itemsize):
        for ld in (D, D + 16, D + 17):
            for scale in (1.0, 3.0):
                out, store = out_view(T, D, ld, start, dtype)
                rc = lib.fw_embed_rows(code, ids.data_ptr(), T, w.data_ptr(), D, V, D, scale, out.data_ptr(), ld, None, stream())
                assert rc == 0
                want = R.embed(ids, w, scale)
                R.within(out, want, want.abs() * R.E32 + R.rounded(want, dtype), (start, ld))
                assert int(store.isnan().sum()) == store.numel() - T * D


# few tokens of a small table; sorted by one cluster; sorted by several launches
@pytest.mark.parametrize("T,V", [(70, 300), (3000, 300), (33000, 300)])
@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("D", [128, 250, 256, 1024])
def test_gradient_into_a_table_at_every_distance(T, V, D, dtype):
    lib, code = capi.load(), capi.DTYPE_CODES[dtype]
    g = R.gen(T + D)
    ids = torch.randint(0, V // 2, (T,), generator=g, device="cuda")  # half the rows have no token
    ids[: T // 2] = V - 1  # and one has a run of many parts
    grad = R.normal((T, D), dtype, g)
    n = lib.fw_embed_grad_workspace(T, V, D)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    ref, total, most = R.embed_grad(ids, grad, V, 3.0)
    for start in range(16 // dtype.itemsize):
        dw, store = out_view(V, D, D, start, dtype)
        rc = lib.fw_embed_grad(code, ids.data_ptr(), T, grad.data_ptr(), D, V, D, 3.0, -1, dw.data_ptr(), ws.data_ptr(), n,
                               None, stream())
        assert rc == 0
        R.within(dw, ref, total * (most + 2) * R.E32 + R.rounded(ref, dtype), start)
        assert int(store.isnan().sum()) == store.numel() - V * D

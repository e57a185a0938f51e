"""What a tensor-core kernel whose waits gave up leaves in its outputs: NaN,
or the right value, never memory that was not written, status word or not."""
import ctypes

import pytest
import torch

import lm_ref as R
from fwloss_b200 import capi
from test_gpu_lm_waits import giving_up

pytestmark = pytest.mark.gpu

UNWRITTEN = 12345.0


def stream():
    return torch.cuda.current_stream().cuda_stream


def nan_or_right(got, want):
    assert not (got == UNWRITTEN).any() and not (want == UNWRITTEN).any()
    lost = got.isnan()
    assert lost.any() and torch.equal(got[~lost], want[~lost])


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("T,N,K", [(1, 5001, 2000), (50, 19003, 704), (300, 1001, 1504), (700, 9001, 608)])
def test_int8_product(T, N, K, dtype):
    lib, g = capi.load(), R.gen(T)
    q = torch.randint(-127, 128, (T, K), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    qs, ws = torch.rand(T, generator=g, device="cuda") * 1e-2, torch.rand(N, generator=g, device="cuda") * 1e-2

    def product():
        store = torch.full((T * N + 64,), UNWRITTEN, dtype=dtype, device="cuda")
        assert lib.fw_int8_linear(capi.DTYPE_CODES[dtype], q.data_ptr(), K, qs.data_ptr(), w.data_ptr(), K, ws.data_ptr(),
                                  T, N, K, store.data_ptr(), N, None, stream()) == 0
        assert bool((store[T * N:] == UNWRITTEN).all())
        return store[: T * N].view(T, N)

    want = product()
    with giving_up():
        got = product()
    nan_or_right(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", [0, 1])
@pytest.mark.parametrize("B,D,V", [(600, 520, 3000), (64, 512, 20000), (33000, 64, 10007)])
def test_cross_entropy_gradients(B, D, V, dtype, reduction):
    """In one piece; dhidden in splits; several pieces of the vocabulary."""
    lib, code, g = capi.load(), capi.DTYPE_CODES[dtype], R.gen(B)
    h, w = R.normal((B, D), dtype, g), R.normal((V, D), dtype, g, 0.1)
    y = torch.randint(0, V, (B,), generator=g, device="cuda")
    y[::5] = -100
    n = B if reduction == 0 else 1
    loss, go = torch.empty(n, device="cuda"), torch.rand(n, generator=g, device="cuda") + 0.5
    ns = lib.fw_xent_state_bytes(B, D, V, ctypes.c_void_p(w.data_ptr()), D)
    nf, nb = lib.fw_xent_workspace(B, D, V, 0), lib.fw_xent_workspace(B, D, V, 1)
    state, ws = torch.zeros(ns, dtype=torch.uint8, device="cuda"), torch.zeros(max(nf, nb), dtype=torch.uint8, device="cuda")
    assert lib.fw_xent_forward(code, h.data_ptr(), D, w.data_ptr(), D, y.data_ptr(), B, D, V, -100, reduction,
                               loss.data_ptr(), state.data_ptr(), ns, ws.data_ptr(), nf, None, stream()) == 0

    def gradients():
        ws.zero_()
        dh, dw = torch.full_like(h, UNWRITTEN), torch.full_like(w, UNWRITTEN)
        assert lib.fw_xent_backward(code, w.data_ptr(), D, B, D, V, reduction, go.data_ptr(), state.data_ptr(), ns,
                                    ws.data_ptr(), nb, dh.data_ptr(), dw.data_ptr(), None, stream()) == 0
        return dh, dw

    want = gradients()
    with giving_up():
        got = gradients()
        torch.cuda.synchronize()
    for a, b in zip(got, want):
        nan_or_right(a, b)
    assert not got[0][::5].any()  # ignored rows
    for a, b in zip(gradients(), want):
        assert torch.equal(a, b)


def test_cross_entropy_loss_without_a_status_word():
    lib, code, B, D, V = capi.load(), 1, 300, 64, 1000
    g = R.gen(1)
    h, w = R.normal((B, D), torch.bfloat16, g), R.normal((V, D), torch.bfloat16, g)
    y = torch.randint(0, V, (B,), generator=g, device="cuda")
    ns, nf = lib.fw_xent_state_bytes(B, D, V, ctypes.c_void_p(w.data_ptr()), D), lib.fw_xent_workspace(B, D, V, 0)
    state, ws = torch.zeros(ns, dtype=torch.uint8, device="cuda"), torch.zeros(nf, dtype=torch.uint8, device="cuda")
    loss = torch.full((B,), UNWRITTEN, device="cuda")
    with giving_up():
        assert lib.fw_xent_forward(code, h.data_ptr(), D, w.data_ptr(), D, y.data_ptr(), B, D, V, -100, 0, loss.data_ptr(),
                                   state.data_ptr(), ns, ws.data_ptr(), nf, None, stream()) == 0
    assert loss.isnan().all()

"""The state that the cross entropy's forward keeps is only read by the gradient."""
import ctypes

import pytest
import torch

import lm_ref as R
from fwloss_b200 import capi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("reduction", [0, 1, 2])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gradient_leaves_the_state_as_it_was(dtype, reduction):
    lib, code, B, D, V = capi.load(), capi.DTYPE_CODES[dtype], 150, 72, 400
    g = R.gen(2)
    h, w = R.normal((B, D), dtype, g), R.normal((V, D), dtype, g, 0.2)
    y = torch.randint(0, V, (B,), generator=g, device="cuda")
    y[::7] = -100
    n = B if reduction == 0 else 1
    loss, go = torch.empty(n, device="cuda"), torch.rand(n, generator=g, device="cuda") * 1000
    ns = lib.fw_xent_state_bytes(B, D, V, ctypes.c_void_p(w.data_ptr()), D)
    state = torch.zeros(ns, dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    nf, nb = lib.fw_xent_workspace(B, D, V, 0), lib.fw_xent_workspace(B, D, V, 1)
    ws = torch.empty(max(nf, nb), dtype=torch.uint8, device="cuda")
    assert lib.fw_xent_forward(code, h.data_ptr(), D, w.data_ptr(), D, y.data_ptr(), B, D, V, -100, reduction,
                               loss.data_ptr(), state.data_ptr(), ns, ws.data_ptr(), nf, None, st) == 0
    kept = state.clone()
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    assert lib.fw_xent_backward(code, w.data_ptr(), D, B, D, V, reduction, go.data_ptr(), state.data_ptr(), ns,
                                ws.data_ptr(), nb, dh.data_ptr(), dw.data_ptr(), None, st) == 0
    assert dh.isfinite().all() and torch.equal(state, kept)

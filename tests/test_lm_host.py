"""The language-model operators' refusals that need no device: CPU tensors in
Python, argument checks of the C entry points before any device work."""
import ctypes

import pytest
import torch

import fwloss_b200 as fw
from fwloss_b200 import capi

P = None
D = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(257)
OFF = ctypes.c_void_p(264)
OK, SHAPE, POINTER, CAPACITY, DTYPE = 0, 1, 2, 4, 5


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 8), torch.ones(8)
    q = torch.zeros(4, 8, dtype=torch.int8)
    y = torch.zeros(4, dtype=torch.int64)
    for call in (lambda: fw.embed_tokens(y, x), lambda: fw.rms_norm(x, w), lambda: fw.rms_norm_int8(x, w),
                 lambda: fw.quantize_rows_int8(x), lambda: fw.int8_linear(q, torch.ones(4), q, torch.ones(4)),
                 lambda: fw.lm_head_cross_entropy(x.bfloat16(), x.bfloat16(), y)):
        with pytest.raises(TypeError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="reduction"):
        fw.lm_head_cross_entropy(x, x, y, reduction="avg")


def test_embedding_arguments():
    lib = capi.load()
    f, g = lib.fw_embed_rows, lib.fw_embed_grad
    assert f(3, D, 4, D, 8, 10, 8, 1.0, D, 8, P, P) == DTYPE
    assert f(0, D, -1, D, 8, 10, 8, 1.0, D, 8, P, P) == SHAPE
    assert f(0, D, 4, D, 7, 10, 8, 1.0, D, 8, P, P) == SHAPE
    assert f(0, D, 4, D, 8, 0, 8, 1.0, D, 8, P, P) == SHAPE
    assert f(0, P, 4, D, 8, 10, 8, 1.0, D, 8, P, P) == POINTER
    assert f(0, D, 4, ODD, 8, 10, 8, 1.0, D, 8, P, P) == POINTER
    assert f(0, P, 0, P, 8, 10, 8, 1.0, P, 8, P, P) == OK
    need = lib.fw_embed_grad_workspace(100, 10, 8)
    assert need > 0 and lib.fw_embed_grad_workspace(-1, 10, 8) == 0
    assert g(0, D, 100, D, 8, 10, 8, 1.0, -1, D, D, need - 1, P, P) == CAPACITY
    assert g(0, D, 100, D, 8, 10, 8, 1.0, -1, P, D, need, P, P) == POINTER
    assert g(0, D, 100, D, 8, 10, 8, 1.0, -1, D, OFF, need, P, P) == POINTER
    assert g(0, D, 100, D, 7, 10, 8, 1.0, -1, D, D, need, P, P) == SHAPE
    assert g(9, D, 100, D, 8, 10, 8, 1.0, -1, D, D, need, P, P) == DTYPE


def test_norm_arguments():
    lib = capi.load()
    f, q, g, r = lib.fw_rms_norm, lib.fw_rms_norm_int8, lib.fw_rms_norm_grad, lib.fw_quantize_rows_int8
    assert f(1, 2, D, 8, P, 0, D, 4, 8, 1e-6, P, 0, D, 8, P, P) == DTYPE
    assert f(0, 0, D, 7, P, 0, D, 4, 8, 1e-6, P, 0, D, 8, P, P) == SHAPE
    assert f(0, 0, D, 8, P, 0, D, 4, 8, -1.0, P, 0, D, 8, P, P) == SHAPE
    assert f(0, 0, D, 8, P, 0, D, 4, 8, float("nan"), P, 0, D, 8, P, P) == SHAPE
    assert f(0, 0, D, 8, D, 8, D, 4, 8, 1e-6, P, 0, D, 8, P, P) == POINTER
    assert f(0, 0, ODD, 8, P, 0, D, 4, 8, 1e-6, P, 0, D, 8, P, P) == POINTER
    assert f(0, 0, P, 8, P, 0, P, 0, 8, 1e-6, P, 0, P, 8, P, P) == OK
    assert q(0, 0, D, 8, P, 0, D, 4, 8, 1e-6, P, 0, D, 8, D, P) == SHAPE
    assert q(0, 0, D, 8, P, 0, D, 4, 8, 1e-6, P, 0, OFF, 16, D, P) == POINTER
    assert r(0, D, 20, 4, 20, D, 16, D, P) == SHAPE
    assert r(0, D, 20, 4, 20, D, 32, P, P) == POINTER
    assert lib.fw_rms_norm_grad_parts(5) == 5 and lib.fw_rms_norm_grad_parts(-5) == 0
    assert g(0, 0, D, 8, D, 8, P, 0, D, D, 4, 8, D, 8, D, 0, D, P) == CAPACITY
    assert g(0, 0, D, 8, D, 8, P, 0, D, D, 4, 8, D, 8, P, 4, D, P) == POINTER
    assert g(0, 0, D, 8, D, 8, P, 0, D, P, 4, 8, D, 8, D, 4, D, P) == POINTER


def test_int8_arguments():
    lib = capi.load()
    f = lib.fw_int8_linear
    assert f(7, D, 32, D, D, 32, D, 4, 10, 20, D, 10, P, P) == DTYPE
    assert f(0, D, 24, D, D, 32, D, 4, 10, 20, D, 10, P, P) == SHAPE
    assert f(0, D, 16, D, D, 32, D, 4, 10, 20, D, 10, P, P) == SHAPE
    assert f(0, D, 32, D, D, 32, D, 4, 10, 20, D, 9, P, P) == SHAPE
    assert f(0, D, 131072, D, D, 131072, D, 4, 10, 131072, D, 10, P, P) == CAPACITY
    assert f(0, OFF, 32, D, D, 32, D, 4, 10, 20, D, 10, P, P) == POINTER
    assert f(0, D, 32, P, D, 32, D, 4, 10, 20, D, 10, P, P) == POINTER
    assert f(0, P, 32, P, P, 32, P, 0, 10, 20, P, 10, P, P) == OK


def test_cross_entropy_arguments():
    lib = capi.load()
    f, b = lib.fw_xent_forward, lib.fw_xent_backward
    ns, nf, nb = lib.fw_xent_state_bytes(4, 8, 10, D, 8), lib.fw_xent_workspace(4, 8, 10, 0), lib.fw_xent_workspace(4, 8, 10, 1)
    assert lib.fw_xent_state_bytes(4, 8, 10, OFF, 8) > ns  # a weight that has to be copied
    assert lib.fw_xent_state_bytes(-1, 8, 10, D, 8) == 0 and lib.fw_xent_workspace(4, 0, 10, 1) == 0
    assert f(0, D, 8, D, 8, D, 4, 8, 10, -100, 1, D, D, ns, D, nf, P, P) == DTYPE
    assert f(1, D, 7, D, 8, D, 4, 8, 10, -100, 1, D, D, ns, D, nf, P, P) == SHAPE
    assert f(1, D, 8, D, 8, D, 4, 8, 10, -100, 3, D, D, ns, D, nf, P, P) == SHAPE
    assert f(1, D, 8, D, 8, P, 4, 8, 10, -100, 1, D, D, ns, D, nf, P, P) == POINTER
    assert f(1, D, 8, ODD, 8, D, 4, 8, 10, -100, 1, D, D, 1 << 20, D, nf, P, P) == POINTER
    assert f(1, D, 8, D, 8, D, 4, 8, 10, -100, 1, D, D, ns - 1, D, nf, P, P) == CAPACITY
    assert f(1, D, 8, D, 8, D, 4, 8, 10, -100, 1, D, D, ns, D, nf - 1, P, P) == CAPACITY
    assert b(1, D, 8, 4, 8, 10, 1, D, D, ns, D, nb - 1, D, D, P, P) == CAPACITY
    assert b(1, D, 8, 4, 8, 10, 1, P, D, ns, D, nb, D, D, P, P) == POINTER
    assert b(1, D, 8, 4, 8, 10, 1, D, D, ns, D, nb, P, P, P, P) == OK

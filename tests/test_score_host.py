"""The scoring and clipping operators' refusals that need no device: CPU
tensors in Python, argument checks of the C entry points before any device work."""
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
    x, y = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: fw.token_log_probs(x, y), lambda: fw.lm_head_log_probs(x.bfloat16(), x.bfloat16(), y),
                 lambda: fw.grad_norm([x]), lambda: fw.grad_norm(x), lambda: fw.clip_grad_norm_([x], 1.0)):
        with pytest.raises(TypeError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="no tensors"):
        fw.grad_norm([])
    with pytest.raises(ValueError, match="every gradient"):
        fw.clip_grad_norm_([x], 1.0, out=[x, x])


def test_token_log_probs_arguments():
    lib = capi.load()
    f, g = lib.fw_token_log_probs, lib.fw_token_log_probs_grad

    def fwd(dtype=0, z=D, ld=8, y=D, B=4, V=8, it=1.0, k=2, logp=D, ent=D, tl=D, ti=D, state=D):
        return f(dtype, z, ld, y, B, V, it, -100, k, logp, ent, tl, ti, state, P, P)

    assert fwd(dtype=3) == DTYPE
    for bad in (dict(ld=7), dict(B=-1), dict(V=0), dict(V=1 << 29, ld=1 << 29), dict(B=1 << 29), dict(it=0.0), dict(it=-1.0),
                dict(it=float("nan")), dict(it=float("inf")), dict(it=3e38), dict(k=-1), dict(k=9)):
        assert fwd(**bad) == SHAPE, bad
    assert fwd(V=100, ld=100, k=33) == CAPACITY
    for bad in (dict(z=P), dict(y=P), dict(logp=P), dict(ent=P), dict(tl=P), dict(ti=P), dict(z=ODD), dict(state=OFF)):
        assert fwd(**bad) == POINTER, bad
    assert fwd(B=0, z=P, y=P, logp=P, ent=P) == OK

    def bwd(dtype=0, z=D, ld=8, B=4, V=8, it=1.0, state=D, grad=D, ldg=8):
        return g(dtype, z, ld, B, V, it, state, P, P, grad, ldg, P)

    assert bwd(dtype=9) == DTYPE
    for bad in (dict(ld=7), dict(ldg=7), dict(V=0), dict(it=0.0)):
        assert bwd(**bad) == SHAPE, bad
    for bad in (dict(z=P), dict(state=P), dict(grad=P), dict(state=OFF), dict(grad=ODD)):
        assert bwd(**bad) == POINTER, bad
    assert bwd(B=0, z=P, state=P, grad=P) == OK


def test_lm_head_log_probs_arguments():
    lib = capi.load()
    f, b = lib.fw_lm_head_log_probs, lib.fw_lm_head_log_probs_grad
    ns = lib.fw_lm_head_log_probs_state(4, 8, 10, D, 8)
    nf, nb = (lib.fw_lm_head_log_probs_workspace(4, 8, 10, i) for i in (0, 1))
    assert lib.fw_lm_head_log_probs_state(4, 8, 10, OFF, 8) > ns  # a weight that has to be copied
    assert lib.fw_lm_head_log_probs_state(-1, 8, 10, D, 8) == 0 and lib.fw_lm_head_log_probs_workspace(4, 0, 10, 1) == 0
    assert ns > lib.fw_xent_state_bytes(4, 8, 10, D, 8)  # the entropies

    def fwd(dtype=1, h=D, ldh=8, w=D, ldw=8, y=D, it=1.0, logp=D, ent=D, state=D, n=ns, ws=D, m=nf, B=4):
        return f(dtype, h, ldh, w, ldw, y, B, 8, 10, it, -100, logp, ent, state, n, ws, m, P, P)

    assert fwd(dtype=0) == DTYPE
    for bad in (dict(ldh=7), dict(ldw=7), dict(it=0.0), dict(it=float("inf")), dict(it=3e38), dict(B=-1), dict(B=(1 << 26) + 1)):
        assert fwd(**bad) == SHAPE, bad
    for bad in (dict(h=P), dict(w=P), dict(y=P), dict(logp=P), dict(ent=P), dict(state=P), dict(ws=P), dict(w=ODD, n=1 << 20),
                dict(state=OFF), dict(ws=OFF)):
        assert fwd(**bad) == POINTER, bad
    assert fwd(n=ns - 1) == CAPACITY and fwd(m=nf - 1) == CAPACITY
    assert fwd(B=0, h=P, y=P, logp=P, ent=P) == OK

    def bwd(dtype=1, w=D, ldw=8, it=1.0, state=D, n=ns, ws=D, m=nb, dh=P, dw=P):
        return b(dtype, w, ldw, 4, 8, 10, it, D, D, state, n, ws, m, dh, dw, P, P)

    assert bwd(dtype=0) == DTYPE and bwd(ldw=7) == SHAPE and bwd(it=-1.0) == SHAPE
    for bad in (dict(w=P), dict(state=P), dict(ws=P), dict(state=OFF), dict(dh=ODD), dict(dw=ODD)):
        assert bwd(**bad) == POINTER, bad
    assert bwd(n=ns - 1) == CAPACITY and bwd(m=nb - 1) == CAPACITY
    assert bwd() == OK  # no gradient asked for


def test_gradient_norm_arguments():
    lib = capi.load()

    def arrays(ptrs, numel, types):
        n = len(ptrs)
        return (ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*numel), (ctypes.c_int32 * n)(*types)

    need = lib.fw_grad_norm_workspace(2)
    assert need > 0 and lib.fw_grad_norm_workspace(-1) == 0 and lib.fw_grad_norm_workspace(1 << 25) == 0

    def norm(ptrs=(256, 512), numel=(8, 8), types=(0, 1), ws=D, n=need, out=D, count=None):
        a, b, c = arrays(ptrs, numel, types)
        return lib.fw_grad_norm(len(ptrs) if count is None else count, a, b, c, ws, n, out, P, P)

    assert norm(types=(0, 3)) == DTYPE
    assert norm(numel=(8, -1)) == SHAPE and norm(numel=(8, 1 << 43)) == SHAPE and norm(count=-1) == SHAPE
    for bad in (dict(ptrs=(256, 0)), dict(ptrs=(258, 512)), dict(ptrs=(256, 513)), dict(out=P), dict(ws=P), dict(ws=OFF)):
        assert norm(**bad) == POINTER, bad
    assert norm(n=need - 1) == CAPACITY
    assert lib.fw_grad_norm(2, P, P, P, D, need, D, P, P) == POINTER

    def clip(ptrs=(256, 512), outs=(256, 512), numel=(8, 8), types=(0, 1), otypes=(0, 1), most=1.0, given=P, ws=D, n=need, out=D):
        a, b, c = arrays(ptrs, numel, types)
        o, _, d = arrays(outs, numel, otypes)
        return lib.fw_grad_clip(len(ptrs), a, o, b, c, d, most, given, ws, n, out, P, P)

    assert clip(otypes=(0, 7)) == DTYPE
    assert clip(most=-1.0) == SHAPE and clip(most=float("nan")) == SHAPE
    for bad in (dict(outs=(256, 0)), dict(outs=(256, 513)), dict(ws=P), dict(out=P), dict(ws=OFF)):
        assert clip(**bad) == POINTER, bad
    assert clip(n=need - 1) == CAPACITY
    assert clip(numel=(0, 0), given=D) == OK  # nothing to scale

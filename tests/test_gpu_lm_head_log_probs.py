"""Log probabilities and entropies of an output layer, and their gradients,
against the 64-bit definition.

Logits: products of 16-bit numbers are exact in fp32, and D additions with
truncation are off by 2 * E32 of the absolute terms each at most (e_z); what
follows from logits that are off so is score_ref's.  A logit gradient is rounded
once to the operands' type (for dhidden the label's entry is not); both sums are
truncating fp32 additions.  float16's logit gradient may be under its range:
half of 2^-24 over 2^13, of the largest factor's next power of two.
"""
import ctypes

import pytest
import torch

import fwloss_b200 as fw
import lm_ref as R
import score_ref as S
from fwloss_b200 import capi
from test_gpu_lm_waits import giving_up

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def reference(hidden, weight, tokens, temperature=1.0, a=None, b=None, ignore=-100):
    dtype = hidden.dtype
    live = tokens != ignore
    h = torch.where(live[:, None], hidden.double(), 0.0)
    w = weight.double()
    D, V, B = h.shape[1], w.shape[0], h.shape[0]
    e_z = 2 * (D + 2) * R.E32 * (h.abs() @ w.abs().t()).amax(1)
    r = S.rows(h @ w.t(), tokens, temperature, ignore, e_z=torch.nan_to_num(e_z, nan=0.0, posinf=0.0))
    G, eG = S.logit_grad(r, a, b)
    scale = torch.zeros(B, dtype=torch.float64, device=h.device)
    for x in (a, b):
        if x is not None:
            scale = torch.maximum(scale, x.double().abs())
    scale = torch.where(live, scale, torch.zeros_like(scale)) / temperature
    # one exponential's argument here is a fused product and difference against the rounded log sum of exponentials
    lse = (r["t"] * 0 + (h @ w.t()).amax(1, keepdim=True) / temperature).abs()
    eG = eG + (r["q"] * 3 * R.E32 * (lse + 40) * (scale[:, None] * (2 + r["logq"].abs().clamp(max=745) + r["h"][:, None])))
    eG = eG + G.abs() * R.U[dtype]
    if dtype == torch.float16 and B:
        eG = eG + 2.0 ** -24 / 2.0 ** 13 * 2 * float(torch.nan_to_num(scale).max())
    eG = torch.where(live[:, None], eG, torch.zeros_like(eG))
    dh, dw = G @ w, G.t() @ h
    e_dh = eG @ w.abs() + (G.abs() @ w.abs()) * (2 * V + 8) * R.E32 + R.rounded(dh, dtype)
    e_dw = eG.t() @ h.abs() + (G.abs().t() @ h.abs()) * (2 * B + 8) * R.E32 + R.rounded(dw, dtype)
    return r, (dh, e_dh), (dw, e_dw)


def check(hidden, weight, tokens, temperature=1.0, kind="both", seed=0, scale=1.0):
    g = R.gen(seed + 5)
    a, b = (torch.randn(len(tokens), generator=g, device="cuda") * scale for _ in range(2))
    a, b = (a if kind != "entropy" else None), (b if kind != "logp" else None)
    r, dh, dw = reference(hidden, weight, tokens, temperature, a, b)
    plain = fw.lm_head_log_probs(hidden, weight, tokens, temperature=temperature)
    R.within(plain[0], r["logp"], r["e_logp"], "logp")
    R.within(plain[1], r["entropy"], r["e_entropy"], "entropy")
    h, w = hidden.detach().requires_grad_(True), weight.detach().requires_grad_(True)
    out = fw.lm_head_log_probs(h, w, tokens, temperature=temperature)
    for p, q in zip(out, plain):
        assert torch.equal(torch.nan_to_num(p.detach(), nan=7.0), torch.nan_to_num(q, nan=7.0))
    outs = [o for o, x in zip(out, (a, b)) if x is not None]
    got = torch.autograd.grad(outs, (h, w), [x for x in (a, b) if x is not None])
    R.within(got[0], *dh, "dhidden")
    R.within(got[1], *dw, "dweight")


def tokens_for(B, V, g, ignored=0.0):
    y = torch.randint(0, V, (B,), generator=g, device="cuda")
    return torch.where(torch.rand(B, generator=g, device="cuda") < ignored, torch.full_like(y, -100), y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,D,V", [(1, 1, 1), (1, 64, 300), (3, 7, 5), (37, 65, 129), (128, 64, 256), (256, 256, 1000),
                                   (300, 520, 3001), (257, 1000, 5001), (64, 512, 20000), (1000, 72, 4099)])
def test_values_and_gradients(B, D, V, dtype):
    g = R.gen(B + D + V)
    h, w = R.normal((B, D), dtype, g), R.normal((V, D), dtype, g, 2.0 * D ** -0.5)
    y = tokens_for(B, V, g, 0.2 if B > 2 else 0.0)
    check(h, w, y)
    check(h, w, y, temperature=0.6, kind="logp", scale=1e-3)
    check(h, w, y, temperature=1.7, kind="entropy", scale=30.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_anywhere(dtype):
    g = R.gen(3)
    hs, ws = R.normal((50, 77), dtype, g), R.normal((700, 83), dtype, g, 0.2)
    y = tokens_for(50, 700, g, 0.1)
    check(hs[:, 3:64], ws[:, 1:62], y)
    check(hs[:, 3:64], ws[:, 1:62].contiguous(), y)
    check(R.normal((64, 50), dtype, g).t(), R.normal((64, 700), dtype, g, 0.2).t(), y)


@pytest.mark.parametrize("dtype", TYPES)
def test_confident_and_flat_rows(dtype):
    """A token that has nearly all of the probability, none of it, and rows without any preference."""
    g = R.gen(4)
    w = R.normal((900, 64), dtype, g)
    h = torch.zeros(40, 64, dtype=dtype, device="cuda")
    h[:20] = w[100:120] * 0.7  # |w|^2 is near 64: 45 nats ahead
    h[20:30] = R.normal((10, 64), dtype, g, 1e-3)
    y = torch.arange(100, 140, device="cuda")
    y[10:20] = 0
    check(h, w, y)
    check(h, w, y, kind="entropy", temperature=0.5)
    out = fw.lm_head_log_probs(h[30:], w, y[30:])
    R.within(out[1], torch.full((10,), 900.0, dtype=torch.float64, device="cuda").log(), 1e-5)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_row_ignored_none_and_bad_ones(dtype):
    g = R.gen(5)
    h, w = R.normal((30, 40), dtype, g), R.normal((200, 40), dtype, g)
    y = torch.full((30,), -100, device="cuda")
    h[3] = float("nan")
    check(h, w, y)
    y[4:] = tokens_for(26, 200, g)
    check(h, w, y)
    none = fw.lm_head_log_probs(h[:0].requires_grad_(True), w, y[:0])
    assert none[0].shape == (0,) and none[1].shape == (0,)
    ww = w.clone().requires_grad_(True)
    (d,) = torch.autograd.grad(fw.lm_head_log_probs(h[:0], ww, y[:0])[0].sum(), ww)
    assert d.shape == ww.shape and not d.any()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    fw.lm_head_log_probs(h, w, y, status=status)
    assert int(status) == 0
    y[8], y[9], y[10] = 200, -1, 5
    h[10, 3] = float("inf")
    hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    out = fw.lm_head_log_probs(hh, ww, y, status=status)
    assert int(status) == 3
    bad = torch.zeros(30, dtype=torch.bool, device="cuda")
    bad[8:11] = True
    for o in out:
        assert o[bad].isnan().all() and not o[~bad].isnan().any() and not o[:4].any()
    dh, dw = torch.autograd.grad(out[0].sum(), (hh, ww))
    assert dh[bad].isnan().all() and not dh[~bad].isnan().any() and not dh[:4].any() and dw.isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_upstream_factors(value, dtype):
    """Of very different sizes, zero, and not finite."""
    g = R.gen(6)
    h, w = R.normal((64, 48), dtype, g), R.normal((500, 48), dtype, g, 0.3)
    y = tokens_for(64, 500, g, 0.1)
    # (float16 takes them relative to the largest: its gradient holds what is 2^-24 of that)
    a, b = (torch.randn(64, generator=g, device="cuda") * 2.0 ** torch.randint(-6, 7, (64,), generator=g, device="cuda") for _ in range(2))
    a[::4], b[::3] = 0.0, 0.0
    hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    got = torch.autograd.grad(fw.lm_head_log_probs(hh, ww, y), (hh, ww), (a, b))
    _, dh, dw = reference(h, w, y, 1.0, a, b)
    R.within(got[0], *dh, "dhidden")
    R.within(got[1], *dw, "dweight")
    zero = torch.zeros_like(a)
    for d in torch.autograd.grad(fw.lm_head_log_probs(hh, ww, y), (hh, ww), (zero, zero)):
        assert not d.any()
    row = int((y != -100).nonzero()[5])
    a[row] = value
    got = torch.autograd.grad(fw.lm_head_log_probs(hh, ww, y), (hh, ww), (a, b))
    rest = torch.arange(64, device="cuda") != row
    assert got[0][row].isnan().all() and got[1].isnan().all()
    R.within(got[0][rest], dh[0][rest], dh[1][rest], "other rows")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,D,V", [(700, 300, 1), (700, 300, 40), (900, 100, 3000), (513, 136, 700)])
def test_labels_met_again_and_again(B, D, V, dtype):
    """Many rows with labels of one 32 rows of the weight, and with one label."""
    g = R.gen(B + V)
    h, w = R.normal((B, D), dtype, g), R.normal((V, D), dtype, g, D ** -0.5)
    y = torch.randint(0, min(V, 45), (B,), generator=g, device="cuda") + (V - min(V, 45))
    check(h, w, y)
    y[: B // 2] = V // 2
    y[::7] = -100
    check(h, w, y, kind="logp")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,D,V", [(1000, 300, 2000), (3000, 129, 70), (2500, 64, 40000)])
def test_common_labels(B, D, V, dtype):
    """Labels that fall off as 1 / rank, runs of one label from 1 to a third of the rows, starting anywhere; one piece
    of the vocabulary and several."""
    g = R.gen(B)
    h, w = R.normal((B, D), dtype, g), R.normal((V, D), dtype, g, D ** -0.5)
    u = torch.rand(B, generator=g, device="cuda", dtype=torch.float64)
    y = ((V + 1.0) ** u - 1.0).long().clamp_(0, V - 1)
    check(h, w, y)
    y[: B // 3] = V - 1
    y[torch.rand(B, generator=g, device="cuda") < 0.1] = -100
    check(h, w, y, temperature=1.3, kind="logp")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,V", [(8192, 300), (8193, 300), (20011, 3), (40000, 511), (9000, 512)])
def test_many_rows(B, V, dtype):
    """Rows counted and rows sorted into the order of their labels; ignored rows and bad labels among them."""
    g = R.gen(B + V)
    h, w = R.normal((B, 40), dtype, g), R.normal((V, 40), dtype, g, 0.3)
    y = tokens_for(B, V, g, 0.2)
    check(h, w, y)
    bad = torch.randint(0, B, (5,), generator=g, device="cuda")
    y[bad] = torch.tensor([V, -1, V + 7, 1 << 40, -(1 << 50)], device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    out = fw.lm_head_log_probs(hh, ww, y, status=status)
    assert int(status) == 1
    r, (dh, e_dh), _ = reference(h, w, y, 1.0, torch.ones(B, device="cuda"))
    R.within(out[0], r["logp"], r["e_logp"], "logp")
    R.within(out[1], r["entropy"], r["e_entropy"], "entropy")
    got = torch.autograd.grad(out[0].sum(), (hh, ww))
    R.within(got[0], dh, e_dh, "dhidden")
    assert got[1].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_rounding_of_the_labels_entry_is_made_good(dtype):
    """A label's gradient is the one large entry of its row; both products have to come out as if it were not rounded:
    within the rounding of the result and a twentieth of the entry's."""
    g = R.gen(21)
    h, w = R.normal((64, 64), dtype, g, 1e-3), R.normal((4096, 64), dtype, g)  # probabilities of 2^-12 each
    y = torch.randperm(4096, generator=g, device="cuda")[:64]
    hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    a = torch.rand(64, generator=g, device="cuda") + 1.0
    dh, dw = torch.autograd.grad(fw.lm_head_log_probs(hh, ww, y)[0], (hh, ww), a)
    _, (eh, _), (ew, _) = reference(h, w, y, 1.0, a)
    term = a.double()[:, None] * w[y].double().abs()
    # the other 4095 entries are 2^-12 of the label's, each rounded: their sum of absolute terms is under w's largest
    R.within(dh, eh, R.rounded(eh, dtype) + term * R.U[dtype] / 20 + R.U[dtype] * 2.0 ** -12 * 64 * 5 * a[:, None] * 2, "dhidden")
    got, want = dw[y], ew[y]
    R.within(got, want, R.rounded(want, dtype) + a[:, None].double() * h.double().abs() * R.U[dtype] / 20
             + R.U[dtype] * 2.0 ** -12 * 64 * 5e-3 * 2, "dweight")


def test_equal_to_the_loss():
    """-logp is lm_head_cross_entropy's loss, both within their bounds of one value; and the entropy's share is apart."""
    g = R.gen(7)
    h, w = R.normal((200, 96), torch.bfloat16, g), R.normal((1500, 96), torch.bfloat16, g, 0.3)
    y = tokens_for(200, 1500, g, 0.1)
    r, _, _ = reference(h, w, y)
    loss = fw.lm_head_cross_entropy(h, w, y, reduction="none")
    R.within(-fw.lm_head_log_probs(h, w, y)[0], loss, 2 * r["e_logp"] + R.xent(h, w, y, "none")["e_loss"])


def test_gradient_against_differences():
    """Directional differences of the values; the error of a difference is the
    values' over the step and the third derivative's part."""
    g = R.gen(8)
    h, w = R.normal((8, 32), torch.bfloat16, g), R.normal((60, 32), torch.bfloat16, g, 0.25)
    y = tokens_for(8, 60, g)
    hh = h.clone().requires_grad_(True)
    a, b = torch.randn(8, device="cuda"), torch.randn(8, device="cuda")
    (d,) = torch.autograd.grad(fw.lm_head_log_probs(hh, w, y), hh, (a, b))
    _, (want, e_d), _ = reference(h, w, y, 1.0, a, b)
    step = 2.0 ** -3  # exact in bfloat16 next to values under 2 once h is on a grid of 2^-6
    base = (h.float() * 64).round().clamp(-127, 127) / 64
    hh = base.bfloat16().requires_grad_(True)
    (d,) = torch.autograd.grad(fw.lm_head_log_probs(hh, w, y), hh, (a, b))
    r, (want, e_d), _ = reference(hh.detach(), w, y, 1.0, a, b)
    for j in (0, 17, 31):
        vals = []
        for sign in (1, -1):
            x = base.clone()
            x[:, j] += sign * step
            assert torch.equal(x.bfloat16().float(), x)
            l, e = fw.lm_head_log_probs(x.bfloat16(), w, y)
            vals.append(a.double() * l.double() + b.double() * e.double())
        near = 4 * (a.abs() * r["e_logp"] + b.abs() * r["e_entropy"]) / (2 * step)
        reach = float(w[:, j].double().abs().max())  # third derivatives: 2 and 8 (1 + H) in units of the largest weight's cube
        third = (2 * a.abs() + b.abs() * 8 * (1 + r["h"] + 2 * step * reach)) * (2 * reach) ** 3 * step ** 2 / 6
        R.within(d[:, j], (vals[0] - vals[1]) / (2 * step), near + third + e_d[:, j], f"column {j}")


def test_nodes():
    g = R.gen(9)
    h = R.normal((100, 64), torch.bfloat16, g).requires_grad_(True)
    w = R.normal((300, 64), torch.bfloat16, g, 0.3).requires_grad_(True)
    y = tokens_for(100, 300, g, 0.1)
    up = torch.randn(100, device="cuda")
    out = fw.lm_head_log_probs(h, w, y)
    want = torch.autograd.grad(out, (h, w), (up, up), retain_graph=True)
    for p, q in zip(want, torch.autograd.grad(out, (h, w), (up, up))):
        assert torch.equal(p, q)
    only = torch.autograd.grad(fw.lm_head_log_probs(h.detach(), w, y), w, (up, up))
    assert torch.equal(only[0], want[1])
    only = torch.autograd.grad(fw.lm_head_log_probs(h, w.detach(), y), h, (up, up))
    assert torch.equal(only[0], want[0])
    (d,) = torch.autograd.grad(fw.lm_head_log_probs(h, w, y)[0].sum(), h, create_graph=True)
    with pytest.raises(RuntimeError, match="again"):
        d.float().sum().backward()
    with torch.autograd.graph.save_on_cpu():
        out = fw.lm_head_log_probs(h, w, y)
    for p, q in zip(want, torch.autograd.grad(out, (h, w), (up, up))):
        assert torch.equal(p, q)
    out = fw.lm_head_log_probs(h, w, y)
    keep = y.clone()
    y.zero_()
    for p, q in zip(want, torch.autograd.grad(out, (h, w), (up, up))):  # packed rows and labels are the operator's own
        assert torch.equal(p, q)
    y.copy_(keep)
    out = fw.lm_head_log_probs(h, w, y)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out[1].sum().backward()
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level(), pytest.raises(NotImplementedError):
        fw.lm_head_log_probs(fwd.make_dual(h.detach(), torch.ones_like(h)), w, y)


def test_weight_restored_with_other_strides():
    """A saved-tensor hook may bring the weight back off the 16-byte boundaries it was saved on."""
    g = R.gen(30)
    h = R.normal((70, 64), torch.bfloat16, g).requires_grad_(True)
    w = R.normal((300, 64), torch.bfloat16, g, 0.3).requires_grad_(True)
    y = tokens_for(70, 300, g, 0.1)
    up = torch.randn(70, device="cuda")

    def off(t):
        if t.dim() != 2:
            return t
        store = torch.empty(t.shape[0], t.shape[1] + 3, dtype=t.dtype, device="cuda")
        store[:, 1:-2] = t
        return store[:, 1:-2]

    want = torch.autograd.grad(fw.lm_head_log_probs(h, w, y), (h, w), (up, up))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, off):
        out = fw.lm_head_log_probs(h, w, y)
        got = torch.autograd.grad(out, (h, w), (up, up))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_gradients_on_two_streams():
    """Two gradients of one retained graph at once, and another forward beside them."""
    g = R.gen(31)
    h = R.normal((600, 128), torch.bfloat16, g).requires_grad_(True)
    w = R.normal((4000, 128), torch.bfloat16, g, 0.2).requires_grad_(True)
    y = tokens_for(600, 4000, g, 0.1)
    up = torch.randn(600, device="cuda")
    out = fw.lm_head_log_probs(h, w, y)
    want = torch.autograd.grad(out, (h, w), (up, up), retain_graph=True)
    torch.cuda.synchronize()
    streams, held = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(4):
        for s in streams[:2]:
            with torch.cuda.stream(s):
                held.append(torch.autograd.grad(out, (h, w), (up, up), retain_graph=True))
        with torch.cuda.stream(streams[2]):
            again = fw.lm_head_log_probs(h, w, y)
    torch.cuda.synchronize()
    for got in held:
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    for a, b in zip(again, out):
        assert torch.equal(a.detach(), b.detach())


def test_refusals():
    h, w = torch.zeros(4, 8, device="cuda", dtype=torch.bfloat16), torch.zeros(9, 8, device="cuda", dtype=torch.bfloat16)
    y = torch.zeros(4, dtype=torch.int64, device="cuda")
    f = fw.lm_head_log_probs
    for bad in ((h.float(), w.float(), y), (h.half(), w, y), (h.cpu(), w, y), (h[0], w, y), (h, w, y.int()), (h, w[:0], y)):
        with pytest.raises(TypeError):
            f(*bad)
    for bad in ((h[:, :7], w, y), (h, w, y[:3]), (h, w, y.cpu()), (h, w, y[:, None])):
        with pytest.raises(ValueError):
            f(*bad)
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-40):
        with pytest.raises(ValueError):
            f(h, w, y, temperature=t)


def test_streams_and_graphs():
    g = R.gen(10)
    h = R.normal((200, 64), torch.bfloat16, g).requires_grad_(True)
    w = R.normal((1000, 64), torch.bfloat16, g, 0.3).requires_grad_(True)
    y = tokens_for(200, 1000, g, 0.1)
    a, b = torch.randn(200, device="cuda"), torch.randn(200, device="cuda")

    def step():
        out = fw.lm_head_log_probs(h, w, y, temperature=0.8)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, (h, w), (a, b))]

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, held = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            held.append(step())
    for seed in (1, 2):
        with torch.no_grad():
            h.copy_(R.normal((200, 64), torch.bfloat16, R.gen(seed)))
        y.copy_(tokens_for(200, 1000, R.gen(seed + 9), 0.3))
        for graph in graphs:
            graph.replay()
        want = step()
        for captured in held:
            for p, q in zip(captured, want):
                assert torch.equal(p, q)


@pytest.mark.parametrize("B,D,V", [(600, 520, 3000), (64, 512, 20000), (33000, 64, 10007)])
def test_waits_that_gave_up_leave_nan(B, D, V):
    """In one piece; dhidden in splits; several pieces of the vocabulary."""
    lib, g = capi.load(), R.gen(B)
    h, w = R.normal((B, D), torch.bfloat16, g), R.normal((V, D), torch.bfloat16, g, 0.1)
    y = tokens_for(B, V, g)
    y[::5] = -100
    a, b = (torch.rand(B, generator=g, device="cuda") + 0.5 for _ in range(2))
    ns = lib.fw_lm_head_log_probs_state(B, D, V, ctypes.c_void_p(w.data_ptr()), D)
    nf, nb = (lib.fw_lm_head_log_probs_workspace(B, D, V, i) for i in (0, 1))
    state, ws = torch.zeros(ns, dtype=torch.uint8, device="cuda"), torch.zeros(max(nf, nb), dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    out = torch.empty(2, B, device="cuda")

    def forward(to, state):
        assert lib.fw_lm_head_log_probs(1, h.data_ptr(), D, w.data_ptr(), D, y.data_ptr(), B, D, V, 1.0, -100, to[0].data_ptr(),
                                        to[1].data_ptr(), state.data_ptr(), ns, ws.data_ptr(), nf, None, st) == 0

    def gradients():
        ws.zero_()
        dh, dw = torch.full_like(h, 12345.0), torch.full_like(w, 12345.0)
        assert lib.fw_lm_head_log_probs_grad(1, w.data_ptr(), D, B, D, V, 1.0, a.data_ptr(), b.data_ptr(), state.data_ptr(), ns,
                                             ws.data_ptr(), nb, dh.data_ptr(), dw.data_ptr(), None, st) == 0
        return dh, dw

    forward(out, state)
    want = gradients()
    lost = torch.full((2, B), 12345.0, device="cuda")
    with giving_up():
        forward(lost, torch.zeros_like(state))
        got = gradients()
        torch.cuda.synchronize()
    live = y != -100
    assert lost[:, live].isnan().all() and not lost[:, ~live].any()
    for x, ref in zip(got, want):
        unwritten = torch.full((), 12345.0, dtype=x.dtype, device="cuda")
        gone = x.isnan()
        assert gone.any() and not (x == unwritten).any() and torch.equal(x[~gone], ref[~gone])
    assert not got[0][::5].any()
    for x, ref in zip(gradients(), want):
        assert torch.equal(x, ref)

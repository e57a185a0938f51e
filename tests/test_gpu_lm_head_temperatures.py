"""Log probabilities of an output layer at low temperatures: rows whose
probabilities are 1, or 1 / 2 twice, whatever the temperature, so that the
gradients are known without the logits.

The winning logit is near 50 and 40 ahead; equal rows of the weight give equal
logits, and every exponential's argument is then 0 or under -40.  The other
columns, taken for 0 here, have probabilities p under exp(-40) < 2^-57, and
entries of the logit gradient under p (|a| + |b| |log p|), where p |log p| is at
most 40 exp(-40) < 2^-52: within 2^-50 of their row's factors.  A
probability's error is that of the logarithm of 1 or 2, of its product with
log2(e) and of the hardware's exponential, 2^-22 + 3 * E32 < 2^-20, whatever
the temperature; l + h cancels within 2 * E32.  What is rounded to the operands'
type are powers of two times 1 or 1 / 2, so that rounding gives no more than that
error again: an entry of the logit gradient is within 2^-19 of its row's factors.
Sums over columns and rows: each step of 16 may truncate by an ulp.  From T = 0.5
on the gradient's own logits may be off from the forward's by d = 2 * D / 16
such ulps over T, hence p and l by 5 / 4 d (exp(d) - 1, d < 1 / 8), and entries
other than the label's are then rounded.
"""
import math

import pytest
import torch

import fwloss_b200 as fw
import lm_ref as R
from test_gpu_lm_head_log_probs import check, tokens_for
from test_gpu_lm_waits import giving_up

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]
D, V, B = 2048, 700, 96


def case(dtype, temperature, seed=0):
    """h, w, tokens, upstream factors, probabilities; the first column of w is 1 / 2 and of h 0, so that the first
    column of dhidden is half the sum of the logit gradient's row"""
    g = R.gen(seed + 40)
    w = R.normal((V, D), dtype, g, (50 / D) ** 0.5)
    w[300:332] = w[:32]
    w[:, 0] = 0.5
    top = torch.cat([torch.arange(100, 148), torch.arange(0, 32), torch.arange(300, 316)]).cuda()
    h = w[top].clone()
    h[:, 0] = 0.0
    y = top.clone()
    y[32:48] = torch.arange(400, 416).cuda()  # a token without probability
    y[60:70] = top[60:70] + 300  # the other one of the two
    p = torch.zeros(B, V, dtype=torch.float64, device="cuda")
    rows = torch.arange(B, device="cuda")
    p[rows, top] = 1.0
    for r in range(48, B):
        p[r, [int(top[r]) % 300, int(top[r]) % 300 + 300]] = 0.5
    scale = 2.0 ** math.floor(math.log2(temperature)) if temperature > 1e-10 else 2.0 ** -112
    a, b = (torch.randint(0, 2, (2, B), generator=g, device="cuda") * 2.0 - 1) * \
        2.0 ** torch.randint(-2, 3, (2, B), generator=g, device="cuda") * scale
    return h, w, y, a, b, p


def compare(got, want, error, terms, steps, dtype, what):
    R.within(got, want, error + 2 * steps * R.E32 * terms + R.rounded(want, dtype) * (1 + 2.0 ** -7), what)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1.0, 0.5, 0.49, 0.1, 0.01, 1e-3, 1e-4, 1e-37])
def test_rows_that_are_sure(temperature, dtype):
    """1e-37: the winning logit over the temperature is past fp32's largest number."""
    h, w, y, a, b, p = case(dtype, temperature)
    h.requires_grad_(True), w.requires_grad_(True)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    logp, entropy = fw.lm_head_log_probs(h, w, y, temperature=temperature, status=status)
    at = p.gather(1, y[:, None])[:, 0]
    R.within(entropy, -(p * p.clamp(min=1e-300).log()).sum(1), 2.0 ** -20, "entropy")
    R.within(logp[at > 0], at[at > 0].log(), 2.0 ** -20, "logp")
    assert (logp[at == 0] < -30 / temperature).all()
    dh, dw = torch.autograd.grad((logp, entropy), (h, w), (a, b))
    assert int(status) == 0
    wd, hd, f = w.detach().double(), h.detach().double(), (a.double() / temperature)[:, None]
    G = (torch.zeros_like(p).scatter_(1, y[:, None], 1.0) - p) * f  # the entropy's share is 0
    hot = (p > 0).double().scatter_(1, y[:, None], 1.0)
    e_p = hot * 2.0 ** -19 + 2.0 ** -50
    if temperature >= 0.5:
        e_p = e_p + hot * 1.25 * 2 * D / 16 * R.E32 * (hd.abs() @ wd.abs().t()) / temperature
        e_p = e_p + R.U[dtype] * hot.scatter(1, y[:, None], 0.0)
    e_g = e_p * ((a.abs() + b.abs()).double() / temperature)[:, None]
    compare(dh, G @ wd, e_g @ wd.abs(), G.abs() @ wd.abs(), V / 16, dtype, "dhidden")
    compare(dw, G.t() @ hd, e_g.t() @ hd.abs(), G.abs().t() @ hd.abs(), B / 16, dtype, "dweight")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,vocab", [(1, 1, 1), (3, 7, 5), (37, 65, 129), (300, 520, 3001), (257, 1000, 5001), (64, 512, 20000),
                                            (1000, 72, 4099)])
def test_values_and_gradients(rows, dim, vocab, dtype):
    """Every path of the gradient at low temperatures, against the 64-bit definition."""
    g = R.gen(rows + dim)
    h, w = R.normal((rows, dim), dtype, g), R.normal((vocab, dim), dtype, g, dim ** -0.5)
    y = tokens_for(rows, vocab, g, 0.2 if rows > 2 else 0.0)
    check(h, w, y, temperature=0.3)
    check(h, w, y, temperature=0.07, kind="logp", scale=1e-3)
    check(h, w, y, temperature=0.4, kind="entropy", scale=30.0)


@pytest.mark.parametrize("temperature", [0.25, 0.75])
def test_waits_that_gave_up_leave_nan(temperature):
    g = R.gen(50)
    h, w = R.normal((600, 520), torch.bfloat16, g), R.normal((3000, 520), torch.bfloat16, g, 0.05)
    y = tokens_for(600, 3000, g, 0.2)
    h.requires_grad_(True), w.requires_grad_(True)
    out = fw.lm_head_log_probs(h, w, y, temperature=temperature)
    up = (torch.ones(600, device="cuda"),) * 2
    want = torch.autograd.grad(out, (h, w), up, retain_graph=True)
    with giving_up():
        got = torch.autograd.grad(out, (h, w), up, retain_graph=True)
        torch.cuda.synchronize()
    for x, ref in zip(got, want):
        gone = x.isnan()
        assert gone.any() and torch.equal(x[~gone], ref[~gone])
    assert not got[0][y == -100].any()
    for x, ref in zip(torch.autograd.grad(out, (h, w), up), want):
        assert torch.equal(x, ref)


def test_graphs_of_both_forms():
    """Steps on either side of T = 0.5 captured one after the other and replayed on new rows."""
    g = R.gen(60)
    h = R.normal((300, 600), torch.bfloat16, g).requires_grad_(True)
    w = R.normal((1000, 600), torch.bfloat16, g, 0.1).requires_grad_(True)
    y = tokens_for(300, 1000, g, 0.1)
    a, b = torch.randn(300, generator=g, device="cuda"), torch.randn(300, generator=g, device="cuda")

    def step(temperature):
        out = fw.lm_head_log_probs(h, w, y, temperature=temperature)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, (h, w), (a, b))]

    temperatures = (0.5, 0.2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(1.0)
    torch.cuda.current_stream().wait_stream(side)
    graphs, held = [torch.cuda.CUDAGraph() for _ in temperatures], []
    for graph, t in zip(graphs, temperatures):
        with torch.cuda.graph(graph):
            held.append(step(t))
    for seed in (1, 2):
        with torch.no_grad():
            h.copy_(R.normal((300, 600), torch.bfloat16, R.gen(seed)))
        y.copy_(tokens_for(300, 1000, R.gen(seed + 9), 0.3))
        for graph in graphs:
            graph.replay()
        for t, captured in zip(temperatures, held):
            for p, q in zip(captured, step(t)):
                assert torch.equal(p, q)

"""What the scoring and clipping operators compute on another stream than the
current one, and with a norm that is given, compared value by value."""
import pytest
import torch

import fwloss_b200 as fw
import lm_ref as R
from test_gpu_lm_head_log_probs import tokens_for

pytestmark = pytest.mark.gpu


def on_side_streams(step, runs=3):
    """Results of `step` on two streams at once, each run's own."""
    streams, held = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(runs):
        for s in streams:
            with torch.cuda.stream(s):
                held.append(step())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    return held


def equal(got, want):
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [200, 9000])
@pytest.mark.parametrize("temperature", [0.8, 0.2])
def test_output_layer(temperature, rows, dtype):
    g = R.gen(rows)
    h = R.normal((rows, 64), dtype, g).requires_grad_(True)
    w = R.normal((1000, 64), dtype, g, 0.3).requires_grad_(True)
    y = tokens_for(rows, 1000, g, 0.1)
    a, b = torch.randn(rows, generator=g, device="cuda"), torch.randn(rows, generator=g, device="cuda")

    def step():
        out = fw.lm_head_log_probs(h, w, y, temperature=temperature)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, (h, w), (a, b))]

    want = step()
    for got in on_side_streams(step):
        equal(got, want)


@pytest.mark.parametrize("top_k", [0, 7])
def test_logits(top_k):
    g = R.gen(3)
    z = R.normal((48, 40000), torch.bfloat16, g, 2.0).requires_grad_(True)
    y = tokens_for(48, 40000, g, 0.1)
    a, b = torch.randn(48, generator=g, device="cuda"), torch.randn(48, generator=g, device="cuda")

    def step():
        out = fw.token_log_probs(z, y, top_k=top_k, temperature=0.8)
        return [*(t.detach() for t in out), *torch.autograd.grad(out[:2], z, (a, b))]

    want = step()
    for got in on_side_streams(step):
        equal(got, want)


def test_clipping():
    g = R.gen(5)
    grads = [R.normal((s,), t, g) for s, t in ((70001, torch.bfloat16), (33, torch.float32), (9000, torch.float16), (0, torch.float32))]
    grads.append(R.normal((100, 90), torch.float32, g)[:, 3:70])

    def step():
        out = [torch.full_like(x, 9.0, dtype=torch.float32) for x in grads]
        return [fw.clip_grad_norm_(grads, 3.0, out=out), *out]

    def inplace():
        mine = [x.clone() for x in grads]
        return [fw.clip_grad_norm_(mine, 3.0), *mine]

    for f in (step, inplace):
        want = f()
        assert float(want[0]) > 100.0
        for got in on_side_streams(f):
            equal(got, want)


def test_a_given_norm():
    """The factor is max_norm over fp32's rounding of the norm instead of over the norm: another E32, and the factor's
    own rounding differs by as much again; the products are rounded on either side of that."""
    g = R.gen(7)
    grads = [R.normal((s,), t, g) for s, t in ((300001, torch.bfloat16), (17, torch.float32), (40000, torch.float16))]
    outs = [[torch.full_like(x, 9.0) for x in grads] for _ in range(2)]
    norm = fw.clip_grad_norm_(grads, 2.0, out=outs[0])
    given = fw.clip_grad_norm_(grads, 2.0, out=outs[1], norm=norm)
    assert given.data_ptr() == norm.data_ptr() and torch.equal(given, fw.grad_norm(grads))
    for x, y in zip(*outs):
        want = x.double()
        R.within(y, want, want.abs() * 4 * R.E32 + 2 * R.rounded(want, x.dtype))
    mine = [x.clone() for x in grads]
    fw.clip_grad_norm_(mine, 2.0, norm=norm)
    equal(mine, outs[1])
    for f in (0.5, 4.0):  # norms that are not the tensors' own: scaled by half, and left as they are
        mine = [x.clone() for x in grads]
        fw.clip_grad_norm_(mine, 2.0, norm=torch.full((1,), 2.0 / f, device="cuda"))
        for x, b in zip(mine, grads):
            assert torch.equal(x, (b.float() * min(f, 1.0)).to(b.dtype))


def test_a_limit_of_infinity():
    """Nothing is scaled, whatever the norm; NaN stays NaN everywhere."""
    x = torch.ones(5000, device="cuda")
    x[7] = float("inf")
    before = x.clone()
    assert float(fw.clip_grad_norm_([x], float("inf"))) == float("inf") and torch.equal(x, before)
    x[9] = float("nan")
    assert fw.clip_grad_norm_([x], float("inf")).isnan() and x.isnan().all()

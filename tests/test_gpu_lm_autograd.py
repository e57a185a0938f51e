"""What the language-model operators' autograd nodes promise beyond values:
second derivatives refused, status words that may be cleared, in-place changes
of saved operands noticed, graph capture, saved-tensor hooks."""
import pytest
import torch

import fwloss_b200 as fw
import lm_ref as R

pytestmark = pytest.mark.gpu


def operands(seed=0):
    g = R.gen(seed)
    h = R.normal((100, 64), torch.bfloat16, g).requires_grad_(True)
    w = R.normal((300, 64), torch.bfloat16, g, 0.3).requires_grad_(True)
    y = torch.randint(0, 300, (100,), generator=g, device="cuda")
    gain = torch.ones(64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    return h, w, y, gain


def losses(h, w, y, gain):
    return {"embed": lambda: fw.embed_tokens(y, w).float().sum(), "norm": lambda: fw.rms_norm(h, gain).float().sum(),
            "xent": lambda: fw.lm_head_cross_entropy(h, w, y)}


@pytest.mark.parametrize("name,at", [("embed", 1), ("norm", 0), ("xent", 0)])
def test_second_derivatives_are_refused(name, at):
    ops = operands()
    (g,) = torch.autograd.grad(losses(*ops)[name](), ops[at], create_graph=True)
    with pytest.raises(RuntimeError, match="again"):
        g.float().sum().backward()


def test_status_may_be_cleared_before_backward():
    h, w, y, _ = operands()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y[3] = 300
    loss = fw.lm_head_cross_entropy(h, w, y, status=status)
    out = fw.embed_tokens(y, w, status=status)
    assert int(status) == 1
    status.zero_()
    torch.autograd.grad(loss, (h, w))
    torch.autograd.grad(out, w, torch.ones_like(out))
    assert int(status) == 1  # the embedding's backward meets the token again


def test_changed_operands_are_noticed():
    h, w, y, gain = operands()
    loss = fw.lm_head_cross_entropy(h, w, y)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    r = R.normal((100, 64), torch.bfloat16, R.gen(4))
    out, stream = fw.rms_norm(h, gain, residual=r)
    with torch.no_grad():
        stream.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.float().sum().backward()


def test_hidden_may_change_after_the_forward():
    """The packed rows are the operator's own."""
    h, w, y, _ = operands()
    want = torch.autograd.grad(fw.lm_head_cross_entropy(h, w, y), (h, w))
    loss = fw.lm_head_cross_entropy(h, w, y)
    with torch.no_grad():
        h.zero_()
    for got, ref in zip(torch.autograd.grad(loss, (h, w)), want):
        assert torch.equal(got, ref)


def test_saved_tensors_on_the_host():
    h, w, y, gain = operands()
    for name, f in losses(h, w, y, gain).items():
        want = torch.autograd.grad(f(), (h, w, gain), allow_unused=True)
        with torch.autograd.graph.save_on_cpu():
            loss = f()
        for got, ref in zip(torch.autograd.grad(loss, (h, w, gain), allow_unused=True), want):
            assert (got is None and ref is None) or torch.equal(got, ref), name


def test_a_step_in_a_cuda_graph():
    g = R.gen(9)
    table = R.normal((300, 64), torch.bfloat16, g, 0.3).requires_grad_(True)
    gain = torch.ones(64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    ids, y = (torch.randint(0, 300, (500,), generator=g, device="cuda") for _ in range(2))

    def step():
        x = fw.embed_tokens(ids, table, scale=2.0)
        out, _ = fw.rms_norm(x, gain, residual=x)
        loss = fw.lm_head_cross_entropy(out, table, y)
        return [loss, *torch.autograd.grad(loss, (table, gain))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2):
        ids.copy_(torch.randint(0, 300, (500,), generator=R.gen(seed), device="cuda"))
        y.copy_(torch.randint(0, 300, (500,), generator=R.gen(seed + 5), device="cuda"))
        graph.replay()
        for got, ref in zip(captured, step()):
            assert torch.equal(got, ref)


def test_serving_step_in_a_cuda_graph():
    g = R.gen(3)
    x, r = R.normal((5, 96), torch.bfloat16, g), R.normal((5, 96), torch.bfloat16, g)
    gain = torch.ones(96, dtype=torch.bfloat16, device="cuda")
    wq, ws = fw.quantize_rows_int8(R.normal((1000, 96), torch.bfloat16, g))

    def step():
        q, s, total = fw.rms_norm_int8(x, gain, residual=r)
        return fw.int8_linear(q, s, wq, ws), total

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    x.copy_(R.normal((5, 96), torch.bfloat16, R.gen(8)))
    graph.replay()
    for got, ref in zip(captured, step()):
        assert torch.equal(got, ref)

"""Log probabilities, entropies, alternatives and their gradient from logits,
against the 64-bit definition."""
import pytest
import torch

import fwloss_b200 as fw
import lm_ref as R
import score_ref as S

pytestmark = pytest.mark.gpu

NEG = float("-inf")


def check(logits, tokens, k=0, temperature=1.0, ignore=-100, grads=("both",), seed=0):
    """forward with alternatives, and the gradient for the upstream factors named"""
    V = logits.shape[1]
    z = logits.double()
    r = S.rows(z, tokens, temperature, ignore)
    plain = fw.token_log_probs(logits, tokens, top_k=k, temperature=temperature, ignore_index=ignore)
    got = list(plain)
    assert got[0].dtype == torch.float32 and len(got) == (4 if k else 2)
    # a token that has probability 0: -inf
    fin = torch.isfinite(r["logp"]) | torch.isnan(r["logp"])
    assert torch.equal(got[0][~fin].double(), r["logp"][~fin])
    R.within(got[0][fin], r["logp"][fin], r["e_logp"][fin], "logp")
    R.within(got[1], r["entropy"], r["e_entropy"], "entropy")
    if k:
        value, ids, bound = S.top(z, r, k)
        assert torch.equal(got[3], ids)
        fin = torch.isfinite(value) | torch.isnan(value)
        assert torch.equal(got[2][~fin].double(), value[~fin])
        R.within(got[2][fin], value[fin], bound[fin], "top")
    g = R.gen(seed + 77)
    for kind in grads:
        x = logits.detach().requires_grad_(True)
        out = fw.token_log_probs(x, tokens, top_k=k, temperature=temperature, ignore_index=ignore)
        for a, b in zip(out, plain):  # recording changes no result
            assert torch.equal(torch.nan_to_num(a.detach(), nan=7.0), torch.nan_to_num(b, nan=7.0))
        a, b = (torch.randn(len(tokens), generator=g, device="cuda") for _ in range(2))
        if kind == "both":
            (d,) = torch.autograd.grad(out[:2], x, (a, b))
        elif kind == "logp":
            (d,) = torch.autograd.grad(out[0], x, a)
        else:
            (d,) = torch.autograd.grad(out[1], x, b)
        want, bound = S.logit_grad(r, a if kind != "entropy" else None, b if kind != "logp" else None)
        assert d.shape == logits.shape and d.dtype == logits.dtype
        R.within(d, want, S.grad_bound(want, bound, logits.dtype), f"gradient of {kind}")
    return plain


def tokens_for(B, V, g, ignored=0.0):
    y = torch.randint(0, V, (B,), generator=g, device="cuda")
    return torch.where(torch.rand(B, generator=g, device="cuda") < ignored, torch.full_like(y, -100), y)


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 7), (9, 8), (70, 33), (300, 257), (33, 1000), (600, 1025), (17, 2051),
                                 (64, 5001), (9, 8192), (5, 16385), (3, 50257), (1, 32000), (2, 128256), (1, 262147)])
def test_values_and_gradients(B, V, dtype):
    g = R.gen(B + V)
    z = R.normal((B, V), dtype, g, 3.0)
    check(z, tokens_for(B, V, g, 0.2), k=min(V, 5), temperature=0.7, grads=("both", "logp", "entropy"))


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("V", [40, 1000, 5001, 40000])
@pytest.mark.parametrize("k", [1, 2, 20, 31, 32])
def test_alternatives(V, k, dtype):
    g = R.gen(V + k)
    z = R.normal((13, V), dtype, g, 2.0)
    check(z, tokens_for(13, V, g), k=k, grads=())


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("V", [64, 1001, 4096, 33333, 100000])
def test_ties_go_to_the_lowest_column(V, dtype):
    g = R.gen(V)
    z = torch.randint(-3, 4, (12, V), generator=g, device="cuda").to(dtype)
    z[0] = 0
    z[1] = -5
    z[2, : V // 2] = -0.0  # equal to 0
    z[2, V // 2:] = 0.0
    z[3, :-1] = NEG
    z[4, ::2] = NEG
    z[5] = torch.finfo(dtype).min
    z[6, V // 3:] = torch.finfo(dtype).min
    z[7] = torch.finfo(dtype).max
    z[8, 5:] = NEG
    check(z, torch.full((12,), 0, device="cuda"), k=32, grads=("both",))
    check(z, torch.full((12,), V - 1, device="cuda"), k=1, grads=("both",), temperature=2.0)


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("V", [1024, 16384, 131072])
@pytest.mark.parametrize("threads", [32, 128, 256, 2048])
def test_the_largest_lie_with_one_thread(V, threads, dtype):
    """Rising columns, and rows whose largest values lie in the slots that one
    thread of `threads` reads."""
    n = 128 // torch.finfo(dtype).bits
    e = torch.arange(V, device="cuda")
    rising = (e.float() * (20.0 / V)).to(dtype)
    mine = (e // n) % threads == 5 % threads
    z = torch.stack([rising, rising.flip(0), torch.where(mine, rising + 25, rising), torch.where(mine, rising.flip(0) + 25, rising),
                     torch.where(mine, torch.full_like(rising, 30), rising)])
    check(z, torch.tensor([0, 1, 2, 3, V - 1], device="cuda"), k=32, grads=("both",))


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("V", [1000, 1003, 9001])
@pytest.mark.parametrize("pad", [0, 1, 3, 8])
@pytest.mark.parametrize("start", [0, 1, 5])
def test_rows_anywhere(V, pad, start, dtype):
    """Rows that start off 16-byte boundaries, in wider matrices whose other columns are NaN."""
    g = R.gen(V + pad)
    store = torch.full((7 * (V + pad) + start + 64,), float("nan"), dtype=dtype, device="cuda")
    z = store[start: start + 7 * (V + pad)].view(7, V + pad)[:, :V]
    z.copy_(R.normal((7, V), dtype, g, 2.0))
    check(z, tokens_for(7, V, g, 0.1), k=4)


def test_column_strides_and_broadcast_rows():
    g = R.gen(4)
    z = R.normal((300, 50), torch.float32, g)
    y = tokens_for(50, 300, g)
    check(z.t(), y, k=3)
    check(R.normal((1, 300), torch.float32, g).expand(50, 300), y, k=3)
    check(z[::2, ::2], tokens_for(150, 25, g), k=3)


def test_leading_shapes():
    g = R.gen(5)
    z, y = R.normal((4, 6, 99), torch.bfloat16, g).requires_grad_(True), torch.randint(0, 99, (4, 6), generator=g, device="cuda")
    out = fw.token_log_probs(z, y, top_k=2)
    flat = fw.token_log_probs(z.reshape(24, 99), y.reshape(24), top_k=2)
    assert [tuple(t.shape) for t in out] == [(4, 6), (4, 6), (4, 6, 2), (4, 6, 2)]
    for a, b in zip(out, flat):
        assert torch.equal(a.reshape(b.shape), b)
    up = torch.randn(4, 6, device="cuda")
    (d,) = torch.autograd.grad(out[0], z, up)
    assert torch.equal(d.reshape(24, 99), torch.autograd.grad(flat[0], z, up.reshape(24))[0].reshape(24, 99))
    one = fw.token_log_probs(z[1, 2], y[1, 2])
    assert one[0].shape == () and torch.equal(one[0], out[0][1, 2]) and torch.equal(one[1], out[1][1, 2])
    x = torch.zeros(0, 9, device="cuda", requires_grad=True)
    none = fw.token_log_probs(x, torch.zeros(0, dtype=torch.int64, device="cuda"), 3)
    assert [tuple(t.shape) for t in none] == [(0,), (0,), (0, 3), (0, 3)]
    assert torch.autograd.grad(none[0].sum(), x)[0].shape == (0, 9)


@pytest.mark.parametrize("dtype", R.FLOATS)
def test_rows_that_are_not_finite(dtype):
    g = R.gen(6)
    z = R.normal((9, 777), dtype, g)
    z[0, 5] = float("nan")
    z[1, 700] = float("inf")
    z[2] = NEG
    z[3, 6] = NEG  # its token: logp -inf, everything else finite
    z[4, 3], z[4, 4] = float("nan"), float("inf")
    z[5] = float("nan")  # ignored
    y = torch.tensor([5, 6, 7, 6, 0, -100, 777, -1, 3], device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(z, y, k=5, grads=("both", "entropy"))
    fw.token_log_probs(z, y, status=status)
    assert int(status) == 3
    status.zero_()
    fw.token_log_probs(z[3:4], y[3:4], status=status)
    fw.token_log_probs(z[5:6], y[5:6], status=status)
    assert int(status) == 0
    out = fw.token_log_probs(z, y)
    assert float(out[0][3]) == NEG and bool(torch.isfinite(out[1][3]))


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("V", [40000, 9000, 2100])
def test_bad_rows_of_few_long_ones(V, dtype):
    """Rows split over CTAs: every alternative of a bad one is written, whatever was there."""
    g = R.gen(V)
    z = R.normal((7, V), dtype, g)
    z[0, V // 2], z[1, 0], z[2] = float("nan"), float("inf"), NEG
    z[3, :] = float("nan")
    z[4, 20:] = NEG  # fewer than 32 columns left
    y = torch.tensor([0, 1, 2, 3, 5, -100, V], device="cuda")
    for _ in range(3):
        torch.full((7, 32), 777, dtype=torch.int64, device="cuda")  # what freed memory holds
        torch.full((7, 32), 777.0, device="cuda")
        check(z, y, k=32, grads=("both",))


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("B,V", [(9, 900), (9, 5001), (5, 40000), (700, 9001), (2400, 3500)])
def test_masks(B, V, dtype):
    """Most columns of one value: -inf, the type's lowest, one between the others; few or many columns above it."""
    g = R.gen(B + V)
    rows = []
    for i in range(9):
        z = R.normal((V,), dtype, g, 2.0)
        mask = (NEG, torch.finfo(dtype).min, -1.0)[i % 3]
        keep = torch.rand(V, generator=g, device="cuda") < (3 / V, 40 / V, 0.3)[i // 3]
        keep[int(torch.randint(0, V, (1,), generator=g, device="cuda"))] = True
        rows.append(torch.where(keep, z, torch.full_like(z, mask)))
    rows[0][: V // 2] = -50.0  # the mask begins late
    z = torch.stack([rows[i % 9] for i in range(B)])
    y = z.argmax(1)
    for k in (1, 5, 32):
        check(z, y, k=k, grads=("both",) if k == 5 else ())


def test_offsets_past_2_31_elements():
    if torch.cuda.get_device_properties(0).total_memory < 60e9:
        pytest.skip("needs 20 GB of device memory")
    B, V, last = 17000, 131072, 7
    z = torch.zeros(B, V, dtype=torch.bfloat16, device="cuda")
    tail = R.normal((last, V), torch.bfloat16, R.gen(2), 2.0)
    z[-last:] = tail
    y = torch.full((B,), -100, device="cuda")
    y[-last:] = tokens_for(last, V, R.gen(3))
    x, xt = z.requires_grad_(True), tail.clone().requires_grad_(True)
    up = torch.ones(B, device="cuda")
    out, ref = fw.token_log_probs(x, y, top_k=4), fw.token_log_probs(xt, y[-last:], top_k=4)
    bound = S.rows(tail.double(), y[-last:], 1.0)
    for i, e in ((0, "e_logp"), (1, "e_entropy")):  # few rows take another way through them
        R.within(out[i][-last:], ref[i].double(), 2 * bound[e])
    assert torch.equal(out[3][-last:], ref[3])
    (d,) = torch.autograd.grad(out[0], x, up)
    want, e = S.logit_grad(bound, up[-last:])
    R.within(d[-last:], want, S.grad_bound(want, e, torch.bfloat16))
    assert not d[: 100].any() and not d[B // 2: B // 2 + 100].any()


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("temperature", [1e-3, 0.25, 3.0, 1e4])
def test_temperature_and_far_logits(temperature, dtype):
    g = R.gen(8)
    z = R.normal((20, 3001), dtype, g, 4.0)
    z[:5] += 1000.0
    if dtype != torch.float16:
        z[5:8] *= 1e30
    check(z, tokens_for(20, 3001, g), k=6, temperature=temperature)


def test_gradient_against_differences():
    """Central differences of the operator itself; their error is the values'
    (e_logp, e_entropy) over the step and the third derivative's part."""
    g = R.gen(10)
    z = R.normal((4, 37), torch.float32, g, 1.5).requires_grad_(True)
    y = tokens_for(4, 37, g)
    logp, entropy = fw.token_log_probs(z, y, temperature=0.8)
    a, b = torch.randn(4, device="cuda"), torch.randn(4, device="cuda")
    (d,) = torch.autograd.grad((logp, entropy), z, (a, b))
    r = S.rows(z.detach().double(), y, 0.8)
    step = 2.0 ** -6
    for j in (0, 5, 36):
        vals = []
        for sign in (1, -1):
            x = z.detach().clone()
            x[:, j] += sign * step
            l, e = fw.token_log_probs(x, y, temperature=0.8)
            vals.append(a.double() * l.double() + b.double() * e.double())
        off = (2 * (a.abs() * r["e_logp"] + b.abs() * r["e_entropy"])) / (2 * step)
        # third derivatives of log softmax and entropy in one logit are under 1 and 8 (1 + H) in units of 1 / T^3
        third = (a.abs() + b.abs() * 8 * (1 + r["h"])) / 0.8 ** 3 * step ** 2 / 6
        R.within(d[:, j], (vals[0] - vals[1]) / (2 * step), off + third + 1e-6, f"column {j}")


def test_state_outlives_changes_of_tokens_and_results():
    g = R.gen(11)
    z = R.normal((40, 500), torch.float32, g).requires_grad_(True)
    y = tokens_for(40, 500, g, 0.2)
    up = torch.randn(40, device="cuda")

    def grads(change):
        t = y.clone()
        out = fw.token_log_probs(z, t)
        loss = (out[0] * up + 0.1 * out[1]).sum()
        if change:
            t.zero_()
            with torch.no_grad():
                out[1].detach().zero_()
        return torch.autograd.grad(loss, z)[0]

    assert torch.equal(grads(False), grads(True))
    x = z.detach().clone().requires_grad_(True)
    out = fw.token_log_probs(x, y)
    with torch.no_grad():
        x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out[0].sum().backward()
    with torch.autograd.graph.save_on_cpu():
        out = fw.token_log_probs(z, y)
    want = torch.autograd.grad(fw.token_log_probs(z, y)[0], z, up)[0]
    assert torch.equal(torch.autograd.grad(out[0], z, up)[0], want)


def test_nodes_refuse_second_derivatives_and_tangents():
    z = torch.randn(4, 30, device="cuda", requires_grad=True)
    y = torch.zeros(4, dtype=torch.int64, device="cuda")
    out = fw.token_log_probs(z, y, top_k=2)
    assert not out[2].requires_grad and not out[3].requires_grad
    (d,) = torch.autograd.grad(out[0].sum() + out[1].sum(), z, create_graph=True)
    with pytest.raises(RuntimeError, match="again"):
        d.sum().backward()
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level(), pytest.raises(NotImplementedError):
        fw.token_log_probs(fwd.make_dual(z.detach(), torch.ones_like(z)), y)


def test_refusals():
    z, y = torch.zeros(4, 30, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    f = fw.token_log_probs
    for bad in ((z.double(), y), (z.long(), y), (z, y.int()), (z.cpu(), y)):
        with pytest.raises(TypeError):
            f(*bad)
    for bad in ((z, y[:3]), (z, y.cpu()), (z, y[:, None]), (z[0], y)):
        with pytest.raises(ValueError):
            f(*bad)
    for kw in ({"top_k": 33}, {"top_k": -1}, {"top_k": 31}, {"temperature": 0.0}, {"temperature": -1.0},
               {"temperature": float("nan")}, {"temperature": float("inf")}, {"temperature": 1e-40}, {"temperature": 3.2e-39}):
        with pytest.raises(ValueError):
            f(z, y, **kw)
    with pytest.raises(RuntimeError):
        f(z, y, status=torch.zeros(1, device="cuda"))


def test_streams_and_graphs():
    g = R.gen(12)
    z = R.normal((50, 4000), torch.bfloat16, g).requires_grad_(True)
    y = tokens_for(50, 4000, g, 0.1)
    a, b = torch.randn(50, device="cuda"), torch.randn(50, device="cuda")

    def step():
        out = fw.token_log_probs(z, y, top_k=7, temperature=0.9)
        return [*(t.detach() for t in out), *torch.autograd.grad(out[:2], z, (a, b))]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            other = step()
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(want, other):
        assert torch.equal(p, q)
    graphs, held = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            held.append(step())
    for seed in (1, 2):
        with torch.no_grad():
            z.copy_(R.normal((50, 4000), torch.bfloat16, R.gen(seed)))
        y.copy_(tokens_for(50, 4000, R.gen(seed + 9), 0.3))
        for graph in graphs:
            graph.replay()
        want = step()
        for captured in held:
            for p, q in zip(captured, want):
                assert torch.equal(p, q)


def test_many_rows():
    """More rows than one grid dimension's old limit, and more units than the gradient's grid."""
    g = R.gen(13)
    z = R.normal((70001, 65), torch.float16, g)
    check(z, tokens_for(70001, 65, g, 0.1), k=3)

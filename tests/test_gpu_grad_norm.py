"""Global gradient norm and clipping against the 64-bit definition.

Tolerances: a thread adds 32 squares in fp32, each product and addition within
E32, so its sum is within 33 * E32; everything behind it is fp64 and the root
halves the relative error: 17 * E32, and one rounding to fp32.  A scaled value
is the factor (the norm's double, one rounding to fp32) times the element, two
roundings in fp32, and one to the result's type.
"""
import pytest
import torch

import fwloss_b200 as fw
import lm_ref as R

pytestmark = pytest.mark.gpu

E_NORM = 18 * R.E32
FACTOR = E_NORM + 3 * R.E32


def norm64(tensors):
    return torch.stack([t.double().square().sum() for t in tensors]).sum().sqrt()


def check_norm(got, want, extra=0.0):
    assert got.shape == () and got.dtype == torch.float32
    R.within(got, want, want.abs() * (E_NORM + R.E32 + extra), "norm")


def check(grads, ratio, out_types=None, make_out=None):
    want = norm64(grads)
    max_norm = float(want) * ratio
    factor = min(1.0, max_norm / float(want)) if float(want) > 0 else 1.0
    before = [g.clone() for g in grads]
    check_norm(fw.grad_norm(grads), want)
    if out_types is not None:
        out = make_out() if make_out else [torch.empty_like(g, dtype=t) for g, t in zip(grads, out_types)]
        check_norm(fw.clip_grad_norm_(grads, max_norm, out=out), want)
        for g, b in zip(grads, before):
            assert torch.equal(g, b)
    else:
        out = grads
        versions = [g._version for g in grads]
        check_norm(fw.clip_grad_norm_(grads, max_norm), want)
        assert all(g._version > v for g, v in zip(grads, versions))
        if ratio >= 1.0:
            for g, b in zip(grads, before):
                assert torch.equal(g, b)
    for o, b in zip(out, before):
        v = b.double() * factor
        R.within(o, v, v.abs() * FACTOR + R.rounded(v, o.dtype) * (1 + 2.0 ** -7) + 2.0 ** -149, "scaled")


SIZES = [1, 2, 3, 7, 8, 9, 255, 256, 257, 2048, 8191, 8192, 8193, 16385, 100003]


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("size", SIZES)
def test_one_tensor(size, dtype):
    g = R.gen(size)
    check([R.normal((size,), dtype, g, 1e-2)], 0.5)
    check([R.normal((size,), dtype, g, 1e-2)], 2.0)
    for to in R.FLOATS:
        check([R.normal((size,), dtype, g, 1e-2)], 0.3, [to])


@pytest.mark.parametrize("n", [2, 63, 64, 65, 511, 512, 513, 1200])
def test_many_tensors(n):
    g = R.gen(n)
    sizes = torch.randint(0, 700, (n,), generator=torch.Generator().manual_seed(n)).tolist()
    sizes[n // 2] = 70001

    def make():
        return [R.normal((s,), R.FLOATS[i % 3], g, 1e-2) for i, s in enumerate(sizes)]

    check(make(), 0.5)
    check(make(), 1.5)
    check(make(), 0.5, [R.FLOATS[(i // 2) % 3] for i in range(n)])
    check(make(), 3.0, [R.FLOATS[(i // 2) % 3] for i in range(n)])


@pytest.mark.parametrize("dtype", R.FLOATS)
@pytest.mark.parametrize("to", R.FLOATS)
@pytest.mark.parametrize("start", [0, 1, 2, 3, 5, 7])
def test_pieces_of_buckets(start, dtype, to):
    """Tensors behind one another at any element; what lies around them stays."""
    g, sizes = R.gen(start), [1, 5, 1000, 8192, 3, 20001, 4096]
    total = sum(sizes)
    pool = R.normal((start + total + 9,), dtype, g, 1e-2)
    store = torch.full((total + 2 * start + 20,), 77.0, dtype=to, device="cuda")
    grads, outs, at = [], [], start
    for s in sizes:
        grads.append(pool[at: at + s])
        outs.append(store[at + start: at + start + s])
        at += s
    check(grads, 0.5, [to] * len(sizes), lambda: outs)
    assert (store[: 2 * start] == 77.0).all() and (store[2 * start + total:] == 77.0).all()
    edge = pool.clone()
    check(grads, 0.5)
    assert torch.equal(pool[:start], edge[:start]) and torch.equal(pool[start + total:], edge[start + total:])


def test_layouts():
    g = R.gen(3)
    wide = R.normal((40, 130), torch.float32, g)
    rest = wide.clone()
    grads = [wide[:, :100], R.normal((30, 50), torch.bfloat16, g).t(), R.normal((4, 5, 6, 7), torch.float16, g).permute(3, 1, 0, 2),
             R.normal((), torch.float32, g), R.normal((3, 1, 5), torch.float32, g)]
    check(grads, 0.5)
    assert torch.equal(wide[:, 100:], rest[:, 100:])
    outs = [torch.empty(40, 100, device="cuda"), torch.empty(50, 30, device="cuda", dtype=torch.float16),
            torch.empty(8, 5, 4, 6, device="cuda")[:7], torch.empty((), device="cuda"), torch.empty(3, 2, 5, device="cuda")[:, :1]]
    check(grads, 0.5, [o.dtype for o in outs], lambda: outs)
    check_norm(fw.grad_norm(torch.ones(1, device="cuda").expand(50, 3)), torch.tensor(150.0, device="cuda", dtype=torch.float64).sqrt())


@pytest.mark.parametrize("scale", [1e-42, 1e-38, 1e-30, 1e-24, 1e-20, 1e-14, 1e15, 1e19, 1e30, 3e35])
def test_squares_outside_the_range(scale):
    """float32 values whose squares do not fit fp32, alone and beside ordinary ones."""
    g = R.gen(2)
    x = torch.rand(20000, generator=g, device="cuda") + 0.5
    small = [(x * scale).float()]
    check(small, 0.5)
    mixed = torch.rand(20000, generator=g, device="cuda")
    mixed[::1000] = scale
    check([mixed, (x * scale).float()], 0.5, [torch.float32] * 2)


def test_zeros_and_empty_tensors():
    z = [torch.zeros(9000, device="cuda"), torch.zeros(0, device="cuda", dtype=torch.bfloat16)]
    assert float(fw.grad_norm(z)) == 0.0
    assert float(fw.clip_grad_norm_(z, 0.0)) == 0.0 and not z[0].any()
    only = [torch.zeros(0, device="cuda")]
    assert float(fw.grad_norm(only)) == 0.0 and float(fw.clip_grad_norm_(only, 1.0)) == 0.0
    x = torch.ones(4, device="cuda")
    assert float(fw.clip_grad_norm_([None, x, None], 1.0)) == 2.0 and (x == 0.5).all()
    assert float(fw.clip_grad_norm_(x, float("inf"))) == 1.0 and (x == 0.5).all()
    assert float(fw.clip_grad_norm_(x, 0.0)) == 1.0 and (x == 0.0).all()
    out = torch.full((4,), 9.0, device="cuda")
    assert float(fw.clip_grad_norm_([None, torch.ones(4, device="cuda")], 5.0, out=[None, out])) == 2.0 and (out == 1.0).all()


@pytest.mark.parametrize("dtype", R.FLOATS)
def test_values_that_are_not_finite(dtype):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.ones(10001, dtype=dtype, device="cuda")
    fw.grad_norm([x], status=status)
    assert int(status) == 0
    x[777] = float("inf")
    assert float(fw.grad_norm([x], status=status)) == float("inf") and int(status) == 2
    status.zero_()
    assert float(fw.clip_grad_norm_([x], 1.0, status=status)) == float("inf") and int(status) == 2
    assert x[777].isnan() and not x[:777].any() and not x[778:].any()
    x = torch.ones(10001, dtype=dtype, device="cuda")
    x[5] = float("nan")
    assert fw.clip_grad_norm_([x], 1.0).isnan() and x.isnan().all()


def test_same_bits_every_time_and_a_given_norm():
    g = R.gen(7)
    grads = [R.normal((s,), torch.bfloat16, g) for s in (300001, 17, 40000)]
    a = fw.grad_norm(grads)
    outs = [[torch.empty_like(x) for x in grads] for _ in range(3)]
    for o in outs[:2]:
        assert torch.equal(fw.clip_grad_norm_(grads, 2.0, out=o), a)
    assert fw.clip_grad_norm_(grads, 2.0, out=outs[2], norm=a) is not None
    for p, q in zip(outs[0], outs[1]):
        assert torch.equal(p, q)
    # two shards: each clipped to the norm of both
    halves = [grads[:1], grads[1:]]
    norm = sum(fw.grad_norm(h).square() for h in halves).sqrt()
    o = [torch.empty_like(x) for x in grads]
    fw.clip_grad_norm_(halves[0], 2.0, out=o[:1], norm=norm)
    fw.clip_grad_norm_(halves[1], 2.0, out=o[1:], norm=norm)
    f = 2.0 / float(norm64(grads))
    for x, y in zip(o, grads):
        v = y.double() * f
        R.within(x, v, v.abs() * (FACTOR + 4 * R.E32) + R.rounded(v, torch.bfloat16) * (1 + 2.0 ** -7))


def test_refusals():
    x, y = torch.ones(8, device="cuda"), torch.ones(8, device="cuda")
    p = torch.ones(8, device="cuda", requires_grad=True)
    for call in (lambda: fw.grad_norm([x.cpu()]), lambda: fw.grad_norm([x.double()]), lambda: fw.grad_norm([x.long()]),
                 lambda: fw.grad_norm([x.to_sparse()]), lambda: fw.clip_grad_norm_([x], 1.0, out=[y.cpu()]),
                 lambda: fw.clip_grad_norm_([x], 1.0, out=[y.double()]), lambda: fw.clip_grad_norm_([x, 3], 1.0)):
        with pytest.raises(TypeError):
            call()
    pool = torch.ones(100, device="cuda")
    for call in (lambda: fw.grad_norm([]), lambda: fw.grad_norm([None]), lambda: fw.clip_grad_norm_([], 1.0),
                 lambda: fw.clip_grad_norm_([x], -1.0), lambda: fw.clip_grad_norm_([x], float("nan")),
                 lambda: fw.clip_grad_norm_([x, x], 1.0), lambda: fw.clip_grad_norm_([p], 1.0), lambda: fw.grad_norm([p]),
                 lambda: fw.clip_grad_norm_([pool[:50], pool[49:]], 1.0), lambda: fw.clip_grad_norm_([pool[49:], pool[:50]], 1.0),
                 lambda: fw.clip_grad_norm_([pool], 1.0, out=[pool.view(torch.bfloat16)[:100]]),
                 lambda: fw.clip_grad_norm_([pool[:50], pool[50:]], 1.0, out=[pool[50:], torch.ones(50, device="cuda")]),
                 lambda: fw.clip_grad_norm_([pool[:50]], 1.0, out=[pool[1:51]]),
                 lambda: fw.clip_grad_norm_([x], 1.0, out=[]), lambda: fw.clip_grad_norm_([x], 1.0, out=[y[:4]]),
                 lambda: fw.clip_grad_norm_([x], 1.0, norm=torch.ones(2, device="cuda")),
                 lambda: fw.clip_grad_norm_([x], 1.0, norm=torch.ones((), device="cuda").double()),
                 lambda: fw.clip_grad_norm_([x], 1.0, norm=torch.ones(()))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        fw.clip_grad_norm_([x[:1].expand(4)], 1.0)
    assert (x == 1).all() and (pool == 1).all() and (p == 1).all()
    with torch.no_grad():
        assert abs(float(fw.grad_norm([p])) - 8 ** 0.5) < 1e-6
    # the same tensor twice counts twice where nothing is written, and may be read twice for other results
    assert float(fw.grad_norm([x, x])) == 4.0
    outs = [torch.empty(8, device="cuda") for _ in range(2)]
    assert float(fw.clip_grad_norm_([x, x], 2.0, out=outs)) == 4.0 and all((o == 0.5).all() for o in outs)
    # a result may be the gradient itself
    assert float(fw.clip_grad_norm_([x, y], 2.0, out=[x, outs[0]])) == 4.0 and (x == 0.5).all() and (y == 1.0).all()


def test_streams_and_graphs():
    g = R.gen(5)
    grads = [R.normal((s,), t, g) for s, t in ((70001, torch.bfloat16), (33, torch.float32), (9000, torch.float16))]
    out = [torch.empty_like(x, dtype=torch.float32) for x in grads]

    def step():
        return fw.clip_grad_norm_(grads, 3.0, out=out)

    want = step()
    held = [o.clone() for o in out]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for f in (1.0, 1e-4, 50.0):
        for x, b in zip(grads, [x.clone() for x in grads]):
            x.copy_(b * f)
        graph.replay()
        norms, values = captured.clone(), [o.clone() for o in out]
        assert torch.equal(step(), norms)
        for o, v in zip(out, values):
            assert torch.equal(o, v)
    assert held[0].shape == out[0].shape


def test_a_long_tensor():
    """Offsets past 2^31 elements."""
    n = (1 << 31) + 12345
    if torch.cuda.get_device_properties(0).total_memory < 40e9:
        pytest.skip("needs 20 GB of device memory")
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    x[-1], x[0], x[1 << 30] = 3.0, 4.0, 12.0
    assert float(fw.clip_grad_norm_([x], 6.5)) == 13.0
    assert float(x[-1]) == 1.5 and float(x[0]) == 2.0 and float(x[1 << 30]) == 6.0 and int((x != 0).sum()) == 3

"""What clipping writes: results that share memory, the given norm's place,
gradients of a graph.  A refused call writes nothing."""
import pytest
import torch

import fwloss_b200 as fw
import lm_ref as R

pytestmark = pytest.mark.gpu


def ones(*shape, dtype=torch.float32):
    return torch.ones(shape, dtype=dtype, device="cuda")


def pair():
    return [ones(50, 60), ones(50, 60)]


OVERLAPPING = [
    lambda m: (pair(), [m[:50, :60], m[:50, 40:100]]),  # columns 40 .. 60 are in both
    lambda m: (pair(), [m[:50, :60], m[49:99, :60]]),  # one row
    lambda m: (pair(), [m[:50, :120:2], m[:50, 2:122:2]]),  # every other column, shifted by one of them
    lambda m: (pair(), [m[:60, :50].t(), m[59:119, 49:99].t()]),  # one element
    lambda m: (pair(), [m[:60, :50].t(), m.view(-1)[: 50 * 60].view(50, 60)]),  # copied and written by the kernel
    lambda m: (pair(), [m.view(torch.bfloat16)[:50, :60], m[:50, 29:89]]),  # one of two halves of an element
    lambda m: ([ones(50, 60), m[:50, 100:160]], [m[:50, 59:119], ones(50, 60)]),  # another gradient's memory
    lambda m: ([m[:50, ::4], m[:50, ::4]], None),  # the same one twice, in place
    lambda m: ([m[:50, :90], m[:50, 89:170]], None),
]


@pytest.mark.parametrize("make", OVERLAPPING)
def test_copied_results_that_overlap_are_refused(make):
    m = ones(200, 200)
    grads, out = make(m)
    with pytest.raises(ValueError, match="overlap"):
        fw.clip_grad_norm_(grads, 1.0, out=out)
    with pytest.raises(ValueError, match="overlap"):
        fw.clip_grad_norm_(grads[::-1], 1.0, out=out and out[::-1])
    assert (m == 1).all() and all((g == 1).all() for g in grads)


APART = [
    lambda m: [m[:50, :60], m[:50, 60:120]],
    lambda m: [m[:50, :120:2], m[:50, 1:121:2]],  # interleaved columns
    lambda m: [m[:100:2, :60], m[1:101:2, :60]],  # and rows
    lambda m: [m[:60, :50].t(), m[60:120, :50].t()],
    lambda m: [m[:60, :50].t(), m[:50, 50:110]],
    lambda m: [m.view(torch.bfloat16)[:50, :60], m[:50, 30:90]],
    lambda m: [m[:150:3, :180:3], m[1:151:3, 1:181:3]],  # a grid inside a grid
]


@pytest.mark.parametrize("make", APART)
def test_copied_results_beside_each_other(make):
    m = torch.full((200, 200), 7.0, device="cuda")
    out = make(m)
    norm = fw.clip_grad_norm_(pair(), 6000 ** 0.5 / 4, out=out)
    assert abs(float(norm) / 6000 ** 0.5 - 1) < 1e-6
    # the factor is within a few ulps of 1 / 4
    for o in out:
        R.within(o, torch.full_like(o, 0.25).double(), 0.25 * (20 * R.E32 + R.U[o.dtype]))
    if out[0].dtype == torch.float32:
        assert int((m == 7.0).sum()) == 200 * 200 - 6000


def test_many_interleaved_results():
    """512 columns of one matrix, each the result of a gradient of its own."""
    m = torch.full((100, 512), 7.0, device="cuda")
    fw.clip_grad_norm_([ones(100) for _ in range(512)], 51200 ** 0.5 / 2, out=[m[:, i] for i in range(512)])
    R.within(m, torch.full_like(m, 0.5).double(), 20 * R.E32)
    g = ones(100, 512)
    fw.clip_grad_norm_([g[:, i] for i in range(512)], 51200 ** 0.5 / 2)
    R.within(g, torch.full_like(g, 0.5).double(), 20 * R.E32)


def test_a_norm_in_what_is_written_is_refused():
    x, m = ones(5000), ones(100, 100)
    calls = [lambda: fw.clip_grad_norm_([x], 0.5, norm=x[:1]), lambda: fw.clip_grad_norm_([ones(7), x], 0.5, norm=x[4999]),
             lambda: fw.clip_grad_norm_([ones(5000)], 0.5, out=[x], norm=x[77:78]),
             lambda: fw.clip_grad_norm_([m[:, ::2]], 0.5, norm=m[3, 4]),
             lambda: fw.clip_grad_norm_([ones(100, 50, dtype=torch.float16)], 0.5, out=[m.t()[::2].t()], norm=m[99, 98]),
             lambda: fw.clip_grad_norm_([m.view(torch.bfloat16)[:, 1::2]], 0.5, norm=m[0, 0])]
    for call in calls:
        with pytest.raises(ValueError, match="norm must not lie"):
            call()
    assert (x == 1).all() and (m == 1).all()
    # beside what is written, or in what is only read
    assert float(fw.clip_grad_norm_([m[:, ::2]], 0.5, norm=m[3, 5])) == 1.0 and (m[:, ::2] == 0.5).all() and (m[:, 1::2] == 1).all()
    out = torch.empty_like(x)
    assert float(fw.clip_grad_norm_([x], 0.25, out=[out], norm=x[:1])) == 1.0 and (out == 0.25).all()
    assert float(fw.clip_grad_norm_([x[1:]], 0.5, norm=x[0])) == 1.0 and (x[1:] == 0.5).all() and float(x[0]) == 1.0


def test_gradients_of_a_graph_are_refused():
    """Their graph would be dropped without a word, as grad_norm says."""
    p, out = ones(8).requires_grad_(True), ones(8)
    for g in (p, p * 2.0):
        with pytest.raises(ValueError, match="not differentiable"):
            fw.clip_grad_norm_([ones(8), g], 1.0, out=[ones(8), out])
        with pytest.raises(ValueError, match="not differentiable"):
            fw.grad_norm([ones(8), g])
    assert (out == 1).all() and (p == 1).all()
    with torch.no_grad():
        fw.clip_grad_norm_([p], 2.0 ** 0.5, out=[out])
    R.within(out, torch.full_like(out, 0.5).double(), 20 * R.E32)
    fw.clip_grad_norm_([p.detach()], 8.0 ** 0.5 / 4, out=[out])
    R.within(out, torch.full_like(out, 0.25).double(), 20 * R.E32)

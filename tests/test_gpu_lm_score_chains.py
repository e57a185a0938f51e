"""The scoring and clipping operators together with those around them: a
training step and a serving step as a user runs them, eager and captured, and
each call reading what the one before it has just written."""
import os
import sys

import pytest
import torch

import fwloss_b200 as fw
import lm_ref as R
import score_ref as S

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def tokens_for(shape, V, g, ignored=0.0):
    y = torch.randint(0, V, shape, generator=g, device="cuda")
    return torch.where(torch.rand(shape, generator=g, device="cuda") < ignored, torch.full_like(y, -100), y)


def make(B, D, V, seed=0, dtype=torch.bfloat16):
    g = R.gen(seed)
    return {"table": R.normal((V, D), dtype, g, 0.5).requires_grad_(True), "gain": torch.ones(D, device="cuda", requires_grad=True),
            "out": R.normal((V, D), dtype, g, 1.5 * D ** -0.5).requires_grad_(True), "ids": tokens_for((B,), V, g),
            "y": tokens_for((B,), V, g, 0.2), "adv": torch.randn(B, generator=g, device="cuda") / B,
            "buffers": [torch.zeros(V, D, device="cuda"), torch.zeros(D, device="cuda"), torch.zeros(V, D, device="cuda")]}


def train_step(s, fused, wait=lambda: None):
    """policy gradient with an entropy bonus; (logp, entropy, norm, clipped gradients)"""
    x = fw.embed_tokens(s["ids"], s["table"])
    wait()
    h = fw.rms_norm(x, s["gain"])
    wait()
    if fused:
        logp, entropy = fw.lm_head_log_probs(h, s["out"], s["y"], temperature=0.9)
    else:
        logp, entropy = fw.token_log_probs(h @ s["out"].t(), s["y"], temperature=0.9)
    wait()
    loss = -(logp * s["adv"]).sum() - 0.01 * entropy.mean()
    grads = torch.autograd.grad(loss, (s["table"], s["gain"], s["out"]))
    wait()
    norm = fw.clip_grad_norm_(grads, 1e-3, out=s["buffers"])
    wait()
    return [logp.detach(), entropy.detach(), norm, *(b.clone() for b in s["buffers"])]


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("B,D,V", [(65, 64, 301), (600, 256, 5001)])
def test_training_step(B, D, V, fused):
    states = [make(B, D, V, i) for i in range(3)]
    want = [train_step(s, fused, torch.cuda.synchronize) for s in states]
    for _ in range(3):
        for s, ref in zip(states, want):
            for a, b in zip(train_step(s, fused), ref):
                assert torch.equal(a, b)
    for s, ref in zip(states, want):  # the clipped gradients have the norm asked for, to the two roundings in between
        total = torch.stack([b.double().square().sum() for b in ref[3:]]).sum().sqrt()
        assert float(ref[2]) > 1e-3 and abs(float(total) / 1e-3 - 1) < 40 * R.E32


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fused_and_materialised_logits_agree(dtype):
    """lm_head_log_probs and token_log_probs on float32 logits of the same operands, each within its bound of the definition."""
    g = R.gen(3)
    h, w = R.normal((130, 200), dtype, g), R.normal((3001, 200), dtype, g, 0.1)
    y = tokens_for((130,), 3001, g, 0.1)
    z = h.double() @ w.double().t()
    e_z = 2 * 202 * R.E32 * (h.double().abs() @ w.double().abs().t()).amax(1)
    r = S.rows(z, y, 1.0, e_z=e_z)
    a, b = fw.lm_head_log_probs(h, w, y), fw.token_log_probs(z.float(), y, top_k=4)
    for i, e in ((0, "e_logp"), (1, "e_entropy")):
        R.within(a[i], b[i], 2 * r[e] + 2 * R.E32 * z.abs().amax(1))
    assert torch.equal(b[3][:, 0][y != -100], z.float().argmax(1)[y != -100])


def test_training_step_in_a_graph():
    s = make(300, 128, 1000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            train_step(s, True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = train_step(s, True)
    for seed in (4, 5):
        new = make(300, 128, 1000, seed)
        with torch.no_grad():
            for k in ("table", "out", "ids", "y", "adv"):
                s[k].copy_(new[k])
        graph.replay()
        got = [t.clone() for t in held]
        for a, b in zip(got, train_step(s, True)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows,D,V", [(1, 256, 5000), (48, 512, 20003)])
def test_serving_step(rows, D, V):
    g = R.gen(V)
    gain = torch.ones(D, dtype=torch.bfloat16, device="cuda")
    wq, ws = fw.quantize_rows_int8(R.normal((V, D), torch.bfloat16, g, 0.1))
    xs = [(R.normal((rows, D), torch.bfloat16, g), R.normal((rows, D), torch.bfloat16, g)) for _ in range(4)]

    def step(x, r, wait=lambda: None):
        q, s, stream = fw.rms_norm_int8(x, gain, residual=r)
        wait()
        logits = fw.int8_linear(q, s, wq, ws)
        wait()
        chosen = logits.argmax(1)
        return [chosen, *fw.token_log_probs(logits, chosen, top_k=8, temperature=0.7)]

    want = [step(x, r, torch.cuda.synchronize) for x, r in xs]
    for _ in range(4):
        for (x, r), ref in zip(xs, want):
            for a, b in zip(step(x, r), ref):
                assert torch.equal(a, b)
    for ref in want:
        assert torch.equal(ref[1], ref[3][:, 0])  # the chosen token is the likeliest
    x, r = (t.clone() for t in xs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(x, r)
    for (a, b), ref in zip(xs, want):
        x.copy_(a)
        r.copy_(b)
        graph.replay()
        for p, q in zip(held, ref):
            assert torch.equal(p, q)


def test_example_runs_with_entropy_and_clipping():
    import lm_ends

    model, losses = lm_ends.train(steps=5, kind="entropy", clip=0.5)
    assert len(losses) == 5 and all(x == x for x in losses) and float(model.norm) > 0
    total = torch.stack([g.double().square().sum() for g in model.grads.values()]).sum().sqrt()
    assert float(total) <= 0.5 * (1 + 40 * R.E32)
    server = lm_ends.Server(model)
    tokens, _ = lm_ends.batch(torch.Generator(device="cuda").manual_seed(7), 9)
    logp, entropy, top_logp, top_ids = server.score(tokens[:, :6], tokens[:, 6])
    r = S.rows(server.logits(tokens[:, :6]).double(), tokens[:, 6], 1.0)
    R.within(logp, r["logp"], r["e_logp"])
    R.within(entropy, r["entropy"], r["e_entropy"])
    assert top_ids.shape == (9, 3) and top_logp.shape == (9, 3)


def test_example_gradients_with_entropy():
    """One step's gradients against the same model in float32 torch operators on the same (bfloat16) parameters."""
    import lm_ends

    model = lm_ends.Model(3)
    tokens, targets = lm_ends.batch(torch.Generator(device="cuda").manual_seed(5), 16)
    model.loss(tokens, targets, "entropy").backward()
    p = {k: v.detach().float().requires_grad_(True) for k, v in model.p.items()}

    def norm(x, gain):
        return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * gain

    x = p["embed"][tokens] * lm_ends.DIM ** 0.5
    h = norm(x, p["gain1"])
    before = torch.nn.functional.pad(h, (0, 0, 1, 0))[..., :-1, :]
    block = torch.nn.functional.gelu(torch.cat([h, before], -1) @ p["mix"]) @ p["out"]
    logq = (norm(block + x, p["gain2"]) @ p["embed"].t()).log_softmax(-1).flatten(0, 1)
    live = (targets != lm_ends.IGNORED).flatten()
    logp = logq.gather(1, targets.flatten().clamp(min=0)[:, None])[:, 0]
    entropy = -(logq.exp() * logq).sum(1)
    (-((logp + lm_ends.BONUS * entropy) * live).sum() / live.sum()).backward()
    for k in p:  # bfloat16 activations between the operators: eight roundings of 2^-8 at most along a path
        got, want = model.p[k].grad.float(), p[k].grad
        assert (got - want).norm() <= 8 * 2.0 ** -8 * want.norm(), k

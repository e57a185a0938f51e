"""The language-model operators together, as examples/lm_ends.py uses them."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("kind", ["softmax", "familywise"])
def test_training_lowers_the_loss(kind):
    import lm_ends

    _, losses = lm_ends.train(steps=120, kind=kind)
    assert all(x == x for x in losses)
    assert sum(losses[-10:]) < 0.8 * sum(losses[:10])


def test_gradients_of_the_whole_model_match_plain_operators():
    """One step's gradients against the same model in float32 torch operators on the same (bfloat16) parameters."""
    import lm_ends

    model = lm_ends.Model(3)
    tokens, targets = lm_ends.batch(torch.Generator(device="cuda").manual_seed(5), 16)
    model.loss(tokens, targets, "softmax").backward()
    p = {k: v.detach().float().requires_grad_(True) for k, v in model.p.items()}

    def norm(x, gain):
        return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * gain

    x = p["embed"][tokens] * lm_ends.DIM ** 0.5
    h = norm(x, p["gain1"])
    before = torch.nn.functional.pad(h, (0, 0, 1, 0))[..., :-1, :]
    block = torch.nn.functional.gelu(torch.cat([h, before], -1) @ p["mix"]) @ p["out"]
    logits = norm(block + x, p["gain2"]) @ p["embed"].t()
    torch.nn.functional.cross_entropy(logits.flatten(0, 1), targets.flatten(), ignore_index=lm_ends.IGNORED).backward()
    for k in p:  # bfloat16 activations between the operators: eight roundings of 2^-8 at most along a path
        got, want = model.p[k].grad.float(), p[k].grad
        assert (got - want).norm() <= 8 * 2.0 ** -8 * want.norm(), k


def test_serving_agrees_with_the_float_output_layer():
    import lm_ends

    model, _ = lm_ends.train(steps=120)
    server = lm_ends.Server(model)
    tokens, _ = lm_ends.batch(torch.Generator(device="cuda").manual_seed(7), 48)
    got = server.logits(tokens)
    with torch.no_grad():
        block, x = model.stream(tokens[:, -2:])
        y, _ = lm_ends.fw.rms_norm(block[:, -1], model.p["gain2"], residual=x[:, -1])
    want = y.float() @ model.p["embed"].float().t()
    # two quantisations of half a step each, 1 / 254 of a row's largest value, and bfloat16's rounding of y
    assert (got - want).norm() <= (2 / 254 * 4 + 2.0 ** -8) * want.norm()
    assert server.generate(tokens[:, :4], 3).shape == (48, 7)

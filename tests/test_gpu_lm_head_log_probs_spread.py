"""Upstream factors of very different sizes in one call of lm_head_log_probs.

bfloat16 holds every entry of the logit gradient relative to itself.  float16
holds the entries relative to the largest factor m of the call, scaled by 2^13
over a power of two of at most 2 m: its numbers under 2^-14 are 2^-24 apart, so
an entry is off by up to 2^-25 * 2^-13 * 2 m = 2^-37 m, over T.  A label's entry
is made good in both gradients (the reference has these bounds, twice that)."""
import pytest
import torch

import fwloss_b200 as fw
import lm_ref as R
from test_gpu_lm_head_log_probs import reference, tokens_for

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [3, 500, 9000])
@pytest.mark.parametrize("temperature", [1.0, 0.3])
def test_wide_spread(temperature, vocab, dtype):
    g = R.gen(vocab)
    h, w = R.normal((256, 72), dtype, g), R.normal((vocab, 72), dtype, g, 0.2)
    y = tokens_for(256, vocab, g, 0.1)
    a, b = (torch.randn(256, generator=g, device="cuda") * 2.0 ** torch.randint(-40, 1, (256,), generator=g, device="cuda")
            for _ in range(2))
    a[0] = 1.0
    hh, ww = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    got = torch.autograd.grad(fw.lm_head_log_probs(hh, ww, y, temperature=temperature), (hh, ww), (a, b))
    _, dh, dw = reference(h, w, y, temperature, a, b)
    R.within(got[0], *dh, "dhidden")
    R.within(got[1], *dw, "dweight")

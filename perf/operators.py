"""Measured cases of the language-model operators around the loss.

Four operators, as a user of the package calls them:

  embed  rows of an embedding table, scaled, and the table's gradient (training step of the input end);
  norm   root-mean-square norm of a residual stream with the addition, and its gradients;
  head   serving: norm with an 8-bit output, then the output layer's logits from 8-bit weights; and the
         8-bit product alone;
  xent   softmax cross entropy of an output layer, with the gradients of hidden states and weight.

`run` computes each in its plain form with elementary torch operations in 32 bits, or, where `own` is set, by the
package's operators.  `exact` restates the definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _package():
    path = os.path.join(_ROOT, "fast-familywise-loss_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fwloss_b200

    return fwloss_b200


def listed():
    return [
        # a short prompt's tokens in a small model, float32: latency
        {"name": "embed-small", "op": "embed", "tokens": 128, "vocab": 1000, "dim": 256, "dtype": "f32", "scale": 1.0},
        # a training step's tokens in an ordinary model, odd token count
        {"name": "embed-ordinary", "op": "embed", "tokens": 8191, "vocab": 32000, "dim": 2048, "dtype": "bf16",
         "scale": 45.25},
        # a large vocabulary: the gradient's zero rows are most of the bytes
        {"name": "embed-large", "op": "embed", "tokens": 32768, "vocab": 128256, "dim": 4096, "dtype": "bf16", "scale": 1.0},
        # a few sequences' worth of rows in a small model: latency
        {"name": "norm-small", "op": "norm", "rows": 64, "dim": 1000, "dtype": "f32", "residual": True},
        # one layer's stream in a training step
        {"name": "norm-large", "op": "norm", "rows": 16384, "dim": 4096, "dtype": "bf16", "residual": True},
        # one sequence generating: a single token through norm and output layer
        {"name": "head-one-token", "op": "head", "tokens": 1, "dim": 2048, "vocab": 32000, "dtype": "bf16", "norm": True},
        # a batch of sequences generating, large vocabulary
        {"name": "head-batch", "op": "head", "tokens": 48, "dim": 4096, "vocab": 128256, "dtype": "bf16", "norm": True},
        # every position of long prompts scored
        {"name": "head-prompt", "op": "head", "tokens": 4096, "dim": 4096, "vocab": 32000, "dtype": "f16", "norm": True},
        # the 8-bit product alone, ragged in every direction, float32 out
        {"name": "int8-ragged", "op": "head", "tokens": 333, "dim": 1000, "vocab": 5001, "dtype": "f32", "norm": False},
        # a small model's loss: latency
        {"name": "xent-small", "op": "xent", "rows": 256, "dim": 256, "vocab": 1000, "dtype": "bf16", "ignored": 0.0,
         "reduction": "mean"},
        # an ordinary model's loss, ragged rows, prompt positions ignored, weights per row from outside
        {"name": "xent-ordinary", "op": "xent", "rows": 2011, "dim": 2048, "vocab": 32000, "dtype": "f16", "ignored": 0.2,
         "reduction": "none"},
        # a large vocabulary
        {"name": "xent-large", "op": "xent", "rows": 4096, "dim": 4096, "vocab": 128256, "dtype": "bf16", "ignored": 0.02,
         "reduction": "mean"},
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["embed", "norm", "head", "head", "xent"])
    if op == "embed":
        return {"op": op, "tokens": _spread(rng, 16, 32768), "vocab": _spread(rng, 500, 128256), "dim": _spread(rng, 64, 4096),
                "dtype": rng.choice(["bf16", "f16", "f32"]), "scale": rng.choice([1.0, 8.0, 45.25])}
    if op == "norm":
        return {"op": op, "rows": _spread(rng, 1, 16384), "dim": _spread(rng, 64, 8192),
                "dtype": rng.choice(["bf16", "f16", "f32"]), "residual": rng.random() < 0.7}
    if op == "head":
        norm = rng.random() < 0.7
        return {"op": op, "tokens": _spread(rng, 1, 4096), "dim": _spread(rng, 64, 4096), "vocab": _spread(rng, 256, 128256),
                "dtype": rng.choice(["bf16", "f16"] if norm else ["bf16", "f16", "f32"]), "norm": norm}
    return {"op": op, "rows": _spread(rng, 16, 4096), "dim": _spread(rng, 64, 4096), "vocab": _spread(rng, 500, 128256),
            "dtype": rng.choice(["bf16", "f16"]), "ignored": rng.choice([0.0, 0.1, 0.5]),
            "reduction": rng.choice(["mean", "sum", "none"])}


def work(case):
    op, e = case["op"], 4 if case["dtype"] == "f32" else 2
    d = case["dim"]
    if op == "embed":  # ids; rows named, once; their copies; upstream gradient; the whole table's gradient
        t, v = case["tokens"], case["vocab"]
        return {"bytes": 8 * t + e * d * (min(t, v) + 2 * t + v), "flops": 2.0 * t * d}
    if op == "norm":  # forward: x (, residual, sum) and y; backward: dy, stored stream (, its gradient) and the gradient
        n = case["rows"] * d
        return {"bytes": e * n * (8 if case["residual"] else 5) + 2 * e * d, "flops": 16.0 * n}
    if op == "head":
        t, v = case["tokens"], case["vocab"]
        io = 3 * e * t * d + e * d if case["norm"] else t * d  # x, residual, sum and gains; or the rows in 8 bits
        return {"bytes": io + v * d + 4 * v + e * t * v, "flops": 2.0 * t * d * v}
    b, v = case["rows"], case["vocab"]
    return {"bytes": 2 * e * d * (b + v) + 8 * b, "flops": 6.0 * b * (1.0 - case["ignored"]) * d * v}


def _rows16(rows, cols, gen):
    """8-bit integers in rows that start on 16-byte boundaries, as the package's own quantiser lays weights out."""
    store = torch.randint(-127, 128, (rows, (cols + 15) // 16 * 16), generator=gen, device="cuda", dtype=torch.int8)
    return store[:, :cols]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dt, d = case["op"], _DTYPES[case["dtype"]], case["dim"]

    def normal(*shape, scale=1.0):
        return torch.empty(shape, dtype=dt, device="cuda").normal_(0.0, scale, generator=g)

    s = {"case": case}
    if op == "embed":
        # frequencies fall off as 1 / rank, as words' do: the commonest tokens take whole percents of the positions
        u = torch.rand(case["tokens"], generator=g, device="cuda", dtype=torch.float64)
        s["ids"] = ((case["vocab"] + 1.0) ** u - 1.0).long().clamp_(0, case["vocab"] - 1)
        s["weight"] = normal(case["vocab"], d, scale=0.02).requires_grad_(True)
        s["grad"] = normal(case["tokens"], d)
    elif op == "norm":
        n = case["rows"]
        s["x"] = normal(n, d).requires_grad_(True)
        s["gain"] = (1.0 + 0.1 * normal(d).float()).to(dt).requires_grad_(True)
        s["dy"] = normal(n, d)
        if case["residual"]:
            s["residual"] = normal(n, d, scale=3.0).requires_grad_(True)
            s["dsum"] = normal(n, d)
    elif op == "head":
        t, v = case["tokens"], case["vocab"]
        s["weight"] = _rows16(v, d, g)
        s["weight_scale"] = torch.rand(v, generator=g, device="cuda") * 1e-3 + 2e-4
        if case["norm"]:
            s["x"], s["residual"] = normal(t, d), normal(t, d, scale=3.0)
            s["gain"] = (1.0 + 0.1 * normal(d).float()).to(dt)
        else:
            s["q"] = _rows16(t, d, g)
            s["q_scale"] = torch.rand(t, generator=g, device="cuda") * 0.02 + 0.01
    else:
        b, v = case["rows"], case["vocab"]
        # logits of a few units' spread, so that some rows are confident
        s["hidden"] = normal(b, d).requires_grad_(True)
        s["weight"] = normal(v, d, scale=2.0 / math.sqrt(d)).requires_grad_(True)
        y = torch.randint(0, v, (b,), generator=g, device="cuda")
        out = torch.rand(b, generator=g, device="cuda") < case["ignored"]
        out[0] = False
        s["target"] = torch.where(out, torch.full_like(y, -100), y)
        if case["reduction"] == "none":
            s["upstream"] = torch.rand(b, generator=g, device="cuda") * 2.0 / b
    return s


EPS = 1e-6


def _own_run(s):
    p, c = _package(), s["case"]
    if c["op"] == "embed":
        out = p.embed_tokens(s["ids"], s["weight"], scale=c["scale"])
        return [out, *torch.autograd.grad(out, s["weight"], s["grad"])]
    if c["op"] == "norm":
        if c["residual"]:
            y, total = p.rms_norm(s["x"], s["gain"], eps=EPS, residual=s["residual"])
            return [y, total, *torch.autograd.grad((y, total), (s["x"], s["residual"], s["gain"]), (s["dy"], s["dsum"]))]
        y = p.rms_norm(s["x"], s["gain"], eps=EPS)
        return [y, *torch.autograd.grad(y, (s["x"], s["gain"]), s["dy"])]
    if c["op"] == "head":
        dt = _DTYPES[c["dtype"]]
        if not c["norm"]:
            return [p.int8_linear(s["q"], s["q_scale"], s["weight"], s["weight_scale"], out_dtype=dt)]
        q, q_scale, total = p.rms_norm_int8(s["x"], s["gain"], eps=EPS, residual=s["residual"])
        return [p.int8_linear(q, q_scale, s["weight"], s["weight_scale"], out_dtype=dt), total]
    loss = p.lm_head_cross_entropy(s["hidden"], s["weight"], s["target"], reduction=c["reduction"])
    return [loss.detach(), *torch.autograd.grad(loss, (s["hidden"], s["weight"]), s.get("upstream"))]


def _normed(s):
    """(sum as it is stored, its values, 1 / root mean square, normed values) in 32 bits"""
    total = s["x"].detach()
    if "residual" in s:
        total = (total.float() + s["residual"].detach().float()).to(total.dtype)
    v = total.float()
    r = torch.rsqrt((v * v).mean(1, keepdim=True) + EPS)
    return total, v, r, v * r * s["gain"].detach().float()


def _plain_norm(s):
    dt = s["x"].dtype
    total, v, r, y = _normed(s)
    dy = s["dy"].float()
    a = dy * s["gain"].detach().float()
    d = r * (a - v * ((a * v).mean(1, keepdim=True) * r * r))
    dgain = (dy * v * r).sum(0).to(dt)
    if "residual" not in s:
        return [y.to(dt), d.to(dt), dgain]
    d = (d + s["dsum"].float()).to(dt)
    return [y.to(dt), total, d, d, dgain]  # both addends have the sum's gradient


def _plain_head(s):
    dt = _DTYPES[s["case"]["dtype"]]
    if not s["case"]["norm"]:
        q, q_scale, rest = s["q"].float(), s["q_scale"], []
    else:
        total, _, _, y = _normed(s)
        q_scale = y.abs().amax(1) / 127.0
        q, rest = torch.round(y / q_scale[:, None]), [total]
    out = (q @ s["weight"].float().t()) * q_scale[:, None] * s["weight_scale"]
    return [out.to(dt), *rest]


def _plain_xent(s):
    h, w, y = s["hidden"].detach().float(), s["weight"].detach().float(), s["target"]
    live = (y != -100)
    at = torch.where(live, y, torch.zeros_like(y))[:, None]
    z = h @ w.t()
    zy = z.gather(1, at)
    top = z.amax(1, keepdim=True)
    z = z.sub_(top).exp_()
    total = z.sum(1, keepdim=True)
    rows = torch.where(live, (total.log() + top - zy)[:, 0], torch.zeros_like(top[:, 0]))
    kind = s["case"]["reduction"]
    count = live.sum().float()
    loss = rows if kind == "none" else rows.sum() / count if kind == "mean" else rows.sum()
    up = s["upstream"] if kind == "none" else 1.0 / count if kind == "mean" else torch.ones_like(count)
    z = z.div_(total).scatter_add_(1, at, torch.full_like(zy, -1.0)).mul_((live * up)[:, None])
    dt = s["hidden"].dtype
    return [loss, (z @ w).to(dt), (z.t() @ h).to(dt)]


def run(state):
    if own:
        return _own_run(state)
    op = state["case"]["op"]
    if op == "embed":
        w, scale = state["weight"].detach(), state["case"]["scale"]
        out = (w[state["ids"]].float() * scale).to(w.dtype)
        dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
        dw.index_add_(0, state["ids"], state["grad"].float() * scale)
        return [out, dw.to(w.dtype)]
    return _plain_norm(state) if op == "norm" else _plain_head(state) if op == "head" else _plain_xent(state)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "embed":
            w, ids, scale = s["weight"].double(), s["ids"], case["scale"]
            out = w.index_select(0, ids).mul_(scale)
            order = torch.argsort(ids, stable=True)
            dw = torch.zeros_like(w)
            dw.index_put_((ids[order],), s["grad"].double()[order] * scale, accumulate=True)
            return [out, dw]
        if op == "norm" or (op == "head" and case["norm"]):
            total = s["x"].double()
            if "residual" in s:  # the stream holds the sum in its own type: that is the definition
                total = (total + s["residual"].double()).to(s["x"].dtype).double()
            n = total.shape[1]
            rms = (total.square().sum(1, keepdim=True) / n + EPS).sqrt()
            unit, gain = total / rms, s["gain"].double()
            y = unit * gain
            if op == "norm":
                a = s["dy"].double() * gain
                d = (a - unit * (a * unit).sum(1, keepdim=True) / n) / rms
                dgain = torch.einsum("nd,nd->d", s["dy"].double(), unit)
                if "residual" not in s:
                    return [y, d, dgain]
                d = d + s["dsum"].double()
                return [y, total, d, d, dgain]
            q_scale = y.abs().max(1).values / 127
            q, rest = (y / q_scale[:, None]).round(), [total]
        elif op == "head":
            q, q_scale, rest = s["q"].double(), s["q_scale"].double(), []
        if op == "head":
            return [torch.einsum("tk,nk->tn", q, s["weight"].double()) * torch.outer(q_scale, s["weight_scale"].double()), *rest]
        h, w, y = s["hidden"].double(), s["weight"].double(), s["target"]
        live = y.ne(-100)
        rows_at = live.nonzero()[:, 0]
        z = h[rows_at] @ w.t()
        lse = torch.logsumexp(z, 1)
        each = torch.zeros(y.shape, dtype=torch.float64, device=y.device)
        each[rows_at] = lse - z[torch.arange(len(rows_at), device=y.device), y[rows_at]]
        kind = case["reduction"]
        loss = each if kind == "none" else each[rows_at].mean() if kind == "mean" else each.sum()
        up = s["upstream"].double()[rows_at] if kind == "none" else torch.full_like(lse, 1.0 / len(rows_at) if kind == "mean" else 1.0)
        z = torch.exp(z - lse[:, None])
        z[torch.arange(len(rows_at), device=y.device), y[rows_at]] -= 1.0
        z = z * up[:, None]
        dh = torch.zeros_like(h)
        dh[rows_at] = z @ w
        return [loss, dh, z.t() @ h[rows_at]]

"""Measured cases of the operators that score tokens and end a training step.

Three operators, as a user of the package calls them:

  score   log probabilities of given tokens from logits, the entropy of each row and its likeliest alternatives
          (serving), or the first two with the gradient of the logits (training on them);
  policy  log probabilities and entropies of an output layer, with the gradients of hidden states and weight;
  clip    the global norm of many gradients, and the gradients clipped to it: in place, in buckets that hold one behind
          another, or into the buffers of an update.

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
IGNORED = -100


def _package():
    path = os.path.join(_ROOT, "fast-familywise-loss_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fwloss_b200

    return fwloss_b200


def listed():
    return [
        # one sequence generating: the token just chosen, with alternatives, from float32 logits: latency
        {"name": "score-one-token", "op": "score", "rows": 1, "vocab": 32000, "dtype": "f32", "top_k": 5,
         "temperature": 1.0, "ignored": 0.0, "padded": 0, "train": False},
        # a batch of sequences generating, large vocabulary whose table is padded, many alternatives
        {"name": "score-batch", "op": "score", "rows": 48, "vocab": 128256, "dtype": "bf16", "top_k": 20,
         "temperature": 0.8, "ignored": 0.0, "padded": 56, "train": False},
        # every position of long prompts scored
        {"name": "score-prompt", "op": "score", "rows": 4096, "vocab": 32000, "dtype": "f32", "top_k": 5,
         "temperature": 1.0, "ignored": 0.02, "padded": 0, "train": False},
        # a small vocabulary, odd sizes, part of the positions ignored, forward and gradient
        {"name": "score-train-ragged", "op": "score", "rows": 333, "vocab": 5001, "dtype": "f16", "top_k": 0,
         "temperature": 0.7, "ignored": 0.2, "padded": 0, "train": True},
        # a training step on the logits of a whole batch
        {"name": "score-train", "op": "score", "rows": 4096, "vocab": 32000, "dtype": "bf16", "top_k": 0,
         "temperature": 1.0, "ignored": 0.05, "padded": 0, "train": True},
        # a small model's step: latency
        {"name": "policy-small", "op": "policy", "rows": 256, "dim": 256, "vocab": 1000, "dtype": "bf16",
         "temperature": 1.0, "ignored": 0.0},
        # an ordinary model's step, ragged rows, prompt positions ignored
        {"name": "policy-ordinary", "op": "policy", "rows": 2011, "dim": 2048, "vocab": 32000, "dtype": "f16",
         "temperature": 0.9, "ignored": 0.2},
        # a large vocabulary
        {"name": "policy-large", "op": "policy", "rows": 4096, "dim": 4096, "vocab": 128256, "dtype": "bf16",
         "temperature": 1.0, "ignored": 0.02},
        # the gradients of a small model in float32: latency
        {"name": "clip-small", "op": "clip", "layers": 2, "dim": 256, "vocab": 1000, "dtype": "f32", "form": "out",
         "ratio": 0.5},
        # odd sizes, float16, gradients that are within the limit: norm and decision, in place
        {"name": "clip-within", "op": "clip", "layers": 12, "dim": 1000, "vocab": 10007, "dtype": "f16", "form": "inplace",
         "ratio": 1.5},
        # an ordinary model: bfloat16 matrices, float32 gains, clipped into the update's float32 buffer
        {"name": "clip-ordinary", "op": "clip", "layers": 8, "dim": 1024, "vocab": 32000, "dtype": "mixed", "form": "out",
         "ratio": 0.25},
        # a large model's gradients
        {"name": "clip-large", "op": "clip", "layers": 24, "dim": 2048, "vocab": 128256, "dtype": "bf16", "form": "out",
         "ratio": 0.5},
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["score", "score", "policy", "clip"])
    if op == "score":
        train, vocab = rng.random() < 0.5, _spread(rng, 64, 128256)
        return {"op": op, "rows": _spread(rng, 1, 4096), "vocab": vocab, "dtype": rng.choice(["bf16", "f16", "f32"]),
                "top_k": 0 if train else rng.choice([0, 1, 5, 20, 32]), "temperature": rng.choice([1.0, 0.6, 1.3]),
                "ignored": rng.choice([0.0, 0.1, 0.5]), "padded": rng.choice([0, 0, vocab // 100]), "train": train}
    if op == "policy":
        return {"op": op, "rows": _spread(rng, 16, 4096), "dim": _spread(rng, 64, 4096), "vocab": _spread(rng, 500, 128256),
                "dtype": rng.choice(["bf16", "f16"]), "temperature": rng.choice([1.0, 0.6, 1.3]),
                "ignored": rng.choice([0.0, 0.1, 0.5])}
    form = rng.choice(["out", "out", "inplace", "norm"])
    return {"op": op, "layers": _spread(rng, 1, 48), "dim": _spread(rng, 32, 1448), "vocab": _spread(rng, 256, 128256),
            "dtype": rng.choice(["bf16", "f16", "f32", "mixed"]), "form": form,
            "ratio": 1.5 if form == "inplace" else rng.choice([0.1, 0.5, 2.0])}


def _shapes(case):
    """Shapes of a model's gradients: embedding, then per layer two gains, four square matrices and two wide ones."""
    d = case["dim"]
    return [(case["vocab"], d)] + [(d,), (d, d), (d, d), (d, d), (d, d), (d,), (4 * d, d), (d, 4 * d)] * case["layers"]


def _grad_types(case):
    mixed = case["dtype"] == "mixed"
    return [(torch.float32 if len(s) == 1 else torch.bfloat16) if mixed else _DTYPES[case["dtype"]] for s in _shapes(case)]


def _buckets(shapes, types):
    """One flat buffer for each type, and the tensors in them, one behind another."""
    size, at = {}, []
    for shape, dt in zip(shapes, types):
        at.append(size.get(dt, 0))
        size[dt] = at[-1] + math.prod(shape)
    flat = {dt: torch.empty(n, dtype=dt, device="cuda") for dt, n in size.items()}
    return list(flat.values()), [flat[dt][a:a + math.prod(s)].view(s) for s, dt, a in zip(shapes, types, at)]


def work(case):
    e = 2 if case["dtype"] in ("bf16", "f16") else 4
    if case["op"] == "score":
        b, v = case["rows"], case["vocab"]
        # forward: the logits and the tokens in, a few numbers a row out; gradient: the logits again, and theirs
        return {"bytes": b * (e * v * (3 if case["train"] else 1) + 16 + 12 * case["top_k"]),
                "flops": b * v * (16.0 if case["train"] else 8.0)}
    if case["op"] == "policy":
        b, d, v = case["rows"], case["dim"], case["vocab"]
        return {"bytes": 2 * e * d * (b + v) + 24 * b, "flops": 8.0 * b * (1.0 - case["ignored"]) * d * v}
    read = wrote = 0
    for shape in _shapes(case):
        n = math.prod(shape)
        read += n * (4 if case["dtype"] == "mixed" and len(shape) == 1 else 2 if case["dtype"] == "mixed" else e)
        wrote += n * (4 if case["dtype"] == "mixed" else e)
    total = sum(math.prod(shape) for shape in _shapes(case))
    out = case["form"] == "out"
    return {"bytes": read + (wrote if out else 0), "flops": total * (3.0 if out else 2.0)}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}

    def normal(*shape, dtype, scale=1.0):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, scale, generator=g)

    def targets(rows, vocab):
        y = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        out = torch.rand(rows, generator=g, device="cuda") < case["ignored"]
        out[0] = False
        return torch.where(out, torch.full_like(y, IGNORED), y)

    if case["op"] == "clip":
        shapes, types = _shapes(case), _grad_types(case)
        # separate tensors, as backward gives them, or pieces of one bucket for each type
        if case["form"] == "inplace":
            s["buckets"], s["grads"] = _buckets(shapes, types)
        else:
            s["grads"] = [torch.empty(shape, dtype=dt, device="cuda") for shape, dt in zip(shapes, types)]
        if case["form"] == "out":
            s["buckets"], s["out"] = _buckets(shapes, [torch.float32] * len(types) if case["dtype"] == "mixed" else types)
        squares = torch.zeros((), dtype=torch.float64, device="cuda")
        for i, x in enumerate(s["grads"]):  # entries differ by tensor: those of matrices are small, those of gains larger
            x.normal_(0.0, (3e-2 if x.dim() == 1 else 1e-3) * (1.0 + 0.1 * (i % 7)), generator=g)
            squares += torch.linalg.vector_norm(x, dtype=torch.float32).double() ** 2
        s["max_norm"] = float(squares.sqrt()) * case["ratio"]
        return s
    dt, b, v = _DTYPES[case["dtype"]], case["rows"], case["vocab"]
    if case["op"] == "score":
        # logits of a few units' spread with some far above the rest, as a trained model's are
        logits = normal(b, v, dtype=dt, scale=2.5)
        likely = torch.randint(0, v - case["padded"], (b, 4), generator=g, device="cuda")
        lift = torch.rand((b, 4), generator=g, device="cuda") * 14.0
        logits.scatter_(1, likely, lift.to(dt))
        if case["padded"]:
            logits[:, v - case["padded"]:] = -math.inf  # columns that no token has
        y = targets(b, v - case["padded"])
        # a token drawn from the row is mostly one of the likely ones
        s["tokens"] = torch.where((y != IGNORED) & (torch.rand(b, generator=g, device="cuda") < 0.7), likely[:, 0], y)
        s["logits"] = logits.requires_grad_(case["train"])
    else:
        d = case["dim"]
        s["hidden"] = normal(b, d, dtype=dt).requires_grad_(True)
        s["weight"] = normal(v, d, dtype=dt, scale=2.0 / math.sqrt(d)).requires_grad_(True)
        s["tokens"] = targets(b, v)
    if case["op"] == "policy" or case["train"]:
        # advantages of either sign, and a small entropy bonus
        s["dlogp"] = torch.randn(b, generator=g, device="cuda") / b
        s["dentropy"] = torch.rand(b, generator=g, device="cuda") * 0.02 / b
    return s


def _own_run(s):
    p, c = _package(), s["case"]
    if c["op"] == "clip":
        if c["form"] == "norm":
            return [p.grad_norm(s["grads"])]
        return [p.clip_grad_norm_(s["grads"], s["max_norm"], out=s.get("out")), *s["buckets"]]
    if c["op"] == "score":
        if not c["train"]:
            return list(p.token_log_probs(s["logits"], s["tokens"], top_k=c["top_k"], temperature=c["temperature"],
                                          ignore_index=IGNORED))
        out = p.token_log_probs(s["logits"], s["tokens"], temperature=c["temperature"], ignore_index=IGNORED)
        return [out[0].detach(), out[1].detach(), *torch.autograd.grad(out, s["logits"], (s["dlogp"], s["dentropy"]))]
    out = p.lm_head_log_probs(s["hidden"], s["weight"], s["tokens"], temperature=c["temperature"], ignore_index=IGNORED)
    return [out[0].detach(), out[1].detach(),
            *torch.autograd.grad(out, (s["hidden"], s["weight"]), (s["dlogp"], s["dentropy"]))]


def _plain_rows(z, tokens, temperature):
    """(log probabilities of all columns, probabilities, live rows, columns of the tokens, logp, entropy); z is used up"""
    live = tokens != IGNORED
    at = torch.where(live, tokens, torch.zeros_like(tokens))[:, None]
    z = z.sub_(z.amax(1, keepdim=True)).div_(temperature)
    p = z.exp()
    total = p.sum(1, keepdim=True)
    z = z.sub_(total.log())
    p = p.div_(total)
    zero = torch.zeros_like(total[:, 0])
    logp = torch.where(live, z.gather(1, at)[:, 0], zero)
    z = z.clamp_(min=-200.0)  # where p is 0 the product with its logarithm is 0
    entropy = torch.where(live, -(p * z).sum(1), zero)
    return z, p, live, at, logp, entropy


def _plain_grad(z, p, live, at, entropy, dlogp, dentropy, temperature):
    """gradient of the logits; z and p are used up"""
    g, e = (dlogp * live / temperature)[:, None], (dentropy * live / temperature)[:, None]
    z = z.add_(entropy[:, None]).mul_(e).add_(g)
    return p.mul_(z).neg_().scatter_add_(1, at, g)


def _plain_top(logits, live, logsum, top, temperature, k):
    """values and columns of the k largest, equal ones by column"""
    v = logits.float() + 0.0  # -0 is 0
    bits = v.view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    key = order * 2 ** 32 + (logits.shape[1] - 1 - torch.arange(logits.shape[1], device=logits.device))
    at = key.topk(k, 1).indices
    values = (v.gather(1, at) - top) / temperature - logsum
    return [torch.where(live[:, None], values, torch.zeros_like(values)), torch.where(live[:, None], at, torch.full_like(at, -1))]


def _plain_clip(s):
    grads, c = s["grads"], s["case"]
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for x in grads:  # a sum of 1e9 squares
        x = x.float()
        total += (x * x).sum(dtype=torch.float64)
    norm = total.sqrt()
    if c["form"] == "norm":
        return [norm.float()]
    factor = (s["max_norm"] / norm).clamp(max=1.0).float()
    for x, to in zip(grads, s.get("out", grads)):
        to.copy_(x.float() * factor)
    return [norm.float(), *s["buckets"]]


def run(state):
    if own:
        return _own_run(state)
    case = state["case"]
    if case["op"] == "clip":
        return _plain_clip(state)
    with torch.no_grad():
        tokens, temperature = state["tokens"], case["temperature"]
        if case["op"] == "score":
            logits = state["logits"]
            z, p, live, at, logp, entropy = _plain_rows(logits.float().clone(), tokens, temperature)
            if case["train"]:
                dz = _plain_grad(z, p, live, at, entropy, state["dlogp"], state["dentropy"], temperature)
                return [logp, entropy, dz.to(logits.dtype)]
            if not case["top_k"]:
                return [logp, entropy]
            top = logits.float().amax(1, keepdim=True)
            logsum = ((logits.float() - top) / temperature).exp().sum(1, keepdim=True).log()
            return [logp, entropy, *_plain_top(logits, live, logsum, top, temperature, case["top_k"])]
        h, w = state["hidden"].float(), state["weight"].float()
        z, p, live, at, logp, entropy = _plain_rows(h @ w.t(), tokens, temperature)
        dz = _plain_grad(z, p, live, at, entropy, state["dlogp"], state["dentropy"], temperature)
        dt = state["hidden"].dtype
        return [logp, entropy, (dz @ w).to(dt), (dz.t() @ h).to(dt)]


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "clip":
            norm = torch.stack([torch.linalg.vector_norm(x, dtype=torch.float64) for x in s["grads"]]).square().sum().sqrt()
            if case["form"] == "norm":
                return [norm]
            factor = min(1.0, s["max_norm"] / float(norm))
            held = {}  # by the type of the bucket, in the order of the tensors
            for x in s["grads"]:
                held.setdefault(torch.float32 if "out" in s and case["dtype"] == "mixed" else x.dtype, []).append(x)
            return [norm, *(torch.cat([x.double().reshape(-1) for x in xs]) * factor for xs in held.values())]
        t, y = case["temperature"], s["tokens"]
        rows = y.ne(IGNORED).nonzero()[:, 0]
        n, at = torch.arange(len(rows), device=y.device), y[rows]
        if case["op"] == "score":
            z = s["logits"][rows].double() / t
        else:
            h, w = s["hidden"].double(), s["weight"].double()
            z = h[rows] @ w.t() / t
        logq = z - torch.logsumexp(z, 1, keepdim=True)
        q = logq.exp()
        inner = torch.where(q > 0, logq, torch.zeros_like(logq))
        h_rows = -torch.einsum("nv,nv->n", q, inner)

        def full(value, fill=0.0):
            out = torch.full((len(y),) + value.shape[1:], fill, dtype=value.dtype, device=y.device)
            out[rows] = value
            return out

        first = [full(logq[n, at]), full(h_rows)]
        if case["op"] == "score" and not case["train"]:
            if not case["top_k"]:
                return first
            order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, : case["top_k"]]
            return [*first, full(logq.gather(1, order)), full(order, -1)]
        onehot_minus_q = -q
        onehot_minus_q[n, at] += 1.0
        dz = onehot_minus_q * (s["dlogp"].double()[rows, None] / t)
        dz -= q * (inner + h_rows[:, None]) * (s["dentropy"].double()[rows, None] / t)
        if case["op"] == "score":
            return [*first, full(dz)]
        return [*first, full(dz @ w), dz.t() @ h[rows]]

"""64-bit definitions of the language-model operators and the units their
tolerances are made of.

U[dtype] is the largest relative error of one rounding to the type, TINY[dtype]
the largest absolute error of one where the type runs out of exponents.  Every
tolerance in the tests is a worst-case bound: n additions in fp32 in any order
are off by at most n * E32 times the sum of the absolute terms.
"""
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
E32 = 2.0 ** -24
FLOATS = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def within(got, want, bound, what=""):
    """|got - want| <= bound everywhere, both in 64 bits; NaN where wanted NaN."""
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(nan, torch.isnan(got)), f"{what}: NaN in other places"
    off = (got - want).abs()[~nan]
    lim = torch.as_tensor(bound, dtype=torch.float64, device=want.device).expand_as(want)[~nan]
    bad = off > lim
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst {float((off / lim).max()):.3g} of the bound"


def rounded(x, dtype):
    """Bound of rounding the 64-bit values x once to dtype."""
    return x.abs() * U[dtype] + TINY[dtype]


def embed(ids, weight, scale):
    w = weight.double()
    ok = (ids >= 0) & (ids < w.shape[0])
    out = w[ids.clamp(0, w.shape[0] - 1)] * scale
    out[~ok] = float("nan")
    return out


def embed_grad(ids, grad, V, scale, padding=None):
    """(gradient, sum of absolute terms, most terms of a row)"""
    i, g = ids.reshape(-1), grad.reshape(-1, grad.shape[-1]).double() * scale
    keep = (i >= 0) & (i < V)
    if padding is not None:
        keep &= i != padding
    i, g = i[keep], g[keep]
    dw = torch.zeros(V, g.shape[1], dtype=torch.float64, device=g.device)
    return dw.index_add(0, i, g), dw.index_add(0, i, g.abs()), int(torch.bincount(i, minlength=1).max()) if len(i) else 0


def norm(x, weight, eps, residual=None):
    s = x.double()
    if residual is not None:
        s = (s + residual.double()).to(x.dtype).double()
    rstd = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    return s, rstd, s * rstd * weight.double()


def norm_grad(dy, s, rstd, weight, dsum=None):
    """(ds, dweight, bound parts of ds, of dweight)"""
    D = s.shape[-1]
    a, n = dy.double() * weight.double(), s * rstd
    ds = rstd * (a - n * (a * n).mean(-1, keepdim=True))
    ds_abs = rstd * (a.abs() + n.abs() * (a * n).abs().mean(-1, keepdim=True))
    if dsum is not None:
        ds, ds_abs = ds + dsum.double(), ds_abs + dsum.double().abs()
    dn = dy.double() * n
    rows = s.numel() // D
    return ds, dn.reshape(-1, D).sum(0), ds_abs * (D + 16) * E32 * 3, dn.reshape(-1, D).abs().sum(0) * (rows + D + 16) * E32


def xent(hidden, weight, target, reduction, ignore=-100, go=None):
    """dict of loss, dh, dw, and worst-case bounds for operands of hidden's dtype."""
    h, w = hidden.double(), weight.double()
    B, D = h.shape
    V = w.shape[0]
    live = target != ignore
    bad = live & ((target < 0) | (target >= V))
    h = torch.where(live[:, None], h, torch.zeros_like(h))
    z = h @ w.t()
    # fp32 products are exact, D additions with truncation are off by 2 * E32 each at most
    dz = (2 * (D + 2) * E32) * (h.abs() @ w.abs().t()).amax(1)
    lse = torch.logsumexp(z, 1)
    at = target.clamp(0, V - 1)[:, None]
    rows = lse - z.gather(1, at)[:, 0]
    rows = torch.where(bad, torch.full_like(rows, float("nan")), rows)
    rows = torch.where(live, rows, torch.zeros_like(rows))
    # exponentials to 2^-21, V positive terms joined pairwise per 32, per tile and over tiles
    e_rows = 2 * dz + 2.0 ** -21 + (64 + V / 256) * 2 * E32 + 4 * E32 * (lse.abs() + rows.abs())
    n = int(live.sum())
    out = {"rows": rows}
    if reduction == "none":
        out["loss"], out["e_loss"] = rows, e_rows * live
        up = torch.ones_like(rows) if go is None else go.double()
    elif reduction == "mean":
        out["loss"] = rows.sum() / n if n else rows.sum() * float("nan")
        out["e_loss"] = (e_rows * live).sum() / max(n, 1) + out["loss"].abs() * 4 * E32
        up = torch.full_like(rows, (1.0 if go is None else float(go)) / max(n, 1))
    else:
        out["loss"], out["e_loss"] = rows.sum(), (e_rows * live).sum() + rows.sum().abs() * 4 * E32
        up = torch.full_like(rows, 1.0 if go is None else float(go))
    p = torch.exp(z - lse[:, None])
    p[torch.arange(B, device=p.device), at[:, 0]] -= 1.0
    p = torch.where(bad[:, None], torch.full_like(p, float("nan")), p)
    G = torch.where(live[:, None], p * up[:, None], torch.zeros_like(p))
    out["dh"], out["dw"] = G @ w, G.t() @ h
    # one rounding of G to the operands' type, the error of the logit and of log-sum-exp in the
    # exponent, and V (or B) additions with truncation
    rel = U[hidden.dtype] + 2 * dz + e_rows + 2.0 ** -20
    # where G underflows the scaled 16-bit range: 2^-24 of 2^15 of the largest upstream factor
    floor = (2.0 ** -25 / 2.0 ** 15) * float(up.abs().max()) if hidden.dtype == torch.float16 and up.numel() else 0.0
    eG = G.abs() * rel[:, None] + floor + up.abs()[:, None] * torch.exp(z - lse[:, None]) * rel[:, None]
    eG = torch.where(live[:, None], eG, torch.zeros_like(eG))
    out["e_dh"] = eG @ w.abs() + (G.abs() @ w.abs()) * (2 * V * E32) + rounded(out["dh"], hidden.dtype)
    out["e_dw"] = eG.t() @ h.abs() + (G.abs().t() @ h.abs()) * (2 * B * E32) + rounded(out["dw"], hidden.dtype)
    return out

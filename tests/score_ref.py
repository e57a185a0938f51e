"""64-bit definitions of the operators that score tokens, with worst-case
bounds on what fp32 arithmetic may make of them.

With t = (z - max z) / T, p the row's probabilities, M1 = sum p |t| and
M2 = sum p t^2: an exponential's argument is the product of a difference and a
factor that is itself the product of two rounded numbers, so it is off by
5 * E32 |t| at most, and the hardware's exponential by 2^-22 of its value.  A
thread adds N = 128 + V / 256 terms at most and rescales its sums at most once
per 16 of them, each time by one more such exponential.  The sum of the
exponentials is therefore off by e_s (relative), log S by e_s and its own
rounding, sum p t by the same factors applied term by term.
"""
import torch

from lm_ref import E32, rounded


def finite(x):
    return torch.where(torch.isinf(x), torch.zeros_like(x), x)


def rows(z, tokens, temperature, ignore=-100, e_z=None):
    """dict of logp, entropy, bounds, and what the gradient needs; z [B, V] in
    64 bits.  e_z: absolute error of each row's logits (0: they are given)."""
    B, V = z.shape
    live = tokens != ignore
    label = (tokens >= 0) & (tokens < V)
    top = z.amax(1)
    bad = live & (~label | ~torch.isfinite(top))
    z = torch.where((live & ~bad)[:, None], z, torch.zeros_like(z))
    top = z.amax(1, keepdim=True)
    t = (z - top) / temperature
    s = t.exp().sum(1, keepdim=True)
    log_s = s.log()
    logq = t - log_s
    q = logq.exp()
    tt = torch.where(q > 0, t, torch.zeros_like(t))
    m1, m2 = -(q * tt).sum(1), (q * tt * tt).sum(1)
    entropy = log_s[:, 0] + m1
    at = torch.where(label & live, tokens, torch.zeros_like(tokens))[:, None]
    logp = logq.gather(1, at)[:, 0]
    n = 128 + V / 256
    own = (n + 32) * E32 + (n / 16 + 16) * 2.0 ** -21
    shift = torch.zeros_like(m1) if e_z is None else 2 * e_z / temperature  # of every t, and so of log S
    e_s = own + 5 * E32 * m1 + shift
    e_log_s = e_s + 4 * E32 * log_s[:, 0].abs()
    # relative to t and logq however large they are: logits of 1e30 at T = 1e-3 make a t of 1e34, whose difference,
    # reciprocal of T and product are each rounded by up to E32 |t| (an infinite one is exact)
    e_t = 5 * E32 * finite(t).abs() + shift[:, None]
    e_logq = e_t + e_log_s[:, None] + 2 * E32 * finite(logq).abs()
    e_entropy = e_log_s + (own + e_s + 9 * E32) * m1 + 5 * E32 * m2 + shift * (1 + m1) + 2 * E32 * entropy.abs()
    nan = torch.full_like(logp, float("nan"))

    def out(x):
        return torch.where(bad, nan, torch.where(live, x, torch.zeros_like(x)))

    return {"logp": out(logp), "entropy": out(entropy), "e_logp": e_logq.gather(1, at)[:, 0] * live, "e_entropy": e_entropy * live,
            "t": t, "q": q, "logq": logq, "e_logq": e_logq, "live": live, "bad": bad, "at": at, "h": entropy, "e_h": e_entropy,
            "temperature": temperature}


def logit_grad(r, dlogp=None, dentropy=None):
    """(gradient of the logits, bound without a final rounding)"""
    zero = torch.zeros_like(r["h"])
    g = (zero if dlogp is None else dlogp.double()) / r["temperature"]
    e = (zero if dentropy is None else dentropy.double()) / r["temperature"]
    g, e = g[:, None], e[:, None]
    q, logq, h = r["q"], r["logq"].clamp(min=-745.0), r["h"][:, None]
    bent = g + e * (logq + h)
    d = -q * bent
    d = d.scatter_add(1, r["at"], g)
    e_q = r["e_logq"].clamp(max=1e3) + 2.0 ** -21 + 3 * E32 * logq.abs()
    size = g.abs() + e.abs() * (logq.abs() + h)  # where the probability is 0 the bound of its relative error is of no account
    bound = q * (size * (e_q + 8 * E32) + e.abs() * (r["e_logq"].clamp(max=1e3) + r["e_h"][:, None])) + 4 * E32 * d.abs()
    bound = bound + 2.0 ** -125 * (g.abs() + 200 * e.abs())  # probabilities under fp32's smallest normal number are 0
    bound = bound.scatter_add(1, r["at"], 4 * E32 * g.abs())
    live = r["live"][:, None]
    d = torch.where(live, d, torch.zeros_like(d))
    d = torch.where(r["bad"][:, None], torch.full_like(d, float("nan")), d)
    return d, torch.where(live, bound, torch.zeros_like(bound))


def top(z, r, k):
    """(log probabilities, columns, bound): the k largest, equal ones by the lowest column"""
    order = torch.sort(z + 0.0, dim=1, descending=True, stable=True).indices[:, :k]
    gone = (r["bad"] | ~r["live"])[:, None]
    value = r["logq"].gather(1, order)
    value = torch.where(r["bad"][:, None], torch.full_like(value, float("nan")), torch.where(gone, torch.zeros_like(value), value))
    return value, torch.where(gone, torch.full_like(order, -1), order), r["e_logq"].gather(1, order)


def grad_bound(d, bound, dtype):
    return bound + rounded(d, dtype)

"""Plain 64-bit forms of the log probability calls, and how far 32-bit results may lie from them."""
import math

import torch


def reference(logits, tokens=None, temperature=1.0, top_n=0, g=None, h=None):
    """dict of logprobs, entropy, ranks, top, ids, grad (float64 / int) for logits (..., V), row by row."""
    V = logits.shape[-1]
    rows = logits.shape[:-1]
    x = logits.detach().reshape(-1, V)
    R = x.shape[0]
    t = tokens.reshape(-1).long() if tokens is not None else torch.zeros(R, dtype=torch.long, device=x.device)
    T = temperature if torch.is_tensor(temperature) else torch.tensor(float(temperature), device=x.device)
    T = T.double()
    if T.dim() == 1 and len(rows) == 2:
        T = T[:, None]
    T = T.expand(rows).reshape(-1, 1)
    x = x.double()
    scored = t >= 0
    at = t.clamp_min(0)[:, None]
    bad = torch.isnan(x).any(1) | (x == math.inf).any(1)
    none = (x == -math.inf).all(1)
    z = x / T
    m = torch.where(none | bad, torch.zeros_like(z[:, 0]), z.amax(1))[:, None]
    e = (z - m).exp()
    s = e.sum(1, keepdim=True)
    logs = torch.where(none[:, None], torch.zeros_like(s), s.log())
    logp = z - m - logs
    p = torch.where(none[:, None], torch.zeros_like(e), e / s)
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    H = -plogp.sum(1, keepdim=True)
    nan = torch.full_like(H[:, 0], math.nan)
    out = {}
    lp = torch.where(none, -math.inf, torch.where(bad, nan, logp.gather(1, at)[:, 0]))
    out["logprobs"] = torch.where(scored, lp, 0.0).reshape(rows)
    out["entropy"] = torch.where(scored, torch.where(bad, nan, torch.where(none, 0.0, H[:, 0])), 0.0).reshape(rows)
    xt = x.gather(1, at)
    before = torch.arange(V, device=x.device)[None, :] < at
    rank = 1 + ((x > xt) | ((x == xt) & before)).sum(1)
    out["ranks"] = torch.where(scored & ~bad, rank, 0).int().reshape(rows)
    if top_n:
        order = x.sort(dim=1, descending=True, stable=True)
        n = min(top_n, V)
        there = (order.values[:, :n] > -math.inf) & scored[:, None] & ~bad[:, None]
        top = torch.full((R, top_n), -math.inf, dtype=torch.float64, device=x.device)
        ids = torch.full((R, top_n), -1, dtype=torch.int32, device=x.device)
        top[:, :n] = torch.where(there, logp.gather(1, order.indices[:, :n]), -math.inf)
        ids[:, :n] = torch.where(there, order.indices[:, :n], -1).int()
        top[bad & scored] = math.nan
        out["top"], out["ids"] = top.reshape(rows + (top_n,)), ids.reshape(rows + (top_n,))
    if g is not None or h is not None:
        zero = torch.zeros(R, 1, dtype=torch.float64, device=x.device)
        g = zero if g is None else g.double().expand(rows).reshape(-1, 1)
        h = zero if h is None else h.double().expand(rows).reshape(-1, 1)
        d = -g * p - h * (plogp + H * p)
        d.scatter_add_(1, at, g)
        d = d / T
        d[none | ~scored] = 0
        d[bad & scored] = math.nan
        out["grad"] = d.reshape(logits.shape)
    return out


# A 32-bit log probability is (x - m)/T - ln s: three roundings relative to the first term, and the relative error of s.
# That is at most 2^-22 (the exponential) + sum p |d| 2^-22 (its argument, three roundings; sum p |d| <= ln V + 1 < 15) + the
# additions on the longest path, 32 in a batch + V / (256 * 16) batches (at most 256) + 12, each 2^-24: below 1.3e-5 in all for
# V = 2^20, and 5e-6 up to V = 2^16.  The second sum behaves alike, relative to its size, the entropy.
def close(got, want, V, tol=None):
    tol = tol or (5e-6 if V <= 65536 else 1.5e-5)
    got, want = got.double(), want.double()
    # (beyond 32 bits' largest value, as a lowest logit over a small temperature, the nearest result is infinite)
    same = (got == want) | (got == want.float().double()) | (torch.isnan(got) & torch.isnan(want))
    off = (got - want).abs() <= tol * (1 + want.abs())
    assert bool((same | off).all()), float(torch.where(same, 0.0, (got - want).abs() / (1 + want.abs())).max())


# A gradient is p (A + D d) / T rounded to the logits' type: p carries the relative error above (tol), and so does the
# bracket, whose terms do not exceed |g| + |h| (H + |ln p|).
def close_grad(got, want, logits, g, h, temperature, ref):
    V = logits.shape[-1]
    tol = 5e-6 if V <= 65536 else 1.5e-5
    T = temperature.double() if torch.is_tensor(temperature) else torch.tensor(float(temperature), dtype=torch.float64, device=got.device)
    if T.dim() == 1 and logits.dim() == 3:
        T = T[:, None]
    size = (g.double().abs() if g is not None else 0.0)
    # p |ln p| <= 1/e and p H <= H: with |h| (H + 1) the bracket is covered for every p
    size = size + (h.double().abs() * (ref["entropy"].abs() + 1) if h is not None else 0.0)
    bound = 3 * tol * (size / T)[..., None]
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * half * 2
    a, b = got.double(), want.double()
    same = (a == b) | (torch.isnan(a) & torch.isnan(b))
    ok = same | ((a - b).abs() <= bound + half * b.abs() * (1 + 1e-6) + tiny)
    assert bool(ok.all()), float(torch.where(ok, 0.0, (a - b).abs()).max())

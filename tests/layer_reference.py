"""64-bit references of the layers around attention, with first-order error bounds.

Each follows the operator's definition in float64 on the CPU. A bound is the sum of
what the operator's documented roundings can change: sums in float32 (gamma = n 2^-24
for n terms one after the other), each float32 operation half a unit, outputs rounded
once to their type (U, and TINY below the normal range).
"""
from __future__ import annotations

import torch

from seq_reference import E32, TINY, U

U = dict(U)


def f64(x):
    return None if x is None else x.detach().cpu().double()


def rounded(value, dtype, err):
    """Bound of a value that carries `err` and is rounded to a type."""
    return err + (value.abs() + err) * U[dtype] + TINY[dtype]


def embedding(tokens, table, scale, dtype):
    """(out, bound); a token outside the table gives NaN."""
    t, tab = tokens.cpu().long(), f64(table)
    inside = (t >= 0) & (t < tab.shape[0])
    out = torch.full((len(t), tab.shape[1]), float("nan"), dtype=torch.float64)
    out[inside] = tab[t[inside]] * scale
    return out, rounded(out.nan_to_num(0.0), dtype, 2 * E32 * out.abs().nan_to_num(0.0))


def embedding_grad(dout, tokens, rows, scale, dtype):
    t, d = tokens.cpu().long(), f64(dout)
    inside = (t >= 0) & (t < rows)
    total, size = (torch.zeros(rows, d.shape[1], dtype=torch.float64) for _ in "ab")
    total.index_add_(0, t[inside], d[inside])
    size.index_add_(0, t[inside], d[inside].abs())
    n = torch.bincount(t[inside], minlength=rows).double()[:, None]
    err = (n + 8) * E32 * size * abs(scale)
    return total * scale, rounded(total * scale, dtype, err)


def stream(x, residual):
    """(h, bound): the sum in float32, rounded to the stream's type."""
    h = f64(x) + f64(residual)
    return h, rounded(h, residual.dtype, E32 * h.abs())


def rms(h, gain, eps):
    """(y, bound before its rounding) of the stream as it was returned."""
    h, D = f64(h), h.shape[1]
    y = h * (h.square().mean(1, keepdim=True) + eps) ** -0.5
    y = y if gain is None else y * f64(gain)
    # half the relative error of the sum of squares; a quotient, root, sum, quotient, and
    # two products
    return y, y.abs() * (0.5 * (D + 4) + 8) * E32


def rms_grad(dy, h, gain, dh, eps):
    """dict of d, dgain (None without a gain) with bounds before their rounding."""
    dy, h, gain, dh = f64(dy), f64(h), f64(gain), f64(dh)
    T, D = h.shape
    rho = (h.square().mean(1, keepdim=True) + eps) ** -0.5
    n, u = h * rho, dy if gain is None else dy * gain
    d = (u - n * (u * n).mean(1, keepdim=True)) * rho
    # rho: as above; the mean of u n: a sum of D rounded products, and rho twice
    r = (0.5 * (D + 4) + 8) * E32
    mean = (u * n).abs().mean(1, keepdim=True)
    err = rho * (u.abs() * (r + 4 * E32) + n.abs() * mean * ((D + 8) * E32 + 4 * r))
    if dh is not None:
        d = d + dh
        err = err + E32 * d.abs()
    out = dict(d=d, d_err=err, dgain=None)
    if gain is not None:
        out["dgain"] = (dy * n).sum(0)
        out["dgain_err"] = (dy * n).abs().sum(0) * ((T + 8) * E32 + r)
    return out


def logprobs(logits, tokens, temperature):
    """dict of lp [T, V], logp, entropy, order and bounds: of one log-probability
    (lp_err [T, V]) and of the entropy."""
    x = f64(logits)
    T, V = x.shape
    z = x / temperature
    lp = z.log_softmax(1)
    p = lp.exp()
    none = (x == float("-inf")).all(1)
    lp[none], p[none] = float("-inf"), 0.0
    t = (z - z.amax(1, keepdim=True))
    t[none] = 0.0
    away = t.abs().masked_fill(p == 0, 0.0)           # of what has weight
    plp = (p * lp.masked_fill(p == 0, 0.0))
    # additions one after the other: a thread's, then across threads
    depth = V if V <= 512 else V // 64 + 16
    # exponents: a difference and products of relative 2^-24 each; the power to 2 units,
    # and exact for the largest
    e = (6 * away + 4 * (away > 0)) * E32
    rest = 1.0 - p.amax(1, keepdim=True)
    rest[none] = 0.0
    # the sum's relative error; what rounding takes from it beside 1 where the rest is
    # more than 2^-6, and from the rest where it is less
    s = (p * e).sum(1, keepdim=True) + depth * E32 * torch.where(
        rest < 2.0 ** -7, 2 * rest, torch.ones_like(rest))
    log_sum = (p.amax(1, keepdim=True).log()).abs().nan_to_num(0.0, posinf=0.0)
    base = s + 3 * E32 * log_sum
    lp_err = base + 5 * E32 * t.abs().nan_to_num(posinf=0.0) + 2 * E32 * lp.abs().nan_to_num(
        posinf=0.0)
    h = -plp.sum(1)
    h_err = base[:, 0] + (p * away * (e + s + (depth + 8) * E32)).sum(1) + 3 * E32 * h
    ids = tokens.cpu().long()
    ok = (ids >= 0) & (ids < V)
    at = torch.where(ok, ids, 0)[:, None]
    logp = torch.where(ok, lp.gather(1, at)[:, 0], float("nan"))
    return dict(lp=lp, p=p, logp=logp, entropy=h, lp_err=lp_err, logp_err=lp_err.gather(1, at)[:, 0],
                entropy_err=h_err, order=x.sort(dim=1, descending=True, stable=True).indices, s=s,
                e=e, rest=rest)


def logprobs_grad(r, tokens, dlogp, dentropy, temperature, dtype):
    """(dlogits, bound) of a case that logprobs gave."""
    p, lp, h = r["p"], r["lp"], r["entropy"][:, None]
    g = torch.zeros_like(h) if dlogp is None else f64(dlogp)[:, None]
    k = torch.zeros_like(h) if dentropy is None else f64(dentropy)[:, None]
    at = tokens.cpu().long()[:, None]
    g = g.masked_fill(r["logp"][:, None] == float("-inf"), 0.0)
    inner = (lp + h).masked_fill(p == 0, 0.0)
    d = -p * (g + k * inner)
    own = torch.zeros_like(p).scatter_(1, at, 1.0)
    d = (d + own * g) / temperature
    lp_err = r["lp_err"].masked_fill(p == 0, 0.0)
    # a power of two below 2^-126 is 0 on the device: p, its multiple by 1 / S <= 1, is off by
    # at most 2^-126 more there
    weight = g.abs() + k.abs() * (lp.nan_to_num(neginf=0.0).abs() + h.abs())
    size = p * weight
    err = size * (r["e"] + r["s"] + 12 * E32) + p * k.abs() * (lp_err + r["entropy_err"][:, None])
    err = err + 2.0 ** -126 * weight
    # the token's own 1 - p is one rounded difference, or the rest where p is the largest
    top = p == p.amax(1, keepdim=True)
    own_size = torch.where(top, (1 - p) * 8 * E32 + 4 * r["s"], 4 * E32 * torch.ones_like(p))
    err = (err + own * g.abs() * own_size) / temperature
    return d, rounded(d, dtype, err)

"""64-bit references of the sequence operators, with first-order error bounds.

Each reference follows the operator's definition in float64 on the CPU, one
sequence (or token) at a time. A bound is the sum of what the operator's
documented roundings can change: probabilities and score gradients rounded to
the tensors' type before a product, outputs rounded to it, products summed in
float32 (gamma = (n + 8) 2^-24 for n terms).
"""
from __future__ import annotations

import math

import torch

# unit roundoff: half a unit of the last of 8, 11 and 24 bits
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# absolute rounding of values below the type's normal range
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
E32 = 2.0 ** -24


def segments(cu_q, cu_k, k_lens):
    cu_q, cu_k = cu_q.tolist(), cu_k.tolist()
    for b in range(len(cu_q) - 1):
        lk = cu_k[b + 1] - cu_k[b] if k_lens is None else int(k_lens[b])
        yield slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b] + lk)


def attention(q, k, v, cu_q, cu_k, k_lens=None, scale=None, do=None):
    """dict of o, lse (and dq, dk, dv) with o_tol ... bounds, all float64."""
    dt = q.dtype
    u, tiny = U[dt], TINY[dt]
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    do = None if do is None else do.detach().cpu().double()
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    G = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    gamma = (d + 8) * E32
    out = {"o": torch.zeros_like(q), "lse": torch.full((hq, q.shape[0]), float("-inf"),
                                                       dtype=torch.float64)}
    out["o_tol"], out["lse_tol"] = torch.zeros_like(q), torch.zeros_like(out["lse"])
    if do is not None:
        for n, x in (("dq", q), ("dk", k), ("dv", v)):
            out[n], out[n + "_tol"] = torch.zeros_like(x), torch.zeros_like(x)
    for rows, keys in segments(cu_q, cu_k, k_lens):
        lq, lk = rows.stop - rows.start, keys.stop - keys.start
        if lq == 0 or lk == 0:
            continue
        see = torch.arange(lk)[None] <= torch.arange(lq)[:, None] + (lk - lq)
        any_key = see.any(1)
        for h in range(hq):
            Q, K, V = q[rows, h], k[keys, h // G], v[keys, h // G]
            S = scale * (Q @ K.T)
            # error of a score: float32 sum, and the exponent's rounding
            es = gamma * scale * (Q.abs() @ K.abs().T) + 4 * E32 * S.abs()
            es = (2 * es.masked_fill(~see, 0.0)).amax(1, keepdim=True) + 8 * E32
            S = S.masked_fill(~see, float("-inf"))
            m = torch.where(any_key, S.amax(1), torch.zeros(lq).double())[:, None]
            P = torch.exp(S - m)
            total = P.sum(1, keepdim=True)
            P = torch.where(total > 0, P / total, torch.zeros_like(P))
            O = P @ V
            av = P @ V.abs()
            n_err = (lk + 8) * E32
            o_tol = u * (av + O.abs()) + (es + n_err) * (av + O.abs()) \
                + 2 * tiny * (1 + V.abs().sum(0))
            out["o"][rows, h], out["o_tol"][rows, h] = O, o_tol
            lse = (m + torch.log(total))[:, 0]
            out["lse"][h, rows] = lse
            out["lse_tol"][h, rows] = es[:, 0] + n_err + 4 * E32 * lse.abs()
            if do is None:
                continue
            DO = do[rows, h]
            DP, delta = DO @ V.T, (DO * O).sum(1, keepdim=True)
            dS = P * (DP - delta)
            # delta comes from the rounded output, dP from a float32 sum
            e_delta = (DO.abs() * (o_tol + u * O.abs())).sum(1, keepdim=True) \
                + gamma * (DO.abs() * O.abs()).sum(1, keepdim=True)
            e_dp = gamma * (DO.abs() @ V.abs().T)
            e_p = 2 * es + n_err + 2 * E32 * (1 + lse.abs().nan_to_num(0, 0, 0))[:, None]
            e_ds = (u + e_p) * dS.abs() + P * (e_delta + e_dp) + tiny
            e_ds = torch.where(see, e_ds, torch.zeros_like(e_ds))
            n_q = (lq * G + 8) * E32
            dq = scale * dS @ K
            out["dq"][rows, h] = dq
            out["dq_tol"][rows, h] = scale * (e_ds + n_err * dS.abs()) @ K.abs() + u * dq.abs()
            out["dk"][keys, h // G] += scale * dS.T @ Q
            out["dk_tol"][keys, h // G] += scale * (e_ds + n_q * dS.abs()).T @ Q.abs()
            out["dv"][keys, h // G] += P.T @ DO
            e_pv = torch.where(see, (u + e_p + n_q) * P + tiny, torch.zeros_like(P))
            out["dv_tol"][keys, h // G] += e_pv.T @ DO.abs()
    for n in ("dq", "dk", "dv"):
        if n in out:
            out[n + "_tol"] += u * out[n].abs() + 2 * tiny
    return out


def rotary(x, positions, rot, f, m, interleaved, inverse):
    """y and its bound; f float64 frequencies, m the table's magnitude."""
    dt = x.dtype
    x = x.detach().cpu().double()
    a = positions.cpu().double()[:, None] * f
    c, s = (m * a.cos())[:, None], (m * a.sin())[:, None]
    s = -s if inverse else s
    y, size = x.clone(), torch.zeros_like(x)
    ia = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    ib = ia + 1 if interleaved else ia + rot // 2
    A, B = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = A * c - B * s, B * c + A * s
    size[..., ia] = size[..., ib] = m * (A.abs() + B.abs())
    # table and products rounded to float32, then the output
    return y, 4 * E32 * size + U[dt] * y.abs() + TINY[dt]


def policy(logits, actions, logp_old, advantages, logp_ref, weights, clip, kl_coef, temperature,
           grad=True):
    """loss, logp, dlogits and bounds, token by token."""
    dt = logits.dtype
    x = logits.detach().cpu().double()
    T, V = x.shape
    loss = loss_tol = 0.0
    logp, logp_tol = torch.zeros(T).double(), torch.zeros(T).double()
    dx, dx_tol = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(T):
        w, a, A = float(weights[t]), int(actions[t]), float(advantages[t])
        if w == 0.0:
            continue
        z = x[t] / temperature
        if math.isinf(z[a]) and z[a] < 0:
            logp[t] = float("-inf")
            if logp_ref is not None and kl_coef:
                loss = float("inf")
            loss += w * -min(0.0, (1 - clip[0]) * A)
            continue
        top = z.max()
        e = torch.exp(z - top)
        p = e / e.sum()
        lp = float(z[a] - top - torch.log(e.sum()))
        spread = float((z[a] - top).abs()) + 1.0
        # the exponents' rounding, a sum of V terms in a tree, the logarithm
        tol = E32 * (6 * spread + 8 * float((p * (top - z).clamp(max=100)).sum()) + 40
                     + 2 * abs(lp))
        logp[t], logp_tol[t] = lp, tol
        gap_old = lp - float(logp_old[t])
        r = math.exp(gap_old)
        er = tol + 4 * E32 * (abs(gap_old) + abs(lp) + 1)
        held = min(max(r, 1 - clip[0]), 1 + clip[1])
        term, slope = -min(r * A, held * A), (-r * A if r * A <= held * A else 0.0)
        e_term = abs(r * A) * er + 4 * E32 * abs(term)
        e_slope = abs(r * A) * er
        if logp_ref is not None:
            g = float(logp_ref[t]) - lp
            term += kl_coef * (math.exp(g) - g - 1)
            slope += kl_coef * (1 - math.exp(g))
            eg = tol + 4 * E32 * (abs(g) + abs(lp))
            e_term += abs(kl_coef) * (abs(math.exp(g) - 1) * eg + 8 * E32 * (math.exp(g) + abs(g) + 1))
            e_slope += abs(kl_coef) * math.exp(g) * (eg + 4 * E32)
        loss += w * term
        loss_tol += abs(w) * e_term + 2 * E32 * abs(w * term)
        if grad:
            s = w * slope / temperature
            es = abs(w) / temperature * e_slope + 4 * E32 * abs(s)
            hot = torch.zeros(V).double()
            hot[a] = 1.0
            dx[t] = s * (hot - p)
            # a probability's relative error: its exponent's rounding and the sum's
            ep = p * (tol + 8 * E32 * ((top - z).clamp(max=100) + 2))
            dx_tol[t] = es * (hot + p) + abs(s) * (ep + 2 * E32 * hot) + U[dt] * dx[t].abs() \
                + TINY[dt] + 1e-38
    return dict(loss=loss, loss_tol=loss_tol + E32 * abs(loss), logp=logp, logp_tol=logp_tol, dlogits=dx,
                dlogits_tol=dx_tol)


def worst(got, want, tol):
    """Largest |got - want| over its bound (equal values, infinities among
    them, count 0)."""
    got = got.detach().cpu().double()
    err = (got - want).abs()
    err = torch.where(got == want, torch.zeros_like(err), err)
    assert not bool(err.isnan().any()), "a value is NaN where the definition has a number"
    return float((err / (tol.double() + 1e-300)).max()) if err.numel() else 0.0

"""Performance cases of the operators of an expression proposer.

A proposer is a causal sequence model that emits prefix programs (the packed
token sequences of a pop.bin population) and is trained by a clipped policy
gradient on the losses that the constant fitter returns for them. Its
operators are measured here one call at a time:

  attention   causal attention over packed sequences, grouped heads; queries
              are whole sequences, or the newest token of each over a cache
  rotary      rotary positions of q and k in one call, and its inverse
  loss        clipped policy loss with a KL term over logits, with gradient

`own` selects the framework's entry points (cusr_amd.kernel.seq_ops) or the
plain form: elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
DEV = "cuda:0"


# ------------------------------------------------------------------- cases

def _attention(name, dtype, hq, hkv, d, n, lo, hi, *, spread="uniform", step=False, grad=False,
               fused=False, lengths=1):
    """n sequences of lo..hi tokens; step: one query each over a cache whose
    segments hold hi keys; fused: q, k, v are slices of one projection."""
    c = dict(op="attention", dtype=dtype, hq=hq, hkv=hkv, d=d, n=n, lo=lo, hi=hi, spread=spread,
             step=step, grad=grad, fused=fused, lengths=lengths)
    return dict(c, name=name) if name else c


def _rotary(name, dtype, hq, hkv, d, rot, tokens, table, *, interleaved=False, inverse=False,
            base=10000.0, scaling="", factor=1.0, original=0):
    c = dict(op="rotary", dtype=dtype, hq=hq, hkv=hkv, d=d, rot=rot, tokens=tokens, table=table,
             interleaved=interleaved, inverse=inverse, base=base, scaling=scaling, factor=factor,
             original=original)
    return dict(c, name=name) if name else c


def _loss(name, dtype, tokens, vocab, *, grad, forbidden=0.0, outside=0, temperature=1.0,
          kl_coef=0.04):
    """forbidden: share of -inf logits; outside: tokens that carry no weight
    (a prompt's, or padding)."""
    c = dict(op="loss", dtype=dtype, tokens=tokens, vocab=vocab, grad=grad, forbidden=forbidden,
             outside=outside, temperature=temperature, kl_coef=kl_coef)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the first steps of sampling one expression after a short prompt: launches and latency
        _attention("step_one", "fp16", 8, 2, 64, 1, 129, 129, step=True),
        # sampling under long contexts (data points and earlier expressions in the
        # prompt): one token for each of 24 sequences, ragged, over a large cache
        _attention("step_long", "bf16", 32, 8, 128, 24, 8000, 65536, step=True),
        # scoring a population: 16,384 expressions of at most 31 nodes (gen_synth C2)
        _attention("score_population", "bf16", 8, 4, 64, 16384, 1, 31),
        # a training step's attention on 8,192 expressions of at most 63 nodes (C3)
        _attention("train_population", "fp16", 8, 8, 64, 8192, 3, 63, grad=True),
        # scoring packed prompts of very different lengths, from one token to long
        _attention("score_prompts", "bf16", 32, 8, 128, 10, 1, 8191, spread="log", lengths=5),
        # a training step's attention on packed long sequences, q, k, v from one projection
        _attention("train_prompts", "bf16", 32, 8, 128, 5, 700, 4801, grad=True, fused=True),
        # positions of one sampling step at far positions, long-context scaling by parts
        _rotary("rotary_step", "bf16", 32, 8, 128, 128, 24, 131072, base=500000.0,
                scaling="parts", factor=16.0, original=8192),
        # positions of a packed batch of prompts
        _rotary("rotary_prompts", "bf16", 32, 8, 128, 128, 32768, 8192),
        # the gradient through positions that turn half of each head, pairs side by side
        _rotary("rotary_grad", "fp32", 12, 12, 96, 48, 8191, 4096, interleaved=True,
                inverse=True, scaling="linear", factor=2.0),
        # scoring a few tokens under a word vocabulary: loss alone
        _loss("loss_few", "fp32", 64, 32001, grad=False, temperature=0.8),
        # a training step's loss on a generation of 65,536 expressions (C5): a token is
        # one of 21 symbols, a third of which the grammar forbids at each place
        _loss("loss_generation", "bf16", 1300001, 21, grad=True, forbidden=0.33),
        # a training step's loss under a word vocabulary, a fifth of the tokens prompt
        _loss("loss_words", "bf16", 8192, 131071, grad=True, outside=1638),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _seconds(c):
    """Rough cost of a case: its work at a large copy's and product's rates."""
    w = work(c)
    return max(w["bytes"] / 4e12, w["flops"] / 5e14)


def _drawn(rng):
    kind = rng.choice(["step", "population", "population", "prompts", "prompts", "rotary",
                       "rotary", "symbols", "words", "words"])
    half = rng.choice(["bf16", "bf16", "fp16"])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 8] if hkv < 8 else [1, 2, 4])
    d = rng.choice([32, 64, 64, 80, 96, 128, 128])
    seed = rng.randint(1, 10 ** 6)
    if kind == "step":
        hi = _log(rng, 16, 65536)
        return _attention(None, half, hq, hkv, d, _log(rng, 1, 256), rng.randint(1, hi), hi,
                          step=True, lengths=seed)
    if kind == "population":
        hi = rng.choice([15, 31, 31, 63, 127])
        return _attention(None, half, hq, hkv, d, _log(rng, 16, 16384), rng.randint(1, 5), hi,
                          grad=rng.random() < 0.5, fused=rng.random() < 0.3, lengths=seed)
    if kind == "prompts":
        hi = _log(rng, 128, 8192)
        return _attention(None, half, hq, hkv, d, _log(rng, 1, 64), 1, hi,
                          spread=rng.choice(["uniform", "log"]), grad=rng.random() < 0.5,
                          fused=rng.random() < 0.3, lengths=seed)
    if kind == "rotary":
        rot = d if rng.random() < 0.5 else 2 * rng.randint(2, d // 2)
        scaling = rng.choice(["", "linear", "base", "parts"])
        return _rotary(None, rng.choice(["bf16", "fp16", "fp32"]), hq, hkv, d, rot,
                       _log(rng, 1, 32768), _log(rng, 1024, 131072),
                       interleaved=rng.random() < 0.5, inverse=rng.random() < 0.3,
                       base=rng.choice([10000.0, 500000.0]), scaling=scaling,
                       factor=rng.choice([2.0, 4.0, 16.0]) if scaling else 1.0, original=1024)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "symbols":
        tokens = _log(rng, 31, 1300001)
        return _loss(None, dtype, tokens, rng.randint(12, 80), grad=rng.random() < 0.7,
                     forbidden=rng.choice([0.0, 0.33]), outside=rng.choice([0, tokens // 10]),
                     temperature=rng.choice([1.0, 0.7]), kl_coef=rng.choice([0.0, 0.04]))
    tokens = _log(rng, 16, 16384)
    return _loss(None, dtype, tokens, _log(rng, 1000, 131072), grad=rng.random() < 0.6,
                 outside=rng.choice([0, tokens // 5]), temperature=rng.choice([1.0, 0.8]),
                 kl_coef=rng.choice([0.0, 0.1]))


def draw(rng):
    """One more case: every operator, direction and type; lengths from one
    token to 65,536 keys, sequences from one to 16,384, vocabularies from 12
    to 131,072 (log-uniform where the range is wide, rarely round)."""
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0.0), _seconds(c))
    while True:
        c = _drawn(rng)
        if _seconds(c) <= most[c["op"]]:
            return c


def _lengths(c):
    """Sequence lengths of an attention case, a function of the case alone."""
    rng = random.Random(c["lengths"])
    if c["spread"] == "log":
        out = [_log(rng, c["lo"], c["hi"]) for _ in range(c["n"])]
        out[0], out[-1] = c["lo"], c["hi"]
        return out
    return [rng.randint(c["lo"], c["hi"]) for _ in range(c["n"])]


def work(c):
    e = BYTES[c["dtype"]]
    if c["op"] == "attention":
        lens = _lengths(c)
        total = sum(lens)
        queries = c["n"] if c["step"] else total
        pairs = total if c["step"] else sum(n * (n + 1) // 2 for n in lens)
        q, kv = queries * c["hq"] * c["d"] * e, total * c["hkv"] * c["d"] * e
        if c["grad"]:      # q, k, v, do in; o, dq, dk, dv out
            return {"bytes": 4 * q + 4 * kv, "flops": 14 * c["d"] * c["hq"] * pairs}
        return {"bytes": 2 * q + 2 * kv, "flops": 4 * c["d"] * c["hq"] * pairs}
    if c["op"] == "rotary":
        heads = c["tokens"] * (c["hq"] + c["hkv"])
        rows = min(c["tokens"], c["table"])
        return {"bytes": 2 * heads * c["d"] * e + rows * c["rot"] * 4 + 4 * c["tokens"],
                "flops": 3 * heads * c["rot"]}
    n = (c["tokens"] - c["outside"]) * c["vocab"]
    # token, old and reference log-probability, advantage, weight in; log-probability out
    small = 24 * c["tokens"]
    if c["grad"]:
        return {"bytes": n * e + c["tokens"] * c["vocab"] * e + small, "flops": 8 * n}
    return {"bytes": n * e + small, "flops": 5 * n}


# ------------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _starts(lens):
    return [0] + torch.tensor(lens, dtype=torch.int64).cumsum(0).tolist()


def _prepare_attention(c, seed):
    g = _generator(seed)
    dt = DTYPES[c["dtype"]]
    lens = _lengths(c)
    random.Random(seed).shuffle(lens)
    n, hq, hkv, d = c["n"], c["hq"], c["hkv"], c["d"]
    s = dict(case=c, lens=lens, k_lens=None)
    if c["step"]:
        cap = c["hi"]
        s["q_starts"], s["k_starts"] = list(range(n + 1)), [b * cap for b in range(n + 1)]
        tq, tk = n, n * cap
        s["k_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    else:
        s["q_starts"] = s["k_starts"] = _starts(lens)
        tq = tk = s["q_starts"][-1]
    s["cu_q"] = torch.tensor(s["q_starts"], dtype=torch.int32, device=DEV)
    s["cu_k"] = torch.tensor(s["k_starts"], dtype=torch.int32, device=DEV) if c["step"] \
        else s["cu_q"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dt) \
            if math.prod(shape) < 1 << 28 else torch.empty(*shape, device=DEV, dtype=dt).normal_(
                generator=g)

    if c["fused"]:
        qkv = normal(tq, hq + 2 * hkv, d)
        s["q"], s["k"], s["v"] = qkv.split([hq, hkv, hkv], dim=1)
    else:
        s["q"], s["k"], s["v"] = normal(tq, hq, d), normal(tk, hkv, d), normal(tk, hkv, d)
    s["q"].mul_(1.5)          # scores with a spread of about 1.5 after the scale
    if c["step"]:             # what a cache holds beyond a sequence's length is not data
        for b in range(n):
            s["k"][s["k_starts"][b] + lens[b]:s["k_starts"][b + 1]] = float("nan")
            s["v"][s["k_starts"][b] + lens[b]:s["k_starts"][b + 1]] = float("nan")
    if c["grad"]:
        s["do"] = normal(tq, hq, d)
    return s


def _frequencies(c):
    """Frequencies in 64 bits and the table's magnitude, from the definition."""
    r = c["rot"]
    base = c["base"]
    if c["scaling"] == "base" and r > 2:
        base = base * c["factor"] ** (r / (r - 2.0))
    f = base ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    if c["scaling"] == "linear":
        return f / c["factor"], 1.0
    if c["scaling"] == "parts":
        keep = ((c["original"] * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        return f * (keep + (1.0 - keep) / c["factor"]), 0.1 * math.log(c["factor"]) + 1.0
    return f, 1.0


def _prepare_rotary(c, seed):
    g = _generator(seed)
    dt = DTYPES[c["dtype"]]
    f, m = _frequencies(c)
    if own:
        from cusr_amd.kernel import seq_ops

        table = seq_ops.rotary_table(c["rot"], c["table"], base=c["base"],
                                     scaling=c["scaling"] or None, factor=c["factor"],
                                     original=c["original"], device=DEV)
    else:
        a = torch.arange(c["table"], dtype=torch.float64, device=DEV)[:, None] * f.to(DEV)
        table = (torch.stack([a.cos(), a.sin()], dim=-1) * m).float()
    q = torch.randn(c["tokens"], c["hq"], c["d"], generator=g, device=DEV).to(dt)
    k = torch.randn(c["tokens"], c["hkv"], c["d"], generator=g, device=DEV).to(dt)
    if c["tokens"] <= 256:        # the newest token of each sequence
        pos = torch.randint(0, c["table"], (c["tokens"],), generator=g, device=DEV,
                            dtype=torch.int32)
    else:                         # packed sequences of a few lengths, each from 0
        rng, parts, left = random.Random(seed), [], c["tokens"]
        while left:
            n = min(left, rng.randint(1, c["table"]))
            parts.append(torch.arange(n, dtype=torch.int32))
            left -= n
        pos = torch.cat(parts).to(DEV)
    return dict(case=c, q=q, k=k, positions=pos, table=table)


def _prepare_loss(c, seed):
    g = _generator(seed)
    dt = DTYPES[c["dtype"]]
    T, V = c["tokens"], c["vocab"]
    logits = torch.empty(T, V, device=DEV, dtype=dt)
    actions = torch.empty(T, device=DEV, dtype=torch.int64)
    logp = torch.empty(T, device=DEV)
    step = max(1, (1 << 27) // V)
    for a in range(0, T, step):   # tokens sampled from the policy that the logits give
        b = min(T, a + step)
        z = torch.randn(b - a, V, generator=g, device=DEV) * 2.5
        if c["forbidden"]:
            no = torch.rand(b - a, V, generator=g, device=DEV) < c["forbidden"]
            no[torch.arange(b - a, device=DEV), torch.arange(a, b, device=DEV) % V] = False
            z.masked_fill_(no, float("-inf"))
        logits[a:b] = z
        z = logits[a:b].float() / c["temperature"]
        u = torch.rand(b - a, V, generator=g, device=DEV).clamp_(1e-7, 1 - 1e-7)
        act = (z - u.log().neg().log()).argmax(1)
        actions[a:b] = act
        logp[a:b] = z.gather(1, act[:, None])[:, 0] - z.logsumexp(1)
        del z, u
    ratio = torch.exp(0.15 * torch.randn(T, generator=g, device=DEV))
    # the loss has no derivative at the edges of the clip: ratios keep off them
    for edge in (0.8, 1.25):
        ratio = torch.where((ratio - edge).abs() < 1e-3, torch.full_like(ratio, 0.002 + edge),
                            ratio)
    logp_ref = logp + 0.2 * torch.randn(T, generator=g, device=DEV)
    advantages = torch.randn(T, generator=g, device=DEV)
    weights = torch.ones(T, device=DEV)
    if c["outside"]:
        weights[torch.randperm(T, generator=g, device=DEV)[:c["outside"]]] = 0.0
    weights /= T - c["outside"]
    return dict(case=c, logits=logits, actions=actions, logp_old=logp - ratio.log(),
                logp_ref=logp_ref, advantages=advantages, weights=weights)


def prepare(case, seed):
    return {"attention": _prepare_attention, "rotary": _prepare_rotary,
            "loss": _prepare_loss}[case["op"]](case, seed)


# --------------------------------------------------------- the framework's calls

def _run_own(s):
    from cusr_amd.kernel import seq_ops

    c = s["case"]
    if c["op"] == "attention":
        if not c["grad"]:
            return seq_ops.attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"],
                                     k_lens=s["k_lens"])
        o, lse = seq_ops.attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"],
                                   return_lse=True)
        return (o, *seq_ops.attention_grad(s["do"], s["q"], s["k"], s["v"], o, lse, s["cu_q"],
                                           s["cu_k"]))
    if c["op"] == "rotary":
        return seq_ops.rotary(s["q"], s["k"], s["positions"], s["table"],
                              interleaved=c["interleaved"], inverse=c["inverse"])
    args = (s["logits"], s["actions"], s["logp_old"], s["advantages"])
    kw = dict(logp_ref=s["logp_ref"], weights=s["weights"], clip=(0.2, 0.25),
              kl_coef=c["kl_coef"], temperature=c["temperature"])
    if c["grad"]:
        return seq_ops.policy_loss_grad(*args, **kw)     # loss, logp, dlogits
    return seq_ops.policy_loss(*args, **kw)              # loss, logp


# ----------------------------------------------------------------- plain forms

def _buckets(s):
    """Groups of sequences of about one length (powers of two) whose padded
    scores stay within a few GB."""
    c = s["case"]
    lq = [b - a for a, b in zip(s["q_starts"], s["q_starts"][1:])]
    by = {}
    for b, n in enumerate(s["lens"]):
        by.setdefault(max(n - 1, 0).bit_length(), []).append(b)
    for group in by.values():
        most = max(s["lens"][b] for b in group)
        rows = max(lq[b] for b in group)
        cost = c["hq"] * rows * most + 2 * c["hkv"] * most * c["d"]
        take = max(1, int(2 ** 31 // max(cost, 1)))
        for i in range(0, len(group), take):
            yield group[i:i + take], lq


def _rows(starts, lens, device):
    """Row numbers [n, longest] of a group's sequences, and which are theirs."""
    at = torch.arange(max(lens), device=device)
    inside = at[None] < torch.tensor(lens, device=device)[:, None]
    idx = torch.tensor(starts, device=device)[:, None] + at[None]
    return torch.where(inside, idx, torch.zeros_like(idx)), inside


def _plain_attention(s):
    c = s["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    G, scale = hq // hkv, 1.0 / math.sqrt(d)
    q, k, v = s["q"], s["k"], s["v"]
    o = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    if c["grad"]:
        dq, dk, dv = (torch.zeros(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
    for group, lq_all in _buckets(s):
        lq, lk = [lq_all[b] for b in group], [s["lens"][b] for b in group]
        n = len(group)
        qi, q_in = _rows([s["q_starts"][b] for b in group], lq, q.device)
        ki, k_in = _rows([s["k_starts"][b] for b in group], lk, q.device)
        Lq, Lk = qi.shape[1], ki.shape[1]

        def heads(x, idx, inside, g):      # [n, hkv, g * L, d] in 32 bits, padding zero
            y = x[idx].float().masked_fill(~inside[:, :, None, None], 0.0)
            return y.view(n, idx.shape[1], hkv, g, d).permute(0, 2, 3, 1, 4).reshape(
                n, hkv, g * idx.shape[1], d)

        Q, K, V = heads(q, qi, q_in, G), heads(k, ki, k_in, 1), heads(v, ki, k_in, 1)
        S = torch.matmul(Q, K.transpose(2, 3).contiguous()) * scale
        S = S.view(n, hkv, G, Lq, Lk)
        shift = torch.tensor(lk, device=q.device) - torch.tensor(lq, device=q.device)
        seen = (torch.arange(Lk, device=q.device)[None, None]
                <= torch.arange(Lq, device=q.device)[None, :, None] + shift[:, None, None])
        seen = (seen & k_in[:, None, :])[:, None, None]
        S.masked_fill_(~seen, float("-inf"))
        m = S.amax(-1, keepdim=True)
        m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
        P = torch.exp(S.sub_(m))
        del S
        total = P.sum(-1, keepdim=True)
        P = P / torch.where(total == 0, torch.ones_like(total), total)
        P = P.view(n, hkv, G * Lq, Lk)
        O = torch.matmul(P, V)

        def put(out, idx, inside, y, g):
            L = idx.shape[1]
            y = y.view(n, hkv, g, L, d).permute(0, 3, 1, 2, 4).reshape(n, L, hkv * g, d)
            out[idx[inside]] = y[inside].to(out.dtype)

        put(o, qi, q_in, O, G)
        if c["grad"]:
            DO = heads(s["do"], qi, q_in, G)
            put(dv, ki, k_in, torch.matmul(P.transpose(2, 3).contiguous(), DO), 1)
            DP = torch.matmul(DO, V.transpose(2, 3).contiguous())
            DS = DP.sub_((DO * O).sum(-1, keepdim=True)).mul_(P).mul_(scale)
            put(dq, qi, q_in, torch.matmul(DS, K), G)
            put(dk, ki, k_in, torch.matmul(DS.transpose(2, 3).contiguous(), Q), 1)
    return (o, dq, dk, dv) if c["grad"] else o


def _plain_rotary(s):
    c = s["case"]
    r = c["rot"]
    cs = s["table"][s["positions"].long()][:, None]
    cos, sin = cs[..., 0], -cs[..., 1] if c["inverse"] else cs[..., 1]
    out = []
    for x in (s["q"], s["k"]):
        y = x.float()
        if c["interleaved"]:
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., :r // 2], y[..., r // 2:r]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        out.append(torch.cat([turned, y[..., r:]], -1).to(x.dtype))
    return tuple(out)


def _plain_loss(s):
    c = s["case"]
    at = s["weights"].nonzero()[:, 0]
    x, w = s["logits"][at].float(), s["weights"][at]
    z = x / c["temperature"] if c["temperature"] != 1.0 else x
    z = z - z.amax(1, keepdim=True)
    act = s["actions"][at]
    e = torch.exp(z)
    total = e.sum(1)
    lp = z.gather(1, act[:, None])[:, 0] - total.log()
    ratio = torch.exp(lp - s["logp_old"][at])
    adv = s["advantages"][at]
    free, held = ratio * adv, ratio.clamp(0.8, 1.25) * adv
    apart = s["logp_ref"][at] - lp
    term = -torch.minimum(free, held) + c["kl_coef"] * (torch.exp(apart) - apart - 1.0)
    loss = (w * term).sum()
    logp = torch.zeros_like(s["weights"])
    logp[at] = lp
    if not c["grad"]:
        return loss, logp
    slope = torch.where(free <= held, -free, torch.zeros_like(free)) \
        + c["kl_coef"] * (1.0 - torch.exp(apart))
    slope = w * slope / c["temperature"]
    dx = e.mul_((-slope / total)[:, None])
    dx.scatter_add_(1, act[:, None], slope[:, None])
    grad = torch.zeros_like(s["logits"])
    grad[at] = dx.to(grad.dtype)
    return loss, logp, grad


def run(state):
    if own:
        return _run_own(state)
    return {"attention": _plain_attention, "rotary": _plain_rotary,
            "loss": _plain_loss}[state["case"]["op"]](state)


# ----------------------------------------------------------------- 64 bits

def _exact_attention(c, s):
    """Sequences of one length at a time, differentiated by autograd."""
    G, scale = c["hq"] // c["hkv"], c["d"] ** -0.5
    q, k, v = s["q"], s["k"], s["v"]
    outs = [torch.zeros(x.shape, dtype=torch.float64, device=DEV)
            for x in ((q, q, k, v) if c["grad"] else (q,))]
    by = {}
    for b, n in enumerate(s["lens"]):
        by.setdefault(n, []).append(b)
    for n, group in by.items():
        lq = 1 if c["step"] else n
        ki = torch.tensor([[s["k_starts"][b] + j for j in range(n)] for b in group], device=DEV)
        qi = ki if not c["step"] else torch.tensor([[s["q_starts"][b]] for b in group],
                                                   device=DEV)
        late = torch.ones(lq, n, dtype=torch.bool, device=DEV).triu(n - lq + 1)
        # a few heads at a time: 64-bit scores of a long sequence are large
        per = max(1, min(c["hkv"], int(2 ** 29 // max(1, len(group) * G * lq * n))))
        for h in range(0, c["hkv"], per):
            hk, hqs = slice(h, min(h + per, c["hkv"])), slice(h * G, min(h + per, c["hkv"]) * G)
            Q = q[qi][:, :, hqs].double().transpose(1, 2).contiguous()
            K = k[ki][:, :, hk].double().transpose(1, 2).contiguous()
            V = v[ki][:, :, hk].double().transpose(1, 2).contiguous()
            for x in (Q, K, V):
                x.requires_grad_(c["grad"])
            scores = (Q @ K.repeat_interleave(G, 1).transpose(2, 3).contiguous()) * scale
            O = scores.masked_fill(late, float("-inf")).softmax(-1) @ V.repeat_interleave(G, 1)
            pairs = [(outs[0], qi, hqs, O.detach())]
            if c["grad"]:
                DO = s["do"][qi][:, :, hqs].double().transpose(1, 2)
                grads = torch.autograd.grad(O, (Q, K, V), DO)
                pairs += [(outs[1], qi, hqs, grads[0]), (outs[2], ki, hk, grads[1]),
                          (outs[3], ki, hk, grads[2])]
            for out, idx, hh, val in pairs:
                out[:, hh][idx.flatten()] = val.transpose(1, 2).flatten(0, 1)
    return tuple(outs) if c["grad"] else outs[0]


def _exact_rotary(c, s):
    f, m = _frequencies(c)
    angle = s["positions"].double()[:, None] * f.to(DEV)
    if c["inverse"]:
        angle = -angle
    turn = torch.polar(torch.full_like(angle, m), angle)[:, None]
    out = []
    for x in (s["q"], s["k"]):
        y = x.double()
        head, tail = y[..., :c["rot"]], y[..., c["rot"]:]
        if c["interleaved"]:
            z = torch.view_as_complex(head.reshape(*head.shape[:2], -1, 2).contiguous()) * turn
            head = torch.view_as_real(z).flatten(-2)
        else:
            a, b = head.chunk(2, -1)
            z = torch.complex(a.contiguous(), b.contiguous()) * turn
            head = torch.cat([z.real, z.imag], -1)
        out.append(torch.cat([head, tail], -1))
    return tuple(out)


def _exact_loss(c, s):
    T, V = s["logits"].shape
    logp = torch.zeros(T, dtype=torch.float64, device=DEV)
    grad = torch.zeros(T, V, dtype=torch.float64, device=DEV) if c["grad"] else None
    loss = torch.zeros((), dtype=torch.float64, device=DEV)
    step = max(1, (1 << 26) // V)
    for a in range(0, T, step):
        b = min(T, a + step)
        x = s["logits"][a:b].double()
        w = s["weights"][a:b].double()
        x[w == 0] = 0.0
        x.requires_grad_(c["grad"])
        lp = (x / c["temperature"]).log_softmax(1)
        lp = lp.gather(1, s["actions"][a:b, None])[:, 0]
        r = (lp - s["logp_old"][a:b].double()).exp()
        adv = s["advantages"][a:b].double()
        gap = s["logp_ref"][a:b].double() - lp
        part = (w * (c["kl_coef"] * (gap.expm1() - gap)
                     - torch.minimum(r * adv, r.clamp(0.8, 1.25) * adv))).sum()
        if c["grad"]:
            grad[a:b] = torch.autograd.grad(part, x)[0]
        loss += part.detach()
        logp[a:b] = torch.where(w == 0, 0.0, lp.detach())
    return (loss, logp, grad) if c["grad"] else (loss, logp)


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "rotary": _exact_rotary,
            "loss": _exact_loss}[case["op"]](case, s)

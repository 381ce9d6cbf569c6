"""Performance cases of the layers around a proposer's attention.

A proposer of expressions (cusr_amd.demonstrator.proposer) is a causal model
over packed prefix programs. Beside attention, rotary positions and its policy
loss (perf/operators.py) a pass through it looks its symbols up, adds to the
residual stream and normalises it, multiplies by its weights, and asks for the
probabilities of the symbols that were written. One call, or one chain of
calls as a layer makes them, is measured at a time:

  embedding  rows of a table by token, scaled; the gradient of the table
  norm       root-mean-square norm of the residual's sum, and its gradient
  product    8-bit integer product with scales for each token and channel;
             its left side given, or quantised by rows, or by the norm before it
  logprobs   log-probabilities of given tokens, entropy and top alternatives,
             and the gradient of the first two

`own` selects the framework's entry points (cusr_amd.kernel.seq_layers) or the
plain form: elementary torch operations in 32 bits, in 64 for long sums.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
DEV = "cuda:0"
EPS = 1e-6


# ------------------------------------------------------------------- cases

def _named(name, c):
    return dict(c, name=name) if name else c


def _embedding(name, dtype, tokens, rows, width, *, grad=False, words=True, scale=1.0):
    """words: tokens spread as words of a text are, few of them very frequent;
    else as the symbols of programs, all about alike. grad: the table's
    gradient, in 32 bits, from a gradient of dtype."""
    return _named(name, dict(op="embedding", dtype=dtype, tokens=tokens, rows=rows, width=width,
                             grad=grad, words=words, scale=scale))


def _norm(name, dtype, tokens, width, *, stream="", out="", gain=True, grad=False):
    """stream: type of the residual stream that x is added to ("": none);
    out: type of the norm ("": x's)."""
    return _named(name, dict(op="norm", dtype=dtype, tokens=tokens, width=width, stream=stream,
                             out=out or dtype, gain=gain, grad=grad))


def _product(name, tokens, inner, outer, *, left="int8", dtype="bf16", out="bf16", stream=""):
    """[tokens, inner] times [inner, outer]. left: "int8" (given with its
    scales), "rows" (quantised from dtype) or "norm" (from the norm's pass)."""
    return _named(name, dict(op="product", tokens=tokens, inner=inner, outer=outer, left=left,
                             dtype=dtype, out=out, stream=stream))


def _logprobs(name, dtype, tokens, vocab, *, grad=False, top=0, forbidden=0.0, temperature=1.0):
    """forbidden: share of -inf logits. grad: the forward pass, then the
    gradient from those of the log-probabilities and entropies."""
    return _named(name, dict(op="logprobs", dtype=dtype, tokens=tokens, vocab=vocab, grad=grad,
                             top=top, forbidden=forbidden, temperature=temperature))


def listed():
    return [
        # one sampling step's symbols of 24 sequences under a word vocabulary: latency
        _embedding("embed_step", "bf16", 24, 131071, 4096, scale=64.0),
        # a training step's table gradient on 65,536 expressions (gen_synth C5) of 22
        # symbols: every row of the table gets tens of thousands of tokens
        _embedding("embed_generation_grad", "fp32", 1300001, 22, 128, grad=True, words=False),
        # a training step's table gradient on packed prompts of words
        _embedding("embed_prompts_grad", "bf16", 16383, 32001, 4096, grad=True, scale=64.0),
        # one sampling step's norm of 24 sequences: attention's output joins the stream
        _norm("norm_step", "bf16", 24, 4096, stream="bf16"),
        # scoring 65,536 expressions at the proposer's width, its stream in 32 bits
        _norm("norm_generation", "bf16", 1300001, 128, stream="fp32", gain=False),
        # a training step's norm on packed prompts, forward and backward
        _norm("norm_prompts_grad", "bf16", 16383, 4096, stream="bf16", grad=True),
        # one sampling step's q, k and v of 24 sequences: the weights' bytes count
        _product("product_step", 24, 4096, 6144, left="norm", stream="bf16"),
        # scoring a population of 16,384 expressions (C2) at the proposer's width
        _product("product_population", 262139, 128, 256, left="norm", stream="fp32"),
        # scoring packed prompts: a gated map's first product
        _product("product_prompts", 8192, 4096, 16384, left="rows"),
        # scoring a few tokens under a word vocabulary, with five alternatives to each
        _logprobs("logprobs_few", "fp32", 64, 32001, top=5, temperature=0.8),
        # an entropy-regularised training step on 65,536 expressions of 21 symbols, a
        # third of which the grammar forbids at each place
        _logprobs("logprobs_generation_grad", "bf16", 1300001, 21, grad=True, forbidden=0.33),
        # the same under a word vocabulary
        _logprobs("logprobs_words_grad", "bf16", 8192, 131071, grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _seconds(c):
    """Rough cost of a case: its work at a large copy's and product's rates."""
    w = work(c)
    return max(w["bytes"] / 4e12, w["flops"] / 2e15)


def _width(rng, lo, hi):
    """A model's width: mostly a multiple of 8 or 64, now and then odd."""
    n = _log(rng, lo, hi)
    step = rng.choice([1, 8, 64, 64])
    return max(step, n // step * step)


def _drawn(rng):
    op = rng.choice(["embedding", "norm", "product", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "embedding":
        words = rng.random() < 0.6
        return _embedding(None, dtype, _log(rng, 1, 1300001),
                          _log(rng, 1000, 131072) if words else rng.randint(12, 80),
                          _width(rng, 32, 8192), grad=rng.random() < 0.6, words=words,
                          scale=rng.choice([1.0, 0.125, 27.7]))
    if op == "norm":
        stream = rng.choice(["", "fp32", dtype])
        return _norm(None, dtype, _log(rng, 1, 1300001), _width(rng, 32, 16384), stream=stream,
                     out=rng.choice([dtype, "bf16"]), gain=rng.random() < 0.7,
                     grad=rng.random() < 0.5)
    if op == "product":
        left = rng.choice(["int8", "rows", "norm"])
        return _product(None, _log(rng, 1, 262139), _width(rng, 64, 16384), _width(rng, 32, 32768),
                        left=left, dtype=dtype, out=rng.choice(["bf16", "fp16", "fp32"]),
                        stream=rng.choice(["", "fp32", dtype]) if left == "norm" else "")
    small = rng.random() < 0.4
    return _logprobs(None, dtype, _log(rng, 1, 1300001 if small else 16384),
                     rng.randint(12, 80) if small else _log(rng, 1000, 131072),
                     grad=rng.random() < 0.5, top=rng.choice([0, 0, 1, 5, 10]),
                     forbidden=rng.choice([0.0, 0.33]), temperature=rng.choice([1.0, 0.7]))


def draw(rng):
    """One more case: every operator, direction and type; from one token to
    1,300,001, vocabularies from 12 to 131,072, widths from 32 to 16,384
    (log-uniform where the range is wide, rarely round)."""
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0.0), _seconds(c))
    while True:
        c = _drawn(rng)
        if _seconds(c) <= most[c["op"]]:
            return c


def work(c):
    n = c["tokens"]
    if c["op"] == "embedding":
        e, cells = BYTES[c["dtype"]], n * c["width"]
        if c["grad"]:              # the output's gradient in, the table's out
            return {"bytes": cells * e + 8 * n + 4 * c["rows"] * c["width"], "flops": 2 * cells}
        read = min(n, c["rows"]) * c["width"]
        return {"bytes": (read + cells) * e + 8 * n, "flops": cells}
    if c["op"] == "norm":
        cells, x, y = n * c["width"], BYTES[c["dtype"]], BYTES[c["out"]]
        h = BYTES[c["stream"]] if c["stream"] else 0
        forward = x + 2 * h + y    # x, the stream in and out, the norm
        if not c["grad"]:
            return {"bytes": cells * forward + 4 * c["width"], "flops": 5 * cells}
        # backward: gradients of the norm and of the stream, what was normalised; out:
        # the stream's gradient, and x's where its type is another
        back = y + (3 * h + (x if c["dtype"] != c["stream"] else 0) if h else 2 * x)
        return {"bytes": cells * (forward + back) + 8 * c["width"], "flops": 13 * cells}
    if c["op"] == "product":
        a, b = n * c["inner"], c["inner"] * c["outer"]
        left = {"int8": 1, "rows": BYTES[c["dtype"]], "norm": BYTES[c["dtype"]]}[c["left"]]
        if c["stream"]:
            left += 2 * BYTES[c["stream"]]
        return {"bytes": a * left + b + n * c["outer"] * BYTES[c["out"]] + 4 * (n + c["outer"]),
                "flops": 2 * n * b}
    cells = n * c["vocab"]
    read = cells * BYTES[c["dtype"]]
    small = 16 * n + 12 * n * c["top"]
    if c["grad"]:
        return {"bytes": 2 * read + small + 8 * n, "flops": 10 * cells}
    return {"bytes": read + small, "flops": 5 * cells}


# ------------------------------------------------------------------- inputs

def _normal(g, shape, dtype, spread=1.0):
    out = torch.empty(shape, device=DEV, dtype=dtype)
    return out.normal_(0.0, spread, generator=g)


def _prepare_embedding(c, g):
    dt, n = DTYPES[c["dtype"]], c["tokens"]
    if c["words"]:            # the frequency of a word falls with its rank
        u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
        tokens = (torch.exp(u * math.log(c["rows"] + 1.0)).long() - 1).clamp_(0, c["rows"] - 1)
    else:
        tokens = torch.randint(0, c["rows"], (n,), generator=g, device=DEV)
    if c["grad"]:
        return dict(tokens=tokens, dout=_normal(g, (n, c["width"]), dt, 0.02))
    return dict(tokens=tokens, table=_normal(g, (c["rows"], c["width"]), dt, 0.02))


def _prepare_norm(c, g):
    dt, shape = DTYPES[c["dtype"]], (c["tokens"], c["width"])
    s = dict(x=_normal(g, shape, dt, 0.5), residual=None, gain=None)
    if c["stream"]:
        s["residual"] = _normal(g, shape, DTYPES[c["stream"]], 1.5)
    if c["gain"]:
        s["gain"] = 1.0 + 0.2 * torch.randn(c["width"], generator=g, device=DEV)
    if c["grad"]:
        s["dy"] = _normal(g, shape, DTYPES[c["out"]], 0.1)
        if c["stream"]:
            s["dh"] = _normal(g, shape, DTYPES[c["stream"]], 0.1)
    return s


def _quantize(x):
    """Rows of 32-bit x as 8-bit integers and a scale each."""
    scale = x.abs().amax(1) / 127.0
    safe = torch.where(scale == 0, torch.ones_like(scale), scale)
    return torch.round(x / safe[:, None]).clamp_(-127, 127).to(torch.int8), scale


def _prepare_product(c, g):
    n, k, m = c["tokens"], c["inner"], c["outer"]
    s = dict(zip(("w", "w_scale"), _quantize(
        torch.randn(m, k, generator=g, device=DEV) / math.sqrt(k))))
    dt = DTYPES[c["dtype"]]
    if c["left"] == "int8":
        parts = [_quantize(torch.randn(min(8192, n - i), k, generator=g, device=DEV))
                 for i in range(0, n, 8192)]
        s["a"], s["a_scale"] = (torch.cat(p) for p in zip(*parts))
        return s
    s["x"] = _normal(g, (n, k), dt)
    if c["left"] == "norm":
        s["gain"] = 1.0 + 0.2 * torch.randn(k, generator=g, device=DEV)
        s["residual"] = _normal(g, (n, k), DTYPES[c["stream"]], 1.5) if c["stream"] else None
    return s


def _prepare_logprobs(c, g):
    dt, T, V = DTYPES[c["dtype"]], c["tokens"], c["vocab"]
    logits = torch.empty(T, V, device=DEV, dtype=dt)
    tokens = torch.empty(T, device=DEV, dtype=torch.int64)
    step = max(1, (1 << 27) // V)
    for a in range(0, T, step):   # tokens sampled from the policy that the logits give
        b = min(T, a + step)
        z = torch.randn(b - a, V, generator=g, device=DEV) * 2.5
        if c["forbidden"]:
            no = torch.rand(b - a, V, generator=g, device=DEV) < c["forbidden"]
            no[torch.arange(b - a, device=DEV), torch.arange(a, b, device=DEV) % V] = False
            z.masked_fill_(no, float("-inf"))
        logits[a:b] = z
        u = torch.rand(b - a, V, generator=g, device=DEV).clamp_(1e-7, 1 - 1e-7)
        tokens[a:b] = (logits[a:b].float() / c["temperature"] - u.log().neg().log()).argmax(1)
        del z, u
    s = dict(logits=logits, tokens=tokens)
    if c["grad"]:                 # a policy gradient with an entropy term, summed
        s["dlogp"] = torch.randn(T, generator=g, device=DEV)
        s["dentropy"] = torch.full((T,), -0.01, device=DEV)
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return dict({"embedding": _prepare_embedding, "norm": _prepare_norm,
                 "product": _prepare_product, "logprobs": _prepare_logprobs}[case["op"]](case, g),
                case=case)


# --------------------------------------------------------- the framework's calls

def _run_own(s):
    from cusr_amd.kernel import seq_layers as ops

    c = s["case"]
    if c["op"] == "embedding":
        if c["grad"]:
            return ops.embedding_grad(s["dout"], s["tokens"], c["rows"], scale=c["scale"])
        return ops.embedding(s["tokens"], s["table"], scale=c["scale"])
    if c["op"] == "norm":
        out = ops.rms_norm(s["x"], s["gain"], residual=s["residual"], eps=EPS,
                           dtype=DTYPES[c["out"]])
        if not c["grad"]:
            return out
        y, h = out if c["stream"] else (out, s["x"])
        d, dx, dgain = ops.rms_norm_grad(s["dy"], h, s["gain"], dh=s.get("dh"), eps=EPS,
                                         x_dtype=s["x"].dtype)
        outs = (y, h, d, dx) if c["stream"] else (y, d)
        return outs if dgain is None else outs + (dgain,)
    if c["op"] == "product":
        h = None
        if c["left"] == "int8":
            a, a_scale = s["a"], s["a_scale"]
        elif c["left"] == "rows":
            a, a_scale = ops.quantize_rows(s["x"])
        elif c["stream"]:
            a, a_scale, h = ops.rms_norm_int8(s["x"], s["gain"], residual=s["residual"], eps=EPS)
        else:
            a, a_scale = ops.rms_norm_int8(s["x"], s["gain"], eps=EPS)
        y = ops.int8_product(a, a_scale, s["w"], s["w_scale"], dtype=DTYPES[c["out"]])
        return y if h is None else (y, h)
    kw = dict(temperature=c["temperature"], top=c["top"])
    if not c["grad"]:
        return ops.token_logprobs(s["logits"], s["tokens"], **kw)
    *out, stats = ops.token_logprobs(s["logits"], s["tokens"], return_stats=True, **kw)
    return (*out, ops.token_logprobs_grad(s["logits"], s["tokens"], stats, out[1], s["dlogp"],
                                          s["dentropy"], temperature=c["temperature"]))


# ----------------------------------------------------------------- plain forms

def _plain_embedding(s):
    c = s["case"]
    if not c["grad"]:
        rows = s["table"][s["tokens"]]
        return rows if c["scale"] == 1.0 else (rows.float() * c["scale"]).to(rows.dtype)
    total = torch.zeros(c["rows"], c["width"], dtype=torch.float64, device=DEV)
    if c["rows"] <= 128:          # few symbols: which token is which, times the gradient
        symbols = torch.arange(c["rows"], device=DEV)
        for i in range(0, c["tokens"], 1 << 16):
            which = (symbols[:, None] == s["tokens"][i:i + (1 << 16)]).float()
            total += torch.matmul(which, s["dout"][i:i + (1 << 16)].float())
        return (total * c["scale"]).float()
    step = max(1, (1 << 27) // c["width"])
    for i in range(0, c["tokens"], step):
        total.index_add_(0, s["tokens"][i:i + step], s["dout"][i:i + step].double())
    return (total * c["scale"]).float()


def _plain_rms(x, residual, gain):
    """The stream's sum, in its type, its norm in 32 bits, and 1 / rms."""
    h = x if residual is None else (x.float() + residual.float()).to(residual.dtype)
    f = h.float()
    r = torch.rsqrt((f * f).mean(1, keepdim=True) + EPS)
    y = f * r
    return h, (y if gain is None else y * gain), r


def _plain_norm(s):
    c = s["case"]
    h, y, r = _plain_rms(s["x"], s["residual"], s["gain"])
    y = y.to(DTYPES[c["out"]])
    if not c["grad"]:
        return (y, h) if c["stream"] else y
    n = h.float() * r
    dy = s["dy"].float()
    dg = None if s["gain"] is None else (dy * n).sum(0, dtype=torch.float64).float()
    if s["gain"] is not None:
        dy = dy * s["gain"]
    d = (dy - n * (dy * n).mean(1, keepdim=True)) * r
    if c["stream"]:
        d = d + s["dh"].float()
        out = (y, h, d.to(h.dtype), d.to(s["x"].dtype))
    else:
        out = (y, d.to(h.dtype))
    return out if dg is None else out + (dg,)


def _plain_product(s):
    c = s["case"]
    h = None
    if c["left"] == "int8":
        a, a_scale = s["a"], s["a_scale"]
    elif c["left"] == "rows":
        a, a_scale = _quantize(s["x"].float())
    else:
        h, y, _ = _plain_rms(s["x"], s["residual"], s["gain"])
        a, a_scale = _quantize(y)
    y = torch.matmul(a.float(), s["w"].float().t().contiguous())
    y = (y * a_scale[:, None] * s["w_scale"]).to(DTYPES[c["out"]])
    return (y, h) if c["stream"] else y


def _ordered(x):
    """64-bit keys in the order of 32-bit values, a lower column before a
    higher one among equals."""
    b = (x + 0.0).view(torch.int32)
    b = torch.where(b < 0, b ^ 0x7fffffff, b).long()
    return (b << 32) - torch.arange(x.shape[1], device=x.device)


def _plain_logprobs(s):
    c = s["case"]
    x = s["logits"].float()
    z = x / c["temperature"] if c["temperature"] != 1.0 else x
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    p = e / total
    lp = z - log_total
    entropy = -(p * lp.masked_fill(p == 0, 0.0)).sum(1)
    logp = lp.gather(1, s["tokens"][:, None])[:, 0]
    out = (logp, entropy)
    if c["top"]:
        at = _ordered(x).topk(c["top"], dim=1).indices
        out += (lp.gather(1, at), at)
    if c["grad"]:
        lp = lp.masked_fill(p == 0, 0.0)
        d = -p * (s["dlogp"][:, None] + s["dentropy"][:, None] * (lp + entropy[:, None]))
        d.scatter_add_(1, s["tokens"][:, None], s["dlogp"][:, None])
        out += ((d / c["temperature"]).to(s["logits"].dtype),)
    return out


def run(state):
    if own:
        return _run_own(state)
    return {"embedding": _plain_embedding, "norm": _plain_norm, "product": _plain_product,
            "logprobs": _plain_logprobs}[state["case"]["op"]](state)


# ----------------------------------------------------------------- 64 bits

def _exact_embedding(c, s):
    if not c["grad"]:
        return s["table"].double().index_select(0, s["tokens"]) * c["scale"]
    # the rows of a token side by side, as differences of running sums would lose bits:
    # tokens in order, then each token's rows added by its segment
    order = s["tokens"].argsort(stable=True)
    counts = torch.bincount(s["tokens"], minlength=c["rows"])
    out = torch.empty(c["rows"], c["width"], dtype=torch.float64, device=DEV)
    step = max(1, (1 << 33) // (8 * c["tokens"]))
    for a in range(0, c["width"], step):
        part = s["dout"][:, a:a + step][order].double()
        out[:, a:a + step] = torch.segment_reduce(part, "sum", lengths=counts, axis=0, initial=0)
    return out * c["scale"]


def _rms64(x, gain):
    y = x * (x.square().sum(1, keepdim=True) / x.shape[1] + EPS) ** -0.5
    return y if gain is None else y * gain


def _exact_norm(c, s):
    parts, dgain = [], None
    step = max(1, (1 << 26) // c["width"])
    for a in range(0, c["tokens"], step):
        b = slice(a, a + step)
        h = s["x"][b].double()
        if c["stream"]:      # the stream holds the sum in its type, and that is normalised
            total = h + s["residual"][b].double()
            h = total.to(DTYPES[c["stream"]]).double()
        gain = None if s["gain"] is None else s["gain"].double()
        if not c["grad"]:
            y = _rms64(h, gain)
            parts.append((y, total) if c["stream"] else (y,))
            continue
        h.requires_grad_()
        if gain is not None:
            gain.requires_grad_()
        y = _rms64(h, gain)
        wanted = (h,) if gain is None else (h, gain)
        grads = torch.autograd.grad(y, wanted, s["dy"][b].double())
        d = grads[0]
        if gain is not None:
            dgain = grads[1] if dgain is None else dgain + grads[1]
        if c["stream"]:
            d = d + s["dh"][b].double()
            parts.append((y.detach(), total, d, d))
        else:
            parts.append((y.detach(), d))
    out = tuple(torch.cat(p) for p in zip(*parts))
    out = out if dgain is None else out + (dgain,)
    return out if len(out) > 1 else out[0]


def _exact_product(c, s):
    w = s["w"].double() * s["w_scale"].double()[:, None]
    w = w.t().contiguous()
    out, stream = [], []
    step = max(1, (1 << 28) // max(c["inner"], c["outer"]))
    for i in range(0, c["tokens"], step):
        b = slice(i, i + step)
        if c["left"] == "int8":
            a = s["a"][b].double() * s["a_scale"][b].double()[:, None]
        else:
            y = s["x"][b].double()
            if c["stream"]:
                y = y + s["residual"][b].double()
                stream.append(y)
                y = y.to(DTYPES[c["stream"]]).double()
            if c["left"] == "norm":
                y = _rms64(y, s["gain"].double())
            unit = y.abs().amax(1, keepdim=True).clamp(min=1e-300) / 127.0
            a = (y / unit).round() * unit
        out.append(a @ w)
    return (torch.cat(out), torch.cat(stream)) if c["stream"] else torch.cat(out)


def _exact_logprobs(c, s):
    T, V = s["logits"].shape
    parts = []
    step = max(1, (1 << 26) // V)
    for a in range(0, T, step):
        b = slice(a, a + step)
        x = s["logits"][b].double()
        if c["grad"]:
            x.requires_grad_()
        lp = (x / c["temperature"]).log_softmax(1)
        at = lp.gather(1, s["tokens"][b, None])[:, 0]
        entropy = torch.special.entr(lp.detach().exp()).sum(1)
        one = (at.detach(), entropy)
        if c["top"]:
            order = x.detach().sort(dim=1, descending=True, stable=True).indices[:, :c["top"]]
            one += (lp.detach().gather(1, order), order)
        if c["grad"]:
            # p log p is 0 where p is, and so is its derivative
            seen = lp > float("-inf")
            h = -(lp.exp() * lp.masked_fill(~seen, 0.0)).sum(1)
            aim = (at * s["dlogp"][b].double() + h * s["dentropy"][b].double()).sum()
            one += (torch.autograd.grad(aim, x)[0],)
        parts.append(one)
    return tuple(torch.cat(p) for p in zip(*parts))


def exact(case, seed):
    s = prepare(case, seed)
    return {"embedding": _exact_embedding, "norm": _exact_norm, "product": _exact_product,
            "logprobs": _exact_logprobs}[case["op"]](case, s)

"""A learned proposer of expressions: search by sampling, fitting, reinforcing.

    python -m cusr_amd.demonstrator.proposer [--rounds 10] [--population 1024] [--fused] [--int8]

A small causal model emits prefix programs symbol by symbol; KernelLM fits
their constants to the data on the device; the fits' losses become rewards,
and a clipped policy gradient with a KL term to the starting model trains the
proposer on them. The reference's search is genetic programming (its
demonstrator, cusr/demonstrator/pipeline.py); this shows the sequence operators
(cusr_amd.kernel.seq_ops) together as a search uses them:

  sampling   one symbol a step for the whole population: rotary positions,
             then attention of single tokens over a cache with room for the
             longest program
  scoring    the population as packed sequences of their own lengths: rotary
             positions, packed attention, the policy loss's log-probabilities
  training   the same under autograd, the policy loss's gradient through them

The layers around attention (cusr_amd.kernel.seq_layers) come in by choice: `fused`
makes each lookup, and each norm with the residual's addition before it, one kernel
in every pass; `int8` samples with 8-bit products; a trainer's entropy_coef holds up the
policy's entropy; alternatives() says what a policy would have written instead.

Symbols are pop.bin's: constants, variables, unary and binary operators. A
symbol that cannot complete a program of the allowed length or number of
constants has the logit -inf, in sampling and in training.
"""
from __future__ import annotations

import argparse
import math

import numpy as np
import torch

from cusr_amd.benchmark import popio
from cusr_amd.demonstrator.co_backend import KernelLM
from cusr_amd.kernel import seq_layers, seq_ops

BINARY = (1, 2, 3, 32)                  # + - * protected /
UNARY = (14, 15, 33, 34)                # sin cos clamped exp, square


class Symbols:
    """The vocabulary: symbol 0 opens a program and is never emitted."""

    def __init__(self, n_vars, unary=UNARY, binary=BINARY):
        nodes = [(popio.NODE_CONST, 0)] + [(popio.NODE_VAR, v) for v in range(n_vars)]
        nodes += [(popio.NODE_UFUNC, f) for f in unary] + [(popio.NODE_BFUNC, f) for f in binary]
        self.nt = np.array([-1] + [t for t, _ in nodes], np.int32)
        self.nv = np.array([0] + [v for _, v in nodes], np.float32)
        self.size = len(self.nt)
        self.const = 1
        arity = {popio.NODE_CONST: 0, popio.NODE_VAR: 0, popio.NODE_UFUNC: 1, popio.NODE_BFUNC: 2}
        self.arity = np.array([0] + [arity[t] for t, _ in nodes], np.int64)

    def program(self, symbols):
        """(nt, nv, ci) of one program's symbols, in prefix order."""
        s = np.asarray(symbols)
        nt = self.nt[s]
        is_const = nt == popio.NODE_CONST
        ci = np.where(is_const, np.cumsum(is_const) - 1, -1).astype(np.int32)
        return nt, self.nv[s], ci


class Population:
    """Sampled programs as packed sequences: symbols [T] end to end, offsets
    [M + 1], positions [T], and which symbols were allowed [T, V]."""

    def __init__(self, symbols, lengths, allowed):
        self.symbols, self.lengths, self.allowed = symbols, lengths, allowed
        cu = torch.zeros(len(lengths) + 1, dtype=torch.int32, device=symbols.device)
        cu[1:] = lengths.cumsum(0)
        self.offsets = cu
        of = torch.repeat_interleave(torch.arange(len(lengths), device=cu.device), lengths)
        self.sequence = of
        self.positions = (torch.arange(len(symbols), device=cu.device)
                          - cu[:-1][of].to(torch.int64)).to(torch.int32)
        # what the model reads: the symbol before, the opening one first
        self.inputs = torch.where(self.positions == 0, 0, symbols.roll(1))


class Proposer:
    """Causal model: layers of attention (grouped heads, rotary positions) and
    a gated map, parameters in float32, products in bfloat16. fused: lookups and norms
    as one kernel each (the same model, other roundings)."""

    def __init__(self, n_vars, *, width=128, layers=2, heads=4, kv_heads=2, longest=31,
                 most_constants=8, seed=0, device="cuda:0", fused=False):
        if width % heads or heads % kv_heads or (width // heads) % 8:
            raise ValueError("width must be heads times a multiple of 8, heads a multiple of "
                             "kv_heads")
        if longest < 1 or most_constants < 0:
            raise ValueError("longest must be positive and most_constants not negative")
        self.symbols = Symbols(n_vars)
        self.heads, self.kv_heads, self.d = heads, kv_heads, width // heads
        self.longest, self.most_constants, self.fused = longest, most_constants, fused
        self.device = torch.device(device)
        g = torch.Generator().manual_seed(seed)
        V, kv = self.symbols.size, kv_heads * self.d

        def matrix(rows, cols, scale=1.0):
            w = torch.randn(rows, cols, generator=g) * (scale / math.sqrt(rows))
            return w.to(self.device).requires_grad_()

        self.parameters = {"embed": matrix(V, width, math.sqrt(V) * 0.5),
                           "out": matrix(width, V, 0.5)}
        for i in range(layers):
            self.parameters.update({f"qkv{i}": matrix(width, width + 2 * kv),
                                    f"o{i}": matrix(width, width, 0.5),
                                    f"up{i}": matrix(width, 4 * width),
                                    f"down{i}": matrix(2 * width, width, 0.5)})
        self.layers, self.width = layers, width
        self.table = seq_ops.rotary_table(self.d, longest, device=self.device)
        arity = torch.from_numpy(self.symbols.arity).to(self.device)
        self.arity = arity

    @staticmethod
    def _norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)

    def _logits(self, inputs, positions, attend):
        """Logits [T, V] of input symbols; attend(layer, q, k, v) -> o."""
        if self.fused:
            return self._fused(inputs, positions, attend, None)
        p, bf = self.parameters, torch.bfloat16
        x = p["embed"][inputs]
        kv = self.kv_heads * self.d
        for i in range(self.layers):
            qkv = self._norm(x).to(bf) @ p[f"qkv{i}"].to(bf)
            q, k, v = (t.unflatten(1, (-1, self.d)) for t in qkv.split([self.width, kv, kv], 1))
            q, k = seq_ops.rotary(q, k, positions, self.table)
            o = attend(i, q, k, v)
            x = x + (o.flatten(1) @ p[f"o{i}"].to(bf)).float()
            a, b = (self._norm(x).to(bf) @ p[f"up{i}"].to(bf)).chunk(2, 1)
            x = x + ((a * torch.sigmoid(a) * b) @ p[f"down{i}"].to(bf)).float()
        return (self._norm(x).to(bf) @ p["out"].to(bf)).float()

    @torch.no_grad()
    def int8_weights(self):
        """The products' weights as 8-bit integers with a scale for each channel."""
        return {k: seq_layers.quantize_rows(v.t()) for k, v in self.parameters.items()
                if k != "embed"}

    def _fused(self, inputs, positions, attend, weights):
        """_logits with a kernel for each lookup, and for each norm and the addition before
        it. weights: None, or int8_weights, for 8-bit products of the norms' and the
        gated maps' outputs and attention's."""
        p, bf = self.parameters, torch.bfloat16

        def product(name, x):
            if weights is None:
                return x @ p[name].to(bf)
            return seq_layers.int8_product(*x, *weights[name])

        def normed(x, residual=None):
            if weights is not None:
                q, scale, *h = seq_layers.rms_norm_int8(x, residual=residual)
                return (q, scale), (h[0] if h else x)
            if residual is None:
                return seq_layers.rms_norm(x, dtype=bf), x
            return seq_layers.rms_norm(x, residual=residual, dtype=bf)

        n, x = normed(seq_layers.embedding(inputs, p["embed"]))
        kv = self.kv_heads * self.d
        for i in range(self.layers):
            qkv = product(f"qkv{i}", n)
            q, k, v = (t.unflatten(1, (-1, self.d)) for t in qkv.split([self.width, kv, kv], 1))
            q, k = seq_ops.rotary(q, k, positions, self.table)
            o = attend(i, q, k, v).flatten(1)
            n, x = normed(product(f"o{i}", o if weights is None else seq_layers.quantize_rows(o)),
                          x)
            a, b = product(f"up{i}", n).chunk(2, 1)
            m = a * torch.sigmoid(a) * b
            n, x = normed(product(f"down{i}", m if weights is None else seq_layers.quantize_rows(m)),
                          x)
        return product("out", n).float()

    def logits(self, pop):
        """Logits [T, V] of a population's symbols, forbidden ones -inf."""
        def attend(_, q, k, v):
            return seq_ops.attention(q, k, v, pop.offsets)

        return self._logits(pop.inputs, pop.positions, attend).masked_fill(~pop.allowed,
                                                                           float("-inf"))

    @torch.no_grad()
    def sample(self, M, generator=None, int8=False):
        """M programs, one symbol a step for all of them. int8: with 8-bit products, whose
        weights are made from the present parameters at the start. Programs come from
        that model's probabilities then, while Trainer and alternatives() take those of
        the bfloat16 one."""
        weights = self.int8_weights() if int8 else None
        dev, V, cap = self.device, self.symbols.size, self.longest
        shape = (self.layers, M, cap, self.kv_heads, self.d)
        keys, values = (torch.empty(shape, dtype=torch.bfloat16, device=dev) for _ in "kv")
        cu_q = torch.arange(M + 1, dtype=torch.int32, device=dev)
        cu_k, here = cu_q * cap, torch.full((M,), 0, dtype=torch.int32, device=dev)
        open_ = torch.ones(M, dtype=torch.int64, device=dev)      # subtrees still to write
        constants = torch.zeros(M, dtype=torch.int64, device=dev)
        last = torch.zeros(M, dtype=torch.int64, device=dev)
        symbols, allowed = [], []
        for t in range(cap):
            def attend(i, q, k, v):
                keys[i, :, t], values[i, :, t] = k, v
                return seq_ops.attention(q, keys[i].flatten(0, 1), values[i].flatten(0, 1), cu_q,
                                         cu_k, k_lens=here + 1)

            z = self._logits(last, here, attend) if weights is None else \
                self._fused(last, here, attend, weights)
            # what is left to write has to fit, with a leaf for every open subtree
            ok = open_[:, None] - 1 + self.arity[None] <= cap - t - 1
            ok[:, 0] = False
            ok[:, self.symbols.const] &= constants < self.most_constants
            z = z.masked_fill(~ok, float("-inf"))
            u = torch.rand(z.shape, generator=generator, device=dev).clamp_(1e-9, 1 - 1e-7)
            pick = (z - u.log().neg().log()).argmax(1)
            live = open_ > 0
            symbols.append(torch.where(live, pick, -1))
            allowed.append(ok)
            constants += live & (pick == self.symbols.const)
            open_ = torch.where(live, open_ - 1 + self.arity[pick], open_)
            last, here = pick, here + 1
            if not bool((open_ > 0).any()):
                break
        grid = torch.stack(symbols, 1)
        written = grid >= 0
        return Population(grid[written], written.sum(1), torch.stack(allowed, 1)[written])

    def programs(self, pop):
        """Each program's prefix arrays, for the fitter."""
        flat, cu = pop.symbols.cpu().numpy(), pop.offsets.cpu().numpy()
        return [self.symbols.program(flat[a:b]) for a, b in zip(cu[:-1], cu[1:])]

    @torch.no_grad()
    def alternatives(self, pop, top=3, temperature=1.0):
        """What the present policy makes of each of the population's symbols: (log-probability
        [T], entropy [T], the `top` likeliest symbols' log-probabilities [T, top], those
        symbols [T, top]); top: as many as there are symbols, and 64, at most. A symbol that is
        not allowed there comes last, at -inf."""
        return seq_layers.token_logprobs(self.logits(pop), pop.symbols, temperature=temperature,
                                         top=min(top, self.symbols.size, seq_layers.SEQ_MAX_TOP))

    @torch.no_grad()
    def log_probabilities(self, pop):
        """[T] of the population's symbols under the present parameters."""
        z, zero = self.logits(pop), torch.zeros(len(pop.symbols), device=self.device)
        return seq_ops.policy_loss(z, pop.symbols, zero, zero)[1]


class Trainer:
    """Clipped policy gradient with a KL term to the starting parameters.

    top: the share of a population, by reward, that is learnt from. A search
    wants the best program rather than a good mean, so it learns from the best
    few, by how far they pass the last of them; 1 learns from all, by how far
    they pass the mean.
    entropy_coef: weight of the policy's mean entropy over the symbols that are learnt
    from, which is added to what is reinforced.
    The ratio that is clipped is to the parameters' own log-probabilities before the step,
    formed with bfloat16 products: for programs that 8-bit products sampled it starts at 1
    too, and what the two models differ by is not made up for."""

    def __init__(self, proposer, *, rate=3e-3, clip=0.2, kl_coef=0.01, epochs=4, top=1.0,
                 entropy_coef=0.0):
        if not 0.0 < top <= 1.0:
            raise ValueError("top must be a share of the population")
        if not math.isfinite(entropy_coef):
            raise ValueError("entropy_coef must be finite")
        self.entropy_coef = entropy_coef
        self.p, self.clip, self.kl_coef, self.epochs = proposer, clip, kl_coef, epochs
        self.top = top
        self.start = {k: v.detach().clone() for k, v in proposer.parameters.items()}
        self.opt = torch.optim.Adam(list(proposer.parameters.values()), lr=rate)

    def _reference(self, pop):
        now = self.p.parameters
        self.p.parameters = self.start
        try:
            return self.p.log_probabilities(pop)
        finally:
            self.p.parameters = now

    def step(self, pop, rewards):
        """Reinforce a population by its programs' rewards [M]; returns the
        loss of each epoch."""
        r = torch.as_tensor(rewards, dtype=torch.float32, device=self.p.device)
        least = r.mean() if self.top == 1.0 else torch.quantile(r, 1.0 - self.top)
        used = torch.ones_like(r) if self.top == 1.0 else (r >= least).float()
        advantage = ((r - least) / (r[used > 0].std(unbiased=False) + 1e-6))[pop.sequence]
        old, ref = self.p.log_probabilities(pop), self._reference(pop)
        # every program that is learnt from counts alike, whatever its length
        weights = (used / pop.lengths.float() / used.sum())[pop.sequence]
        losses = []
        for _ in range(self.epochs):
            z = self.p.logits(pop)
            loss, _ = seq_ops.policy_loss(z, pop.symbols, old, advantage,
                                          logp_ref=ref, weights=weights,
                                          clip=(self.clip, self.clip), kl_coef=self.kl_coef)
            if self.entropy_coef:
                entropy = seq_layers.token_logprobs(z, pop.symbols)[1]
                loss = loss - self.entropy_coef * (weights * entropy).sum()
            self.opt.zero_grad(set_to_none=True)
            loss.backward()
            self.opt.step()
            losses.append(loss.detach())
        return [float(x) for x in losses]


def rewards_of(losses, y):
    """1 / (1 + normalised root mean square error), 0 for a failed fit."""
    spread = float(np.std(y)) or 1.0
    rmse = np.sqrt(np.maximum(np.asarray(losses, np.float64), 0.0))
    return np.where(np.isfinite(rmse), 1.0 / (1.0 + rmse / spread), 0.0)


def search(X, y, *, rounds=10, population=1024, max_iter=10, seed=0, proposer=None, trainer=None,
           backend=None, log=print, fused=False, int8=False):
    """Rounds of sampling (int8: with 8-bit products), fitting and training; fused: of the
    proposer that is made here when none is given. Returns (best, history): the
    best program as (loss, (nt, nv, ci), constants), (inf, None, None) when none
    was fitted, and each round's mean and best reward."""
    X, y = np.asarray(X, np.float64), np.asarray(y, np.float64)
    p = proposer or Proposer(X.shape[1], seed=seed, fused=fused)
    tr = trainer or Trainer(p, top=0.1, kl_coef=0.05)
    lm = backend or KernelLM(max_iter=max_iter)
    g = torch.Generator(device=p.device).manual_seed(seed)
    rng = np.random.default_rng(seed)
    best, history = (math.inf, None, None), []
    for i in range(rounds):
        pop = p.sample(population, generator=g, **({"int8": True} if int8 else {}))
        native = p.programs(pop)
        inits = [rng.normal(size=int(np.sum(n[0] == popio.NODE_CONST))) for n in native]
        fits = lm.fit_batch(None, inits, X, y, native=native)
        losses = np.array([f.final_loss for f in fits])
        r = rewards_of(losses, y)
        j = int(np.argmax(r))
        if losses[j] < best[0]:
            best = (float(losses[j]), native[j], fits[j].constants)
        history.append((float(r.mean()), float(r.max())))
        tr.step(pop, r)
        if log:
            log(f"round {i}: mean reward {r.mean():.3f}, best {r.max():.4f}, best loss so far "
                f"{best[0]:.3g}, mean length {float(pop.lengths.float().mean()):.1f}")
    return best, history


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--rounds", type=int, default=10)
    ap.add_argument("--population", type=int, default=1024)
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--fused", action="store_true", help="lookups and norms as one kernel each")
    ap.add_argument("--int8", action="store_true", help="sample with 8-bit products")
    a = ap.parse_args(argv)
    rng = np.random.default_rng(a.seed)
    X = rng.uniform(-2, 2, size=(512, 2))
    y = 1.5 * np.sin(0.8 * X[:, 0]) * X[:, 1] + 0.5
    best, _ = search(X, y, rounds=a.rounds, population=a.population, seed=a.seed, fused=a.fused,
                     int8=a.int8)
    if best[1] is None:
        print("no program was fitted")
        return
    nt, nv, _ = best[1]
    print(f"best loss {best[0]:.3g}: nodes {nt.tolist()}, values {nv.tolist()}, constants "
          f"{np.round(best[2], 4).tolist()}")


if __name__ == "__main__":
    main()

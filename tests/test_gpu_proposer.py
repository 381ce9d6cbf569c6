"""The learned proposer: sampling, scoring and training with the sequence
operators, and the fitter in between."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from cusr_amd.benchmark import popio
from cusr_amd.demonstrator import proposer as pr

gpu = pytest.mark.gpu


def test_symbols_and_rewards():
    s = pr.Symbols(2)
    assert s.size == 1 + 1 + 2 + 4 + 4 and s.arity[0] == 0
    # (c0 * x1) + sin(c1)
    add, mul, sin = (int(np.flatnonzero((s.nt == t) & (s.nv == f))[0]) for t, f in
                     ((popio.NODE_BFUNC, 1), (popio.NODE_BFUNC, 3), (popio.NODE_UFUNC, 14)))
    x1 = int(np.flatnonzero((s.nt == popio.NODE_VAR) & (s.nv == 1))[0])
    nt, nv, ci = s.program([add, mul, s.const, x1, sin, s.const])
    assert nt.tolist() == [3, 3, 1, 0, 2, 1] and nv.tolist() == [1, 3, 0, 1, 14, 0]
    assert ci.tolist() == [-1, -1, 0, -1, -1, 1]
    r = pr.rewards_of([0.0, 4.0, np.inf, np.nan], np.array([-2.0, 2.0]))
    assert r.tolist() == [1.0, 0.5, 0.0, 0.0]
    with pytest.raises(ValueError):
        pr.Proposer(2, width=100, heads=3, device="cpu")
    with pytest.raises(ValueError):
        pr.Trainer(None, top=0.0)


@gpu
def test_sampled_programs_are_whole():
    p = pr.Proposer(3, longest=21, most_constants=3, seed=2)
    pop = p.sample(500, generator=torch.Generator(device="cuda").manual_seed(1))
    lengths = pop.lengths.tolist()
    assert len(lengths) == 500 and min(lengths) >= 1 and max(lengths) <= 21
    for nt, nv, ci in p.programs(pop):
        need = 1
        for i, t in enumerate(nt):
            assert need > 0
            need += {0: -1, 1: -1, 2: 0, 3: 1}[int(t)]
        assert need == 0 and int(np.sum(nt == popio.NODE_CONST)) <= 3
    assert bool(pop.allowed.gather(1, pop.symbols[:, None]).all())
    assert pop.positions.max() < 21 and int(pop.offsets[-1]) == len(pop.symbols)


@gpu
def test_single_tokens_agree_with_packed_sequences():
    """The probabilities of the symbols as they were sampled, one token at a
    time over the cache, and of the packed population: two orders of the same
    bfloat16 products."""
    p = pr.Proposer(2, longest=31, seed=3)
    seen = {}

    def keep(inputs, positions, attend, real=p._logits):
        z = real(inputs, positions, attend)
        seen.setdefault(int(positions[0]), z)
        return z

    p._logits = keep
    pop = p.sample(64, generator=torch.Generator(device="cuda").manual_seed(5))
    del p._logits
    packed = p.logits(pop)
    steps = torch.stack([seen[t] for t in range(len(seen))], 1)
    at = steps[pop.sequence, pop.positions.long()].masked_fill(~pop.allowed, float("-inf"))
    a, b = packed.log_softmax(1), at.log_softmax(1)
    # a layer's bfloat16 roundings (eight of 2^-8 a layer, relative) on logits of order 1
    far, size = (x[pop.allowed].abs().max().item() for x in (a - b, packed))
    assert far <= 2 * 8 * 2.0 ** -8 * max(size, 1.0)
    lp = p.log_probabilities(pop)
    want = a.gather(1, pop.symbols[:, None])[:, 0]
    assert torch.allclose(lp, want, atol=1e-4)


@gpu
def test_training_favours_what_is_rewarded():
    """Programs that use the sine are rewarded: their share grows."""
    p = pr.Proposer(2, longest=15, seed=1)
    tr = pr.Trainer(p)
    g = torch.Generator(device="cuda").manual_seed(7)
    sin = int(np.flatnonzero((p.symbols.nt == popio.NODE_UFUNC) & (p.symbols.nv == 14))[0])
    share = []
    for _ in range(6):
        pop = p.sample(512, generator=g)
        has = torch.zeros(512, device="cuda").index_add_(
            0, pop.sequence, (pop.symbols == sin).float()) > 0
        share.append(float(has.float().mean()))
        losses = tr.step(pop, has.float())
        assert all(np.isfinite(losses))
    print("share of programs with a sine:", [round(s, 3) for s in share], flush=True)
    assert share[-1] > share[0] + 0.1
    for v in p.parameters.values():
        assert bool(v.isfinite().all()) and v.grad is not None and bool(v.grad.isfinite().all())


@gpu
def test_search_fits_what_it_samples():
    rng = np.random.default_rng(0)
    X = rng.uniform(-2, 2, size=(128, 2))
    y = 1.25 * X[:, 0] - 0.5
    best, history = pr.search(X, y, rounds=3, population=256, seed=4, log=None)
    assert len(history) == 3 and best[0] < 1e-8        # c0 * x0 + c1 is among the first
    assert all(0 <= m <= b <= 1 for m, b in history)
    nt, nv, ci = best[1]
    assert int(np.sum(nt == popio.NODE_CONST)) == len(best[2])

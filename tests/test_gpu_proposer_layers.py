"""The learned proposer with the layers around attention, which come in by choice."""
from __future__ import annotations

import pytest
import torch

from cusr_amd.demonstrator import proposer as pr

pytestmark = pytest.mark.gpu


def test_fused_layers_are_the_same_model():
    """Lookups and norms as one kernel each: the same logits and gradients but for the
    roundings of two orders of the same products."""
    a, b = (pr.Proposer(2, longest=31, seed=3, fused=f) for f in (False, True))
    pop = a.sample(200, generator=torch.Generator(device="cuda").manual_seed(5))
    za, zb = a.logits(pop), b.logits(pop)
    size = max(za[pop.allowed].abs().max().item(), 1.0)
    # a layer's bfloat16 roundings (eight of 2^-8 a layer, relative), on both sides
    tol = 2 * 8 * 2.0 ** -8 * size
    assert (za - zb)[pop.allowed].abs().max().item() <= tol
    w = torch.randn(len(pop.symbols), generator=torch.Generator().manual_seed(1)).cuda()
    for z in (za, zb):
        lp = z.log_softmax(1).gather(1, pop.symbols[:, None])[:, 0]
        (lp * w).sum().backward()
    for n, x in a.parameters.items():
        g, h = x.grad.double(), b.parameters[n].grad.double()
        # sixteen roundings of 2^-8 forward and as many back, at random among many terms
        assert float((g - h).norm()) <= 32 * 2.0 ** -8 * float(g.norm()), n


def test_sampling_with_8_bit_products():
    """Whole programs as ever, and logits near those of bfloat16."""
    p = pr.Proposer(3, longest=21, most_constants=3, seed=2, fused=True)
    pop = p.sample(300, generator=torch.Generator(device="cuda").manual_seed(1), int8=True)
    for nt, _, _ in p.programs(pop):
        need = 1
        for t in nt:
            assert need > 0
            need += {0: -1, 1: -1, 2: 0, 3: 1}[int(t)]
        assert need == 0
    assert bool(pop.allowed.gather(1, pop.symbols[:, None]).all())

    def attend(_, q, k, v):
        from cusr_amd.kernel import seq_ops
        return seq_ops.attention(q, k, v, pop.offsets)

    with torch.no_grad():
        z = p._fused(pop.inputs, pop.positions, attend, None).double()
        z8 = p._fused(pop.inputs, pop.positions, attend, p.int8_weights()).double()
    # Both sides of a product are off by up to half a step of 127 in their rows' largest value,
    # which is some three times the others' size: 3 sqrt(2) / (127 sqrt(12)), about 1 %,
    # of each of nine products one after the other.
    assert float((z8 - z).norm()) <= 9 * 0.01 * 1.5 * float(z.norm())


def test_alternatives_and_entropy():
    p = pr.Proposer(2, longest=15, seed=1, fused=True)
    pop = p.sample(128, generator=torch.Generator(device="cuda").manual_seed(3))
    logp, entropy, tl, ti = p.alternatives(pop, top=4)
    z = p.logits(pop).detach().double()
    lp = z.log_softmax(1)
    want = lp.gather(1, pop.symbols[:, None])[:, 0]
    assert torch.allclose(logp.double(), want, atol=1e-5)
    h = -(lp.exp() * lp.masked_fill(~pop.allowed, 0.0)).sum(1)
    assert torch.allclose(entropy.double(), h, atol=1e-5)
    assert torch.equal(ti, z.sort(dim=1, descending=True, stable=True).indices[:, :4])
    assert torch.allclose(tl.double(), lp.gather(1, ti), atol=1e-5)
    assert p.alternatives(pop, top=99)[3].shape[1] == p.symbols.size


def test_training_with_an_entropy_term():
    """The term's gradient goes to the parameters: the same step with and without it
    differs, and its value is what autograd takes off the loss."""
    losses = []
    for coef in (0.0, 0.5):
        p = pr.Proposer(2, longest=15, seed=1, fused=True)
        pop = p.sample(128, generator=torch.Generator(device="cuda").manual_seed(3))
        entropy = float(p.alternatives(pop)[1][pop.positions == 0].mean())
        tr = pr.Trainer(p, entropy_coef=coef, epochs=1)
        losses.append(tr.step(pop, torch.rand(128, generator=torch.Generator().manual_seed(2)))[0])
        assert all(bool(v.grad.isfinite().all()) for v in p.parameters.values())
    assert entropy > 0 and losses[1] < losses[0]
    with pytest.raises(ValueError):
        pr.Trainer(None, entropy_coef=float("nan"))


def test_gradient_of_the_entropy_term():
    """What the term adds to the parameters' gradients is its own gradient, formed by torch from
    the same logits, with the sign that raises the entropy."""
    coef = 4.0

    def fresh():
        p = pr.Proposer(2, longest=15, seed=1, fused=True)
        return p, p.sample(128, generator=torch.Generator(device="cuda").manual_seed(3))

    def gradients(p):
        return {n: v.grad.double() for n, v in p.parameters.items()}

    def entropy_of(p, pop):
        lp = p.logits(pop).log_softmax(1)
        h = -(lp.exp() * lp.masked_fill(~pop.allowed, 0.0)).sum(1)
        weights = (1.0 / pop.lengths.float() / len(pop.lengths))[pop.sequence]
        return (weights * h).sum()

    grads, after = [], []
    for c in (0.0, coef):
        p, pop = fresh()
        rewards = torch.rand(128, generator=torch.Generator().manual_seed(2))
        pr.Trainer(p, entropy_coef=c, epochs=1, rate=1e-3).step(pop, rewards)
        grads.append(gradients(p))
        with torch.no_grad():
            after.append(float(entropy_of(p, pop)))
    p, pop = fresh()
    before = entropy_of(p, pop)
    (-coef * before).backward()
    for n, own in gradients(p).items():
        a, b = grads[0][n], grads[1][n]
        # three passes back, each with sixteen roundings of 2^-8
        tol = 16 * 2.0 ** -8 * float(a.norm() + b.norm() + own.norm())
        assert tol < 0.5 * float(own.norm()), n      # a gradient that is not there would show
        assert float((b - a - own).norm()) <= tol, n
    assert after[1] > before.item() and after[1] > after[0]


def test_the_command_line(capsys):
    """One small round with everything by choice."""
    pr.main(["--rounds", "1", "--population", "64", "--fused", "--int8"])
    out = capsys.readouterr().out
    assert "round 0" in out and ("best loss" in out or "no program" in out)

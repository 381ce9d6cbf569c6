"""Sequence operators where layouts, launches and values meet their edges: groups
as wide as a tile, other orders of arguments and memory, values that have no
finite term."""
from __future__ import annotations

import pytest
import torch

import seq_reference as ref
from test_gpu_seq import BF, DEV, F32, FP, _say, check, cu, normal, policy_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from cusr_amd.kernel import seq_ops
    return seq_ops


# ------------------------------------------------------------------ attention

# many query heads a key head, lengths of the long kernels: a copy's rows then begin
# inside a query's heads
WIDE_GROUPS = [
    ([300, 90], 32, 1, 128, BF),
    ([257], 32, 1, 80, FP),
    ([200, 120], 64, 2, 96, BF),
    ([130, 131], 32, 1, 64, BF),
    ([140, 200], 32, 1, 24, FP),
    ([190], 64, 1, 128, BF),
    ([100, 85], 48, 2, 128, FP),
    ([160], 128, 1, 96, BF),
    ([90] * 70, 128, 4, 128, FP),          # enough blocks of 128 keys to fill the chip
]


@pytest.mark.parametrize("lens,hq,hkv,d,dtype", WIDE_GROUPS)
def test_attention_wide_groups(ops, lens, hq, hkv, d, dtype):
    T, c = sum(lens), cu(lens)
    _say("wide groups", lens[:4], hq, hkv, d, dtype)
    q, k, v, do = (normal((T, h, d), dtype, i + 1) for i, h in enumerate((hq, hkv, hkv, hq)))
    o, lse = ops.attention(q, k, v, c, return_lse=True)
    g = ops.attention_grad(do, q, k, v, o, lse, c)
    r = ref.attention(q, k, v, c, c, do=do)
    for n, x in zip(("o", "lse", "dq", "dk", "dv"), (o, lse, *g)):
        check(n, x, r[n], r[n + "_tol"])


# ---------------------------------------------------------------- policy loss

@pytest.mark.parametrize("dtype", [F32, BF, FP])
@pytest.mark.parametrize("V", [24, 700, 9001])
def test_policy_without_a_kl_term(ops, V, dtype):
    """A KL coefficient of 0 is no KL term, however far the reference's
    log-probabilities lie: the same bits as without them."""
    c = policy_case(8, V, dtype, 3)
    c["logp_ref"][0] += 100.0
    c["logp_ref"][1] = float("inf")
    c["logits"][2, c["actions"][2]] = float("-inf")
    for fn in (ops.policy_loss, ops.policy_loss_grad):
        got, want = fn(**c, kl_coef=0.0), fn(**dict(c, logp_ref=None))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert bool(got[0].isfinite()) and bool(got[-1][3:].isfinite().all())
    assert bool(got[2].isfinite().all())


@pytest.mark.parametrize("V", [24, 700, 9001])
def test_policy_action_that_every_policy_forbids(ops, V):
    """An action at -inf whose old or reference log-probability is -inf too: ratio
    0, no gradient, and a KL term that is infinite, not NaN."""
    c = policy_case(8, V, BF, 5)
    c["logits"][2, c["actions"][2]] = float("-inf")
    want = ops.policy_loss_grad(**dict(c, logp_ref=None))
    assert bool(want[0].isfinite()) and not bool(want[2][2].any())
    old = c["logp_old"].clone()
    old[2] = float("-inf")
    got = ops.policy_loss_grad(**dict(c, logp_ref=None, logp_old=old))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    ref_ = c["logp_ref"].clone()
    ref_[2] = float("-inf")
    want = ops.policy_loss_grad(**c, kl_coef=0.1)
    got = ops.policy_loss_grad(**dict(c, logp_ref=ref_, logp_old=old), kl_coef=0.1)
    assert float(got[0]) == float("inf") == float(want[0])
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


# ------------------------------------------------------------------- launches

def test_more_rows_than_one_axis_of_threads(ops):
    """Log-probabilities of more than 2^22 rows, 1,024 threads to each: every row
    has those of the same row of a small call."""
    few, V, T = policy_case(1024, 300, BF, 9), 300, (1 << 22) + 5
    at = torch.arange(T, device=DEV) % 1024
    c = {n: x[at] for n, x in few.items()}
    want = ops.policy_loss(**few, kl_coef=0.1)
    loss, logp = ops.policy_loss(**c, kl_coef=0.1)
    assert torch.equal(logp, want[1][at])
    rest = ops.policy_loss(**{n: x[:5] for n, x in few.items()}, kl_coef=0.1)[0].double()
    total = want[0].double() * (T // 1024) + rest
    # each loss is rounded once to float32, from a sum in 64 bits
    tol = ref.E32 * (want[0].double().abs() * (T // 1024) + rest.abs() + total.abs())
    check("loss", loss, total.cpu(), tol.cpu())


def test_more_sequences_than_one_axis_of_threads(ops):
    """2^24 sequences, four key heads, nearly all empty: the last are worked on
    like the first."""
    n = (1 << 24) + 40
    c = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
    lens = [3, 1, 2]
    c[1:], c[-2], c[-1] = 3, 4, 6
    q, k, v, do = (normal((6, h, 64), BF, i + 1) for i, h in enumerate((8, 4, 4, 8)))
    o, lse = ops.attention(q, k, v, c, return_lse=True)
    g = ops.attention_grad(do, q, k, v, o, lse, c)
    r = ref.attention(q, k, v, cu(lens), cu(lens), do=do)
    for name, x in zip(("o", "lse", "dq", "dk", "dv"), (o, lse, *g)):
        check(name, x, r[name], r[name + "_tol"])

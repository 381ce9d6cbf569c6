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


# ------------------------------------------------------------- gradient's sums

# (queries, keys) of one sequence, and of how many short ones beside it
SKEWED = [
    ((700, 700), (10, 10), 40, 4, 4, 64),
    ((150, 150), (5, 5), 100, 4, 2, 128),
    ((45, 45), (5, 5), 100, 8, 2, 64),
    ((40, 60), (2, 3), 30, 32, 4, 64),
    ((40, 100), (40, 100), 5, 4, 4, 128),
    ((129, 129), (1, 1), 300, 1, 1, 32),
]


def skewed(long, short, n, hq, hkv, d):
    """Sharp attention, whose outputs are as large as single values: what rounding
    them takes away is then large beside the gradients of scores."""
    lq, lk = [short[0]] * n, [short[1]] * n
    lq.insert(n // 2, long[0])
    lk.insert(n // 2, long[1])
    cq = cu(lq)
    ck = cq if lq == lk else cu(lk)
    q, do = normal((sum(lq), hq, d), BF, 1, 4.0), normal((sum(lq), hq, d), BF, 2)
    k, v = (normal((sum(lk), hkv, d), BF, i) for i in (3, 4))
    rows = slice(sum(lq[:n // 2]), sum(lq[:n // 2]) + long[0])
    keys = slice(sum(lk[:n // 2]), sum(lk[:n // 2]) + long[1])
    return (q, k, v), do, cq, ck, rows, keys


def off_by(got, want):
    """Root mean square error over that of rounding the exact values alone."""
    def rms(x):
        return float(x.square().mean().sqrt())
    return rms(got.cpu().double() - want) / rms(want.to(got.dtype).double() - want)


@pytest.mark.parametrize("long,short,n,hq,hkv,d", SKEWED)
def test_gradient_of_a_long_sequence_among_short_ones(ops, long, short, n, hq, hkv, d):
    """Each sequence's gradient is as good as its type, whatever the others': the
    roundings of P, dS and the result are sqrt(2) of one, and 1.75 leaves a fifth."""
    x, do, cq, ck, rows, keys = skewed(long, short, n, hq, hkv, d)
    o, lse = ops.attention(*x, cq, ck, return_lse=True)
    got = ops.attention_grad(do, *x, o, lse, cq, ck)
    r = ref.attention(*x, cq, ck, do=do)
    for name, g, at in zip(("dq", "dk", "dv"), got, (rows, keys, keys)):
        f = off_by(g[at], r[name][at])
        _say(f"  {long} among {n} of {short} {name}: {f:.3f} of a rounding")
        assert f <= 1.75, name
        check(name, g, r[name], r[name + "_tol"])


def test_gradient_from_a_copy_of_lse(ops):
    """lse may be copied, moved or saved: the gradient has the same bits, and
    loses nothing of its precision."""
    x, do, cq, ck, rows, keys = skewed((300, 300), (12, 12), 9, 4, 2, 64)
    for c, a in ((cq, x), (cu([300]), [t[rows] for t in x])):
        d = do if c is cq else do[rows]
        o, lse = ops.attention(*a, c, return_lse=True)
        want = ops.attention_grad(d, *a, o, lse, c)
        for copy in (lse.clone(), lse.detach(), lse.cpu().to(DEV)):
            got = ops.attention_grad(d, *a, o, copy, c)
            assert all(torch.equal(p, q) for p, q in zip(got, want))


# --------------------------------------------------------------------- rotary

@pytest.mark.parametrize("d,rot", [(48, 32), (20, 6)])
def test_rotary_positions_beyond_32_bits(ops, d, rot):
    """A 64-bit position outside the table gives NaN also where its low 32 bits lie
    inside it; one inside turns like the same in 32 bits."""
    table = ops.rotary_table(rot, 64)
    far = [2 ** 32, 2 ** 32 + 5, -2 ** 32, -2 ** 32 + 1, 2 ** 40 + 63, -2 ** 63, 2 ** 63 - 1]
    q, k = normal((len(far) + 3, 2, d), BF, 1), normal((len(far) + 3, 1, d), BF, 2)
    near = [0, 63, 5]
    pos = torch.tensor(near + far, device=DEV)
    a, b = ops.rotary(q, k, pos, table)
    assert bool(a[3:, :, :rot].isnan().all()) and bool(b[3:, :, :rot].isnan().all())
    assert torch.equal(a[..., rot:], q[..., rot:]) and torch.equal(b[..., rot:], k[..., rot:])
    few = ops.rotary(q[:3], k[:3], pos[:3].to(torch.int32), table)
    assert torch.equal(a[:3], few[0]) and torch.equal(b[:3], few[1])
    step = torch.tensor(near + [9], device=DEV).repeat(2)[::2]      # every other of them
    want = ops.rotary(q[:4], None, step.to(torch.int32), table)
    assert torch.equal(ops.rotary(q[:4], None, step, table), want)


def test_rotary_in_place_is_seen_by_autograd(ops):
    """What an earlier graph saved and rotary overwrites makes its backward raise,
    as torch's own operations in place do."""
    table, pos = ops.rotary_table(32, 64), torch.arange(4, device=DEV)
    for which in "qk":
        q, k = normal((4, 2, 32), F32, 1), normal((4, 1, 32), F32, 2)
        x = q if which == "q" else k
        w = torch.ones_like(x, requires_grad=True)
        y = (w * x).sum()
        before = x._version
        ops.rotary(q, k, pos, table, inplace=True)
        assert x._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.backward()
    with torch.inference_mode():
        q = normal((4, 2, 32), F32, 1).clone()
        want = ops.rotary(q, None, pos, table)
        assert torch.equal(ops.rotary(q, None, pos, table, inplace=True), want)


# --------------------------------------------------------------- empty layouts

def test_attention_empty_tensors_of_any_layout(ops):
    """No rows or no keys, as slices whose strides the kernels would not read."""
    def odd(n, h):
        return torch.empty(n, h, 67, dtype=BF, device=DEV)[..., 3:]

    q, k = normal((7, 4, 64), BF, 1), odd(0, 2)
    o, lse = ops.attention(q, k, odd(0, 2), cu([7]), cu([0]), return_lse=True)
    assert not bool(o.any()) and bool((lse == float("-inf")).all())
    g = ops.attention_grad(q, q, k, k, o, lse, cu([7]), cu([0]))
    assert [x.shape for x in g] == [q.shape, k.shape, k.shape] and not bool(g[0].any())
    q, k = odd(0, 4), normal((5, 2, 64), BF, 2)
    o, lse = ops.attention(q, k, k, cu([0]), cu([5]), return_lse=True)
    assert o.shape == (0, 4, 64) and lse.shape == (4, 0)
    g = ops.attention_grad(odd(0, 4), q, k, k, odd(0, 4), lse, cu([0]), cu([5]))
    assert [x.shape for x in g] == [q.shape, k.shape, k.shape]
    assert not any(bool(x.any()) for x in g)


# ------------------------------------------------------------- hidden values

# (queries, keys) of sequences, heads, head size, type: every kernel and split, with
# queries that see no key among them
HIDDEN = [
    ([(40, 40), (9, 9), (64, 64), (33, 33)], 2, 2, 64, BF),        # short, formed once
    ([(31, 31), (20, 20), (64, 64), (7, 7)], 8, 2, 64, FP),        # short, up to 256 rows
    ([(60, 40), (10, 64), (30, 50), (5, 3)], 4, 2, 40, BF),
    ([(100, 100), (3, 3), (2, 2), (5, 5)], 16, 1, 32, BF),         # rows of many waves
    ([(25, 25), (64, 64), (50, 50)], 3, 1, 128, FP),
    ([(300, 300), (140, 140), (97, 97)], 4, 2, 64, BF),            # long
    ([(260, 260), (200, 200)], 8, 1, 128, FP),
    ([(90, 200), (150, 100), (130, 130)], 4, 1, 96, BF),
    ([(129, 129)] * 40, 16, 8, 128, BF),                           # blocks of 128 keys
    ([(5, 1500), (2, 900), (40, 700)], 8, 2, 64, BF),              # few rows, split
    ([(3, 1111), (7, 600)], 4, 1, 128, FP),
    ([(6, 300), (2, 260)], 32, 8, 96, BF),
]


def planted(x, rows, value, seed):
    """x with `value` in one column of each of its `rows`, in some of its heads."""
    y = x.clone()
    g = torch.Generator().manual_seed(seed)
    for r in rows:
        h = int(torch.randint(x.shape[1], (1,), generator=g))
        y[r, h, int(torch.randint(x.shape[2], (1,), generator=g))] = value
    return y


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("pairs,hq,hkv,d,dtype", HIDDEN)
def test_hidden_values_do_not_reach(ops, pairs, hq, hkv, d, dtype, value):
    """A key or value that is not finite leaves the outputs and gradients of queries
    before it as they are without it, and a query or output gradient those of keys
    after it: all of them, to the bounds of finite inputs."""
    _say("hidden", pairs[:4], hq, hkv, d, dtype, value)
    lq, lk = [a for a, _ in pairs], [b for _, b in pairs]
    cq = cu(lq)
    ck = cq if lq == lk else cu(lk)
    q, do = (normal((sum(lq), hq, d), dtype, i) for i in (1, 2))
    k, v = (normal((sum(lk), hkv, d), dtype, i) for i in (3, 4))
    r = ref.attention(q, k, v, cq, ck, do=do)
    q_at = torch.repeat_interleave(torch.arange(len(lq)), torch.tensor(lq))
    k_at = torch.repeat_interleave(torch.arange(len(lk)), torch.tensor(lk))
    # what query row i sees: keys of its sequence up to number lim (within it)
    lim = torch.cat([torch.arange(a) + b - a for a, b in pairs])
    number = torch.cat([torch.arange(b) for _, b in pairs])
    sees = (q_at[:, None] == k_at[None]) & (number[None] <= lim[:, None])
    G = hq // hkv

    def run(q, k, v, do):
        o, lse = ops.attention(q, k, v, cq, ck, return_lse=True)
        assert torch.equal(o.isnan(), ops.attention(q, k, v, cq, ck).isnan())
        return (o, lse) + ops.attention_grad(do, q, k, v, o, lse, cq, ck)

    def hold(got, name, clean):
        """Checks the elements that nothing visible makes other than finite."""
        x = got.detach().cpu().double()
        assert bool(x[clean].isfinite().all()), name
        check(name, torch.where(clean, x, r[name]), r[name], r[name + "_tol"])

    # the last keys of each sequence, and one that half of the queries see
    keys, rows = [], []
    for b, n in enumerate(lk):
        keys += sorted({sum(lk[:b]) + n - 1, sum(lk[:b]) + max(n - 1 - min(lq[b], n) // 2, 0)})
    for b, n in enumerate(lq):
        rows += sorted({sum(lq[:b]), sum(lq[:b]) + n // 3, sum(lq[:b]) + n // 2})
    for name, x, at in (("k", k, keys), ("v", v, keys), ("q", q, rows), ("do", do, rows)):
        a = dict(q=q, k=k, v=v, do=do)
        a[name] = planted(x, at, value, len(at))
        odd = ~a[name].cpu().float().isfinite()
        o, lse, dq, dk, dv = run(**a)
        if name in "kv":
            # [row, key head]: sees such a place; with a value only its columns of o
            hit = (sees.double() @ odd.any(2).double()) > 0
            col = (sees.double() @ odd.double().flatten(1)).view(len(q_at), hkv, d) > 0
            row_hit = hit.repeat_interleave(G, 1)[..., None].expand(-1, -1, d)
            o_hit = col.repeat_interleave(G, 1) if name == "v" else row_hit
            hold(o, "o", ~o_hit)
            hold(dq, "dq", ~row_hit)
            if name == "v":
                assert not bool(o.cpu()[o_hit].isfinite().any())
                hold(dv, "dv", torch.ones_like(r["dv"], dtype=torch.bool))
                check("lse", lse, r["lse"], r["lse_tol"])
            # a key is clean when no row that sees it is hit
            key_hit = (sees.double().T @ hit.double()) > 0
            hold(dk, "dk", ~key_hit[..., None].expand(-1, -1, d))
            if name == "k":
                hold(dv, "dv", ~key_hit[..., None].expand(-1, -1, d))
        else:
            hit = odd.any(2)                                     # [row, head]
            by_head = hit.view(len(q_at), hkv, G).any(2)
            key_hit = (sees.double().T @ by_head.double()) > 0
            row_hit = hit[..., None].expand(-1, -1, d)
            hold(o, "o", ~row_hit if name == "q" else torch.ones_like(row_hit))
            hold(dq, "dq", ~row_hit)
            clean = ~key_hit[..., None].expand(-1, -1, d)
            hold(dk, "dk", clean)
            hold(dv, "dv", clean)

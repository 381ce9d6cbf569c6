"""Sequence operators against their 64-bit definitions, through the public
entry points (cusr_amd.kernel.seq_ops), at the sizes, masks, strides and types
where they can go wrong."""
from __future__ import annotations

import math

import pytest
import torch

import seq_reference as ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from cusr_amd.kernel import seq_ops
    return seq_ops


def _say(*a):
    print(*a, flush=True)


def cu(lens):
    return torch.tensor([0] + list(lens), dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)


def normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def check(name, got, want, tol):
    w = ref.worst(got, want, tol)
    _say(f"  {name}: {w:.3f} of its bound")
    assert w <= 1.0, (name, w)


# ------------------------------------------------------------------ attention

# lengths of packed sequences, query heads, key heads, head size, type
PACKED = [
    ([1], 1, 1, 64, BF),
    ([1, 2, 3], 2, 1, 64, FP),
    ([31, 32, 33], 4, 2, 32, BF),
    ([64, 65, 1, 0, 127], 3, 1, 128, FP),
    ([0, 0, 5, 0], 8, 8, 8, BF),
    ([300, 0, 5], 6, 2, 80, BF),
    ([17] * 70, 4, 4, 64, FP),
    ([3, 1, 2] * 50, 5, 1, 96, BF),
    ([511, 257], 8, 2, 128, BF),
    ([600], 4, 1, 64, FP),
    ([129, 128, 127], 2, 2, 40, BF),
    ([1025, 40], 2, 1, 128, BF),
    ([33, 95], 7, 1, 64, BF),
    ([900, 333, 1], 8, 8, 128, FP),
    ([200] * 40, 8, 8, 128, BF),           # enough blocks of 128 keys to fill the chip
    ([130, 300, 1] * 14, 16, 8, 96, FP),
    ([128, 0, 129, 193] * 9, 6, 6, 64, BF),
]


@pytest.mark.parametrize("lens,hq,hkv,d,dtype", PACKED)
def test_attention_packed(ops, lens, hq, hkv, d, dtype):
    T = sum(lens)
    _say("attention", lens[:8], hq, hkv, d, dtype)
    q, k, v, do = (normal((T, h, d), dtype, i + 1) for i, h in enumerate((hq, hkv, hkv, hq)))
    c = cu(lens)
    o, lse = ops.attention(q, k, v, c, return_lse=True)
    dq, dk, dv = ops.attention_grad(do, q, k, v, o, lse, c)
    r = ref.attention(q, k, v, c, c, do=do)
    for n, x in (("o", o), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        check(n, x, r[n], r[n + "_tol"])


# (queries, keys) of each sequence, room beyond the keys
STEPS = [
    ([(1, 1)], 0, 4, 2, 64, FP),
    ([(1, 129)], 7, 8, 2, 64, FP),
    ([(1, 5), (1, 64), (1, 65), (1, 1000)], 24, 8, 2, 128, BF),
    ([(1, 3000), (1, 1)], 0, 16, 1, 128, BF),
    ([(1, 700)] * 5, 9, 3, 3, 80, BF),
    ([(1, 257), (1, 0), (1, 32)], 3, 6, 2, 32, FP),
    ([(1, 4100)], 100, 32, 8, 128, BF),
    ([(5, 70), (2, 2), (3, 1), (0, 9)], 4, 4, 2, 64, BF),
    ([(40, 333), (7, 0), (100, 20)], 2, 4, 1, 128, FP),
    ([(1, 50)] * 300, 14, 8, 4, 64, BF),
    ([(4, 2100), (1, 33)], 5, 20, 1, 128, BF),
]


@pytest.mark.parametrize("pairs,room,hq,hkv,d,dtype", STEPS)
def test_attention_newest_tokens(ops, pairs, room, hq, hkv, d, dtype):
    """Queries that are the last of their keys, over cache segments whose spare
    rows hold NaN; queries without a key give 0 and -inf."""
    _say("newest", pairs[:4], room, hq, hkv, d, dtype)
    lq, lk = [a for a, _ in pairs], [b for _, b in pairs]
    cq, ck = cu(lq), cu([n + room for n in lk])
    kl = torch.tensor(lk, dtype=torch.int32, device=DEV)
    q, do = (normal((sum(lq), hq, d), dtype, i) for i in (1, 2))
    k, v = (normal((int(ck[-1]), hkv, d), dtype, i) for i in (3, 4))
    rows = torch.zeros(int(ck[-1]), dtype=torch.bool, device=DEV)
    for s, n in zip(ck.tolist(), lk):
        rows[s:s + n] = True
    k[~rows], v[~rows] = float("nan"), float("nan")
    o, lse = ops.attention(q, k, v, cq, ck, k_lens=kl, return_lse=True)
    dq, dk, dv = ops.attention_grad(do, q, k, v, o, lse, cq, ck, k_lens=kl)
    r = ref.attention(q, k, v, cq, ck, kl, do=do)
    for n, x in (("o", o), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        check(n, x, r[n], r[n + "_tol"])
    assert not bool(dk[~rows].any()) and not bool(dv[~rows].any())


# up to 64 rows and keys: one tile or two of each, fewer keys than queries among them
SHORT = [
    ([(60, 40), (64, 64), (33, 20), (20, 50), (1, 64), (64, 1), (40, 33)], 0, 2, 2, 64, BF),
    ([(30, 20), (32, 32), (16, 16), (17, 17), (9, 31), (1, 1)], 5, 4, 2, 64, FP),
    ([(64, 60), (31, 31), (32, 3), (50, 50)], 4, 1, 1, 128, BF),
    ([(7, 7), (8, 2), (3, 33), (8, 40)], 1, 16, 2, 40, FP),
]


@pytest.mark.parametrize("pairs,room,hq,hkv,d,dtype", SHORT)
def test_attention_short_pairs(ops, pairs, room, hq, hkv, d, dtype):
    test_attention_newest_tokens(ops, pairs, room, hq, hkv, d, dtype)


def test_attention_strides_and_order(ops):
    """q, k, v as slices of one projection, heads before rows, and a layout
    that the kernels do not read directly give the same bits."""
    lens, hq, hkv, d = [70, 3, 130], 4, 2, 64
    T, c = sum(lens), cu(lens)
    qkv = normal((T, hq + 2 * hkv, d), BF, 5)
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    do = normal((T, hq, d), BF, 6)
    o, lse = ops.attention(q.contiguous(), k.contiguous(), v.contiguous(), c, return_lse=True)
    g = ops.attention_grad(do, q, k, v, o, lse, c)

    def other(x, how):
        if how == "slices":
            return x
        if how == "heads first":
            return x.transpose(0, 1).contiguous().transpose(0, 1)
        y = torch.empty(x.shape[0], x.shape[1], d + 1, dtype=x.dtype, device=DEV)[..., 1:]
        y.copy_(x)                       # rows off 16-byte boundaries
        return y

    for how in ("slices", "heads first", "off boundary"):
        a = [other(x, how) for x in (q, k, v)]
        o2, l2 = ops.attention(*a, c, return_lse=True)
        assert torch.equal(o, o2) and torch.equal(lse, l2), how
        g2 = ops.attention_grad(other(do, how), *a, other(o, how), lse, c)
        assert all(torch.equal(x, y) for x, y in zip(g, g2)), how


def test_attention_far_strides(ops):
    """Rows and heads beyond 2^16 elements apart, where offsets take 64 bits."""
    lens, hq, hkv, d = [40, 9, 64, 25], 4, 2, 64
    T, c = sum(lens), cu(lens)
    q, k, v, do = (normal((T, h, d), BF, i + 40) for i, h in enumerate((hq, hkv, hkv, hq)))

    def far(x):
        y = torch.empty(x.shape[0], 70000, dtype=x.dtype, device=DEV)[:, :x.shape[1] * d]
        return y.view(x.shape[0], x.shape[1], d).copy_(x)

    def far_heads(x):
        y = torch.empty(x.shape[1], 1100, d, dtype=x.dtype, device=DEV)[:, :x.shape[0]]
        return y.transpose(0, 1).copy_(x)

    r = ref.attention(q, k, v, c, c, do=do)
    for how in (far, far_heads):
        x, y, z, w = (how(t) for t in (q, k, v, do))
        o, lse = ops.attention(x, y, z, c, return_lse=True)
        g = ops.attention_grad(w, x, y, z, o, lse, c)
        for n, got in zip(("o", "lse", "dq", "dk", "dv"), (o, lse, *g)):
            check(n, got, r[n], r[n + "_tol"])


def test_attention_same_bits_and_streams(ops):
    """The same call gives the same bits, on a side stream too, ordered after
    work queued there."""
    lens = [900, 31, 1, 260]
    c = cu(lens)
    q, k, v, do = (normal((sum(lens), h, 128), BF, i) for i, h in enumerate((8, 2, 2, 8)))
    first = None
    side = torch.cuda.Stream()
    for i in range(4):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            a = torch.rand(1024, 1024, device=DEV)
            for _ in range(10):
                a = a @ a * 1e-3
            q2 = q + 0 * a[0, 0].to(BF)
            o, lse = ops.attention(q2, k, v, c, return_lse=True)
            out = (o, lse, *ops.attention_grad(do, q2, k, v, o, lse, c))
        torch.cuda.synchronize()
        first = first or out
        assert all(torch.equal(x, y) for x, y in zip(first, out))


def test_long_attention_same_bits(ops):
    """Long enough that every wave runs many tiles without an edge: the same
    call, between writes of other memory, gives the same bits each time."""
    lens = [4100, 1900, 3000]
    c = cu(lens)
    q, k, v, do = (normal((sum(lens), h, 128), BF, i, 1.5) for i, h in enumerate((16, 4, 4, 16)))
    first = None
    for _ in range(10):
        junk = torch.full((1 << 26,), float("nan"), device=DEV)
        del junk
        o, lse = ops.attention(q, k, v, c, return_lse=True)
        out = (o, lse, lse.o_low, *ops.attention_grad(do, q, k, v, o, lse, c))
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_attention_extreme_scores(ops):
    """Scores far apart and far from zero: no overflow, no NaN, and rows whose
    largest score comes last."""
    lens, hq, hkv, d = [200, 64], 2, 1, 64
    c = cu(lens)
    q, k, v, do = (normal((sum(lens), h, d), BF, i + 9, 1.0) for i, h in
                   enumerate((hq, hkv, hkv, hq)))
    ramp = torch.linspace(-30, 30, sum(lens), device=DEV)[:, None, None].to(BF)
    k = k * 0.1 + ramp
    o, lse = ops.attention(q * 4, k, v, c, return_lse=True)
    g = ops.attention_grad(do, q * 4, k, v, o, lse, c)
    r = ref.attention(q * 4, k, v, c, c, do=do)
    for n, x in (("o", o), ("lse", lse), ("dq", g[0]), ("dk", g[1]), ("dv", g[2])):
        check(n, x, r[n], r[n + "_tol"])


def test_attention_gradient_by_differences(ops):
    """Directional derivatives of the 64-bit forward against the gradients."""
    lens, hq, hkv, d = [37, 70], 4, 2, 64
    c = cu(lens)
    q, k, v, do = (normal((sum(lens), h, d), BF, i + 20) for i, h in
                   enumerate((hq, hkv, hkv, hq)))
    o, lse = ops.attention(q, k, v, c, return_lse=True)
    g = ops.attention_grad(do, q, k, v, o, lse, c)
    r = ref.attention(q, k, v, c, c, do=do)
    x = [t.cpu().double() for t in (q, k, v)]

    def f(*a):
        ref.U[torch.float64], ref.TINY[torch.float64] = 0.0, 0.0
        return float((ref.attention(*a, c, c)["o"] * do.cpu().double()).sum())

    for i, n in enumerate(("dq", "dk", "dv")):
        u = torch.randn(x[i].shape, generator=torch.Generator().manual_seed(i)).double()
        eps = 1e-5
        lo, hi = list(x), list(x)
        lo[i], hi[i] = x[i] - eps * u, x[i] + eps * u
        slope = (f(*hi) - f(*lo)) / (2 * eps)
        got = float((g[i].cpu().double() * u).sum())
        tol = float((r[n + "_tol"] * u.abs()).sum()) + 1e-6 * abs(slope)
        _say(f"  {n}: {got:.6f} by differences {slope:.6f}, bound {tol:.2e}")
        assert abs(got - slope) <= tol


def test_attention_autograd(ops):
    lens = [40, 9]
    c = cu(lens)
    q, k, v, do = (normal((sum(lens), h, 64), BF, i) for i, h in enumerate((4, 2, 2, 4)))
    o, lse = ops.attention(q, k, v, c, return_lse=True)
    want = ops.attention_grad(do, q, k, v, o, lse, c)
    a = [x.clone().requires_grad_() for x in (q, k, v)]
    out = ops.attention(*a, c)
    assert torch.equal(out, o)
    out.backward(do)
    assert all(torch.equal(x.grad, w) for x, w in zip(a, want))


def test_attention_gradient_is_as_good_as_its_type(ops):
    """The row sums that the gradient needs are not those of the rounded output:
    over many values the error is that of rounding P, dS and the result, about
    sqrt(2) roundings of the type, with delta's part (as large again) gone."""
    for lens, hq, hkv in (([30] * 40, 4, 4), ([50, 61] * 10, 4, 2), ([700, 300], 4, 2),
                          ([40] * 12, 16, 1)):
        c = cu(lens)
        q, k, v, do = (normal((sum(lens), h, 64), BF, i + 3, 1.5 if i == 0 else 1.0)
                       for i, h in enumerate((hq, hkv, hkv, hq)))
        o, lse = ops.attention(q, k, v, c, return_lse=True)
        got = ops.attention_grad(do, q, k, v, o, lse, c)
        r = ref.attention(q, k, v, c, c, do=do)
        for n, g in zip(("dq", "dk", "dv"), got):
            want = r[n]
            rms = lambda x: float(x.square().mean().sqrt())  # noqa: E731
            off = rms(g.cpu().double() - want) / rms(want)
            rounded = rms(want.to(BF).double() - want) / rms(want)
            _say(f"  {lens[:2]} {n}: error {off:.5f}, of rounding alone {rounded:.5f}")
            assert off <= 1.75 * rounded, (lens[:2], n)


def test_graph_replays(ops):
    """Attention, its gradient, rotary positions and the policy loss captured in
    a graph, replayed on changed inputs with eager work in between."""
    lens = [70, 3, 200, 31]
    c, T = cu(lens), sum(lens)
    table, pos = ops.rotary_table(64, 256), torch.arange(T, device=DEV) % 200
    q, k, v, do = (normal((T, h, 64), BF, i) for i, h in enumerate((4, 2, 2, 4)))
    pc = policy_case(T, 40, BF, 3, forbidden=0.2)
    step = [normal((4, 4, 64), BF, 7), torch.tensor([70, 3, 200, 31], dtype=torch.int32,
                                                    device=DEV)]

    def work():
        a, b = ops.rotary(q, k, pos, table)
        o, lse = ops.attention(a, b, v, c, return_lse=True)
        g = ops.attention_grad(do, a, b, v, o, lse, c)
        s = ops.attention(step[0], b, v, torch.arange(5, dtype=torch.int32, device=DEV), c,
                          k_lens=step[1])
        return (o, *g, s, *ops.policy_loss_grad(**pc, kl_coef=0.1))

    work()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for i in range(4):
        q.copy_(normal(q.shape, BF, 50 + i))
        do.copy_(normal(do.shape, BF, 60 + i))
        pc["advantages"].copy_(normal(pc["advantages"].shape, F32, 70 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        want = work()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_attention_offsets_out_of_range(ops):
    """Offsets beyond the tensors or out of order stay inside them."""
    q, k, v = (normal((50, h, 64), BF, i) for i, h in enumerate((4, 2, 2)))
    for bad in ([0, 20, 70], [0, 30, 10, 50], [0, -5, 50], [0, 50, 2 ** 31 - 1]):
        c = torch.tensor(bad, dtype=torch.int32, device=DEV)
        o, lse = ops.attention(q, k, v, c, return_lse=True)
        ops.attention_grad(q, q, k, v, o, lse, c)
    torch.cuda.synchronize()
    c = cu([20, 20])                     # ten rows in no sequence
    o, lse = ops.attention(q, k, v, c, return_lse=True)
    assert not bool(o[40:].any()) and bool((lse[:, 40:] == float("-inf")).all())
    g = ops.attention_grad(q, q, k, v, o, lse, c)
    assert not any(bool(x[40:].any()) for x in g)


def test_nothing_to_do(ops):
    """No tokens, no keys, no sequences."""
    for T, K in ((0, 0), (0, 5), (7, 0)):
        q, k = normal((T, 4, 64), BF, 1), normal((K, 2, 64), BF, 2)
        cq, ck = cu([T]), cu([K])
        o, lse = ops.attention(q, k, k, cq, ck, return_lse=True)
        assert o.shape == q.shape and not bool(o.any())
        g = ops.attention_grad(q, q, k, k, o, lse, cq, ck)
        assert [x.shape for x in g] == [q.shape, k.shape, k.shape]
        assert not any(bool(x.any()) for x in g)
    q, k = normal((9, 4, 64), BF, 1), normal((9, 2, 64), BF, 2)
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    o, lse = ops.attention(q, k, k, none, return_lse=True)
    assert not bool(o.any()) and bool((lse == float("-inf")).all())
    assert not any(bool(x.any()) for x in ops.attention_grad(q, q, k, k, o, lse, none))
    table, pos = ops.rotary_table(64, 9), torch.zeros(0, dtype=torch.int64, device=DEV)
    assert ops.rotary(q[:0], None, pos, table).shape == (0, 4, 64)
    f = torch.zeros(0, device=DEV)
    loss, logp, dx = ops.policy_loss_grad(torch.zeros(0, 7, device=DEV), pos, f, f)
    assert float(loss) == 0.0 and logp.shape == (0,) and dx.shape == (0, 7)


def test_attention_uneven_rows_over_a_cache(ops):
    """Most sequences bring one query, one brings many: more rows than a split has
    room for, beside splits."""
    lq, lk = [1] * 11 + [200, 1], [900] * 11 + [1500, 2000]
    q, do = (normal((sum(lq), 8, 64), BF, i) for i in (1, 2))
    k, v = (normal((sum(lk), 2, 64), BF, i) for i in (3, 4))
    cq, ck = cu(lq), cu(lk)
    o, lse = ops.attention(q, k, v, cq, ck, return_lse=True)
    g = ops.attention_grad(do, q, k, v, o, lse, cq, ck)
    r = ref.attention(q, k, v, cq, ck, do=do)
    for n, x in zip(("o", "lse", "dq", "dk", "dv"), (o, lse, *g)):
        check(n, x, r[n], r[n + "_tol"])


def test_attention_rows_past_32_bits(ops):
    """A cache whose element offsets pass 2^31: the last segment is read where
    it lies."""
    hkv, d, cap = 8, 128, 1 << 20
    rows = 2 * cap + 4096
    k = torch.zeros(rows, hkv, d, dtype=BF, device=DEV)
    v = torch.zeros(rows, hkv, d, dtype=BF, device=DEV)
    assert k.numel() > 2 ** 31
    n = 150
    k[2 * cap:2 * cap + n], v[2 * cap:2 * cap + n] = (normal((n, hkv, d), BF, i) for i in (1, 2))
    q = normal((3, 16, d), BF, 3)
    ck = torch.tensor([0, cap, 2 * cap, rows], dtype=torch.int32, device=DEV)
    kl = torch.tensor([1, 0, n], dtype=torch.int32, device=DEV)
    o = ops.attention(q, k, v, cu([1, 1, 1]), ck, k_lens=kl)
    r = ref.attention(q[2:], k[2 * cap:2 * cap + n], v[2 * cap:2 * cap + n], cu([1]), cu([n]))
    check("o", o[2:], r["o"], r["o_tol"])
    assert not bool(o[:2].any())


# --------------------------------------------------------------------- rotary

@pytest.mark.parametrize("T,hq,hkv,d,rot,dtype,inter,inv,scaling", [
    (1, 1, 1, 64, 64, BF, False, False, None),
    (24, 32, 8, 128, 128, BF, False, False, "parts"),
    (7, 3, 1, 80, 32, FP, True, False, "linear"),
    (300, 4, 4, 96, 48, F32, True, True, "base"),
    (33, 2, 2, 10, 6, F32, False, True, None),
    (65, 5, 1, 7, 2, BF, True, False, None),
    (1000, 8, 2, 128, 128, FP, True, False, "parts"),
    (129, 6, 3, 64, 62, BF, False, True, "linear"),
    (50, 2, 1, 40, 0, F32, False, False, None),
])
def test_rotary(ops, T, hq, hkv, d, rot, dtype, inter, inv, scaling):
    _say("rotary", T, hq, hkv, d, rot, dtype, inter, inv, scaling)
    P, factor, original = 5000, 4.0, 512
    base = 10000.0 * (factor ** (rot / (rot - 2)) if scaling == "base" and rot > 2 else 1.0)
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    m = 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        keep = ((original * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f, m = f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1
    table = ops.rotary_table(rot, P, scaling=scaling, factor=factor if scaling else 1.0,
                             original=original)
    pos = torch.randint(0, P, (T,), generator=torch.Generator().manual_seed(T)).to(DEV)
    pos[-1] = P - 1
    q, k = normal((T, hq, d), dtype, 1), normal((T, hkv, d), dtype, 2)
    out = ops.rotary(q, k, pos, table, interleaved=inter, inverse=inv)
    for n, x, y in (("q", q, out[0]), ("k", k, out[1])):
        want, tol = ref.rotary(x, pos, rot, f, m, inter, inv)
        check(n, y, want, tol)
        assert torch.equal(y[..., rot:], x[..., rot:])
    # strided inputs, one tensor alone, int32 positions, and in place: the same bits
    wide = torch.cat([q, k, k], 1)
    a, b, _ = wide.split([hq, hkv, hkv], 1)
    o2 = ops.rotary(a, b, pos.to(torch.int32), table, interleaved=inter, inverse=inv)
    assert torch.equal(o2[0], out[0]) and torch.equal(o2[1], out[1])
    assert torch.equal(ops.rotary(q, None, pos, table, interleaved=inter, inverse=inv), out[0])
    ops.rotary(a, b, pos, table, interleaved=inter, inverse=inv, inplace=True)
    assert torch.equal(a, out[0]) and torch.equal(b, out[1])
    assert torch.equal(wide[:, hq + hkv:], k)


def test_rotary_odd_layouts(ops):
    """Rows off 16-byte boundaries and heads before rows read and write the
    same values."""
    table = ops.rotary_table(64, 100)
    pos = torch.arange(20, device=DEV)
    q, k = normal((20, 4, 64), BF, 1), normal((20, 2, 64), BF, 2)
    want = ops.rotary(q, k, pos, table)
    q2 = torch.empty(20, 4, 65, dtype=BF, device=DEV)[..., 1:]
    q2.copy_(q)
    k2 = k.transpose(0, 1).contiguous().transpose(0, 1)
    got = ops.rotary(q2, k2, pos, table)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_rotary_positions_outside_and_gradient(ops):
    table = ops.rotary_table(32, 64)
    q, k = normal((4, 2, 48), F32, 1), normal((4, 1, 48), F32, 2)
    pos = torch.tensor([0, 64, -1, 2 ** 31 - 1], device=DEV)
    a, b = ops.rotary(q, k, pos, table)
    assert bool(a[1:, :, :32].isnan().all()) and bool(b[1:, :, :32].isnan().all())
    assert torch.equal(a[:, :, 32:], q[:, :, 32:]) and torch.equal(a[0], q[0])
    pos = torch.tensor([1, 5, 63, 0], device=DEV)
    x, y = q.clone().requires_grad_(), k.clone().requires_grad_()
    gq, gk = normal((4, 2, 48), F32, 3), normal((4, 1, 48), F32, 4)
    out = ops.rotary(x, y, pos, table)
    torch.autograd.backward(out, (gq, gk))
    want = ops.rotary(gq, gk, pos, table, inverse=True)
    assert torch.equal(x.grad, want[0]) and torch.equal(y.grad, want[1])
    # <g, R(x + e u) - R(x - e u)> / 2e = <R^-1 g, u>: the turn is linear
    u = normal((4, 2, 48), F32, 5)
    got = float((want[0].double() * u.double()).sum())
    slope = float((gq.double() * (ops.rotary(q + u, None, pos, table).double()
                                  - ops.rotary(q - u, None, pos, table).double())).sum()) / 2
    assert abs(got - slope) <= 1e-5 * float((gq.abs() * (q.abs() + u.abs())).sum())


# ---------------------------------------------------------------- policy loss

def policy_case(T, V, dtype, seed, forbidden=0.0, zero=0, scale=3.0, lowest=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, V, generator=g) * scale
    if forbidden:
        no = torch.rand(T, V, generator=g) < forbidden
        no[torch.arange(T), torch.arange(T) % V] = False
        x[no] = torch.finfo(dtype).min if lowest else float("-inf")
    x = x.to(dtype)
    z = x.float().masked_fill(x.float() < -1e4, float("-inf"))
    act = torch.multinomial(z.softmax(1), 1, generator=g)[:, 0]
    lp = z.double().log_softmax(1).gather(1, act[:, None])[:, 0]
    old = (lp + 0.2 * torch.randn(T, generator=g)).float()
    r = (lp - old.double()).exp()
    for edge in (0.8, 1.25):             # off the edges, where there is no derivative
        old = torch.where((r - edge).abs() < 1e-3, old - 0.01, old)
    w = torch.rand(T, generator=g) / T
    w[torch.randperm(T, generator=g)[:zero]] = 0.0
    return dict(logits=x.to(DEV), actions=act.to(DEV), logp_old=old.to(DEV),
                advantages=torch.randn(T, generator=g).to(DEV),
                logp_ref=(lp + 0.3 * torch.randn(T, generator=g)).float().to(DEV),
                weights=w.to(DEV))


@pytest.mark.parametrize("T,V,dtype,forbidden,zero,kl,temp", [
    (1, 1, F32, 0.0, 0, 0.1, 1.0),
    (1, 2, BF, 0.0, 0, 0.0, 1.0),
    (37, 21, BF, 0.3, 4, 0.04, 1.0),
    (513, 32, FP, 0.3, 0, 0.04, 0.7),
    (200, 33, F32, 0.5, 20, 0.1, 1.3),
    (65, 64, BF, 0.0, 65, 0.1, 1.0),
    (50, 65, FP, 0.2, 5, 0.0, 1.0),
    (30, 127, F32, 0.0, 0, 0.1, 0.5),
    (19, 1000, BF, 0.1, 3, 0.1, 1.0),
    (17, 4097, FP, 0.0, 2, 0.1, 1.0),
    (9, 8193, F32, 0.9, 0, 0.1, 1.0),
    (6, 32001, F32, 0.0, 1, 0.1, 0.8),
    (5, 50001, BF, 0.0, 1, 0.1, 0.8),
    (4, 131071, BF, 0.0, 1, 0.04, 1.0),
    (3, 131072, FP, 0.2, 0, 0.04, 1.0),
    (2, 200003, F32, 0.0, 0, 0.0, 1.0),
    (3, 300007, BF, 0.0, 0, 0.1, 1.0),
])
def test_policy_loss(ops, T, V, dtype, forbidden, zero, kl, temp):
    _say("policy", T, V, dtype, forbidden, zero, kl, temp)
    c = policy_case(T, V, dtype, T + V, forbidden, zero)
    if zero:                             # what carries no weight is not read
        c["logits"][c["weights"] == 0] = float("nan")
    if not kl:
        c["logp_ref"] = None
    kw = dict(clip=(0.2, 0.25), kl_coef=kl, temperature=temp)
    loss, logp, dx = ops.policy_loss_grad(**c, **kw)
    clean = dict(c, logits=c["logits"].nan_to_num(0.0, neginf=float("-inf")))
    r = ref.policy(*(clean[n] for n in ("logits", "actions", "logp_old", "advantages", "logp_ref",
                                        "weights")), (0.2, 0.25), kl, temp)
    check("loss", loss, torch.tensor(r["loss"]).double(), torch.tensor(r["loss_tol"]))
    check("logp", logp, r["logp"], r["logp_tol"])
    check("dlogits", dx, r["dlogits"], r["dlogits_tol"])
    assert not bool(dx[c["weights"] == 0].any())
    l2, p2 = ops.policy_loss(**c, **kw)
    check("loss alone", l2, torch.tensor(r["loss"]).double(), torch.tensor(r["loss_tol"]))
    check("logp alone", p2, r["logp"], r["logp_tol"])
    again = ops.policy_loss_grad(**c, **kw)
    assert all(torch.equal(a, b) for a, b in zip((loss, logp, dx), again))


def test_policy_masks(ops):
    """Rows that a mask empties, actions it forbids, masks of the type's lowest
    value, actions outside the vocabulary."""
    for dtype in (F32, BF, FP):
        for V in (24, 700, 9001):
            c = policy_case(8, V, dtype, 3, forbidden=0.5, lowest=True)
            low = ops.policy_loss_grad(**c, kl_coef=0.1)
            r = ref.policy(*(c[n] for n in ("logits", "actions", "logp_old", "advantages",
                                            "logp_ref", "weights")), (0.2, 0.2), 0.1, 1.0)
            check("lowest", low[1], r["logp"], r["logp_tol"])
            check("lowest grad", low[2], r["dlogits"], r["dlogits_tol"])
            c["logits"][0] = torch.finfo(dtype).min        # all lowest: uniform
            c["logits"][1] = float("-inf")                 # nothing allowed
            c["logits"][2, c["actions"][2]] = float("-inf")
            c["actions"][3] = V
            c["actions"][4] = -1
            loss, logp, dx = ops.policy_loss_grad(**dict(c, logp_ref=None))
            want = -math.log(V)
            assert abs(float(logp[0]) - want) <= 1e-5 * abs(want)
            assert float(logp[1]) == float("-inf") and float(logp[2]) == float("-inf")
            assert not bool(dx[1].any()) and not bool(dx[2].any())
            assert bool(logp[3:5].isnan().all()) and bool(logp[5:].isfinite().all())
            assert bool(dx[5:].isfinite().all()) and bool(loss.isnan())
            c["actions"][3:5] = 0
            c["logits"][3:5, 0] = 0.0
            c["weights"][1] = 0.0
            loss, _, dx = ops.policy_loss_grad(**dict(c, logp_ref=None))
            assert bool(loss.isfinite()) and bool(dx.isfinite().all())
            loss, _, dx = ops.policy_loss_grad(**c, kl_coef=0.1)
            assert float(loss) == float("inf") and not bool(dx[2].any())


def test_policy_strides_gradient_and_autograd(ops):
    c = policy_case(23, 50, BF, 1, forbidden=0.2)
    want = ops.policy_loss_grad(**c, kl_coef=0.1)
    wide = torch.full((23, 61), float("nan"), dtype=BF, device=DEV)
    wide[:, 3:53] = c["logits"]
    got = ops.policy_loss_grad(**dict(c, logits=wide[:, 3:53]), kl_coef=0.1)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    got = ops.policy_loss_grad(**dict(c, logits=c["logits"].T.contiguous().T), kl_coef=0.1)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    x = c["logits"].clone().requires_grad_()
    loss, logp = ops.policy_loss(**dict(c, logits=x), kl_coef=0.1)
    assert torch.equal(loss, want[0]) and torch.equal(logp, want[1])
    (loss * 2.0).backward()
    assert torch.equal(x.grad, want[2] * 2)              # a power of two: the same bits
    # by differences of the 64-bit loss
    c = policy_case(11, 40, F32, 2)
    names = ("logits", "actions", "logp_old", "advantages", "logp_ref", "weights")
    dx = ops.policy_loss_grad(**c, kl_coef=0.1)[2].cpu().double()
    r = ref.policy(*(c[n] for n in names), (0.2, 0.2), 0.1, 1.0)
    u = torch.randn(dx.shape, generator=torch.Generator().manual_seed(1)).double()
    ref.U[torch.float64], ref.TINY[torch.float64] = 0.0, 0.0
    x0 = c["logits"].cpu().double()
    f = [ref.policy(x0 + s * 1e-6 * u, *(c[n] for n in names[1:]), (0.2, 0.2), 0.1, 1.0,
                    grad=False)["loss"] for s in (1, -1)]
    slope = (f[0] - f[1]) / 2e-6
    tol = float((r["dlogits_tol"] * u.abs()).sum()) + 1e-7 * float((dx.abs() * u.abs()).sum())
    assert abs(float((dx * u).sum()) - slope) <= tol

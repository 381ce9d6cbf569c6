"""The layers around attention against their 64-bit definitions, through the public
entry points (cusr_amd.kernel.seq_layers), at the sizes, values, strides and types
where they can go wrong."""
from __future__ import annotations

import math
import threading

import pytest
import torch

import layer_reference as ref
from seq_reference import E32
from test_gpu_seq import BF, DEV, F32, FP, _say, check, normal

pytestmark = pytest.mark.gpu
I8 = torch.int8


@pytest.fixture(scope="module")
def ops():
    from cusr_amd.kernel import seq_layers
    return seq_layers


def ids(n, rows, seed, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, max(rows, 1), (n,), generator=g).to(dtype).to(DEV)


def layouts(x):
    """x's values in other layouts: rows with room behind, off a 16-byte boundary, and
    transposed memory."""
    T, D = x.shape
    wide = torch.full((T, D + 11), float("nan") if x.is_floating_point() else 77, dtype=x.dtype,
                      device=DEV)
    wide[:, 3:D + 3] = x
    return x, wide[:, 3:D + 3], x.t().contiguous().t()


# ------------------------------------------------------------------ embedding

EMBED = [
    # tokens, rows, width, table's type, out's type
    (1, 1, 1, F32, None), (5, 3, 8, BF, None), (300, 22, 128, F32, BF), (24, 1000, 4096, BF, None),
    (77, 513, 40, FP, F32), (1000, 7, 33, BF, FP), (3, 70000, 2056, F32, None),
    (2, 4, 65536, BF, F32), (9, 5, 1025, FP, None), (0, 5, 16, BF, None),
]


@pytest.mark.parametrize("T,V,D,dt,out", EMBED)
def test_embedding(ops, T, V, D, dt, out):
    _say("embedding", T, V, D, dt)
    table, tokens = normal((V, D), dt, 1), ids(T, V, 2, torch.int32)
    for tab in layouts(table):
        got = ops.embedding(tokens, tab, scale=1.25, dtype=out)
        want, tol = ref.embedding(tokens, table, 1.25, out or dt)
        assert got.dtype is (out or dt)
        check("out", got, want, tol)
    assert torch.equal(ops.embedding(tokens.long(), table), table[tokens.long()])


def test_embedding_outside_the_table(ops):
    table = normal((4, 24), BF, 1)
    for dt in (torch.int32, torch.int64):
        tokens = torch.tensor([0, -1, 3, 4, -2 ** 31, 2 ** 31 - 1], device=DEV, dtype=dt)
        out = ops.embedding(tokens, table)
        assert out.isnan().all(1).tolist() == [False, True, False, True, True, True]
        assert torch.equal(out[[0, 2]], table[[0, 3]])
        d = ops.embedding_grad(torch.ones(6, 24, device=DEV), tokens, 4)
        assert d.sum(1).tolist() == [24.0, 0.0, 0.0, 24.0]
    far = torch.tensor([2 ** 32, 2 ** 32 + 1, -2 ** 63], device=DEV)
    assert bool(ops.embedding(far, table).isnan().all())
    assert not bool(ops.embedding_grad(torch.ones(3, 24, device=DEV), far, 4).any())
    none = ops.embedding(torch.zeros(3, dtype=torch.int64, device=DEV), table[:0])
    assert none.shape == (3, 24) and bool(none.isnan().all())
    assert ops.embedding_grad(torch.ones(3, 24, device=DEV), far, 0).shape == (0, 24)


EMBED_GRAD = [
    (1, 1, 1, F32, F32), (1, 40, 8, BF, F32), (31, 5, 16, FP, F32), (32, 1, 128, BF, BF),
    (33, 1, 24, F32, FP), (500, 22, 128, F32, F32), (2049, 511, 64, BF, F32),
    (4097, 512, 8, F32, F32), (3000, 70000, 16, BF, F32), (5000, 300000, 2, F32, F32),
    (700, 40, 2056, BF, F32), (640, 3, 333, FP, F32), (66000, 22, 40, BF, F32),
    (70001, 9, 8, F32, F32), (600000, 1000, 1, F32, F32), (530000, 2, 16, BF, F32),
    (3, 4, 65536, BF, F32), (0, 5, 16, BF, F32), (40000, 128, 130, BF, F32), (9001, 129, 130, F32, F32),
    (33000, 32, 257, FP, F32), (33000, 33, 257, FP, F32), (5000, 20, 1024, BF, BF),
    (200, 129, 65536, BF, F32), (256, 700, 33, BF, BF), (257, 700, 40, FP, F32),
    (255, 100000, 8, F32, F32), (256, 1, 2056, BF, F32), (64, 5, 300, FP, FP),
    (33000, 5000, 264, F32, F32), (32768, 513, 9, BF, F32), (80000, 200, 136, BF, F32),
]


@pytest.mark.parametrize("T,V,D,dt,out", EMBED_GRAD)
def test_embedding_grad(ops, T, V, D, dt, out):
    _say("embedding_grad", T, V, D, dt)
    d, tokens = normal((T, D), dt, 3), ids(T, V, 4)
    if T > 100:
        tokens[T // 3:T // 2] = V // 2              # one token far more often than others
    want, tol = ref.embedding_grad(d, tokens, V, 0.75, out)
    first = None
    for x in layouts(d):
        got = ops.embedding_grad(x, tokens, V, scale=0.75, dtype=out)
        assert got.dtype is out and got.shape == (V, D)
        check("dtable", got, want, tol)
        first = got if first is None else first
    assert torch.equal(first, ops.embedding_grad(d, tokens.int(), V, scale=0.75, dtype=out))


@pytest.mark.parametrize("V", [11, 32, 33, 3000])
def test_embedding_grad_same_bits(ops, V):
    """The same call gives the same bits, whatever else runs; a token's rows do not depend on
    the other tokens' values."""
    T, D = 50000, 72
    d, tokens = normal((T, D), F32, 5), ids(T, V, 6)
    first = ops.embedding_grad(d, tokens, V)
    other = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(other):
            ops.embedding_grad(d, tokens // 2, V)
        assert torch.equal(first, ops.embedding_grad(d, tokens, V))
    d[tokens != 5] = float("nan")
    again = ops.embedding_grad(d, tokens, V)
    assert torch.equal(again[5], first[5]) and bool(again[6].isnan().all())


def test_embedding_autograd(ops):
    table = normal((50, 32), BF, 1).requires_grad_()
    tokens, w = ids(200, 50, 2), normal((200, 32), F32, 3)
    (ops.embedding(tokens, table, scale=3.0, dtype=F32) * w).sum().backward()
    want, tol = ref.embedding_grad(w, tokens, 50, 3.0, BF)
    assert table.grad.dtype is BF
    check("dtable", table.grad, want, tol)


# ----------------------------------------------------------------------- norm

NORM = [
    # tokens, width, x, stream, gain, out
    (1, 1, F32, None, None, None), (3, 8, BF, None, BF, None), (5, 128, BF, F32, None, None),
    (17, 128, BF, F32, F32, FP), (33, 136, FP, FP, FP, F32), (9, 512, F32, F32, F32, BF),
    (4, 1000, BF, BF, F32, None), (7, 1024, FP, F32, BF, None), (24, 4096, BF, BF, F32, None),
    (3, 8192, F32, F32, None, None), (2, 16384, BF, F32, F32, None), (3, 16392, BF, BF, F32, None),
    (2, 65536, F32, None, F32, BF), (5, 7, BF, F32, F32, None), (6, 129, FP, None, None, None),
    (3, 513, BF, BF, BF, None), (2, 2049, F32, F32, F32, None), (2, 16383, BF, F32, F32, None),
    (2, 16385, FP, FP, FP, None), (1025, 64, BF, BF, F32, None), (0, 64, BF, BF, F32, None),
]


@pytest.mark.parametrize("T,D,dt,st,gt,out", NORM)
def test_rms_norm(ops, T, D, dt, st, gt, out):
    _say("rms_norm", T, D, dt, st)
    x, eps = normal((T, D), dt, 1), 1e-5
    res = None if st is None else normal((T, D), st, 2, 2.0)
    gain = None if gt is None else normal((D,), gt, 3)
    for i, xx in enumerate(layouts(x)):
        rr = None if res is None else layouts(res)[i]
        got = ops.rms_norm(xx, gain, residual=rr, eps=eps, dtype=out)
        y, h = got if res is not None else (got, x)
        assert y.dtype is (out or dt)
        if res is not None:
            assert h.dtype is st
            check("h", h, *ref.stream(x, res))
        want, err = ref.rms(h, gain, eps)
        check("y", y, want, ref.rounded(want, out or dt, err))


@pytest.mark.parametrize("T,D,dt,st,gt,out", NORM)
def test_rms_norm_int8(ops, T, D, dt, st, gt, out):
    x, eps = normal((T, D), dt, 1), 1e-5
    res = None if st is None else normal((T, D), st, 2, 2.0)
    gain = None if gt is None else normal((D,), gt, 3)
    first = None
    for i, xx in enumerate(layouts(x)):
        rr = None if res is None else layouts(res)[i]
        q, s, *h = ops.rms_norm_int8(xx, gain, residual=rr, eps=eps)
        assert q.dtype is I8 and s.shape == (T,)
        want, err = ref.rms(h[0] if h else x, gain, eps)
        quantized(q, s, want, err)
        if res is not None:
            check("h", h[0], *ref.stream(x, res))
        first = first or (q, s)
    if T:
        assert int(q.abs().max()) == 127


def quantized(q, s, want, err):
    """Scales and integers of rows `want`, known to `err`."""
    if not len(want):
        return
    most = want.abs().amax(1)
    check("scale", s, most / 127, err.amax(1) / 127 + 2 * E32 * most / 127)
    scale = ref.f64(s)[:, None]
    # the quotient's distance from its integer: half, the value's error, and the rounding
    # of the two factors and the product, of 127 at most
    tol = 0.5 * scale + err + err.amax(1, keepdim=True) + 127 * 5 * E32 * scale
    check("q", q.double() * s.double()[:, None], want, tol + 1e-45)
    assert int(q.min()) >= -127


@pytest.mark.parametrize("T,D,dt", [(5, 64, BF), (300, 4096, F32), (3, 77, FP), (1, 1, BF),
                                    (40, 16385, F32), (0, 8, BF)])
def test_quantize_rows(ops, T, D, dt):
    x = normal((T, D), dt, 7, 3.0)
    for xx in layouts(x):
        q, s = ops.quantize_rows(xx)
        quantized(q, s, ref.f64(x), torch.zeros(T, D).double())


def test_quantize_edges(ops):
    for D in (40, 37, 20000):
        x = torch.zeros(8, D, device=DEV)
        x[1, 0] = 1e-30
        x[2, :3] = torch.tensor([1e-38, -5e-39, 2e-45])
        x[3, D - 1] = float("inf")
        x[4, 1] = float("nan")
        x[5, :2] = torch.tensor([3e38, -3.4e38])
        x[6, :6] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -3.5])
        q, s = ops.quantize_rows(x)
        assert s[0] == 0 and not bool(q[0].any()) and not bool(q[7].any())
        assert q[1, 0] == 127 and abs(float(s[1]) * 127 / 1e-30 - 1) < 1e-6
        assert q[2, 0] == 127 and q[2, 1] in (-63, -64)
        assert bool(s[3:5].isnan().all()) and not bool(q[3:5].any())
        assert q[5, 1] == -127 and q[5, 0] == 112 and bool(s[5].isfinite())
        assert q[6, :6].tolist() == [127, 0, 2, 2, 0, -4]          # halves to even


def test_norm_of_nothing_and_of_what_is_not_finite(ops):
    for D in (128, 51, 17000):
        x = torch.zeros(4, D, device=DEV, dtype=BF)
        x[1, 3] = float("nan")
        x[2, 3] = float("inf")
        x[3] = 1.0
        y = ops.rms_norm(x, eps=1e-6)
        assert not bool(y[0].any()) and bool(y[1].isnan().all()) and bool(y[2, 3].isnan())
        assert bool(y[3].isfinite().all())
        assert bool(ops.rms_norm(x, eps=0.0)[0].isnan().all())     # 0 / 0
        q, s = ops.rms_norm_int8(x)
        assert s[0] == 0 and bool(s[1:3].isnan().all()) and not bool(q[:3].any())


NORM_GRAD = [
    # tokens, width, dy, h, x, gain, dh
    (1, 1, F32, F32, None, None, False), (3, 8, BF, BF, None, BF, True),
    (50, 128, BF, F32, BF, F32, True), (50, 128, BF, F32, BF, None, True),
    (5, 256, FP, FP, None, FP, False), (33, 512, F32, F32, None, F32, True),
    (40, 1000, BF, BF, None, F32, True), (9, 2048, BF, F32, BF, F32, True),
    (2500, 4096, BF, BF, None, F32, True), (3, 8192, F32, F32, None, F32, False),
    (300, 16384, BF, F32, BF, F32, True), (5, 16392, BF, BF, None, F32, True),
    (70, 65536, F32, F32, FP, F32, True), (70, 20001, BF, BF, None, None, True),
    (21, 7, BF, F32, BF, F32, True), (30, 129, FP, F32, FP, FP, True),
    (3, 513, BF, BF, None, BF, True), (3, 2049, F32, F32, None, F32, True),
    (300, 16383, BF, F32, BF, F32, True), (20001, 64, BF, BF, None, F32, True),
    (40003, 12, F32, F32, None, F32, False), (0, 24, BF, BF, None, F32, True),
]


@pytest.mark.parametrize("T,D,yt,ht,xt,gt,with_dh", NORM_GRAD)
def test_rms_norm_grad(ops, T, D, yt, ht, xt, gt, with_dh):
    _say("rms_norm_grad", T, D, yt, ht)
    eps = 1e-5
    dy, h = normal((T, D), yt, 1), normal((T, D), ht, 2, 2.0)
    gain = None if gt is None else normal((D,), gt, 3)
    dh = normal((T, D), ht, 4) if with_dh else None
    r = ref.rms_grad(dy, h, gain, dh, eps)
    for i in range(3):
        d, dx, dgain = ops.rms_norm_grad(layouts(dy)[i], layouts(h)[i], gain,
                                         dh=None if dh is None else layouts(dh)[i], eps=eps,
                                         x_dtype=xt)
        check("d", d, r["d"], ref.rounded(r["d"], ht, r["d_err"]))
        assert (dx is d) == (xt is None or xt is ht)
        check("dx", dx, r["d"], ref.rounded(r["d"], xt or ht, r["d_err"]))
        if gain is not None:
            assert dgain.dtype is F32
            check("dgain", dgain, r["dgain"], ref.rounded(r["dgain"], F32, r["dgain_err"]))
        else:
            assert dgain is None


@pytest.mark.parametrize("st", [None, F32, BF])
def test_norm_autograd(ops, st):
    T, D, eps = 40, 96, 1e-6
    x, gain = normal((T, D), BF, 1).requires_grad_(), normal((D,), BF, 2).requires_grad_()
    res = None if st is None else normal((T, D), st, 3).requires_grad_()
    wy, wh = normal((T, D), F32, 4), normal((T, D), F32, 5)
    out = ops.rms_norm(x, gain, residual=res, eps=eps, dtype=F32)
    y, h = out if st is not None else (out, None)
    loss = (y * wy).sum() + (0 if h is None else (h.float() * wh).sum())
    loss.backward()
    r = ref.rms_grad(wy, x if h is None else h, gain, None if h is None else wh.to(st), eps)
    check("dx", x.grad, r["d"], ref.rounded(r["d"], BF, r["d_err"]))
    check("dgain", gain.grad, r["dgain"],
          ref.rounded(r["dgain"], BF, r["dgain_err"] + E32 * r["dgain"].abs()))
    if res is not None:
        check("dresidual", res.grad, r["d"], ref.rounded(r["d"], st, r["d_err"]))
        assert res.grad.data_ptr() != x.grad.data_ptr()
        # the stream alone, the norm alone, and neither
        for pick in ("y", "h"):
            for t in (x, gain, res):
                t.grad = None
            y, h = ops.rms_norm(x, gain, residual=res, eps=eps, dtype=F32)
            (y if pick == "y" else h).float().sum().backward()
            assert x.grad is not None and res.grad is not None
            if pick == "h":
                assert gain.grad is None and torch.equal(x.grad, torch.ones_like(x))


# -------------------------------------------------------------- 8-bit product

PRODUCT = [
    (1, 1, 1), (1, 64, 16), (3, 17, 5), (16, 128, 256), (24, 4096, 384), (33, 100, 130),
    (128, 64, 128), (129, 65, 127), (200, 1000, 72), (257, 256, 300), (7, 16, 1000),
    (300, 131, 33), (64, 2064, 260), (1000, 512, 520), (32, 131071, 17), (5, 0, 7), (0, 8, 4),
    (4, 8, 0), (17, 1280, 640), (2, 5008, 2050), (260, 4100, 258), (65, 48, 100), (64, 528, 31),
    # enough tiles of 128 and of 256 to be taken, whole and cut ones
    (1500, 128, 1450), (1536, 16, 1408), (4000, 80, 4100), (4096, 208, 4104),
]


def int8s(shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=g).to(I8).to(DEV)


def product_case(M, K, N):
    a, w = int8s((M, K), 1), int8s((N, K), 2)
    sa, sw = normal((M,), F32, 3).abs(), normal((N,), F32, 4).abs()
    exact = a.cpu().double() @ w.cpu().double().t()              # below 2^53: exact
    want = exact * ref.f64(sa)[:, None] * ref.f64(sw)
    return a, sa, w, sw, want


@pytest.mark.parametrize("M,K,N", PRODUCT)
def test_int8_product(ops, M, K, N):
    _say("int8_product", M, K, N)
    a, sa, w, sw, want = product_case(M, K, N)
    for dt in (F32, BF, FP):
        # the integer's conversion and two products, half a unit each
        tol = ref.rounded(want, dt, 3.1 * E32 * want.abs())
        big = want.abs() * (1 + 2.0 ** -8) >= 65504 if dt is FP else torch.zeros_like(want) > 0
        first = None
        for i in range(3 if M and N and K else 1):
            got = ops.int8_product(layouts(a)[i] if K else a, sa, layouts(w)[i] if K else w, sw,
                                   dtype=dt)
            assert got.dtype is dt and got.shape == (M, N)
            check("o", got.cpu().masked_fill(big, 0.0), want.masked_fill(big, 0.0),
                  tol.masked_fill(big, 0.0))
            assert first is None or torch.equal(first, got)
            first = got


# long sums of few outputs, which are cut among blocks: sides of 64 and 128, odd and ragged
CUT = [(40, 16384, 72), (33, 8208, 1001), (100, 12000, 255), (17, 65536, 9), (3, 70001, 50),
       (512, 16384, 136), (64, 131071, 8), (1, 131071, 1), (130, 4112, 7), (700, 20480, 1500)]


@pytest.mark.parametrize("M,K,N", CUT)
def test_int8_product_of_long_sums(ops, M, K, N):
    _say("int8_product, cut", M, K, N)
    a, sa, w, sw, want = product_case(M, K, N)
    for dt in (F32, BF):
        tol = ref.rounded(want, dt, 3.1 * E32 * want.abs())
        got = ops.int8_product(a, sa, w, sw, dtype=dt)
        check("o", got, want, tol)
        assert torch.equal(got, ops.int8_product(layouts(a)[1], sa, w, sw, dtype=dt))
    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        out = ops.int8_product(a, sa, w, sw)
    for seed in range(2):
        a.copy_(int8s((M, K), 10 + seed))
        got = ops.int8_product(a, sa, w, sw)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, got)


def test_int8_product_extremes(ops):
    """The largest sums there are, of one sign and the other."""
    K = ops.SEQ_MAX_INNER
    a = torch.full((2, K), -128, dtype=I8, device=DEV)
    a[1] = 127
    one = torch.ones(2, device=DEV)
    o = ops.int8_product(a, one, a, one, dtype=F32)
    want = torch.tensor([[K * 16384.0, -K * 128.0 * 127.0], [-K * 128.0 * 127.0, K * 127.0 ** 2]])
    check("o", o, want.double(), want.double().abs() * E32)
    # a scale that is not finite, or 0, stays in its row or column
    s = torch.tensor([float("nan"), 0.0], device=DEV)
    o = ops.int8_product(a, s, a, one, dtype=F32)
    assert bool(o[0].isnan().all()) and not bool(o[1].any())
    o = ops.int8_product(a, one, a, s, dtype=BF)
    assert bool(o[:, 0].isnan().all()) and not bool(o[:, 1].any())


def test_int8_product_in_views(ops):
    """Operands that are rows of one larger weight, and a broadcast row."""
    w = int8s((300, 256), 5)
    sw = normal((300,), F32, 6).abs()
    a, sa = w[:1].expand(40, 256), sw[:1].expand(40)
    got = ops.int8_product(a[:, 64:192], sa, w[20:150, 64:192], sw[20:150], dtype=F32)
    want = (a[:, 64:192].cpu().double() @ w[20:150, 64:192].cpu().double().t()) \
        * ref.f64(sa)[:, None] * ref.f64(sw[20:150])
    check("o", got, want, 4 * E32 * want.abs())


# ----------------------------------------------------------- log-probabilities

LOGPROBS = [
    # tokens, vocabulary, type, alternatives, share of -inf, temperature
    (1, 1, F32, 1, 0.0, 1.0), (5, 2, BF, 2, 0.0, 0.7), (300, 21, BF, 5, 0.33, 1.0),
    (257, 22, FP, 0, 0.3, 1.3), (100, 32, F32, 3, 0.0, 1.0), (100, 64, BF, 10, 0.2, 0.8),
    (130, 100, BF, 1, 0.0, 1.0), (70, 128, F32, 64, 0.5, 1.0), (65, 250, FP, 7, 0.0, 2.0),
    (9, 256, BF, 64, 0.0, 1.0), (9, 257, BF, 20, 0.1, 1.0), (40, 300, F32, 5, 0.0, 0.5),
    (33, 1000, FP, 10, 0.3, 1.0), (7, 4099, BF, 64, 0.0, 1.0), (5, 8193, F32, 3, 0.0, 0.8),
    (4, 32001, F32, 5, 0.0, 0.8), (3, 32001, BF, 20, 0.9, 1.0), (1030, 5003, BF, 2, 0.0, 1.0),
    (2, 131071, BF, 64, 0.0, 1.0), (2, 200000, F32, 2, 0.0, 0.1), (0, 50, BF, 2, 0.0, 1.0),
    # enough rows for a block each
    (520, 9001, F32, 7, 0.1, 1.0), (600, 33000, FP, 64, 0.0, 0.9), (512, 4104, F32, 1, 0.9, 1.0),
    (1, 600000, F32, 64, 0.0, 1.0), (511, 8200, BF, 3, 0.0, 1.0),
]


def logits_case(T, V, dt, share, seed=1, spread=2.5):
    x, tokens = normal((T, V), dt, seed, spread), ids(T, V, seed + 1)
    if share:
        g = torch.Generator().manual_seed(seed + 2)
        no = torch.rand(T, V, generator=g) < share
        no[torch.arange(T), torch.arange(T) % V] = False
        x.masked_fill_(no.to(DEV), float("-inf"))
    return x, tokens


def check_logprobs(out, r, top, stats=False):
    check("logp", out[0], r["logp"], r["logp_err"])
    check("entropy", out[1], r["entropy"], r["entropy_err"])
    if top:
        order = r["order"][:, :top]
        assert torch.equal(out[3].cpu(), order)
        check("top", out[2], r["lp"].gather(1, order), r["lp_err"].gather(1, order))


@pytest.mark.parametrize("T,V,dt,top,share,temperature", LOGPROBS)
def test_token_logprobs(ops, T, V, dt, top, share, temperature):
    _say("token_logprobs", T, V, dt, top)
    x, tokens = logits_case(T, V, dt, share)
    r = ref.logprobs(x, tokens, temperature)
    for xx in layouts(x):
        check_logprobs(ops.token_logprobs(xx, tokens, temperature=temperature, top=top), r, top)
    if T:
        a = ops.token_logprobs(x, tokens.int(), temperature=temperature)
        b = ops.token_logprobs(x, tokens, temperature=temperature, top=top)
        assert len(a) == 2 and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("T,V,dt,top,share,temperature", LOGPROBS)
def test_token_logprobs_grad(ops, T, V, dt, top, share, temperature):
    _say("token_logprobs_grad", T, V, dt)
    x, tokens = logits_case(T, V, dt, share)
    r = ref.logprobs(x, tokens, temperature)
    g, k = normal((T,), F32, 5), normal((T,), F32, 6)
    *_, entropy, stats = ops.token_logprobs(x, tokens, temperature=temperature, return_stats=True)
    for dl, dh in ((g, k), (g, None), (None, k)):
        want, tol = ref.logprobs_grad(r, tokens, dl, dh, temperature, dt)
        for xx in layouts(x):
            got = ops.token_logprobs_grad(xx, tokens, stats, entropy, dl, dh,
                                          temperature=temperature)
            assert got.dtype is dt
            check("dlogits", got, want, tol + 1e-38)
    assert not bool(ops.token_logprobs_grad(x, tokens, stats, entropy,
                                            temperature=temperature).any())


@pytest.mark.parametrize("V,T", [(21, 12), (256, 12), (3001, 12), (40000, 12), (6001, 520),
                                 (131001, 12)])
@pytest.mark.parametrize("dt", [F32, BF])
def test_logprobs_of_sure_rows(ops, V, T, dt):
    """Rows of nearly all weight on one symbol keep the relative precision of the rest, in
    the log-probability, in the entropy and in the gradient."""
    x, _ = logits_case(T, V, dt, 0.0, spread=1.0)
    tokens = (torch.arange(T, device=DEV) * 7) % V
    gap = torch.linspace(4.0, 40.0, T, device=DEV) + math.log(V)
    x[torch.arange(T, device=DEV), tokens] = (x.float().amax(1) + gap).to(dt)
    z = ref.f64(x)
    r = ref.logprobs(x, tokens, 1.0)
    # the rest from the other columns alone: 1 - p has lost it in 64 bits too
    others = z.clone().scatter_(1, tokens.cpu()[:, None], float("-inf"))
    t = others - z.amax(1, keepdim=True)
    rest = t.exp().sum(1)
    logp = -torch.log1p(rest)
    entropy = -logp - (t.exp() * t.masked_fill(t == float("-inf"), 0.0)).sum(1) / (1 + rest)
    depth = V if V <= 512 else V // 64 + 16
    rel = (8 * float(t[t > float("-inf")].abs().max()) + depth + 24) * E32
    got = ops.token_logprobs(x, tokens, return_stats=True)
    check("logp", got[0], logp, rel * logp.abs())
    check("entropy", got[1], entropy, rel * entropy)
    one = torch.ones(T, device=DEV)
    d = ops.token_logprobs_grad(x, tokens, got[2], got[1], one)
    at = torch.arange(T), tokens.cpu()
    want = rest / (1 + rest)
    check("own gradient", d.cpu()[at], want, want * (rel + ref.U[dt]))
    assert r["p"].shape == (T, V)


@pytest.mark.parametrize("V,reps", [(7, 1), (256, 1), (700, 1), (5000, 1), (5000, 60), (33000, 1),
                                    (33000, 60), (100001, 1), (300001, 1)])
@pytest.mark.parametrize("dt", [F32, BF, FP])
def test_logprobs_of_odd_rows(ops, V, reps, dt):
    """All -inf, all the same, all but one -inf, NaN, +inf, the type's lowest value, tokens
    outside the vocabulary, and a token that is not allowed."""
    low = torch.finfo(dt).min
    x = normal((10, V), dt, 3)
    x[0] = float("-inf")
    x[1] = 3.0
    x[2] = float("-inf")
    x[2, V // 2] = -7.0
    x[3, V - 1] = float("nan")
    x[4, 0] = float("inf")
    x[5] = low
    x[6, 1:] = low
    x[9, 2] = float("-inf")
    tokens = torch.tensor([0, V - 1, V // 2, 0, 1, 2, 0, -1, V, 2], device=DEV)
    top = min(V, 9)
    x, tokens = x.repeat(reps, 1), tokens.repeat(reps)
    out = ops.token_logprobs(x, tokens, top=top, return_stats=True)
    assert all(torch.equal(o[:10].nan_to_num(7.0), o[-10:].nan_to_num(7.0)) for o in out)
    x, tokens = x[-10:], tokens[-10:]
    logp, entropy, tl, ti, stats = (o[-10:] for o in out)
    ninf = float("-inf")
    assert logp[0] == ninf and entropy[0] == 0 and ti[0].tolist() == list(range(top))
    assert bool((tl[0] == ninf).all())
    for i in (1, 5):
        assert abs(float(logp[i]) + math.log(V)) < 1e-5 * math.log(V) + 1e-7
        assert abs(float(entropy[i]) - math.log(V)) < 1e-5 * math.log(V)
        assert ti[i].tolist() == list(range(top))
    assert logp[2] == 0 and entropy[2] == 0 and ti[2, 0] == V // 2 and tl[2, 0] == 0
    rest = [j for j in range(V) if j != V // 2][:top - 1]
    assert ti[2, 1:].tolist() == rest and bool((tl[2, 1:] == ninf).all())
    assert bool(logp[3:5].isnan().all()) and bool(entropy[3:5].isnan().all())
    assert bool(((ti[3:5] >= 0) & (ti[3:5] < V)).all())
    assert all(len(set(ti[i].tolist())) == top for i in (3, 4))
    assert logp[6] == 0 and entropy[6] == 0 and ti[6].tolist() == list(range(top))
    assert bool(logp[7:9].isnan().all()) and bool(entropy[7:9].isfinite().all())
    assert logp[9] == ninf and bool(entropy[9].isfinite())
    one = torch.ones(10, device=DEV)
    d = ops.token_logprobs_grad(x, tokens, stats, entropy, one, one)
    assert not bool(d[0].any()) and not bool(d[2].any())
    assert bool(d[3:5].isnan().all()) and bool(d[7:9].isnan().all())
    assert bool(d[[1, 5, 6, 9]].isfinite().all()) and d[9, 2] == 0
    alone = ops.token_logprobs_grad(x, tokens, stats, entropy, None, one)
    assert torch.equal(d[9], alone[9])               # a logp of -inf gives nothing
    assert bool(alone[7:9].isfinite().all())
    part = one.clone()
    part[[3, 4, 7]] = 0.0                            # tokens that take no part are not read
    d = ops.token_logprobs_grad(x, tokens, stats, entropy, part)
    assert not bool(d[[3, 4, 7]].any())


def test_logprobs_ties(ops):
    """Equal values by column, -0 and +0 among them, over pieces, threads and edges."""
    for T, V in ((6, 40), (6, 300), (6, 5001), (6, 70000), (515, 9000)):
        g = torch.Generator().manual_seed(V)
        x = torch.randint(-1, 2, (T, V), generator=g).to(BF)
        x[x == 0] *= -1.0
        x[:, ::3] = x[:, ::3].abs()
        x = x.to(DEV)
        for xx in layouts(x):
            ti = ops.token_logprobs(xx, ids(T, V, 1), top=40)[3]
            want = (x.double() + 0.0).cpu().sort(dim=1, descending=True, stable=True).indices
            assert torch.equal(ti.cpu(), want[:, :40])


def test_logprobs_alternatives_side_by_side(ops):
    """The largest values in one thread's pieces, in falling and rising order."""
    for T, V in ((2, 600), (2, 9000), (512, 9000), (2, 131071)):
        x = torch.linspace(5, -5, V, device=DEV)[None].repeat(T, 1)
        x[1] = x[1].flip(0)
        x[:, 2048:2048 + 64] += 20.0
        out = ops.token_logprobs(x, ids(T, V, 1), top=64)
        assert torch.equal(out[3].cpu(), x.cpu().sort(dim=1, descending=True, stable=True)
                           .indices[:, :64])


def test_logprobs_autograd(ops):
    x, tokens = logits_case(50, 300, F32, 0.2)
    x.requires_grad_()
    g, k = normal((50,), F32, 5), normal((50,), F32, 6)
    logp, entropy, tl, ti = ops.token_logprobs(x, tokens, temperature=0.9, top=3)
    assert logp.requires_grad and entropy.requires_grad and not tl.requires_grad
    ((logp * g).masked_fill(logp == float("-inf"), 0.0) + entropy * k).sum().backward()
    r = ref.logprobs(x, tokens, 0.9)
    want, tol = ref.logprobs_grad(r, tokens, g, k, 0.9, F32)
    check("dlogits", x.grad, want, tol)
    for pick in (0, 1):
        x.grad = None
        ops.token_logprobs(x, tokens, temperature=0.9)[pick].nan_to_num(neginf=0.0).sum().backward()
        one = torch.ones(50, device=DEV)
        want, tol = ref.logprobs_grad(r, tokens, *((one, None) if pick == 0 else (None, one)),
                                      0.9, F32)
        check("dlogits", x.grad, want, tol)


# --------------------------------------------------------------------- together

def model(ops, c):
    """One layer's steps in a row, forward, 8-bit and backward, as a pass makes them."""
    e = ops.embedding(c["tokens"], c["table"], scale=4.0, dtype=F32)
    y, h = ops.rms_norm(c["x"], c["gain"], residual=e, dtype=BF)
    q, s, h2 = ops.rms_norm_int8(c["x"], c["gain"], residual=h)
    z = ops.int8_product(q, s, c["w"], c["w_scale"], dtype=F32)
    logp, entropy, tl, ti, stats = ops.token_logprobs(z, c["ids"], top=4, return_stats=True)
    dz = ops.token_logprobs_grad(z, c["ids"], stats, entropy, c["g"], c["g"])
    d, dx, dgain = ops.rms_norm_grad(c["x"], h, c["gain"], dh=h2, x_dtype=BF)
    dt = ops.embedding_grad(d, c["tokens"], len(c["table"]), scale=4.0)
    return e, y, h, q, s, h2, z, logp, entropy, tl, ti, dz, d, dx, dgain, dt


def model_case(ops, seed, T=700, D=128, V=50, N=77):
    w, w_scale = ops.quantize_rows(normal((N, D), F32, seed))
    return dict(tokens=ids(T, V, seed), table=normal((V, D), BF, seed + 1),
                x=normal((T, D), BF, seed + 2), gain=normal((D,), F32, seed + 3), w=w,
                w_scale=w_scale, ids=ids(T, N, seed + 4), g=normal((T,), F32, seed + 5))


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_run_of_them(ops):
    """The steps in a row against the same steps in 64 bits, each from what the one before
    gave; twice the same bits."""
    c = model_case(ops, 3)
    e, y, h, q, s, h2, z, logp, entropy, tl, ti, dz, d, dx, dgain, dt = out = model(ops, c)
    check("e", e, *ref.embedding(c["tokens"], c["table"], 4.0, F32))
    check("h", h, *ref.stream(c["x"], e))
    want, err = ref.rms(h, c["gain"], 1e-6)
    check("y", y, want, ref.rounded(want, BF, err))
    want, err = ref.rms(h2, c["gain"], 1e-6)
    quantized(q, s, want, err)
    want = (q.cpu().double() @ c["w"].cpu().double().t()) * ref.f64(s)[:, None] * ref.f64(
        c["w_scale"])
    check("z", z, want, 4 * E32 * want.abs())
    r = ref.logprobs(z, c["ids"], 1.0)
    check_logprobs((logp, entropy, tl, ti), r, 4)
    want, tol = ref.logprobs_grad(r, c["ids"], c["g"], c["g"], 1.0, F32)
    check("dz", dz, want, tol)
    r = ref.rms_grad(c["x"], h, c["gain"], h2, 1e-6)
    check("d", d, r["d"], ref.rounded(r["d"], F32, r["d_err"]))
    want, tol = ref.embedding_grad(d, c["tokens"], 50, 4.0, F32)
    check("dtable", dt, want, tol)
    assert same(out, model(ops, c))


def test_streams_and_threads(ops):
    """Calls on streams of their own, from threads of their own, at the same time."""
    cases = [model_case(ops, s, T=300 + 200 * s) for s in range(3)]
    want = [model(ops, c) for c in cases]
    torch.cuda.synchronize()
    got, errors = [None] * 3, []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(4):
                    got[i] = model(ops, cases[i])
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    assert all(same(a, b) for a, b in zip(want, got))


def test_captured_and_replayed(ops):
    """Two captured graphs that share a pool, replayed in turn with other inputs and eager
    calls between."""
    cases = [model_case(ops, 11), model_case(ops, 12, T=900)]
    new = [model_case(ops, 21), model_case(ops, 22, T=900)]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for c in cases:
            model(ops, c)
    stream.synchronize()
    graphs, outs, pool = [], [], None
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool, stream=stream):
            outs.append(model(ops, c))
        pool = g.pool()
        graphs.append(g)
    for turn in range(3):
        for i in (0, 1):
            if turn == 1:
                for k, v in new[i].items():
                    cases[i][k].copy_(v)
            want = model(ops, cases[i])
            graphs[i].replay()
            torch.cuda.synchronize()
            assert same(outs[i], want), (turn, i)


def test_a_large_product_captured(ops):
    """The largest tiles, and rows that are laid out anew, in a graph that is replayed with other
    operands."""
    for M, K, N in ((4096, 272, 4104), (700, 401, 300)):
        a, sa, w, sw, _ = product_case(M, K, N)
        stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            ops.int8_product(a, sa, w, sw)
        stream.synchronize()
        with torch.cuda.graph(g, stream=stream):
            out = ops.int8_product(a, sa, w, sw)
        for seed in range(3):
            a.copy_(int8s((M, K), 10 + seed))
            want = ops.int8_product(a, sa, w, sw)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_refuses_nothing_silently(ops):
    """Gradients that are asked for are formed or refused, under a graph of a graph too."""
    x = normal((4, 64), BF, 1).requires_grad_()
    for fn in (lambda: ops.quantize_rows(x), lambda: ops.rms_norm_int8(x),
               lambda: ops.rms_norm_int8(x.detach(), x[0])):
        with pytest.raises(ValueError):
            fn()
    with torch.no_grad():
        ops.quantize_rows(x)
    y = ops.rms_norm(x, dtype=F32)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()
    z = x.float().detach().requires_grad_()
    logp, entropy = ops.token_logprobs(z, ids(4, 64, 1))
    entropy.add_(1.0)                                # what the backward pass reads has changed
    with pytest.raises(RuntimeError):
        logp.sum().backward()


def test_far_offsets(ops):
    """Rows beyond 2^31 elements have the results of the same rows alone."""
    T, D = 525000, 4096 + 8
    x = torch.empty((T, D), dtype=BF, device=DEV)
    tail = normal((40, D), BF, 1)
    x.zero_()
    x[-40:] = tail
    gain = normal((D,), F32, 2)
    y, h = ops.rms_norm(x, gain, residual=x)
    a, b = ops.rms_norm(tail, gain, residual=tail)
    assert torch.equal(y[-40:], a) and torch.equal(h[-40:], b)
    del y
    d = ops.rms_norm_grad(x, h, dh=h)[0]
    assert torch.equal(d[-40:], ops.rms_norm_grad(tail, b, dh=b)[0])
    del d, h
    q, s = ops.quantize_rows(x)
    tq, ts = ops.quantize_rows(tail)
    assert torch.equal(q[-40:], tq) and torch.equal(s[-40:], ts)
    w, sw = ops.quantize_rows(normal((24, D), F32, 3))
    o = ops.int8_product(q, s, w, sw)
    assert torch.equal(o[-40:], ops.int8_product(tq, ts, w, sw))
    del q, o
    tokens = torch.full((T,), 3, dtype=torch.int64, device=DEV)
    tokens[-40:] = torch.arange(40, device=DEV) % 3
    dt = ops.embedding_grad(x, tokens, 4)
    want, tol = ref.embedding_grad(tail, tokens[-40:], 4, 1.0, F32)
    check("dtable", dt, want, tol)
    out = ops.embedding(torch.arange(T, device=DEV) % 40, tail)
    assert torch.equal(out[-40:], tail[torch.arange(T - 40, T, device=DEV) % 40])
    del out
    at = tokens * 0 + 5
    lp = ops.token_logprobs(x, at, top=2, return_stats=True)
    small = ops.token_logprobs(tail, at[:40], top=2, return_stats=True)
    assert all(torch.equal(p[-40:], r) for p, r in zip(lp, small))
    one = torch.ones(T, device=DEV)
    g = ops.token_logprobs_grad(x, at, lp[4], lp[1], one, one)
    assert torch.equal(g[-40:], ops.token_logprobs_grad(tail, at[:40], small[4], small[1],
                                                        one[:40], one[:40]))


def test_copies_of_operands_live_until_the_launch(ops, monkeypatch):
    """Operands that a call copies first are kept until its kernels are queued: memory that
    another thread allocates and fills in between is not theirs."""
    T, D, V = 3000, 96, 200
    tokens, x, gain = ids(2 * T, V, 1)[::2], normal((T, 2 * D), BF, 2)[:, ::2], normal((2 * D,), F32, 3)
    table, dy, dh = (normal((n, 2 * D), F32, 4 + n)[:, ::2] for n in (V, T, T + 1))
    logits, g = normal((T, 2 * V), F32, 5)[:, ::2], normal((2 * T,), F32, 6)[::2]
    a, w = int8s((T, 2 * D), 7)[:, ::2], int8s((V, 2 * D), 8)[:, ::2]

    def calls():
        _, entropy, *_, stats = ops.token_logprobs(logits, tokens, top=3, return_stats=True)
        return (ops.embedding(tokens, table), ops.embedding_grad(dy, tokens, V),
                *ops.rms_norm(x, gain[::2], residual=dy), *ops.rms_norm_int8(x, gain[::2]),
                *ops.rms_norm_grad(x, dy, gain[::2], dh=dh[:T]),
                ops.int8_product(a, g.abs(), w, gain[:1].expand(V)),
                *ops.token_logprobs(logits, tokens, top=3),
                ops.token_logprobs_grad(logits, tokens, stats, entropy, g, g))

    want = calls()
    real = ops._run

    def run(*args):
        taken = [torch.zeros(n, dtype=torch.uint8, device=DEV)
                 for n in 4 * [8 * T, 4 * T, 2 * T * D, 4 * T * D, 4 * V * D, 4 * T * V, T * D, V * D,
                               4 * D, 4 * V]]
        real(*args)
        del taken

    monkeypatch.setattr(ops, "_run", run)
    assert same(want, calls())

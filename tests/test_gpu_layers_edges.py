"""The layers around attention at values and lengths where one kernel's order of
additions, or one value's place among others, shows."""
from __future__ import annotations

import pytest
import torch

import layer_reference as ref
from seq_reference import E32
from test_gpu_layers import ids, layouts
from test_gpu_seq import BF, DEV, F32, FP, _say, check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from cusr_amd.kernel import seq_layers
    return seq_layers


# ------------------------------------------------- alternatives of rows with NaN

# symbols in LDS, a wave and four waves a row, a row cut into parts
NAN_ROWS = [(1, 1, 1), (7, 3, 7), (64, 5, 64), (21, 300, 9), (64, 300, 64), (700, 3, 64),
            (9001, 3, 40), (40003, 2, 64), (40003, 80, 5), (80001, 2, 5)]


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("V,T,top", NAN_ROWS)
def test_alternatives_of_rows_with_nan(ops, V, T, top, dt):
    """A NaN comes before every number, wherever it stands, and the lower column first among
    them: every column at most once, and none outside the row."""
    _say("nan", V, T, top, dt)
    g = torch.Generator().manual_seed(V)
    x = torch.randn(T, V, generator=g).to(dt)
    nan, inf = float("nan"), float("inf")
    x[0, 0] = nan                                    # in the first column alone
    if T > 1:
        x[1] = nan                                   # everywhere
    if T > 2:
        x[2, 0] = x[2, -1] = nan
        x[2, V // 2] = inf
    if T > 3:
        x[3] = -inf
        x[3, 0] = nan
    if T > 4:
        x[4] = nan
        x[4, 0] = -inf
    x = x.to(DEV)
    want = x.cpu().float().sort(dim=1, descending=True, stable=True).indices[:, :top]
    for xx in layouts(x):
        logp, entropy, top_logp, top_ids = ops.token_logprobs(xx, ids(T, V, 1), top=top)
        assert bool(((top_ids >= 0) & (top_ids < V)).all())
        assert torch.equal(top_ids.cpu(), want)
        odd = x.isnan().any(1)
        assert bool(top_logp[odd].isnan().all()) and bool(logp[odd].isnan().all())
        assert not bool(top_logp[~odd].isnan().any())


# --------------------------------------------------- scales far from each other

# few tokens' kernel, tiles of 64, 128 and 256, terms cut among blocks, rows laid out anew,
# columns that no eights fill
PRODUCTS = [(1, 64, 33), (20, 128, 96), (70, 96, 100), (700, 64, 520), (3000, 64, 2056),
            (2048, 128, 4096), (24, 16384, 96), (64, 16384, 1001), (33, 77, 40)]


@pytest.mark.parametrize("out", [F32, BF])
@pytest.mark.parametrize("M,K,N", PRODUCTS)
def test_int8_product_of_scales_far_apart(ops, M, K, N, out):
    """A sum times one scale may pass float32 where the whole product does not; the rows
    beside such a one keep their bits."""
    _say("scales", M, K, N, out)
    g = torch.Generator().manual_seed(M + N)
    a, w = (torch.randint(-127, 128, s, generator=g).to(torch.int8).to(DEV) for s in ((M, K), (N, K)))
    a[:, 0], w[:, 0] = 127, 127
    usual = torch.rand(M, generator=g).to(DEV) + 0.5
    sa, sw = usual.clone(), (torch.rand(N, generator=g) + 0.5).to(DEV) * 1e-36
    far = torch.arange(M, device=DEV) % 3 == 0
    sa[far] *= 2e38
    sums = a.cpu().double() @ w.cpu().double().t()
    want = sums * sa.cpu().double()[:, None] * sw.cpu().double()
    got = ops.int8_product(a, sa, w, sw, dtype=out)
    assert bool(got.isfinite().all())
    # an integer's rounding to float32 and two products', and the output's
    least = torch.full_like(want, 2.0 ** -149 if out is F32 else 2.0 ** -133)
    check("o", got, want, ref.rounded(want, out, 4 * E32 * want.abs()) + least)
    plain = ops.int8_product(a, usual, w, sw, dtype=out)
    assert torch.equal(got[~far], plain[~far])
    # the whole product passes float32: infinite, and 0 where the sum is 0
    a[:, 1:], w[:, 1:] = 0, 0
    w[::2, 0] = 0
    got = ops.int8_product(a, torch.full_like(sa, 3e38), w, sw * 1e36, dtype=out)
    assert bool(got[:, 1::2].isinf().all()) and not bool(got[:, ::2].any())
    got = ops.int8_product(a, sa * float("inf"), w, sw, dtype=out)
    assert bool(got[:, 1::2].isinf().all()) and bool(got[:, ::2].isnan().all())


# ----------------------------------------------------------- sums that are exact

EXACT = [
    # tokens, rows, width, type
    (300, 22, 128, F32), (2049, 511, 64, BF), (66000, 22, 40, BF), (70001, 9, 8, F32),
    (600000, 1000, 1, F32), (530000, 2, 16, BF), (40000, 128, 130, BF), (33000, 32, 257, FP),
    (33000, 33, 257, FP), (33000, 5000, 264, F32), (32768, 513, 9, BF), (80000, 200, 136, BF),
    (256, 1, 2056, BF), (257, 700, 40, FP), (20000, 31, 2056, BF), (700, 40, 2056, BF),
    (100000, 3, 1160, FP),
]


@pytest.mark.parametrize("T,V,D,dt", EXACT)
def test_embedding_grad_of_whole_numbers(ops, T, V, D, dt):
    """Sums of small whole numbers are exact in float32 in any order: every token counts,
    once."""
    _say("whole", T, V, D, dt)
    g = torch.Generator().manual_seed(T)
    d = torch.randint(1, 4, (T, D), generator=g).to(dt).to(DEV)
    tokens = ids(T, V + 2, 4) - 1                    # a few outside the table
    tokens[T // 3:T // 2] = V // 2
    inside = (tokens >= 0) & (tokens < V)
    want = torch.zeros(V, D, dtype=torch.float64, device=DEV)
    want.index_add_(0, tokens[inside], d[inside].double())
    for x in layouts(d):
        got = ops.embedding_grad(x, tokens, V, scale=0.5)
        assert torch.equal(got.double(), want * 0.5)


@pytest.mark.parametrize("T,D,dt", [(1, 8, F32), (301, 1, BF), (20001, 96, BF), (40003, 128, F32),
                                    (30001, 250, FP), (9001, 512, BF), (5003, 1024, F32),
                                    (20001, 2048, BF), (4099, 4096, FP), (2051, 8192, BF),
                                    (1501, 16384, F32), (700, 16400, BF)])
def test_norm_gain_grad_of_whole_numbers(ops, T, D, dt):
    """Rows of ones of either sign are their own norm, and the gain's gradient a sum of whole
    numbers: every row counts, once."""
    _say("whole", T, D, dt)
    g = torch.Generator().manual_seed(T)
    h = (torch.randint(0, 2, (T, D), generator=g) * 2 - 1).to(dt).to(DEV)
    dy = torch.randint(-3, 6, (T, D), generator=g).to(dt).to(DEV)
    gain = torch.ones(D, device=DEV)
    want = (dy.double() * h.double()).sum(0)
    for x, y in zip(layouts(h), layouts(dy)):
        got = ops.rms_norm_grad(y, x, gain, eps=0.0)[2]
        assert torch.equal(got.double(), want)


# --------------------------------------------------- long sums of one sign

def one_row(D, dt, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(1, D, generator=g) * 0.5 + 0.5).to(dt).to(DEV)


# what follows one another in float32: a wave's or a chunk's additions, 4,096 at most, and the
# few that join them
DEPTH = 4096 + 64


@pytest.mark.parametrize("T,V,D", [(1200000, 32, 16384), (1200000, 20, 1027), (9000000, 7, 128),
                                   (3000000, 5, 40000), (70000000, 32, 120),
                                   (4000000, 33, 136), (6000000, 40, 24), (60000000, 33, 24)])
def test_embedding_grad_of_one_sign(ops, T, V, D):
    """One row's gradient over and over, whose roundings do not cancel: the error does not grow
    with the tokens."""
    _say("one sign", T, V, D)
    d = one_row(D, F32, 1)
    tokens = torch.full((T,), 3, dtype=torch.int32, device=DEV)
    tokens[::7] = torch.arange(len(tokens[::7]), device=DEV, dtype=torch.int32) % V
    got = ops.embedding_grad(d.expand(T, D), tokens, V)
    want = torch.bincount(tokens.long(), minlength=V).double()[:, None] * d.double()
    check("dtable", got, want.cpu(), want.cpu() * DEPTH * E32)


@pytest.mark.parametrize("T,D", [(3000000, 8200), (1000000, 16392), (12000000, 1032)])
def test_norm_gain_grad_of_one_sign(ops, T, D):
    """The same of the gain's gradient, whose groups add 2,048 rows at most."""
    _say("one sign", T, D)
    h, dy, gain = one_row(D, BF, 1), one_row(D, F32, 2), torch.ones(D, device=DEV)
    got = ops.rms_norm_grad(dy.expand(T, D), h.expand(T, D), gain)[2]
    n = h.double() * (h.double().square().mean(1, keepdim=True) + 1e-6) ** -0.5
    want = (T * dy.double() * n)[0].cpu()
    # the norm of a row: half the relative error of its sum of squares, and some products
    check("dgain", got, want, want * (2048 + 64 + 0.5 * (D / 64 + 16) + 8) * E32)

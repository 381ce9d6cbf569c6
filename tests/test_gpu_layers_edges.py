"""The layers around attention at values and lengths where one kernel's order of
additions, or one value's place among others, shows."""
from __future__ import annotations

import pytest
import torch

from test_gpu_layers import ids, layouts
from test_gpu_seq import BF, DEV, F32, _say

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

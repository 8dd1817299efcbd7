"""The paged cache at its edges: values that are not finite."""
import math

import pytest
import torch

from test_cache import BF16, DEV, F16, Batch, cache, near


# ---- values that are not finite ----------------------------------------------------------------------
def peaked_batch(new, past, dim, dtype, low):
    """All scores 0, those of the keys `low(j)` 300 powers of two below: their weights are zero in 32 bits."""
    b = Batch(new, past, 8, 2, dim, dtype, 16, seed=5)
    b.q.fill_(1.0)
    for r, (a, p) in enumerate(zip(new, past)):
        t = torch.arange(a + p, device=DEV)
        k = torch.where(low(t), -300.0 * math.log(2.0) / math.sqrt(dim), 0.0)
        b.k[b.table[r].long()[t // 16], t % 16] = k[:, None, None].expand(-1, 2, dim).to(dtype)
    return b


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("what, bad", [("k", "nan"), ("k", "inf"), ("v", "nan"), ("v", "inf")])
def test_a_value_a_row_sees_reaches_it_whatever_its_weight(what, bad, new, dim, dtype):
    # 4 rows a kv head, and 160: both kernels; keys far below the best ones in pieces of their own (the first
    # ones, and the first half of the request), and within a tile (sixteen of 64, what one warp takes)
    for low, at in ((lambda t: t < 192, 100), (lambda t: t < 2500, 100), (lambda t: (t // 16) % 4 == 1, 4949)):
        b = peaked_batch([new, new], [5000, 5000], dim, dtype, low)
        clean = b.run(cache(8, 2, dim, 16, 2, 512, dtype), max_new=new)
        near(clean, b.want(), dtype)
        getattr(b, what)[int(b.table[0, at // 16]), at % 16] = float(bad)
        c = cache(8, 2, dim, 16, 2, 512, dtype)
        got = b.run(c, max_new=new)
        c.status()
        assert not bool(got[:new].isfinite().any())
        assert torch.equal(got[new:], clean[new:])      # the request that does not see it


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_score_of_minus_infinity_is_a_weight_of_zero(dim, new):
    b = Batch([new, new], [900, 30], 8, 2, dim, BF16, 16)
    b.q.abs_()
    b.k[int(b.table[0, 50]), 3] = -math.inf
    b.k[b.table[1][b.table[1] >= 0].long()] = -math.inf   # no key of the second request has a weight: zeros
    got = b.run(cache(8, 2, dim, 16, 2, 512, BF16), max_new=new)
    b.k.nan_to_num_(0, 0, 0)
    want = b.want(drop=[(0, 803)])
    near(got[:new], tuple(x[:new] for x in want), BF16)
    assert bool((got[new:] == 0).all())

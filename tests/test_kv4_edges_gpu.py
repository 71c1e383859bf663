"""Edges of attention over the 4-bit cache on the GPU: shares of the work without any keys, lengths that take a block more
than a second, recorded errors, rows that are not finite, weights spread over many small probabilities. Bounds: tests/_kv4.py."""

import math

import numpy as np
import pytest
import torch
from _kv4 import attend64, cumulative, ints, make_cache
from test_kv4_gpu import BF, HF, randn, run_case, takes_many

from tfimage import kv4

pytestmark = pytest.mark.gpu


NOTHING = [  # lens, rows, (Hq, Hk), dim, page, causal: row blocks that see keys in front of row blocks that see none
    ([3000] + [0] * 255, [16] * 256, (32, 8), 128, 64, False),     # one request among the empty places of a full batch
    ([256], [4096], (128, 128), 64, 64, True),                     # the first 3840 rows lie before the first key
    ([0] * 40 + [700, 0, 0, 0, 0, 900] + [0] * 60, [70] * 106, (16, 4), 64, 32, False),
    ([900 if i % 7 == 3 else 0 for i in range(300)], [20 if i % 5 else 0 for i in range(300)], (64, 8), 64, 16, True)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", NOTHING)
def test_row_blocks_that_see_nothing(dev, dtype, case):
    """A block's share with keys, then several without any: all are written (zeros, lse -inf) and no wait runs out."""
    lens, rows, heads, dim, page, causal = case
    assert takes_many(lens, rows, heads, page)
    run_case(dev, lens, rows, heads, dim, page, dtype, causal, False, seed=len(rows) + dim, behind=2)


@pytest.mark.parametrize("rows", [[64] * 6, [64, 200]])
def test_a_share_longer_than_a_second(dev, rows):
    """A block whose first row block has 96 million keys and 64 rows (its other query tile has none), behind it short ones:
    five that are handed out when the first is done, or one with rows in both query tiles. 148 heads are 148 equal shares, and
    one page serves all positions: the exact result is that of 256 keys. Of the long rows it is the sum that is compared
    (750000 tiles, each a rounding of 2^-24 at most), the outputs only for being there."""
    long, heads, dim, page = 96_000_000 // 256 * 256, 148, 64, 256
    lens = [long] + [page] * (len(rows) - 1)
    assert takes_many(lens, rows, (heads, heads), page)
    cache, _, (one,) = make_cache(dev, [page], heads, dim, page, seed=41, spare=0)
    table = torch.zeros((len(rows), long // page), dtype=torch.int32, device=dev)
    q = randn((sum(rows), heads, dim), 42, HF)
    out, lse = kv4.attention(q.to(dev), cache, table, ints(lens, dev), cu=ints(cumulative(rows), dev), return_lse=True)
    ref, ref_lse, tol, tol_lse = attend64(q.double().numpy(), [one] * len(rows), rows, dim ** -0.5, False, half_step=2.0 ** -11)
    ref_lse[:64] += math.log(long // page)
    tol_lse[:64] += long / 128 * 2.0 ** -24
    got = out.double().cpu().numpy()
    assert (np.abs(got[64:] - ref[64:]) <= tol[64:]).all() and np.isfinite(got).all() and (got[:64] != 0).all()
    assert (np.abs(lse.double().cpu().numpy() - ref_lse) <= tol_lse).all()

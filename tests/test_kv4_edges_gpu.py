"""Edges of attention over the 4-bit cache on the GPU: shares of the work without any keys, lengths that take a block more
than a second, recorded errors, rows that are not finite, weights spread over many small probabilities. Bounds: tests/_kv4.py."""

import pytest
import torch
from test_kv4_gpu import BF, HF, run_case, takes_many

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

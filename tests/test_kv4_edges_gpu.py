"""Edges of attention over the 4-bit cache on the GPU: shares of the work without any keys, lengths that take a block more
than a second, recorded errors, rows that are not finite, weights spread over many small probabilities. Bounds: tests/_kv4.py."""

import ctypes
import math

import numpy as np
import pytest
import torch
from _kv4 import attend64, cumulative, ints, make_cache
from test_kv4_gpu import BF, HF, randn, run_case, takes_many

from tfimage import _lib, kernels as K, kv4

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


@pytest.mark.parametrize("rows", [1, 4, 150])
def test_calls_after_a_recorded_error(dev, rows):
    """With a code in the device error word (a wait of another kernel that nothing satisfies, as in test_failure_gpu) an
    attention call returns, whatever its waits find; with the word cleared it gives the bits it gave before."""
    heads, dim, page = (16, 4), 128, 64
    cache, table, _ = make_cache(dev, [9000, 3000], heads[1], dim, page, seed=51)
    lens = ints([9000, 3000], dev)
    assert takes_many([9000, 3000], [rows, rows], heads, page) == (rows == 150)
    calls = []
    for fresh in (False, True):
        q, k, v = (randn((2 * rows, h, dim), 52 + i, BF).to(dev) for i, h in enumerate((heads[0], heads[1], heads[1])))
        calls.append(lambda q=q, new=dict(k_new=k, v_new=v) if fresh else {}: kv4.attention(q, cache, table, lens, **new))
    want = [call() for call in calls]
    nbytes, _ = _lib.tp_layout(2, 1024, 256)
    own, silent = (torch.zeros(nbytes, dtype=torch.uint8, device=dev) for _ in range(2))
    comm = _lib.TpComm(2, 0, (ctypes.c_void_p * _lib.TP_MAX_WORLD)(own.data_ptr(), silent.data_ptr()), 1024, 256)
    assert _lib.device_status(reset=True) == 0
    _lib.tp_wait(comm, 1024, 256, 1, dev)
    for call in calls:
        call()
    assert _lib.device_status(reset=True) == 0x304           # the first code stays
    assert all(torch.equal(call(), w) for call, w in zip(calls, want))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("seqs,rows", [(500, 1), (40, 64)])
def test_many_small_weights_beside_a_large_one(dev, dtype, seqs, rows):
    """A key that takes nearly all of the weight and has a value of 0, and 16383 keys of 2^-26.5 of its weight each, whose
    values have one sign: the result is theirs alone. Probabilities may be lost below 2^-32 of the largest, not before.
    As many sequences (on the same pages) as leave each to one block, so that the large weight is everyone's base."""
    heads, dim, page, n = 4, 64, 64, 16384
    assert takes_many([n] * seqs, [rows] * seqs, (heads, heads), page) == (rows == 64)
    g = torch.Generator().manual_seed(61)
    k, v = (torch.randn((n, heads, dim), generator=g) * s for s in (0.25, 0.2))
    v += 1
    k[..., 0], k[5], v[5] = 0, 0, 0
    k[5, :, 0] = 6
    q = torch.randn((rows, heads, dim), generator=g) * 0.2
    q[..., 0] = 26.5 * math.log(2) * dim ** 0.5 / 6
    cache = kv4.Kv4Cache.empty(n // page, page, heads, dim, kv4.global_for(6.0), kv4.global_for(2.0), dev)
    table = torch.arange(n // page, dtype=torch.int32, device=dev).expand(seqs, -1).contiguous()
    kv4.write(cache, table[:1], ints([0], dev), k.to(dev), v.to(dev))
    held = torch.empty((2, n, heads, dim), device=dev)
    kv4.read(cache, table[:1], ints([0], dev), held[0], held[1])
    seq = tuple(h.double().cpu().numpy() for h in held)
    assert (seq[0][5, :, 0] > 5.5).all() and (seq[1][5] == 0).all()
    q = q.to(dtype)
    half = torch.finfo(dtype).eps / 2
    ref, ref_lse, tol, tol_lse = attend64(q.double().numpy(), [seq], [rows], dim ** -0.5, False, half_step=half, least_p=2.0 ** -32)
    assert (tol / np.abs(ref)).max() < 0.04             # 2^-32 of 16384 keys beside 2^-12.5: 2.2 %, and two roundings of 2^-8
    out, lse = kv4.attention(q.to(dev).repeat(seqs, 1, 1), cache, table, ints([n] * seqs, dev), return_lse=True)
    got, e = (t.double().cpu().numpy().reshape(seqs, *r.shape) for t, r in ((out, ref), (lse, ref_lse)))
    assert (np.abs(got - ref) <= tol).all(), f"worst {np.max(np.abs(got - ref) / tol):.2f} of the bound"
    assert (np.abs(e - ref_lse) <= tol_lse).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens,rows,heads,causal,fresh", [
    ([300, 0], [3, 2], (8, 2), False, False), ([3, 700], [5, 9], (4, 4), True, False), ([200, 1], [6, 3], (4, 2), True, True),
    ([9000], [2], (2, 1), False, False), ([40, 500], [200, 300], (24, 8), True, False), ([0, 2500], [130, 120], (16, 8), False, True),
    ([3000], [200], (8, 2), False, False), ([1, 0], [1, 260], (32, 32), True, True)])
def test_query_rows_that_are_not_finite(dev, dtype, lens, rows, heads, causal, fresh):
    """A NaN or an infinity anywhere in a query row: NaN in its output and lse, or 0 and -inf if it sees nothing. Rows beside it
    are right."""
    (Hq, Hk), dim, page = heads, 128, 64
    cache, table, seqs = make_cache(dev, lens, Hk, dim, page, seed=71, poison=False)
    T = sum(rows)
    q = randn((T, Hq, dim), 72, dtype)
    kn, vn = (randn((T, Hk, dim), 73 + i, dtype) for i in range(2)) if fresh else (None, None)
    n64 = lambda t: None if t is None else t.double().numpy()   # noqa: E731
    half = torch.finfo(dtype).eps / 2
    ref, ref_lse, tol, tol_lse = attend64(n64(q), seqs, rows, dim ** -0.5, causal, n64(kn), n64(vn), new_p=half, half_step=half)
    bad = torch.zeros((T, Hq), dtype=torch.bool)
    for i, x in enumerate((float("nan"), float("inf"), -float("inf"))):
        for j, c in enumerate((0, 37, 64, 127)):
            r, h = (29 * i + 17 * j) % T, (5 * i + 3 * j) % Hq
            q[r, h, c] = x
            bad[r, h] = True
    q[T - 1, Hq - 1] = float("inf")
    bad[T - 1, Hq - 1] = True
    up = lambda t: None if t is None else t.to(dev)   # noqa: E731
    out, lse = kv4.attention(up(q), cache, table, ints(lens, dev), cu=ints(cumulative(rows), dev), causal=causal, k_new=up(kn),
                             v_new=up(vn), return_lse=True)
    got, e, bad = out.double().cpu().numpy(), lse.double().cpu().numpy(), bad.numpy()
    nothing = np.isneginf(ref_lse)
    assert np.isnan(got[bad & ~nothing]).all() and np.isnan(e[bad & ~nothing]).all()
    assert (got[nothing] == 0).all() and np.isneginf(e[nothing]).all()
    fine = ~bad & ~nothing
    assert (np.abs(got[fine] - ref[fine]) <= tol[fine]).all() and (np.abs(e[fine] - ref_lse[fine]) <= tol_lse[fine]).all()


def test_strides_of_a_single_row_or_head_do_not_matter(dev):
    """One token out of rows that are not a multiple of 16 bytes long, and one head out of such heads, each on a 16-byte boundary:
    the same as contiguous ones."""
    H, D, page = 4, 64, 16
    cache, table, _ = make_cache(dev, [40], H, D, page, seed=81, poison=False)
    rows = randn((3, H * D + 4), 82, BF).to(dev)
    third = lambda t: torch.as_strided(t, (1, H, D), (H * D + 4, D, 1), 2 * (H * D + 4))   # noqa: E731 (520 bytes a row)
    x = third(rows)
    assert x.stride(0) % 8 and x.data_ptr() % 16 == 0
    same = x.contiguous()
    lens, pos = ints([40], dev), ints([17], dev)
    want = kv4.attention(same, cache, table, lens, k_new=same, v_new=same)
    assert torch.equal(kv4.attention(x, cache, table, lens, k_new=x, v_new=x), want)
    kv4.read(cache, table, pos, back := torch.empty_like(same), torch.empty_like(same))
    wide = torch.zeros_like(rows)
    kv4.read(cache, table, pos, third(wide), torch.empty_like(same))
    assert torch.equal(wide[2, :H * D].view(1, H, D), back) and (wide[:2] == 0).all() and (wide[2, H * D:] == 0).all()
    kv4.write(cache, table, pos, x, x)
    kv4.read(cache, table, pos, first := torch.empty_like(same), torch.empty_like(same))
    kv4.write(cache, table, pos, same, same)
    kv4.read(cache, table, pos, back, torch.empty_like(same))
    assert torch.equal(first, back)
    ids = torch.tensor([[3.0, 4.0, 5.0]], device=dev)
    want = K.rope_axes(same[None], None, ids, (16, 24, 24))[0]
    assert torch.equal(K.rope_axes(x[None], None, ids, (16, 24, 24))[0], want)
    one = torch.as_strided(randn((5, 208), 83, BF).to(dev), (5, 1, D), (208, D + 4, 1), 2 * (D + 4))   # the third of such heads
    assert one.data_ptr() % 16 == 0 and one.stride(1) % 8
    assert torch.equal(K.rope_axes(one[None], None, ids.expand(5, 3).contiguous(), (16, 24, 24))[0],
                       K.rope_axes(one.contiguous()[None], None, ids.expand(5, 3).contiguous(), (16, 24, 24))[0])


# A product's fp32 accumulator is not rounded but cut: taken as 4 units at most (2^-21 of the sum so far) for each addition of 16
# keys, half of that over a sum that grows evenly. Sums begin again every 128 tiles of 128 keys: 1024 additions.
CUT = 1024 * 2.0 ** -21 / 2


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_sums_of_one_sign(dev, dim, dtype):
    """A million keys in one block's share, all values of one sign: the sums hold (without carrying, 0.7 % was lost). One page
    serves all positions: the exact result is that of 256 keys."""
    heads, rows, page, n = 148, 64, 256, 1 << 20
    assert takes_many([n], [rows], (heads, heads), page)
    cache, one_table, _ = make_cache(dev, [page], heads, dim, page, seed=91, spare=0)
    v = (randn((page, heads, dim), 92, torch.float32) * 0.2 + 1).to(dev)
    k = torch.empty_like(v)
    kv4.read(cache, one_table, ints([0], dev), k, torch.empty_like(v))
    kv4.write(cache, one_table, ints([0], dev), k, v)
    kv4.read(cache, one_table, ints([0], dev), k, v)
    q = randn((rows, heads, dim), 93, dtype)
    table = torch.zeros((1, n // page), dtype=torch.int32, device=dev)
    out, lse = kv4.attention(q.to(dev), cache, table, ints([n], dev), return_lse=True)
    half = torch.finfo(dtype).eps / 2
    ref, ref_lse, tol, tol_lse = attend64(q.double().numpy(), [(k.double().cpu().numpy(), v.double().cpu().numpy())], [rows],
                                          dim ** -0.5, False, half_step=half)
    err = np.abs(out.double().cpu().numpy() - ref)
    tol += CUT * np.abs(ref)
    assert (err <= tol).all(), f"worst {np.max(err / tol):.2f} of the bound"
    # 8192 roundings of 2^-24 each between two carries' 64, half of that over an even sum
    off = np.abs(lse.double().cpu().numpy() - (ref_lse + math.log(n // page)))
    assert (off <= tol_lse + 128 * 2.0 ** -25 + 64 * 2.0 ** -24).all(), off.max()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,new,causal,fresh", [(16384, 300, False, True), (16384, 300, True, True), (16300, 300, False, True),
                                                (16640, 100, True, True), (33000, 129, True, False), (100, 17000, False, True)])
def test_sums_carried_over_cached_and_new_keys(dev, dtype, n, new, causal, fresh):
    """Shares of more than 128 tiles: sums are carried in front of, at and behind the border between cached and new keys. As many
    sequences (on the same pages, with the same rows) as leave row blocks whole; the first one's rows are compared, all are alike."""
    heads, dim, page = 2, 64, 256
    seqs = 74 if new < 1000 else 2
    pages = -(-n // page)
    assert takes_many([n] * seqs, [new] * seqs, (heads, heads), page)
    cache, table, seq = make_cache(dev, [n], heads, dim, page, seed=95)
    q, k, v = (randn((new, heads, dim), 96 + i, dtype) for i in range(3))
    rep = lambda t: t.to(dev).repeat(seqs, 1, 1)   # noqa: E731
    own = dict(k_new=rep(k), v_new=rep(v)) if fresh else {}
    out, lse = kv4.attention(rep(q), cache, table.expand(seqs, pages).contiguous(), ints([n] * seqs, dev), causal=causal, return_lse=True,
                             **own)
    out, lse = out.view(seqs, new, heads, dim), lse.view(seqs, new, heads)
    if new < 1000:
        assert (out == out[:1]).all() and (lse == lse[:1]).all()
    some = slice(None) if new < 1000 else slice(0, new, 211)                 # (not causal there: rows do not depend on one another)
    half = torch.finfo(dtype).eps / 2
    n64 = lambda t: t.double().numpy()   # noqa: E731
    kc, vc = seq[0]
    if new < 1000:
        ref, ref_lse, tol, tol_lse = attend64(n64(q), seq, [new], dim ** -0.5, causal, *((n64(k), n64(v)) if fresh else ()), new_p=half,
                                              half_step=half)
    else:
        both = [(np.concatenate([kc, n64(k)]), np.concatenate([vc, n64(v)]))]
        ref, ref_lse, tol, tol_lse = attend64(n64(q[some]), both, [len(q[some])], dim ** -0.5, False, cached_p=half, half_step=half)
    err = np.abs(out[0, some].double().cpu().numpy() - ref)
    tol += CUT * np.abs(ref)
    assert (err <= tol).all(), f"worst {np.max(err / tol):.2f} of the bound"
    assert (np.abs(lse[0, some].double().cpu().numpy() - ref_lse) <= tol_lse + 192 * 2.0 ** -24).all()

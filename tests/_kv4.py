"""Shared pieces of the 4-bit cache tests: a seeded cache with its values in float64, the packed batch's page tables,
and attention in float64 with an error bound from the kernels' roundings."""

import numpy as np
import torch

from oracle import nvfp4 as onv
from tfimage import kv4


def values64(codes, sf, g):
    """float64 values of numpy codes [..., D / 2] and scale bytes [..., D / 16]."""
    n = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])
    v = onv.E2M1_LUT[n].astype(np.float64).reshape(*sf.shape, 16)
    return (v * onv.E4M3_TABLE[sf].astype(np.float64)[..., None]).reshape(n.shape) * float(np.float32(g))


def make_cache(dev, lens, heads, dim, page, seed, spare=2, k_global=6.0 / 2688, v_global=5.0 / 2688, poison=True):
    """A cache whose sequences have ``lens`` rows in shuffled pages. With ``poison`` every row behind a length (and every
    spare page) has NaN scales. -> (cache on dev, table on dev, [(k, v) float64 [len, heads, dim] per sequence])."""
    rng = np.random.default_rng(seed)
    need = [max(1, -(-n // page)) for n in lens]
    pages = sum(need) + spare
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((len(lens), max(need)), -7, dtype=np.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    buf, seqs = {}, [[] for _ in lens]
    for name, g in (("k", k_global), ("v", v_global)):
        x = rng.standard_normal((pages * heads * page, dim)).astype(np.float32)
        codes, sf = onv.quantize(x, np.float32(g))
        codes, sf = codes.reshape(pages, heads, page, dim // 2), sf.reshape(pages, heads, page, dim // 16)
        live = np.zeros((pages, page), bool)
        for b, n in enumerate(lens):
            p = np.arange(n)
            live[table[b, p // page], p % page] = True
            seqs[b].append(values64(codes[table[b, p // page], :, p % page], sf[table[b, p // page], :, p % page], g))
        if poison:
            sf = np.where(live[:, None, :, None], sf, np.uint8(0x7F))
        buf[name] = torch.from_numpy(codes).to(dev), torch.from_numpy(np.ascontiguousarray(sf)).to(dev)
    cache = kv4.Kv4Cache(*buf["k"], *buf["v"], k_global, v_global)
    return cache, torch.from_numpy(table).to(dev), seqs


def ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def cumulative(rows):
    return [0, *np.cumsum(rows).tolist()]


def attend64(q, seqs, rows, scale, causal, k_new=None, v_new=None, cached_p=2.0 ** -11, new_p=2.0 ** -8, half_step=2.0 ** -8,
             least_p=2.0 ** -25):
    """float64 attention of packed q [T, Hq, D] (and new rows), and the bound of a kernel's error: half a step of the
    output, half a step of each probability in front of the second product (``cached_p`` / ``new_p``, relative, with
    ``least_p`` of the largest for fp16's smallest ones), and fp32 dot products of D terms in the exponent (each score off by
    at most (D + 8) 2^-24 sum |q k|, an e-fold as much in the probabilities and their sum; exp2 and the final division
    are within the 8 extra units).
    -> out, lse, bound of out, bound of lse (numpy)."""
    T, Hq, D = q.shape
    out, lse = np.zeros((T, Hq, D)), np.full((T, Hq), -np.inf)
    tol, tol_lse = np.zeros((T, Hq, D)), np.zeros((T, Hq))
    lo = 0
    for (kc, vc), n in zip(seqs, rows):
        L = kc.shape[0]
        k, v = kc, vc
        if k_new is not None:
            k, v = np.concatenate([kc, k_new[lo:lo + n]]), np.concatenate([vc, v_new[lo:lo + n]])
        i = np.arange(n)[:, None]
        last = np.full((n, 1), len(k) - 1)
        if causal:
            last = L + i if k_new is not None else L - n + i
        seen = np.arange(len(k))[None] <= last
        part = np.where(np.arange(len(k)) < L, cached_p, new_p)
        for h in range(Hq):
            kh, vh, qh = k[:, h // (Hq // kc.shape[1])], v[:, h // (Hq // kc.shape[1])], q[lo:lo + n, h]
            s = np.where(seen, scale * (qh @ kh.T), -np.inf)
            top = s.max(-1, keepdims=True, initial=-np.inf)
            top = np.where(np.isfinite(top), top, 0.0)
            p = np.exp(s - top)
            total = p.sum(-1, keepdims=True)
            some = total > 0
            w = p / np.where(some, total, 1.0)
            ds = (D + 8) * 2.0 ** -24 * abs(scale) * np.max(np.where(seen, np.abs(qh) @ np.abs(kh).T, 0.0), -1, initial=0.0)
            ds = ds[:, None] + 2.0 ** -22 * (1 + np.abs(top))
            out[lo:lo + n, h] = w @ vh
            spread = w @ np.abs(vh)
            tiny = least_p / np.where(some, total, 1.0) * np.abs(vh).sum(0, keepdims=True)
            tol[lo:lo + n, h] = (half_step * np.abs(out[lo:lo + n, h]) + (w * part) @ np.abs(vh) + 2 * np.e * ds * spread
                                 + tiny)
            lse[lo:lo + n, h] = np.where(some, top + np.log(np.where(some, total, 1.0)), -np.inf)[:, 0]
            tol_lse[lo:lo + n, h] = (2 * ds)[:, 0] + 2.0 ** -23 * np.abs(np.where(some[:, 0], lse[lo:lo + n, h], 0.0))
        lo += n
    return out, lse, tol, tol_lse

"""A 4-bit key / value cache (NVFP4, in pages) and attention over it: ``write`` quantises rows into the cache,
``read`` takes them out again, ``attention`` attends over cached positions and, if given, the call's own keys and
values behind them. This build's addition (the reference keeps its prompt prefix in bf16 and calls torch SDPA,
qwen_image21.py:180-199): a cached token takes 9/16 byte a value instead of 2, so 3.6 times the prompts fit, and one
set of pages can serve every image of a batch.

The packed batch of the three calls: ``table`` int32 [B, max_pages] gives the pages of each sequence; rows
``[cu[b], cu[b + 1])`` of the row tensors belong to sequence b (``cu`` int32 [B + 1]; None: the rows divide evenly).
Rows behind ``cu[B]`` are neither read nor written. Tables, lengths and ``cu`` stay on the device: nothing here
synchronises, and all three calls can be captured into a CUDA graph and replayed with other lengths.
"""

from __future__ import annotations

import ctypes
import operator

import torch

from . import _lib

FP4_TOP, E4M3_TOP = 6.0, 448.0


class Kv4Cache:
    """One layer's cache: codes uint8 [pages, heads, page_size, D / 2] (two E2M1 values a byte, the even one low) and
    scales uint8 [pages, heads, page_size, D / 16] (one E4M3 byte per 16 values) of keys and of values, with one fp32
    factor each: value = lut[code] * e4m3(scale) * global. page_size: a power of two from 16 to 256; D: 64 or 128.

    The calls go by the addresses and factors of the constructor, so they cannot be assigned to: a pool that grows, or
    gets other factors, is a new Kv4Cache (captured graphs keep the old one's)."""

    __slots__ = ("_k_codes", "_k_sf", "_v_codes", "_v_sf", "_k_global", "_v_global", "_pages", "_heads", "_page_size",
                 "_dim", "index", "struct", "ref")

    def __init__(self, k_codes: torch.Tensor, k_sf: torch.Tensor, v_codes: torch.Tensor, v_sf: torch.Tensor,
                 k_global: float, v_global: float):
        shape = k_codes.shape
        if len(shape) != 4:
            raise _lib.TfbError("Kv4Cache: codes must be [pages, heads, page_size, D / 2]")
        self._pages, self._heads, self._page_size, half = shape
        self._dim = 2 * half
        sf_shape = (self._pages, self._heads, self._page_size, half // 8)
        self.index, u8 = k_codes.get_device(), torch.uint8
        for t, want in ((k_codes, shape), (v_codes, shape), (k_sf, sf_shape), (v_sf, sf_shape)):
            if t.dtype is not u8 or t.shape != want or not t.is_contiguous() or t.get_device() != self.index:
                raise _lib.TfbError("Kv4Cache: codes and scales must be contiguous uint8 [pages, heads, page_size, "
                                    "D / 2] and [..., D / 16] on one device")
        self._k_codes, self._k_sf, self._v_codes, self._v_sf = k_codes, k_sf, v_codes, v_sf
        self._k_global, self._v_global = k_global, v_global
        self.struct = _lib.Kv4CacheStruct(k_codes.data_ptr(), k_sf.data_ptr(), v_codes.data_ptr(), v_sf.data_ptr(),
                                          self._pages, self._heads, self._page_size, self._dim, k_global, v_global)
        self.ref = ctypes.byref(self.struct)

    k_codes, k_sf, v_codes, v_sf, k_global, v_global, pages, heads, page_size, dim = (
        property(operator.attrgetter("_" + n)) for n in
        ("k_codes", "k_sf", "v_codes", "v_sf", "k_global", "v_global", "pages", "heads", "page_size", "dim"))

    @classmethod
    def empty(cls, pages: int, page_size: int, heads: int, dim: int, k_global: float, v_global: float,
              device="cuda") -> Kv4Cache:
        """A cache of zeros."""
        new = lambda n: torch.zeros((pages, heads, page_size, n), dtype=torch.uint8, device=device)   # noqa: E731
        return cls(new(dim // 2), new(dim // 16), new(dim // 2), new(dim // 16), k_global, v_global)

    def nbytes(self) -> int:
        return 2 * (self._k_codes.numel() + self._k_sf.numel())


def global_for(amax: float) -> float:
    """The global scale with which values up to ``amax`` just reach the largest code and scale."""
    return max(amax, 1e-12) / (FP4_TOP * E4M3_TOP)


def _batch(what: str, cache: Kv4Cache, table: torch.Tensor, first: torch.Tensor, cu: torch.Tensor | None):
    """The table's (sequences, pages, row stride), all tensors checked."""
    i32, dev = torch.int32, cache.index
    shape, st = table.shape, table.stride()
    if len(shape) != 2 or table.dtype is not i32 or st[1] != 1:
        raise _lib.TfbError(f"{what}: the page table must be int32 [B, max_pages] with contiguous rows")
    B = shape[0]
    if first.dtype is not i32 or first.shape != (B,) or not first.is_contiguous():
        raise _lib.TfbError(f"{what}: starts / lengths must be int32 [{B}]")
    if cu is not None and (cu.dtype is not i32 or cu.shape != (B + 1,) or not cu.is_contiguous() or cu.get_device() != dev):
        raise _lib.TfbError(f"{what}: cu must be int32 [{B + 1}] on the cache's device")
    if dev < 0 or table.get_device() != dev or first.get_device() != dev:
        raise _lib.TfbError(f"{what} takes CUDA tensors on one device (there is no CPU path)")
    return B, shape[1], st[0]


def _rows(what: str, cache: Kv4Cache, t: torch.Tensor, T: int, heads: int, dtype) -> tuple:
    """(address, row stride, head stride) of rows [T, heads, D]."""
    st = t.stride()
    if t.shape != (T, heads, cache._dim) or st[2] != 1 or t.dtype is not dtype or t.get_device() != cache.index:
        raise _lib.TfbError(f"{what}: rows must be {dtype} [{T}, {heads}, {cache._dim}] with contiguous heads on the "
                            f"cache's device (got {t.dtype} {tuple(t.shape)})")
    return t.data_ptr(), st[0], st[1]


def _move(what: str, fn, cache: Kv4Cache, table: torch.Tensor, start: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
          cu: torch.Tensor | None) -> None:
    B, pages, ld = _batch(what, cache, table, start, cu)
    code = _lib.OUT_DTYPES.get(k.dtype)
    if code is None or k.dim() != 3:
        raise _lib.TfbError(f"{what}: k and v must both be bf16, fp16 or fp32 [T, heads, D]")
    T = k.shape[0]
    kr, vr = _rows(what, cache, k, T, cache._heads, k.dtype), _rows(what, cache, v, T, cache._heads, k.dtype)
    _lib.launch(cache.index, fn, cache.ref, table.data_ptr(), ld, B, pages, start.data_ptr(),
                None if cu is None else cu.data_ptr(), T, *kr, *vr, code)


def write(cache: Kv4Cache, table: torch.Tensor, start: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
          cu: torch.Tensor | None = None) -> None:
    """Quantise rows k, v [T, heads, D] (bf16, fp16 or fp32; any strides with contiguous heads and 16-byte aligned
    rows) into the cache: row i of sequence b goes to position ``start[b] + i`` (``start`` int32 [B]), with the bits
    of the NVFP4 quantizer (``quant_nvfp4``) under the cache's globals. Rows whose position lies outside the table,
    or in a page outside the pool, are skipped. Values must be finite; two rows written to the same place in one call
    leave either's bytes there."""
    _move("kv4.write", _lib.load().tfb_kv4_write, cache, table, start, k, v, cu)


def read(cache: Kv4Cache, table: torch.Tensor, start: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor,
         cu: torch.Tensor | None = None) -> None:
    """The values at positions ``start[b] + i`` into rows k_out, v_out [T, heads, D] (bf16, fp16 or fp32): fp32
    products, rounded once. Rows that ``write`` would skip are left as they were."""
    _move("kv4.read", _lib.load().tfb_kv4_read, cache, table, start, k_out, v_out, cu)


def attention(q: torch.Tensor, cache: Kv4Cache, table: torch.Tensor, lengths: torch.Tensor,
              cu: torch.Tensor | None = None, scale: float | None = None, causal: bool = False,
              k_new: torch.Tensor | None = None, v_new: torch.Tensor | None = None, out: torch.Tensor | None = None,
              return_lse: bool = False):
    """softmax(scale * q k^T) v for q [T, Hq, D] (bf16 or fp16) over the cached positions [0, lengths[b]) of each
    sequence (``lengths`` int32 [B]); query head h reads cache head h // (Hq / heads); scale defaults to D^-1/2.

    ``k_new`` / ``v_new`` [T, heads, D] (q's type): this call's own keys and values, attended behind the cached ones
    in full precision (they are not written to the cache). ``causal``: with them, row i of a sequence sees its new
    rows up to i; without them the queries are the last rows of the cache, row i of n sees positions up to
    lengths[b] - n + i. A row that sees nothing gives 0 (and lse -inf); else a NaN or an infinity in a query row
    gives NaN (and lse NaN). What lies behind a sequence's length is never looked at; keys and values in front of it must
    be finite. Page numbers are taken into the pool: one outside of it (which ``write`` and ``read`` skip) reads the first
    or last page's rows. Row tensors may have any strides with contiguous heads and 16-byte aligned rows.
    -> out [T, Hq, D], or (out, lse fp32 [T, Hq]: natural logarithm of the row's sum of exponentials)."""
    what = "kv4.attention"
    B, pages, ld = _batch(what, cache, table, lengths, cu)
    dtype, shape = q.dtype, q.shape
    if len(shape) != 3 or (dtype is not torch.bfloat16 and dtype is not torch.float16):
        raise _lib.TfbError(f"{what}: q must be bf16 or fp16 [T, Hq, D]")
    T, Hq, D = shape
    rows = _rows(what, cache, q, T, Hq, dtype)
    new = (None, 0, 0, None, 0, 0)
    if k_new is not None and v_new is not None:
        new = _rows(what, cache, k_new, T, cache._heads, dtype) + _rows(what, cache, v_new, T, cache._heads, dtype)
    elif k_new is not None or v_new is not None:
        raise _lib.TfbError(f"{what}: k_new and v_new go together")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        res = (out.data_ptr(), Hq * D, D)
    else:
        res = _rows(what, cache, out, T, Hq, dtype)
    lse = q.new_empty((T, Hq), dtype=torch.float32) if return_lse else None
    lib = _lib.load()
    need = _lib.on_device(cache.index, lib.tfb_kv4_attention_ws, cache.ref, B, pages, T, Hq)   # goes by its SMs
    ws = q.new_empty((need,), dtype=torch.uint8) if need > 0 else None
    _lib.launch(cache.index, lib.tfb_kv4_attention, cache.ref, table.data_ptr(), ld, B, pages, lengths.data_ptr(),
                None if cu is None else cu.data_ptr(), T, Hq, *rows, _lib.OUT_DTYPES[dtype], *new,
                D ** -0.5 if scale is None else scale, causal, *res, None if lse is None else lse.data_ptr(),
                None if ws is None else ws.data_ptr(), need)
    return (out, lse) if return_lse else out

// The 4-bit key / value cache: shared argument checks and the packed batch's row -> sequence map.
#pragma once

#include "tfb_common.cuh"

namespace tfb {

// The packed batch and page table of one call, as the kernels see it.
struct Kv4Batch {
  const int32_t* table;
  int64_t table_ld;
  const int32_t* cu;     // nullable: every sequence has `rows` rows
  const int32_t* first;  // start (write / read) or lengths (attention), [B]
  int B, rows;
  int64_t T;
  int max_pages, page_shift;
  int64_t pages;
  int heads;
};

// Rows [*lo, *hi) of sequence b, clamped into [0, T].
__device__ __forceinline__ void kv4_rows(const Kv4Batch& a, int b, int64_t& lo, int64_t& hi) {
  if (a.cu) {
    lo = min(max((int64_t)__ldg(a.cu + b), (int64_t)0), a.T);
    hi = min(max((int64_t)__ldg(a.cu + b + 1), lo), a.T);
  } else {
    lo = (int64_t)b * a.rows;
    hi = lo + a.rows;
  }
}

// Sequence of row t (the last b with cu[b] <= t), or -1 behind the last sequence.
__device__ __forceinline__ int kv4_sequence(const Kv4Batch& a, int64_t t) {
  if (!a.cu) return static_cast<int>(t / a.rows);
  if (t >= __ldg(a.cu + a.B) || t < __ldg(a.cu)) return -1;
  int lo = 0, hi = a.B;          // cu[lo] <= t < cu[hi]
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (__ldg(a.cu + m) <= t) lo = m; else hi = m;
  }
  return lo;
}

inline tfb_status kv4_check(const char* what, const tfb_kv4_cache* c, const int32_t* table, int64_t table_ld, int64_t B,
                            int64_t max_pages, const int32_t* first, const int32_t* cu, int64_t T, Kv4Batch* a) {
  if (!c || !c->k_codes || !c->k_sf || !c->v_codes || !c->v_sf || !table || !first)
    return fail(TFB_BAD_ARG, "%s: null pointer", what);
  if (c->dim != 64 && c->dim != 128) return fail(TFB_BAD_SHAPE, "%s: head dim must be 64 or 128 (got %lld)", what,
                                                 (long long)c->dim);
  int shift = 4;
  while (shift < 8 && (1 << shift) < c->page_size) ++shift;
  if (c->page_size != 1 << shift)
    return fail(TFB_BAD_SHAPE, "%s: page size must be a power of two from 16 to 256 (got %lld)", what,
                (long long)c->page_size);
  if (c->pages < 1 || c->pages > INT32_MAX || c->heads < 1 || c->heads > 1024)
    return fail(TFB_BAD_SHAPE, "%s: needs 1 or more pages and 1 to 1024 heads", what);
  if (B < 1 || B > 65535 || max_pages < 1 || max_pages > ((1 << 30) >> shift) || table_ld < (B > 1 ? max_pages : 0))
    return fail(TFB_BAD_SHAPE, "%s: bad page table [%lld, %lld] with stride %lld (1 to 65535 sequences)", what,
                (long long)B, (long long)max_pages, (long long)table_ld);
  if (T < 0 || T > INT32_MAX || (!cu && T % B))
    return fail(TFB_BAD_SHAPE, "%s: %lld rows do not divide over %lld sequences (pass cu)", what, (long long)T,
                (long long)B);
  if (!aligned(c->k_codes, 16) || !aligned(c->k_sf, 16) || !aligned(c->v_codes, 16) || !aligned(c->v_sf, 16) ||
      !aligned(table, 4) || !aligned(first, 4) || (cu && !aligned(cu, 4)))
    return fail(TFB_BAD_ALIGN, "%s: cache buffers must be 16-byte aligned, table, lengths and cu 4-byte", what);
  if (!(c->k_global > 0.0f) || !(c->v_global > 0.0f) || !isfinite(c->k_global) || !isfinite(c->v_global))
    return fail(TFB_BAD_ARG, "%s: the cache's global scales must be positive and finite", what);
  *a = Kv4Batch{table, table_ld, cu, first, static_cast<int>(B), static_cast<int>(T / B), T,
                static_cast<int>(max_pages), shift, c->pages, static_cast<int>(c->heads)};
  return TFB_OK;
}

// Every head of every row on a 16-byte boundary (the stride of a single row or head is never used).
inline bool kv4_rows_aligned(const void* p, int64_t st, int64_t sh, int item, int64_t T, int64_t heads) {
  return aligned(p, 16) && (T == 1 || st * item % 16 == 0) && (heads == 1 || sh * item % 16 == 0);
}

}  // namespace tfb

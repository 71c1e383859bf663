// Attention over a 4-bit paged cache (and a call's own keys / values in 16 bits behind it):
// checks of a call and the choice between the kernels for few rows (kv4_decode.cu) and for many (kv4_prefill.cu).
#include <math.h>

#include "kv4_attn.cuh"

namespace tfb {
namespace {

// Which kernel: two scores to compare. They are not times (large calls take half to two thirds of them, small ones more): only
// which is smaller was fitted. The kernel for few rows takes 16 rows at a time through the keys, (row block, key) steps over
// the whole GPU and 200 keys' worth to begin each; the one for many takes 256 rows, tiles of 128 keys over a B200's 148 SMs,
// and does not split a sequence below 4 tiles. Up to 8 rows the first one always runs: they fill one fragment of it. Over
// 204 sizes (2 to 768 sequences x heads, 60 to 32000 keys, 16 to 512 rows a head) the rule was 1.0 % above the better one on
// average. Few / many in us, 64 rows a head: 16 / 24 (8 sequences x heads, 4000 keys), 111 / 62 (96, 4000), 320 / 214
// (64, 32000), and the wrong way round 21 / 25 (2, 32000); 16 rows: 41 / 59 (96, 4000); 256 rows: 99 / 39 (24, 4000).
// The lengths are on the device, so the keys are those that the table has room for. A table that is far larger than what the
// sequences hold is judged as if full: 1000 keys, 256 rows a head, 8 sequences x heads take 23 / 26, of which a table for 1024
// keys gets the first and one for 131072 the second; 500 keys, 64 rows, 64 take 25 / 18, a table for 512 the first, one for
// 32768 the second. The worst found: 1000 keys, 32 rows, 256, which gets the first of 63 / 42 from either table.
bool few_rows(int64_t B, int64_t heads, int64_t max_keys, int64_t T, int64_t group) {
  const double rows = static_cast<double>(T) * group / B, keys = static_cast<double>(max_keys) + static_cast<double>(T) / B;
  const double pairs = static_cast<double>(B) * heads, tiles = ceil(keys / 128);
  if (rows <= 8) return true;
  const double few = pairs * ceil(rows / 16) * (keys + 200) / 15000;
  const double many = 2 + 2.8 * fmax(pairs * ceil(rows / 256) * tiles / 148, fmin(tiles, 4));
  return few <= many;
}

}  // namespace
}  // namespace tfb

extern "C" {

int64_t tfb_kv4_attention_ws(const tfb_kv4_cache* c, int64_t B, int64_t max_pages, int64_t T, int64_t Hq) {
  if (!c || B < 1 || max_pages < 1 || T < 0 || Hq < 1 || c->heads < 1) return -1;
  const int64_t keys = max_pages * c->page_size, group = Hq / c->heads;
  return tfb::few_rows(B, c->heads, keys, T, group) ? tfb::attn_few_ws(c->dim, c->heads, B, keys, T, group)
                                    : tfb::attn_many_ws(c->dim, c->heads, B, keys, T, group);
}

tfb_status tfb_kv4_attention(const tfb_kv4_cache* c, const int32_t* table, int64_t table_ld, int64_t B,
                             int64_t max_pages, const int32_t* lengths, const int32_t* cu, int64_t T, int64_t Hq,
                             const void* q, int64_t q_st, int64_t q_sh, int dtype, const void* k_new, int64_t kn_st,
                             int64_t kn_sh, const void* v_new, int64_t vn_st, int64_t vn_sh, float scale, int causal,
                             void* out, int64_t o_st, int64_t o_sh, float* lse, void* ws, int64_t ws_bytes,
                             void* stream) {
  using namespace tfb;
  AttnParams p;
  tfb_status st = kv4_check("kv4_attention", c, table, table_ld, B, max_pages, lengths, cu, T, &p.a);
  if (st != TFB_OK) return st;
  if (dtype != TFB_DT_F16 && dtype != TFB_DT_BF16)
    return fail(TFB_BAD_ARG, "kv4_attention: queries must be fp16 or bf16 (element type %d)", dtype);
  if (Hq < 1 || Hq % c->heads || Hq > 65535)
    return fail(TFB_BAD_SHAPE, "kv4_attention: %lld query heads do not divide over %lld cache heads", (long long)Hq,
                (long long)c->heads);
  if (T * Hq > (int64_t)1 << 30) return fail(TFB_BAD_SHAPE, "kv4_attention: more than 2^30 query rows in a call");
  if (!isfinite(scale)) return fail(TFB_BAD_ARG, "kv4_attention: scale must be finite");
  if (T == 0) return TFB_OK;
  if (!q || !out || (k_new == nullptr) != (v_new == nullptr))
    return fail(TFB_BAD_ARG, "kv4_attention: null pointer (k_new and v_new go together)");
  if (!kv4_rows_aligned(q, q_st, q_sh, 2, T, Hq) || !kv4_rows_aligned(out, o_st, o_sh, 2, T, Hq) ||
      (k_new && (!kv4_rows_aligned(k_new, kn_st, kn_sh, 2, T, c->heads) ||
                 !kv4_rows_aligned(v_new, vn_st, vn_sh, 2, T, c->heads))) ||
      (lse && !aligned(lse, 4)))
    return fail(TFB_BAD_ALIGN, "kv4_attention: q, out, k_new and v_new must have 16-byte aligned pointers and strides");
  const DeviceInfo* di;
  st = device_info(&di);
  if (st != TFB_OK) return st;
  p.c = *c;
  p.Hq = static_cast<int>(Hq);
  p.group = static_cast<int>(Hq / c->heads);
  p.q = q, p.q_st = q_st, p.q_sh = q_sh;
  p.kn = k_new, p.kn_st = kn_st, p.kn_sh = kn_sh;
  p.vn = v_new, p.vn_st = vn_st, p.vn_sh = vn_sh;
  p.scale_log2 = scale * 1.44269504089f, p.causal = causal;
  p.out = out, p.o_st = o_st, p.o_sh = o_sh, p.lse = lse;
  p.err = di->err_word;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return few_rows(B, c->heads, max_pages * c->page_size, T, p.group) ? attn_few(p, dtype, c->dim, di, ws, ws_bytes, s)
                                 : attn_many(p, dtype, c->dim, di, ws, ws_bytes, s);
}

}  // extern "C"

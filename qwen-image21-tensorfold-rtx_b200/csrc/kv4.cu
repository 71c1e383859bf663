// Writing rows of keys and values into a 4-bit paged cache (NVFP4: E2M1 codes, an E4M3 scale per 16 values along the
// head, an fp32 global) and reading them back. Both are bound by HBM: 2 or 4 bytes a value on one side, 9/16 byte on
// the other. A token's heads follow one another in the 16-bit rows while a page keeps each head's rows together, so a
// warp reads (writes) whole lines of rows and 64-byte pieces of pages. Measured on one B200: 100002 tokens x 8 heads x 64 out of
// the cache in fp16 48.0 us (5.5 TB/s); 13054 tokens x 24 heads x 128 written and read back in bf16 81.9 us (5.0 TB/s).
#include <math.h>

#include <algorithm>

#include "kv4.cuh"
#include "tfb_dtype.cuh"

namespace tfb {
namespace {

constexpr int kKv4Threads = 256;

// Place of sequence b's position pos: the row's index in [pages * heads * page_size] for head 0, or -1.
__device__ __forceinline__ int64_t kv4_place(const Kv4Batch& a, int b, int64_t pos) {
  if (pos < 0 || pos >= (int64_t)a.max_pages << a.page_shift) return -1;
  const int64_t page = __ldg(a.table + b * a.table_ld + (pos >> a.page_shift));
  if (page < 0 || page >= a.pages) return -1;
  return ((page * a.heads) << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
}

// What a block of both kernels does with its tokens: thread i < tokens finds where token t0 + i lies (the search, the
// sequence's start and its page are loads that depend on one another: once a token, not once a head). A token's heads and
// pieces are spread over the threads, several tokens at a time where there are few of them.
struct Kv4Spread {
  int tokens;                            // of a block
  int pieces_log;                        // pieces of a head, as a power of two
  int per_token, side;                   // heads * pieces; tokens at a time (0: a token takes more than one round)
};
__device__ __forceinline__ void kv4_find_rows(const Kv4Batch& a, int64_t t0, int tokens, int64_t* place) {
  for (int i = threadIdx.x; i < tokens; i += kKv4Threads) {
    const int64_t t = t0 + i;
    int64_t row = -1;
    const int b = t < a.T ? kv4_sequence(a, t) : -1;
    if (b >= 0) {
      int64_t lo, hi;
      kv4_rows(a, b, lo, hi);
      row = kv4_place(a, b, (int64_t)__ldg(a.first + b) + t - lo);
    }
    place[i] = row;
  }
}
constexpr int kMaxTokens = 64;

// A piece: the 16 values of one scale.
template <typename T>
__global__ void __launch_bounds__(kKv4Threads) kv4_write_kernel(Kv4Batch a, Kv4Spread sp, const T* __restrict__ k,
                                                                int64_t k_st, int64_t k_sh, const T* __restrict__ v,
                                                                int64_t v_st, int64_t v_sh, tfb_kv4_cache c) {
  __shared__ int64_t place[kMaxTokens];
  pdl_trigger();
  pdl_wait();
  const int64_t t0 = blockIdx.x * (int64_t)sp.tokens;
  kv4_find_rows(a, t0, sp.tokens, place);
  __syncthreads();
  const Nvfp4Enc ek = nvfp4_enc(c.k_global), ev = nvfp4_enc(c.v_global);
  const int step = max(sp.side, 1);
  for (int u = threadIdx.x; u < sp.per_token * step; u += kKv4Threads) {
    const int off = u / sp.per_token, x = u - off * sp.per_token;
    const int h = x >> sp.pieces_log, blk = x & ((1 << sp.pieces_log) - 1);
    const T* ks = k + (t0 + off) * k_st + h * k_sh + blk * 16;
    const T* vs = v + (t0 + off) * v_st + h * v_sh + blk * 16;
    for (int i = off; i < sp.tokens; i += step, ks += step * k_st, vs += step * v_st) {
      if (place[i] < 0) continue;
      const int64_t at = ((place[i] + ((int64_t)h << a.page_shift)) << sp.pieces_log) + blk;
      Raw8<T> raw[4];
      raw[0].load(ks), raw[1].load(ks + 8), raw[2].load(vs), raw[3].load(vs + 8);
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        float y[16];
        raw[2 * part].get(y);
        raw[2 * part + 1].get(y + 8);
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(y[j]));
        const Nvfp4Enc e = part ? ev : ek;
        const uint32_t s = nvfp4_scale(amax, e);
        const float inv = nvfp4_inv(s, e);
        uint2 code;
        code.x = nvfp4_codes8(y, inv);
        code.y = nvfp4_codes8(y + 8, inv);
        reinterpret_cast<uint2*>(part ? c.v_codes : c.k_codes)[at] = code;
        (part ? c.v_sf : c.k_sf)[at] = static_cast<uint8_t>(s);
      }
    }
  }
}

// 8 codes under a scale byte as fp32 values, rounded once: lut * scale is exact in fp16, the global's product in fp32.
__device__ __forceinline__ void kv4_values(uint32_t code, uint32_t sf, float g, float* x) {
  const uint32_t h2 = e4m3x2_to_f16x2(sf | sf << 8);
  uint32_t o[4];
  e2m1x8_scaled(code, h2, o);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&o[j]));
    x[2 * j] = __fmul_rn(f.x, g);
    x[2 * j + 1] = __fmul_rn(f.y, g);
  }
}

// A piece: 8 values (half a scale's), 16 bytes of a 16-bit row.
template <typename T>
__global__ void __launch_bounds__(kKv4Threads) kv4_read_kernel(Kv4Batch a, Kv4Spread sp, T* __restrict__ k, int64_t k_st,
                                                               int64_t k_sh, T* __restrict__ v, int64_t v_st,
                                                               int64_t v_sh, tfb_kv4_cache c) {
  constexpr int U = 4;
  __shared__ int64_t place[kMaxTokens];
  pdl_trigger();
  pdl_wait();
  const int64_t t0 = blockIdx.x * (int64_t)sp.tokens;
  kv4_find_rows(a, t0, sp.tokens, place);
  __syncthreads();
  const int step = max(sp.side, 1);
  for (int u = threadIdx.x; u < sp.per_token * step; u += kKv4Threads) {
    const int off = u / sp.per_token, x = u - off * sp.per_token;
    const int h = x >> sp.pieces_log, piece = x & ((1 << sp.pieces_log) - 1);
    T* kd = k + (t0 + off) * k_st + h * k_sh + piece * 8;
    T* vd = v + (t0 + off) * v_st + h * v_sh + piece * 8;
    for (int i0 = off; i0 < sp.tokens; i0 += U * step) {
      uint32_t code[U][2], sf[U][2];
      bool live[U];
#pragma unroll
      for (int w = 0; w < U; ++w) {
        const int i = i0 + w * step;
        const int64_t row = i < sp.tokens ? place[i] : -1;
        live[w] = row >= 0;
        if (live[w]) {
          const int64_t at = ((row + ((int64_t)h << a.page_shift)) << sp.pieces_log) + piece;
          code[w][0] = __ldg(reinterpret_cast<const uint32_t*>(c.k_codes) + at);
          code[w][1] = __ldg(reinterpret_cast<const uint32_t*>(c.v_codes) + at);
          sf[w][0] = __ldg(c.k_sf + (at >> 1));
          sf[w][1] = __ldg(c.v_sf + (at >> 1));
        }
      }
#pragma unroll
      for (int w = 0; w < U; ++w, kd += step * k_st, vd += step * v_st)
        if (live[w]) {
          float y[8];
          kv4_values(code[w][0], sf[w][0], c.k_global, y);
          store8(kd, y);
          kv4_values(code[w][1], sf[w][1], c.v_global, y);
          store8(vd, y);
        }
    }
  }
}

// Tokens of a block: enough rounds to keep loads in flight, as long as every SM gets a few blocks.
Kv4Spread kv4_spread(const Kv4Batch& a, int pieces_log, int rounds, int sms) {
  Kv4Spread sp;
  sp.pieces_log = pieces_log;
  sp.per_token = a.heads << pieces_log;
  sp.side = kKv4Threads / sp.per_token;
  const int64_t want = (int64_t)rounds * std::max(sp.side, 1), share = (a.T + 4 * sms - 1) / (4 * sms);
  sp.tokens = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, share), kMaxTokens)));
  sp.side = std::min(sp.side, sp.tokens);
  return sp;
}

template <typename T>
tfb_status launch_write(const Kv4Batch& a, const tfb_kv4_cache* c, const void* k, int64_t k_st, int64_t k_sh,
                        const void* v, int64_t v_st, int64_t v_sh, int sms, cudaStream_t s) {
  const Kv4Spread sp = kv4_spread(a, c->dim == 128 ? 3 : 2, 8, sms);
  TFB_CUDA(launch_pdl(kv4_write_kernel<T>, dim3(static_cast<unsigned>((a.T + sp.tokens - 1) / sp.tokens)),
                      dim3(kKv4Threads), 0, s, a, sp, static_cast<const T*>(k), k_st, k_sh, static_cast<const T*>(v),
                      v_st, v_sh, *c));
  return TFB_OK;
}

template <typename T>
tfb_status launch_read(const Kv4Batch& a, const tfb_kv4_cache* c, void* k, int64_t k_st, int64_t k_sh, void* v,
                       int64_t v_st, int64_t v_sh, int sms, cudaStream_t s) {
  const Kv4Spread sp = kv4_spread(a, c->dim == 128 ? 4 : 3, 8, sms);
  TFB_CUDA(launch_pdl(kv4_read_kernel<T>, dim3(static_cast<unsigned>((a.T + sp.tokens - 1) / sp.tokens)),
                      dim3(kKv4Threads), 0, s, a, sp, static_cast<T*>(k), k_st, k_sh, static_cast<T*>(v), v_st, v_sh,
                      *c));
  return TFB_OK;
}

tfb_status check_rows(const char* what, const Kv4Batch& a, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                      int64_t v_st, int64_t v_sh, int dtype) {
  if (dtype != TFB_DT_F32 && dtype != TFB_DT_F16 && dtype != TFB_DT_BF16)
    return fail(TFB_BAD_ARG, "%s: unknown element type %d", what, dtype);
  if (!k || !v) return fail(TFB_BAD_ARG, "%s: null pointer", what);
  const int item = dtype == TFB_DT_F32 ? 4 : 2;
  if (!kv4_rows_aligned(k, k_st, k_sh, item, a.T, a.heads) || !kv4_rows_aligned(v, v_st, v_sh, item, a.T, a.heads))
    return fail(TFB_BAD_ALIGN, "%s: k and v must have 16-byte aligned pointers and strides", what);
  if (a.T * a.heads > (int64_t)1 << 34) return fail(TFB_BAD_SHAPE, "%s: more than 2^34 head rows in a call", what);
  return TFB_OK;
}

}  // namespace
}  // namespace tfb

extern "C" {

tfb_status tfb_kv4_write(const tfb_kv4_cache* c, const int32_t* table, int64_t table_ld, int64_t B, int64_t max_pages,
                         const int32_t* start, const int32_t* cu, int64_t T, const void* k, int64_t k_st, int64_t k_sh,
                         const void* v, int64_t v_st, int64_t v_sh, int dtype, void* stream) {
  using namespace tfb;
  Kv4Batch a;
  tfb_status st = kv4_check("kv4_write", c, table, table_ld, B, max_pages, start, cu, T, &a);
  if (st == TFB_OK && T == 0) return TFB_OK;
  if (st == TFB_OK) st = check_rows("kv4_write", a, k, k_st, k_sh, v, v_st, v_sh, dtype);
  const DeviceInfo* di;
  if (st == TFB_OK) st = device_info(&di);
  if (st != TFB_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == TFB_DT_F32) return launch_write<float>(a, c, k, k_st, k_sh, v, v_st, v_sh, di->sm_count, s);
  if (dtype == TFB_DT_F16) return launch_write<__half>(a, c, k, k_st, k_sh, v, v_st, v_sh, di->sm_count, s);
  return launch_write<__nv_bfloat16>(a, c, k, k_st, k_sh, v, v_st, v_sh, di->sm_count, s);
}

tfb_status tfb_kv4_read(const tfb_kv4_cache* c, const int32_t* table, int64_t table_ld, int64_t B, int64_t max_pages,
                        const int32_t* start, const int32_t* cu, int64_t T, void* k, int64_t k_st, int64_t k_sh, void* v,
                        int64_t v_st, int64_t v_sh, int dtype, void* stream) {
  using namespace tfb;
  Kv4Batch a;
  tfb_status st = kv4_check("kv4_read", c, table, table_ld, B, max_pages, start, cu, T, &a);
  if (st == TFB_OK && T == 0) return TFB_OK;
  if (st == TFB_OK) st = check_rows("kv4_read", a, k, k_st, k_sh, v, v_st, v_sh, dtype);
  const DeviceInfo* di;
  if (st == TFB_OK) st = device_info(&di);
  if (st != TFB_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == TFB_DT_F32) return launch_read<float>(a, c, k, k_st, k_sh, v, v_st, v_sh, di->sm_count, s);
  if (dtype == TFB_DT_F16) return launch_read<__half>(a, c, k, k_st, k_sh, v, v_st, v_sh, di->sm_count, s);
  return launch_read<__nv_bfloat16>(a, c, k, k_st, k_sh, v, v_st, v_sh, di->sm_count, s);
}

}  // extern "C"

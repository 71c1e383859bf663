// Rotary positions on several axes: y = R(angle) x on pairs of a head's values, optionally after the head's RMSNorm,
// with the angles computed here from the positions instead of read from a table.
//
// Pair p of a head belongs to one axis a and turns by ids[n, a] * theta^(-2 i / w): i and w are the pair's place in
// its axis and that axis's width, or (sections) the pair's place in the whole rotated part and its width. A frequency is
// handed over in turns (theta^(-2i/w) / 2 pi, fp64, from the host); position * frequency and its reduction to the
// nearest whole turn stay in fp64, so a position of a million is as exact as a small one, and the remainder in
// [-1/2, 1/2] turns goes to sincospif in fp32.
//
// The work is bound by HBM: every value is read once and written once. A block takes a few tokens, computes their
// cos / sin once into shared memory for all of their query and key heads, and a lane holds 8 values of a head.
// Measured on one B200: 20790 tokens x 32 heads x 80 in fp16 39.7 us (5.4 TB/s); 4096 tokens x 48 heads x 128 in bf16
// with the norm 22.0 us (4.6 TB/s; latencies at 44 % of an SM's warps: the norm's shuffles and the loads of cos / sin from shared
// memory hold a warp for 3.5 cycles an instruction, loads from memory for 2.5; issue slots 58 %); 8 tokens 2.8 us (a launch
// and three loads that depend on one another).
#include <math.h>
#include <string.h>

#include <algorithm>

#include "tfb_common.cuh"
#include "tfb_dtype.cuh"

namespace tfb {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kMaxPairs = 128, kMaxAxes = 4;

struct RopeParams {
  const void* src[2];                  // q, k
  void* dst[2];
  int64_t sb[2], sn[2], sh[2];         // element strides of src
  int64_t db[2], dn[2], dh[2];         // of dst
  const float* w[2];                   // RMSNorm weights [D], or null
  int heads[2];
  int D, half, log_lph;                // 2^log_lph lanes a head, at least D / 8
  int64_t B, N;
  const void* ids;
  int64_t ids_sb, ids_sn;
  float eps;
  int tokens, chunks;                  // tokens of a block, blocks of a batch element
  int ids_i32;
  double freq[kMaxPairs];              // turns per unit of position
  uint8_t axis[kMaxPairs];
};

// One token's cos / sin of a pair.
__device__ __forceinline__ float2 pair_turn(const RopeParams& p, int64_t b, int64_t n, int pair, bool inverse) {
  const int64_t at = b * p.ids_sb + n * p.ids_sn + p.axis[pair];
  const double id = p.ids_i32 ? static_cast<double>(__ldg(static_cast<const int32_t*>(p.ids) + at))
                              : static_cast<double>(__ldg(static_cast<const float*>(p.ids) + at));
  const double turns = id * p.freq[pair];
  const float r = static_cast<float>(turns - rint(turns));
  float s, c;
  sincospif(2.0f * r, &s, &c);
  return make_float2(c, inverse ? -s : s);
}

// Thread (slot, l): values [8 l, 8 l + 8) of heads slot, slot + slots, ... (query heads first, then key heads), one head
// after another over the block's tokens, U tokens at a time with their loads before their arithmetic. Head by head the
// addresses are a stride apart and the norm weights stay in registers: with the tokens outside, addresses and weight
// choices were most of 274 instructions a warp and 16-byte piece, and the image tokens (4096 x 48 heads x 128) took 36 us.
template <typename T, bool INTERLEAVED, bool NORM>
__global__ void __launch_bounds__(kRopeThreads) rope_axes_kernel(const __grid_constant__ RopeParams p, bool inverse) {
  constexpr int U = sizeof(T) == 2 ? 4 : 2;
  extern __shared__ __align__(16) float turn[];           // [tokens][half padded to 8] cos, then sin
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x / p.chunks, n0 = (blockIdx.x - b * p.chunks) * p.tokens;
  const int nt = min(p.tokens, static_cast<int>(p.N) - n0);
  const int ld = (p.half + 7) & ~7;
  float* cosp = turn;
  float* sinp = turn + p.tokens * ld;
  for (int i = threadIdx.x; i < nt * ld; i += kRopeThreads) {
    const int k = i / ld, pair = i - k * ld;
    const float2 cs = pair < p.half ? pair_turn(p, b, n0 + k, pair, inverse) : make_float2(1.0f, 0.0f);
    cosp[i] = cs.x;
    sinp[i] = cs.y;
  }
  const int lph = 1 << p.log_lph, l = threadIdx.x & (lph - 1), slot = threadIdx.x >> p.log_lph;
  const int slots = kRopeThreads >> p.log_lph, heads = p.heads[0] + p.heads[1];
  const bool lane_live = l < (p.D >> 3);
  const float inv_d = 1.0f / static_cast<float>(p.D);
  __syncthreads();
  // half-split pairs: value j < half pairs with j + half, held by the lane half / 8 further on
  const int hl = p.half >> 3;
  const bool low = l < hl, rot = l < 2 * hl;
  const int from = (threadIdx.x & 31) + (rot ? (low ? hl : -hl) : 0);
  const int first = INTERLEAVED ? l * 4 : (low ? l : rot ? l - hl : 0) * 8;   // this lane's first pair
  const bool turns = INTERLEAVED ? first < ld : rot;
  const float* tc = cosp + (turns ? first : 0);
  const float* tn = sinp + (turns ? first : 0);
  for (int h0 = 0; h0 < heads; h0 += slots) {              // whole blocks go round together (the shuffles below)
    const int h = h0 + slot;
    const bool live = h < heads && lane_live, key = h >= p.heads[0];
    const int part = key ? 1 : 0, ph = h - (key ? p.heads[0] : 0);
    const int64_t sn = p.sn[part], dn = p.dn[part];
    const T* src = static_cast<const T*>(p.src[part]) + b * p.sb[part] + n0 * sn + ph * p.sh[part] + l * 8;
    T* dst = static_cast<T*>(p.dst[part]) + b * p.db[part] + n0 * dn + ph * p.dh[part] + l * 8;
    float wv[8];
    bool norm = false;
    if (NORM) {
      const float* w = p.w[part];
      norm = w != nullptr;
#pragma unroll
      for (int i = 0; i < 8; ++i) wv[i] = norm && live ? __ldg(w + l * 8 + i) : 1.0f;
    }
    for (int k0 = 0; k0 < nt; k0 += U) {
      Raw8<T> raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (live && k0 + u < nt) raw[u].load(src + u * sn); else raw[u].clear();
      }
      src += U * sn;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (k0 + u >= nt) break;
        float x[8], y[8];
        raw[u].get(x);
        if (NORM) {
          float2 s2 = __fmul2_rn(make_float2(x[0], x[1]), make_float2(x[0], x[1]));
#pragma unroll
          for (int i = 2; i < 8; i += 2) s2 = __ffma2_rn(make_float2(x[i], x[i + 1]), make_float2(x[i], x[i + 1]), s2);
          float ss = s2.x + s2.y;
#pragma unroll
          for (int o = 16; o; o >>= 1)
            if (o < lph) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float rr = norm ? rsqrtf(ss * inv_d + p.eps) : 1.0f;
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const float2 z = __fmul2_rn(__fmul2_rn(make_float2(x[i], x[i + 1]), make_float2(rr, rr)),
                                        make_float2(wv[i], wv[i + 1]));
            x[i] = z.x;
            x[i + 1] = z.y;
          }
        }
        const int at = (k0 + u) * ld;
        if (INTERLEAVED) {
          float4 c = *reinterpret_cast<const float4*>(tc + at), s = *reinterpret_cast<const float4*>(tn + at);
          if (!turns) c = make_float4(1.0f, 1.0f, 1.0f, 1.0f), s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[2 * i] = cv[i] * x[2 * i] - sv[i] * x[2 * i + 1];
            y[2 * i + 1] = sv[i] * x[2 * i] + cv[i] * x[2 * i + 1];
          }
        } else {
          const float sg = low ? -1.0f : 1.0f;
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            float4 c = *reinterpret_cast<const float4*>(tc + at + i), s = *reinterpret_cast<const float4*>(tn + at + i);
            if (!turns) c = make_float4(1.0f, 1.0f, 1.0f, 1.0f), s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float other = __shfl_sync(0xffffffffu, x[i + j], from);
              y[i + j] = cv[j] * x[i + j] + sg * sv[j] * other;
            }
          }
        }
        if (live) store8(dst + u * dn, y);
      }
      dst += U * dn;
    }
  }
}

template <typename T>
cudaError_t launch_rope(const RopeParams& p, bool interleaved, bool inverse, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(p.B * p.chunks)), block(kRopeThreads);
  const size_t smem = 2 * sizeof(float) * p.tokens * ((p.half + 7) & ~7);
  if (p.w[0] || p.w[1])
    return interleaved ? launch_pdl(rope_axes_kernel<T, true, true>, grid, block, smem, s, p, inverse)
                       : launch_pdl(rope_axes_kernel<T, false, true>, grid, block, smem, s, p, inverse);
  return interleaved ? launch_pdl(rope_axes_kernel<T, true, false>, grid, block, smem, s, p, inverse)
                     : launch_pdl(rope_axes_kernel<T, false, false>, grid, block, smem, s, p, inverse);
}

// The pairs' frequencies and axes. A program calls with the same axes and base again and again, and 64 powers cost more
// than a launch: the last ones are kept per host thread.
void rope_table(RopeParams& p, int n_axes, const int* axes, double theta, bool sections, int64_t width) {
  struct Table {
    int n_axes = 0, axes[kMaxAxes];
    double theta;
    bool sections;
    double freq[kMaxPairs];
    uint8_t axis[kMaxPairs];
  };
  static thread_local Table t;
  if (t.n_axes != n_axes || t.theta != theta || t.sections != sections || memcmp(t.axes, axes, n_axes * sizeof(int))) {
    t.n_axes = n_axes;
    t.theta = theta;
    t.sections = sections;
    memcpy(t.axes, axes, n_axes * sizeof(int));
    for (int a = 0, pair = 0; a < n_axes; ++a)
      for (int i = 0; i < axes[a] / 2; ++i, ++pair) {
        const double e = sections ? 2.0 * pair / width : 2.0 * i / axes[a];
        t.freq[pair] = pow(theta, -e) * 0.15915494309189533577;   // 1 / (2 pi)
        t.axis[pair] = static_cast<uint8_t>(a);
      }
  }
  memcpy(p.freq, t.freq, sizeof(double) * p.half);
  memcpy(p.axis, t.axis, p.half);
}

}  // namespace
}  // namespace tfb

extern "C" tfb_status tfb_rope_axes(const void* q, void* q_out, int64_t Hq, const void* k, void* k_out, int64_t Hk,
                                    int dtype, int64_t B, int64_t N, int64_t D, const int64_t* strides,
                                    const void* ids, int ids_i32, int64_t ids_sb, int64_t ids_sn, int n_axes,
                                    const int* axes, double theta, const float* wq, const float* wk, float eps,
                                    int flags, void* stream) {
  using namespace tfb;
  if (!strides || !axes || n_axes < 1 || n_axes > kMaxAxes)
    return fail(TFB_BAD_ARG, "rope_axes: 1 to %d axes (got %d)", kMaxAxes, n_axes);
  if (B < 0 || N < 0 || Hq < 1 || Hk < 0 || Hq + Hk > 8192 || D < 8 || D > 256 || D % 8)
    return fail(TFB_BAD_SHAPE, "rope_axes: head dim must be a multiple of 8 up to 256, at most 8192 heads (D=%lld)",
                (long long)D);
  if (dtype != TFB_DT_F32 && dtype != TFB_DT_F16 && dtype != TFB_DT_BF16)
    return fail(TFB_BAD_ARG, "rope_axes: unknown element type %d", dtype);
  if (!(theta > 0.0) || !isfinite(theta)) return fail(TFB_BAD_ARG, "rope_axes: theta must be positive and finite");
  const bool inverse = flags & TFB_ROPE_INVERSE, interleaved = flags & TFB_ROPE_INTERLEAVED;
  if (inverse && (wq || wk)) return fail(TFB_BAD_ARG, "rope_axes: the inverse rotation takes no norm weights");
  int64_t width = 0;
  for (int a = 0; a < n_axes; ++a) {
    if (axes[a] < 2 || axes[a] % 2 || axes[a] > D)
      return fail(TFB_BAD_SHAPE, "rope_axes: an axis width must be even, from 2 to the head dim (got %d)", axes[a]);
    width += axes[a];
  }
  if (width > D || (!interleaved && width % 16))
    return fail(TFB_BAD_SHAPE, "rope_axes: the axes' sum (%lld) must be at most the head dim%s", (long long)width,
                interleaved ? "" : " and a multiple of 16 for half-split pairs");
  if (B == 0 || N == 0) return TFB_OK;                      // (empty tensors have no address)
  if (!q || !q_out || !ids || (Hk > 0 && (!k || !k_out))) return fail(TFB_BAD_ARG, "rope_axes: null pointer");
  const int item = dtype == TFB_DT_F32 ? 4 : 2;
  const void* ptrs[4] = {q, q_out, k, k_out};
  for (int i = 0; i < (Hk > 0 ? 4 : 2); ++i) {
    bool ok = aligned(ptrs[i], 16);
    const int64_t sizes[3] = {B, N, i < 2 ? Hq : Hk};
    for (int j = 0; j < 3; ++j) ok = ok && (sizes[j] == 1 || strides[3 * i + j] * item % 16 == 0);   // (one: never used)
    if (!ok) return fail(TFB_BAD_ALIGN, "rope_axes: pointers and strides must be 16-byte aligned");
  }
  if (!aligned(ids, 4) || (wq && !aligned(wq, 4)) || (wk && !aligned(wk, 4)))
    return fail(TFB_BAD_ALIGN, "rope_axes: positions and weights must be 4-byte aligned");
  if (B * N >= (int64_t)1 << 31) return fail(TFB_BAD_SHAPE, "rope_axes: fewer than 2^31 tokens");
  const DeviceInfo* di;
  tfb_status st = device_info(&di);
  if (st != TFB_OK) return st;
  RopeParams p;
  p.w[0] = p.w[1] = nullptr;
  for (int i = 0; i < 2; ++i) {
    p.src[i] = ptrs[2 * i];
    p.dst[i] = const_cast<void*>(ptrs[2 * i + 1]);
    p.sb[i] = strides[6 * i];
    p.sn[i] = strides[6 * i + 1];
    p.sh[i] = strides[6 * i + 2];
    p.db[i] = strides[6 * i + 3];
    p.dn[i] = strides[6 * i + 4];
    p.dh[i] = strides[6 * i + 5];
  }
  p.w[0] = wq;
  p.w[1] = wk;
  p.heads[0] = static_cast<int>(Hq);
  p.heads[1] = static_cast<int>(Hk);
  p.D = static_cast<int>(D);
  p.half = static_cast<int>(width / 2);
  p.log_lph = 0;
  while ((8 << p.log_lph) < D) ++p.log_lph;
  p.B = B;
  p.N = N;
  p.ids = ids;
  p.ids_sb = ids_sb;
  p.ids_sn = ids_sn;
  p.eps = eps;
  rope_table(p, n_axes, axes, theta, flags & TFB_ROPE_SECTIONS, width);
  // one wave of four blocks an SM where there are so many tokens, up to 16 tokens a block (8 KB of cos / sin at half 64)
  p.tokens = static_cast<int>(std::min<int64_t>(std::min<int64_t>(16, N), (B * N + 4 * di->sm_count - 1) / (4 * di->sm_count)));
  p.chunks = static_cast<int>((N + p.tokens - 1) / p.tokens);
  p.ids_i32 = ids_i32;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == TFB_DT_F32   ? launch_rope<float>(p, interleaved, inverse, s)
                        : dtype == TFB_DT_F16 ? launch_rope<__half>(p, interleaved, inverse, s)
                                              : launch_rope<__nv_bfloat16>(p, interleaved, inverse, s);
  TFB_CUDA(e);
  return TFB_OK;
}

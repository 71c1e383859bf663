// Attention of few query rows (decode steps, drafted tokens) over the 4-bit cache. Its floor is the cache's bytes, 9/16 of a
// byte per value. At HBM's rate an SM has 6 cycles for the 256 values of a key and head; a key takes 20 warp instructions,
// most of them conversions and the shifts that bring their bytes up, on the ALU pipe at one every two cycles. No pipe is full
// (ALU 54 % busy, issue slots 58 %): what bounds it are those instructions' latencies at 12 warps an SM, which their registers
// allow. Measured on one B200: 32 ragged sequences of up to 16384 keys, 8 heads x 128: 82 us (3.8 TB/s, floor 48 us); one
// sequence of 262143 keys, 4 heads: 44 us (3.4 TB/s, floor 23 us); one of 300 keys, 24 heads: 6.8 us. Tiles of 64 keys: 16
// warps on tiles of 32 or 48 keys took 95 us for the first (spilled registers, a tile's fixed costs), byte shifts by
// multiplications 97 us.
//
// A work item is a run of 64-key tiles of one sequence and cache head and up to 8 * NT query rows (the heads of the group,
// times the sequence's rows). Its four warps take the tiles in turn; each warp keeps a ring of two tiles in shared memory,
// filled by bulk copies (a head's rows of a page are contiguous), and its own running maximum, sum and accumulator; the
// warps' results are joined at the end, the items' by a second kernel.
//
// Both products run with the cache as the left operand of mma.m16n8k16 (fp16 in, fp32 accumulators), so that a
// dequantised fragment serves every query row: S^T = K Q^T (16 keys x 8 rows) and O^T = V^T P^T (16 channels x 8
// rows). The contraction index of the first and the row index of the second may be permuted freely, which gives each
// thread whole 16-byte (8-byte) pieces of a key's (value's) codes:
//   thread (g, t) = (lane / 4, lane % 4) holds channels [t D/4, (t+1) D/4) of the keys of rows g and g + 8, and
//   channels [g D/8, (g+1) D/8) of four values; row r of a 16-key tile is key 4 (r % 2 + 2 (r / 8)) + (r % 8) / 2, so
//   that the four values of a thread are keys t, 4 + t, 8 + t, 12 + t (shared-memory rows of different banks).
// A value fragment pairs two keys of one channel: the nibbles of two keys' words are interleaved before the
// conversion. P^T reaches the second product's layout by movmatrix. E2M1 times its E4M3 scale is exact in fp16; a
// bf16 query row is brought to fp16 by a power of two (row_exponent). P is rounded to fp16 (by 2^-11 of it or 2^-32 of the
// row's largest, see kHead), over new keys to q's type. The products cut off where they add to fp32: a sum of values of one
// sign loses about 1e-8 of itself for every key of a warp, that is a quarter of an item's (5e-4, half a step of fp16, where an
// item has 200000 keys).
#include <math.h>

#include <algorithm>
#include <atomic>

#include "kv4_attn.cuh"
#include "tfb_async.cuh"

namespace tfb {
namespace {

constexpr int kTile = 64;        // keys of a tile
constexpr int kSub = kTile / 16;  // 16-key pieces
constexpr int kWarps = 4;
constexpr int kBlocksPerSm = 3;
constexpr int kFills = 4;         // a quarter of the items may be the sequences' short last runs
constexpr int kStages = 2;
constexpr int kErrDecode = 0x400;

template <int D>
constexpr int kTileBytes = kTile * (D + D / 8);     // keys: codes, scales; values: codes, scales
template <int D>
constexpr int kSmemBytes = kWarps * kStages * kTileBytes<D> + kWarps * kStages * 8;

template <typename T>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if (sizeof(T) == 2 && __is_same(T, __half))
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Key of row r of a 16-key tile (see the top of the file).
__device__ __forceinline__ int key_of_row(int r) { return 4 * ((r & 1) + 2 * (r >> 3)) + ((r & 7) >> 1); }

// A warp's state of its 8 * NT query rows: thread (g, t) has rows 2t and 2t + 1 of each 8 in m (the base of the row's powers)
// and l (its own share of the sum), and for them channels [g D/8, (g+1) D/8) in o: o[i][n][0], [2] are channels 2i, 2i+1 of row 2t, [1], [3] of
// row 2t + 1.
template <int D, int NT>
struct RowState {
  float o[D / 16][NT][4];
  float m[NT][2], l[NT][2];
};

// The softmax of a tile's scores s[16-key tile][n][4] (raw products; `mul` turns them into powers of two), with keys at or
// behind a row's limit left out, and P^T of each 16 keys as the second product's fragments.
template <typename PT, int D, int NT>
__device__ __forceinline__ void tile_softmax(RowState<D, NT>& st, float (*s)[NT][4], const float (*mul)[2], bool masked,
                                             int key0, const int (*limit)[2], uint32_t (*pf)[NT][2]) {
  const int g = (threadIdx.x & 31) >> 2;
  float top[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) top[n][0] = top[n][1] = -INFINITY;
#pragma unroll
  for (int j = 0; j < kSub; ++j)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v = s[j][n][i] * mul[n][i & 1];
        if (masked && key0 + 16 * j + key_of_row(g + (i >> 1) * 8) >= limit[n][i & 1]) v = -INFINITY;
        s[j][n][i] = v;
        top[n][i & 1] = fmaxf(top[n][i & 1], v);
      }
  bool rise = false;
#pragma unroll
  for (int n = 0; n < NT; ++n) rise = rise || top[n][0] > st.m[n][0] + kLazy || top[n][1] > st.m[n][1] + kLazy;
  if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float v = top[n][r];
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
        const float mn = fmaxf(st.m[n][r], v - kHead), c = exp2_fast(st.m[n][r] - mn);
        st.m[n][r] = mn;
        st.l[n][r] *= c;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          st.o[i][n][r] *= c;
          st.o[i][n][2 + r] *= c;
        }
      }
  }
#pragma unroll
  for (int j = 0; j < kSub; ++j)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = exp2_fast(s[j][n][i] - st.m[n][i & 1]);
        st.l[n][i & 1] += e[i];
      }
      pf[j][n][0] = transpose8x8(pack2<PT>(e[0], e[1]));
      pf[j][n][1] = transpose8x8(pack2<PT>(e[2], e[3]));
    }
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? kBlocksPerSm : 2) attn_few_kernel(const __grid_constant__ AttnParams p) {
  constexpr int KW = D / 32;             // 32-bit code words of a thread's piece of a key
  constexpr int VW = D / 64;             // of a value
  constexpr int ROWS = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kWarps * kStages * kTileBytes<D>) + warp * kStages;
  uint8_t* ring = smem + warp * kStages * kTileBytes<D>;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) bar_init(bars + i, 1);
    bar_init_fence();
  }
  pdl_trigger();
  pdl_wait();
  Item w;
  if (!find_item<ROWS, kTile, kWarps, kFills, false>(p, blockIdx.x, w)) return;
  const int h = blockIdx.y;
  const int rows = w.nq * p.group;       // of the sequence and cache head
  const int row0 = w.rt * ROWS;
  const int cached_tiles = (w.len + kTile - 1) / kTile;
  const int mid = min(max(cached_tiles, w.tile0), w.tile1);
  __syncwarp();

  // ---- copies of a cached tile: lane 4 * piece + array
  const int pshift = min(kTile == 64 ? 6 : 5, p.a.page_shift), pieces = kTile >> pshift;
  const int arr = lane & 3, piece = lane >> 2;
  const uint8_t* base = arr == 0 ? p.c.k_codes : arr == 1 ? p.c.k_sf : arr == 2 ? p.c.v_codes : p.c.v_sf;
  const int row_bytes = arr & 1 ? D / 16 : D / 2;
  const int dst_off = (arr >= 2 ? kTile * (D / 2 + D / 16) : 0) + (arr & 1 ? kTile * (D / 2) : 0) +
                      (piece << pshift) * row_bytes;
  const int32_t* table = p.a.table + w.b * p.a.table_ld;
  auto page_at = [&](int tile) -> int {  // this lane's page of a tile (0 where it has none)
    const int key = tile * kTile + (piece << pshift);
    if (tile >= mid || piece >= pieces || key >= w.len) return 0;
    return min(max(__ldg(table + (key >> p.a.page_shift)), 0), static_cast<int>(p.a.pages - 1));
  };
  auto issue = [&](int tile, int stage, int page) {
    const int key = tile * kTile + (piece << pshift);
    const int valid = min(pieces, (w.len - tile * kTile + (1 << pshift) - 1) >> pshift);
    if (lane == 0) bar_arrive_tx(bars + stage, (valid << pshift) * (D + D / 8));
    __syncwarp();
    if (piece < valid) {
      const int64_t row = (((int64_t)page * p.a.heads + h) << p.a.page_shift) + (key & ((1 << p.a.page_shift) - 1));
      copy_bulk(ring + stage * kTileBytes<D> + dst_off, base + row * row_bytes, row_bytes << pshift, bars + stage);
    }
  };
  int next = w.tile0 + warp;             // next tile to fetch
#pragma unroll
  for (int i = 0; i < kStages; ++i, next += kWarps)
    if (next < mid) issue(next, i, page_at(next));
  int page = page_at(next);

  // ---- queries: row g (+ 8) of the tile, channels [t D/4, (t+1) D/4), as the first product's fragments
  uint32_t qf[NT][D / 8];
  float mul[NT][2];
  int limit[NT][2], least = w.len;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = row0 + 8 * n + g;
    float x[D / 4], amax = 0.0f, bad = 0.0f;
    const T* src = static_cast<const T*>(p.q) + (w.lo + r / p.group) * p.q_st + (h * p.group + r % p.group) * p.q_sh +
                   t * (D / 4);
#pragma unroll
    for (int i = 0; i < D / 4; i += 8) {
      if (r < rows)
        load8(src + i, x + i);
      else
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i + j] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < D / 4; ++i) bad = fmaf(x[i], 0.0f, bad);         // NaN if one of them is not finite
    bad += __shfl_xor_sync(0xffffffffu, bad, 1);
    bad += __shfl_xor_sync(0xffffffffu, bad, 2);
    int e = 0;
    if (!__is_same(T, __half)) {
#pragma unroll
      for (int i = 0; i < D / 4; ++i) amax = fmaxf(amax, fabsf(x[i]));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      e = row_exponent(amax);
    }
    const float f = pow2i(-e);
#pragma unroll
    for (int i = 0; i < D / 8; ++i) qf[n][i] = pack_f16x2(x[2 * i] * f, x[2 * i + 1] * f);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float unit = __shfl_sync(0xffffffffu, bad == 0.0f ? pow2i(e) : bad_row(), (2 * t + k) * 4);
      mul[n][k] = p.scale_log2 * p.c.k_global * unit;
      const int rr = row0 + 8 * n + 2 * t + k;
      limit[n][k] = p.causal && !p.kn && rr < rows ? min(w.len, w.len - w.nq + rr / p.group + 1) : w.len;
      least = min(least, limit[n][k]);
    }
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, o));

  RowState<D, NT> st;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      st.m[n][k] = kNoMax;
      st.l[n][k] = 0.0f;
      if (isnan(mul[n][k]) && (limit[n][k] > 0 || p.kn)) st.l[n][k] = bad_row();
#pragma unroll
      for (int i = 0; i < D / 16; ++i) st.o[i][n][k] = st.o[i][n][2 + k] = 0.0f;
    }

  // ---- cached tiles
  bool ok = true;
  int stage = 0, phase = 0;
  for (int tile = w.tile0 + warp; tile < mid; tile += kWarps) {
    ok = warp_wait(bars + stage, phase, p.err, kErrDecode);   // (shuffles and products of the whole warp follow)
    if (!ok) break;
    const uint8_t* kc = ring + stage * kTileBytes<D>;
    const uint8_t* ks = kc + kTile * (D / 2);
    const uint8_t* vc = ks + kTile * (D / 16);
    const uint8_t* vs = vc + kTile * (D / 2);
    const int key0 = tile * kTile;
    const bool masked = key0 + kTile > least;
    float s[kSub][NT][4];
#pragma unroll
    for (int j = 0; j < kSub; ++j) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[j][n][0] = s[j][n][1] = s[j][n][2] = s[j][n][3] = 0.0f;
      uint32_t kf[2][D / 8];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int key = 16 * j + key_of_row(g + 8 * r);
        uint32_t cw[KW], sc[KW / 2];
        if (D == 128) {
          const uint4 u = *reinterpret_cast<const uint4*>(kc + key * (D / 2) + t * (D / 8));
          cw[0] = u.x, cw[1] = u.y, cw[KW - 2] = u.z, cw[KW - 1] = u.w;
          const uint32_t h2 = e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(ks + key * (D / 16) + 2 * t));
          sc[0] = __byte_perm(h2, 0, 0x1010);
          sc[KW / 2 - 1] = __byte_perm(h2, 0, 0x3232);
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(kc + key * (D / 2) + t * (D / 8));
          cw[0] = u.x, cw[1] = u.y;
          const uint32_t h2 = e4m3x2_to_f16x2(ks[key * (D / 16) + t]);
          sc[0] = __byte_perm(h2, 0, 0x1010);
        }
#pragma unroll
        for (int i = 0; i < KW; ++i) e2m1x8_scaled(cw[i], sc[i / 2], kf[r] + 4 * i);
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const uint32_t a[4] = {kf[0][2 * i], kf[1][2 * i], kf[0][2 * i + 1], kf[1][2 * i + 1]};
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<__half>(s[j][n], a, qf[n][2 * i], qf[n][2 * i + 1]);
      }
    }
    uint32_t pf[kSub][NT][2];
    tile_softmax<__half, D, NT>(st, s, mul, masked, key0, limit, pf);
    const bool ragged = key0 + kTile > w.len;   // rows behind the length: any bytes, NaN scales among them
#pragma unroll
    for (int j = 0; j < kSub; ++j) {
      uint32_t cw[4][VW], sc[2];
      uint32_t sb[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = 16 * j + 4 * r + t;
        if (D == 128) {
          const uint2 u = *reinterpret_cast<const uint2*>(vc + key * (D / 2) + g * (D / 16));
          cw[r][0] = u.x, cw[r][VW - 1] = u.y;
          sb[r] = vs[key * (D / 16) + g];
        } else {
          cw[r][0] = *reinterpret_cast<const uint32_t*>(vc + key * (D / 2) + g * (D / 16));
          sb[r] = vs[key * (D / 16) + (g >> 1)];
        }
        if (ragged && key0 + key >= w.len) sb[r] = 0;
      }
      sc[0] = e4m3x2_to_f16x2(sb[0] | sb[1] << 8);
      sc[1] = e4m3x2_to_f16x2(sb[2] | sb[3] << 8);
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        uint32_t f[2][2][4];             // [keys 0, 1 | 2, 3][even, odd channel][channel pair]
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t x = cw[2 * r][i], y = cw[2 * r + 1][i];
          e2m1x8_scaled((x & 0x0F0F0F0Fu) | ((y << 4) & 0xF0F0F0F0u), sc[r], f[r][0]);
          e2m1x8_scaled(((x >> 4) & 0x0F0F0F0Fu) | (y & 0xF0F0F0F0u), sc[r], f[r][1]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a[4] = {f[0][0][k], f[0][1][k], f[1][0][k], f[1][1][k]};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<__half>(st.o[4 * i + k][n], a, pf[j][n][0], pf[j][n][1]);
        }
      }
    }
    __syncwarp();                        // every lane has read the stage
    if (next < mid) issue(next, stage, page);
    next += kWarps;
    page = page_at(next);
    if (++stage == kStages) stage = 0, phase ^= 1;
  }
  if (!ok) {                             // copies still in flight land before the block's shared memory goes away
    for (int i = 0; i < kStages; ++i) bar_drain(bars + (stage + i) % kStages, stage + i >= kStages ? phase ^ 1 : phase);
  }
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) st.o[i][n][k] *= p.c.v_global;

  // ---- the call's own keys and values, straight from memory, in q's type
  if (ok && p.kn && mid < w.tile1) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = row0 + 8 * n + g;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const T*>(p.q) + (w.lo + r / p.group) * p.q_st +
                                                              (h * p.group + r % p.group) * p.q_sh + t * (D / 4));
#pragma unroll
      for (int i = 0; i < D / 8; ++i) qf[n][i] = r < rows ? __ldg(src + i) : 0u;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int rr = row0 + 8 * n + 2 * t + k;
        mul[n][k] = p.scale_log2;
        limit[n][k] = p.causal && rr < rows ? rr / p.group + 1 : w.nq;
      }
    }
    const T* kn = static_cast<const T*>(p.kn) + w.lo * p.kn_st + h * p.kn_sh;
    const T* vn = static_cast<const T*>(p.vn) + w.lo * p.vn_st + h * p.vn_sh;
    for (int tile = mid + (warp + kWarps - (mid - w.tile0) % kWarps) % kWarps; tile < w.tile1; tile += kWarps) {
      const int key0 = (tile - cached_tiles) * kTile;
      float s[kSub][NT][4];
#pragma unroll
      for (int j = 0; j < kSub; ++j) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[j][n][0] = s[j][n][1] = s[j][n][2] = s[j][n][3] = 0.0f;
        uint32_t kf[2][D / 8];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int key = key0 + 16 * j + key_of_row(g + 8 * r);
#pragma unroll
          for (int i = 0; i < D / 8; i += 4) {
            uint4 u = make_uint4(0, 0, 0, 0);
            if (key < w.nq) u = __ldg(reinterpret_cast<const uint4*>(kn + key * p.kn_st + t * (D / 4) + 2 * i));
            kf[r][i] = u.x, kf[r][i + 1] = u.y, kf[r][i + 2] = u.z, kf[r][i + 3] = u.w;
          }
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint32_t a[4] = {kf[0][2 * i], kf[1][2 * i], kf[0][2 * i + 1], kf[1][2 * i + 1]};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<T>(s[j][n], a, qf[n][2 * i], qf[n][2 * i + 1]);
        }
      }
      uint32_t pf[kSub][NT][2];
      tile_softmax<T, D, NT>(st, s, mul, true, key0, limit, pf);
#pragma unroll
      for (int j = 0; j < kSub; ++j) {
        uint32_t x[4][D / 16];           // four values' channels [g D/8, (g+1) D/8)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = key0 + 16 * j + 4 * r + t;
#pragma unroll
          for (int i = 0; i < D / 16; i += 4) {
            uint4 u = make_uint4(0, 0, 0, 0);
            if (key < w.nq) u = __ldg(reinterpret_cast<const uint4*>(vn + key * p.vn_st + g * (D / 8) + 2 * i));
            x[r][i] = u.x, x[r][i + 1] = u.y, x[r][i + 2] = u.z, x[r][i + 3] = u.w;
          }
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint32_t a[4] = {__byte_perm(x[0][i], x[1][i], 0x5410), __byte_perm(x[0][i], x[1][i], 0x7632),
                                 __byte_perm(x[2][i], x[3][i], 0x5410), __byte_perm(x[2][i], x[3][i], 0x7632)};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<T>(st.o[i][n], a, pf[j][n][0], pf[j][n][1]);
        }
      }
    }
  }

  // ---- the four warps' results: rows of o in shared memory (the ring is free once every warp is done), then joined
  float* so = reinterpret_cast<float*>(smem);                       // [warp][row][D]
  float* sm = so + kWarps * ROWS * D;                               // [warp][row] (maximum, sum)
  static_assert(kWarps * ROWS * (D + 2) * 4 <= kWarps * kStages * kTileBytes<D>, "the join fits the ring");
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float l = st.l[n][k];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const int r = 8 * n + 2 * t + k;
      float* dst = so + (warp * ROWS + r) * D + g * (D / 8);
#pragma unroll
      for (int i = 0; i < D / 16; i += 2)
        *reinterpret_cast<float4*>(dst + 2 * i) =
            make_float4(st.o[i][n][k], st.o[i][n][2 + k], st.o[i + 1][n][k], st.o[i + 1][n][2 + k]);
      if (g == 0) {
        sm[(warp * ROWS + r) * 2] = st.m[n][k];
        sm[(warp * ROWS + r) * 2 + 1] = l;
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < ROWS * (D / 8); i += kWarps * 32) {
    const int r = i / (D / 8), c = (i % (D / 8)) * 8, row = row0 + r;
    if (row >= rows) continue;
    float m = kNoMax, l = 0.0f, o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = 0.0f;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) m = fmaxf(m, sm[(x * ROWS + r) * 2]);
#pragma unroll
    for (int x = 0; x < kWarps; ++x) {
      const float f = exp2_fast(sm[(x * ROWS + r) * 2] - m);
      l += f * sm[(x * ROWS + r) * 2 + 1];
      const float4* src = reinterpret_cast<const float4*>(so + (x * ROWS + r) * D + c);
      const float4 a = src[0], b = src[1];
      o[0] += f * a.x, o[1] += f * a.y, o[2] += f * a.z, o[3] += f * a.w;
      o[4] += f * b.x, o[5] += f * b.y, o[6] += f * b.z, o[7] += f * b.w;
    }
    if (w.nsplit == 1) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] *= inv;
      const int64_t tok = w.lo + row / p.group;
      const int hq = h * p.group + row % p.group;
      store8(static_cast<T*>(p.out) + tok * p.o_st + hq * p.o_sh + c, o);
      if (p.lse && c == 0) p.lse[tok * p.Hq + hq] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718056f;
    } else {
      const int64_t slot = ((int64_t)h * p.items + blockIdx.x) * ROWS + r;
      store8(p.part + slot * D + c, o);
      if (c == 0) {
        float* ml = p.part + (int64_t)p.a.heads * p.items * ROWS * D + slot * 2;
        ml[0] = m;
        ml[1] = l;
      }
    }
  }
}

// 8 query rows a work item where a sequence has no more on average, else 16.
int row_blocks(int64_t B, int64_t T, int64_t group) { return T * group <= 8 * B ? 1 : 2; }

struct FewPlan {
  int nt, items, row_blocks, slots, min_tiles;
  bool join;
  int64_t ws;
};
FewPlan few_plan(int64_t dim, int64_t heads, int64_t B, int64_t max_keys, int64_t T, int64_t group, int sms) {
  FewPlan f;
  f.nt = row_blocks(B, T, group);
  f.min_tiles = 512 / kTile;
  const int64_t tiles = (max_keys + kTile - 1) / kTile + (T + kTile - 1) / kTile;
  f.join = tiles > f.min_tiles;
  f.slots = f.join ? static_cast<int>(std::max<int64_t>(1, (f.nt == 1 ? kBlocksPerSm : 2) * (int64_t)sms / heads)) : 0;
  f.row_blocks = static_cast<int>(T * group / (8 * f.nt) + B);
  f.items = static_cast<int>(item_bound(kFills, f.row_blocks, f.slots));
  f.ws = f.join ? heads * f.items * 8 * f.nt * (dim + 2) * 4 : 0;
  return f;
}

template <typename T, int D, int NT>
tfb_status launch_few(AttnParams& p, const FewPlan& f, const DeviceInfo* di, cudaStream_t s) {
  static std::atomic<bool> ready[64];
  if (!ready[di->device].load(std::memory_order_acquire)) {
    TFB_CUDA(cudaFuncSetAttribute(attn_few_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes<D>));
    ready[di->device].store(true, std::memory_order_release);
  }
  const dim3 grid(f.items, p.a.heads);
  TFB_CUDA(launch_pdl(attn_few_kernel<T, D, NT>, grid, dim3(kWarps * 32), kSmemBytes<D>, s, p));
  if (f.join) {
    const int per = join_rows(8 * NT, (int64_t)f.row_blocks * p.a.heads, di->sm_count);
    TFB_CUDA(launch_pdl(attn_join_kernel<T, D, 8 * NT, kTile, kWarps, kFills>, dim3(f.row_blocks, p.a.heads, 8 * NT / per),
                        dim3(256), 0, s, p, per));
  }
  return TFB_OK;
}
template <typename T>
tfb_status launch_few_t(AttnParams& p, const FewPlan& f, int64_t dim, const DeviceInfo* di, cudaStream_t s) {
  if (dim == 128) return f.nt == 1 ? launch_few<T, 128, 1>(p, f, di, s) : launch_few<T, 128, 2>(p, f, di, s);
  return f.nt == 1 ? launch_few<T, 64, 1>(p, f, di, s) : launch_few<T, 64, 2>(p, f, di, s);
}

}  // namespace

int64_t attn_few_ws(int64_t dim, int64_t heads, int64_t B, int64_t max_keys, int64_t T, int64_t group) {
  const DeviceInfo* di;
  if (device_info(&di) != TFB_OK) return -1;
  return few_plan(dim, heads, B, max_keys, T, group, di->sm_count).ws;
}

tfb_status attn_few(AttnParams& p, int dtype, int64_t dim, const DeviceInfo* di, void* ws, int64_t ws_bytes, cudaStream_t s) {
  const FewPlan f = few_plan(dim, p.a.heads, p.a.B, (int64_t)p.a.max_pages << p.a.page_shift, p.a.T, p.group, di->sm_count);
  if (f.ws > 0 && (!ws || ws_bytes < f.ws || !aligned(ws, 16)))
    return fail(TFB_BAD_ARG, "kv4_attention: needs a 16-byte aligned workspace of %lld bytes", (long long)f.ws);
  p.items = f.items;
  p.slots = f.slots;
  p.min_tiles = f.min_tiles;
  p.part = static_cast<float*>(ws);
  return dtype == TFB_DT_F16 ? launch_few_t<__half>(p, f, dim, di, s) : launch_few_t<__nv_bfloat16>(p, f, dim, di, s);
}

}  // namespace tfb

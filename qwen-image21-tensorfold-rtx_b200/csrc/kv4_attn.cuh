// What the attention kernels over the 4-bit cache share: the call's parameters, E2M1 decoding, the exponential.
#pragma once

#include <cuda_fp16.h>

#include <algorithm>

#include "kv4.cuh"
#include "tfb_dtype.cuh"

namespace tfb {

struct AttnParams {
  Kv4Batch a;            // a.first: lengths
  tfb_kv4_cache c;
  int Hq, group;         // group: query heads of a cache head
  const void* q;
  int64_t q_st, q_sh;
  const void *kn, *vn;   // the call's own keys / values, or null
  int64_t kn_st, kn_sh, vn_st, vn_sh;
  float scale_log2;      // scale * log2(e): the softmax works on powers of two
  int causal;
  void* out;
  int64_t o_st, o_sh;
  float* lse;
  int* err;
  int items;             // few rows: upper bound of work items of a cache head; many rows: the grid's blocks
  int slots;             // blocks that the GPU holds at a time, per cache head (0: no sequence is split)
  int min_tiles;         // a work item has at least this many tiles of keys
  float* carry;          // many rows: sums taken out of TMEM on the way, or null where no row block is that long
  float* part;           // partial results; few rows: [heads][items][rows][dim], many: [2 items][dim / 4][rows][4]; then
                         // their rows' (maximum, sum) pairs
};

constexpr float kNoMax = -1e30f;   // a row's base before its first key: finite, so that exp2(-inf - kNoMax) = 0
// A row's powers are taken over a base kHead below its running maximum, which follows only a rise by more than 2^8: at their
// rounding to 16 bits they reach 2^(kHead + 8) = 2^15 (fp16 holds 65504). So a probability keeps its 11 bits in fp16 down to
// 2^-21 of the row's largest and is lost below 2^-32 of it, where 262144 keys together weigh 2^-14 (without the head 2^-7).
// Exponents around 7 are rounded by 2^-22, about as much as the powers themselves: lse is off by up to 9e-7 where it is near 0.
constexpr float kHead = 7.0f;
constexpr float kLazy = 15.0f;     // the base stays while the maximum is at most this far above it

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Number of the last power of two at or below a query row's largest value: the row times 2^-e fits fp16 without loss
// above 2^-14 of that value (below, within 2^-25 of it).
__device__ __forceinline__ int row_exponent(float amax) {
  const int e = static_cast<int>((__float_as_uint(amax) >> 23) & 255u) - 127;
  return amax == 0.0f ? 0 : max(-100, min(100, e));
}
// A query row with NaN or an infinity has NaN as its result where it sees a key: its sum starts as NaN, which every
// sum, factor and logarithm behind it keeps. (Its scores alone would not do: all of them may be -inf.)
__device__ __forceinline__ float bad_row() { return __uint_as_float(0x7FFFFFFFu); }
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return __is_same(T, __half) ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
}

// ---------------------------------------------------------------------------------------------- work items
struct Item {
  int b, rt, item, split, nsplit, tile0, tile1;
  int64_t lo;                    // first row of the sequence
  int nq;                        // its rows
  int len;                       // its cached keys
};

// Tiles of TILE keys of a sequence: its cached keys', then its own new keys'.
template <int TILE>
__device__ __forceinline__ int seq_tiles(const AttnParams& p, int nq, int len) {
  return (len + TILE - 1) / TILE + (p.kn ? (nq + TILE - 1) / TILE : 0);
}
__device__ __forceinline__ void seq_sizes(const AttnParams& p, int b, int& nq, int& len, int64_t& lo) {
  int64_t hi;
  kv4_rows(p.a, b, lo, hi);
  nq = static_cast<int>(hi - lo);
  len = static_cast<int>(min(max((int64_t)__ldg(p.a.first + b), (int64_t)0), (int64_t)p.a.max_pages << p.a.page_shift));
}

// The work items of a cache head: every sequence's rows in blocks of ROWS, its tiles in runs of one length for all, at
// least min_tiles and a multiple of STEP, such that the items fill `slots` (the blocks that the GPU holds at a time,
// shared out over the heads) once, or FILLS times the row blocks' share of them; slots 0 or more than FILLS times as many
// row blocks: nothing is split. item_bound is the host's side of it: never fewer than the items there are.
inline int64_t item_bound(int64_t fills, int64_t row_blocks, int64_t slots) {
  if (slots == 0) return row_blocks;
  return row_blocks <= fills * slots ? fills * row_blocks + slots : std::max(row_blocks, (fills * fills + 1) * slots);
}

// Work item `index`, or with JOIN row block `index` (w.item: its first item). Every warp goes over the sequences, 32 at a
// time, on its own.
template <int ROWS, int TILE, int STEP, int FILLS, bool JOIN>
__device__ bool find_item(const AttnParams& p, int index, Item& w) {
  const int lane = threadIdx.x & 31;
  const int B = p.a.B;
  long long total = 0;
  int blocks = 0, nq, len;
  int64_t lo;
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int b = b0 + lane;
    int rts = 0;
    long long mine = 0;
    if (b < B) {
      seq_sizes(p, b, nq, len, lo);
      rts = (nq * p.group + ROWS - 1) / ROWS;
      mine = (long long)rts * max(1, seq_tiles<TILE>(p, nq, len));
    }
    if (p.slots > 0) {                   // (otherwise the run's length does not depend on the sequences)
      blocks += __reduce_add_sync(0xffffffffu, rts);
#pragma unroll
      for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
      total += mine;
    }
  }
  long long run = 1LL << 40;
  if (p.slots > 0 && blocks <= FILLS * p.slots) {
    const int fills = max(1, (FILLS * blocks + p.slots - 1) / p.slots);
    const int most = max(1, fills * p.slots - blocks);       // total / run + blocks items stay within the fills
    run = max(((total + most - 1) / most + STEP - 1) / STEP * STEP, (long long)p.min_tiles);
  }
  int before = 0, before_items = 0;
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int b = b0 + lane;
    int tiles = 0, rts = 0, nsplit = 0;
    if (b < B) {
      if (B > 32) seq_sizes(p, b, nq, len, lo);
      tiles = max(1, seq_tiles<TILE>(p, nq, len));
      rts = (nq * p.group + ROWS - 1) / ROWS;
      nsplit = run >= tiles ? 1 : (tiles + static_cast<int>(run) - 1) / static_cast<int>(run);
    }
    int upto = JOIN ? rts : rts * nsplit, items = rts * nsplit;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
      if (JOIN) {
        const int x = __shfl_up_sync(0xffffffffu, items, o);
        if (lane >= o) items += x;
      }
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > index);
    if (hit) {
      const int src = __ffs(hit) - 1;
      w.b = b0 + src;
      w.nq = __shfl_sync(0xffffffffu, nq, src);
      w.len = __shfl_sync(0xffffffffu, len, src);
      w.lo = __shfl_sync(0xffffffffu, lo, src);
      const int ns = __shfl_sync(0xffffffffu, nsplit, src), nt = __shfl_sync(0xffffffffu, tiles, src);
      const int rt = __shfl_sync(0xffffffffu, rts, src);
      const int rest = index - before - __shfl_sync(0xffffffffu, upto, src) + (JOIN ? rt : rt * ns);
      const int block = JOIN ? rest : rest / ns;
      w.nsplit = ns;
      w.split = JOIN ? 0 : rest % ns;
      w.rt = rt - 1 - block;             // the last rows see most: first
      w.item = JOIN ? before_items + __shfl_sync(0xffffffffu, items, src) - (rt - block) * ns : index;
      // even runs
      w.tile0 = static_cast<int>((long long)nt * w.split / ns);
      w.tile1 = static_cast<int>((long long)nt * (w.split + 1) / ns);
      w.tile1 = min(w.tile1, seq_tiles<TILE>(p, w.nq, w.len));
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
    if (JOIN) before_items += __shfl_sync(0xffffffffu, items, 31);
  }
  return false;
}

// Joins the items of a row block: a block of eight warps takes `per` rows of it, two at a time, four warps a row, each with
// every fourth item, eight of them in flight.
template <typename T, int D, int ROWS, int TILE, int STEP, int FILLS>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ AttnParams p, int per) {
  constexpr int V = D / 32, CHUNK = 8, kPer = 4;
  __shared__ float acc_s[8][D], ml_s[8][2];
  __shared__ Item w;
  __shared__ bool some;
  pdl_trigger();
  pdl_wait();
  if (threadIdx.x < 32) {
    Item x;
    const bool found = find_item<ROWS, TILE, STEP, FILLS, true>(p, blockIdx.x, x) && x.nsplit > 1;
    if (threadIdx.x == 0) w = x, some = found;
  }
  __syncthreads();
  if (!some) return;
  const int h = blockIdx.y, row0 = w.rt * ROWS, end = min((int)(blockIdx.z + 1) * per, w.nq * p.group - row0);
  const int64_t first = (int64_t)h * p.items + w.item;
  const int ns = min(w.nsplit, p.items - w.item);            // (a cu that does not ascend)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % kPer;
  const float2* ml = reinterpret_cast<const float2*>(p.part + (int64_t)p.a.heads * p.items * ROWS * D);
  for (int r0 = blockIdx.z * per; r0 < end; r0 += 8 / kPer) {
    const int row = min(r0 + warp / kPer, end - 1);          // (an odd last row is joined twice)
    auto at = [&](int i) { return (first + i) * ROWS + row; };
    float acc[V], m = kNoMax, l = 0.0f;                      // of the warp's parts
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.0f;
    for (int i0 = part; i0 < ns; i0 += CHUNK * kPer) {      // CHUNK loads in flight
      float2 s[CHUNK];
      float v[CHUNK][V];
      float top = m;
#pragma unroll
      for (int x = 0; x < CHUNK; ++x) {
        const int i = i0 + x * kPer;
        s[x] = make_float2(kNoMax, 0.0f);
#pragma unroll
        for (int j = 0; j < V; ++j) v[x][j] = 0.0f;
        if (i >= ns) continue;
        s[x] = ml[at(i)];
        const float* src = p.part + at(i) * D + lane * V;
        if (V == 4) {
          const float4 y = *reinterpret_cast<const float4*>(src);
          v[x][0] = y.x, v[x][1] = y.y, v[x][V - 2] = y.z, v[x][V - 1] = y.w;
        } else {
          const float2 y = *reinterpret_cast<const float2*>(src);
          v[x][0] = y.x, v[x][1] = y.y;
        }
      }
#pragma unroll
      for (int x = 0; x < CHUNK; ++x) top = fmaxf(top, s[x].x);
      const float c = exp2_fast(m - top);
      m = top;
      l *= c;
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] *= c;
#pragma unroll
      for (int x = 0; x < CHUNK; ++x) {
        const float f = exp2_fast(s[x].x - m);
        l += f * s[x].y;
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += f * v[x][j];
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) acc_s[warp][lane * V + j] = acc[j];
    if (lane == 0) ml_s[warp][0] = m, ml_s[warp][1] = l;
    __syncthreads();
    if (part == 0) {
      float top = m;
#pragma unroll
      for (int x = 1; x < kPer; ++x) top = fmaxf(top, ml_s[warp + x][0]);
      l = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] = 0.0f;
#pragma unroll
      for (int x = 0; x < kPer; ++x) {
        const float f = exp2_fast(ml_s[warp + x][0] - top);
        l += f * ml_s[warp + x][1];
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += f * acc_s[warp + x][lane * V + j];
      }
      m = top;
    }
    __syncthreads();
    if (part == 0) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int64_t tok = w.lo + (row0 + row) / p.group;
      const int hq = h * p.group + (row0 + row) % p.group;
      T* dst = static_cast<T*>(p.out) + tok * p.o_st + hq * p.o_sh + lane * V;
#pragma unroll
      for (int j = 0; j < V; j += 2)
        *reinterpret_cast<uint32_t*>(dst + j) = pack2<T>(acc[j] * inv, acc[j + 1] * inv);
      if (p.lse && lane == 0) p.lse[tok * p.Hq + hq] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718056f;
    }
  }
}

// Rows of a join block (an even share of ROWS): two rows take about 1.3 us, so many blocks where the row blocks are few.
inline int join_rows(int64_t rows, int64_t blocks, int sms) {
  int64_t z = 1;
  while (z < rows / 2 && blocks * z * 2 <= 16 * (int64_t)sms) z *= 2;
  return static_cast<int>(rows / z);
}

// Few rows: kv4_decode.cu. Many rows: kv4_prefill.cu. *_ws: bytes of workspace.
tfb_status attn_few(AttnParams& p, int dtype, int64_t dim, const DeviceInfo* di, void* ws, int64_t ws_bytes, cudaStream_t s);
int64_t attn_few_ws(int64_t dim, int64_t heads, int64_t B, int64_t max_keys, int64_t T, int64_t group);
tfb_status attn_many(AttnParams& p, int dtype, int64_t dim, const DeviceInfo* di, void* ws, int64_t ws_bytes, cudaStream_t s);
int64_t attn_many_ws(int64_t dim, int64_t heads, int64_t B, int64_t max_keys, int64_t T, int64_t group);

}  // namespace tfb

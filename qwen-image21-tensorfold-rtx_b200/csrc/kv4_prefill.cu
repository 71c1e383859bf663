// Attention of many query rows over the 4-bit cache and the call's own keys / values. Its floor is the tensor cores' time,
// 2048 cycles for a block's tile, which the exponentials between the two products match on the special function units
// (16 a cycle and SM). What bounds it is the chain scores -> softmax -> probabilities -> products of a query tile, about
// 4000 cycles long, of which the other query tile's hides a part: the tensor pipe is active 46 % of the time, no other pipe
// more. Measured on one B200: 4096 rows x 24 heads over 256 cached and 4096 new keys 240 us (0.91 PFLOP/s, 56 % of the
// measured bf16 rate), 270 us over and over, with the clock at the board's 1000 W down from 1.96 to 1.76 GHz; a ragged
// causal chunk over up to 9000 cached keys, 16 heads on 4, 190 to 206 us (0.86 to 0.93 PFLOP/s).
//
// A block, one an SM, works through its share of the work (below), at any time on 256 query rows of one sequence and cache
// head (row r: query r / group of the sequence, head r % group of the group, so that grouped heads share every tile of
// keys) as two 128-row tiles, and walks the keys 128 at a time:
//   warps 0-7, 8-15 : softmax of query tile 0 / 1. Two threads own a row, one for the first 64 keys of a tile, one for the
//                     others: each reads its scores from TMEM, the two tell one another their maxima (shared memory, a
//                     barrier of their two warps), and each writes its probabilities back into the scores' columns as the
//                     packed 16-bit left operand of the second product. The powers' base follows the maximum only at a
//                     rise by more than 2^8 (kHead, kLazy); then (seldom) they rescale the accumulator row in TMEM, half
//                     of it each. (One thread a row, eight warps in all, left an SM's schedulers with two warps that
//                     mostly waited for their own instructions: 4700 cycles a tile instead of 2048 for its powers.)
//   warps 16-19     : keys (16, 17) and values (18, 19). Cached tiles: a thread dequantises two rows' codes (E2M1 times E4M3
//                     is exact in fp16) into shared memory; new tiles: TMA, and 16-byte copies with zeros behind them for
//                     a sequence's last rows. Keys and values have the same layout (rows of 128 bytes, 128-byte
//                     swizzle): K-major for Q K^T, MN-major for P V.
//   warp 20         : one thread issues tcgen05.mma (M = 128, fp32 accumulators): for tile j of query tile w the product
//                     P_w V_j and right behind it Q_w K_{j+1}^T, so that one query tile's products run under the other's
//                     softmax. (Scores in halves of 64 keys with a product each, to have a query tile's next scores at
//                     hand earlier, were slower: the left operand costs 64 cycles a step whatever N is.)
//   warp 21         : finds the block's shares of the work and hands them out, up to four ahead of the other warps, so that
//                     the next share's tiles and first scores are under way while a share's results are written.
// TMEM: scores of the two query tiles at columns 0 and 128, accumulators at 256 and 384. Products over cached tiles run in
// fp16 (bf16 query rows brought there by a power of two, see row_exponent), over new tiles in q's type: a softmax thread
// writes its query row to shared memory, at the border once more, and scales its accumulator by the cache's global value
// scale. Probabilities are rounded to those types for the second product (by 2^-11 and, in bf16, 2^-8 of themselves: as much
// as the result's own rounding; in fp16 or by 2^-32 of the row's largest); maxima, sums and accumulators are fp32.
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kv4_attn.cuh"
#include "tfb_async.cuh"

namespace tfb {
namespace {

constexpr int kRows = 256;               // query rows of a block
constexpr int kKeys = 128;               // keys of a tile
constexpr int kThreadsP = 768;           // 80 registers a thread
constexpr int kErrPrefill = 0x500;
constexpr uint32_t kColO = 256;          // accumulators' first TMEM column

template <int D>
struct Smem {
  static constexpr int kHalf = kKeys * 128;             // 128 rows x 64 16-bit values
  static constexpr int kTileB = (D / 64) * kHalf;
  static constexpr int kQ = 0;                           // two query tiles
  static constexpr int kK = 2 * kTileB;                  // two stages
  static constexpr int kV = 4 * kTileB;
  static constexpr int kPair = 6 * kTileB;               // [2][query tile][half][128]: what a row's two threads tell
  static constexpr int kBar = kPair + 2 * 2 * 2 * 128 * 4;
  static constexpr int kSeg = kBar + 32 * 8;
  static constexpr int kBytes = kSeg + 4 * 64 + 16 + 1024;   // + alignment of the dynamic buffer
};
// KFULL .. VEMPTY: + stage; SFULL, QFULL, ODONE: + query tile; PFULL: + 2 * query tile + part; GFULL, GEMPTY: + place.
enum Bar {
  KFULL = 0, KEMPTY = 2, VFULL = 4, VEMPTY = 6, SFULL = 8, QFULL = 10, PFULL = 12, ODONE = 16, IDLE = 18, GFULL = 20,
  GEMPTY = 24
};
// The tensor core adds to its fp32 accumulators by cutting off, not by rounding: a sum of values of one sign loses about
// 6e-9 of itself for every key (0.16 % after 262144, 10 % after 16 million). So every kCarry tiles a share's accumulators and
// row sums are added to their sums in memory, with rounding, and begin again at zero: 1e-4 is lost at most, a fifth of half a
// step of fp16. 128 KB a block, which stay in L2; a kernel of its own where the table and the new rows have room for more
// tiles (4.33 -> 4.49 ms for 2048 rows x 32 heads on 8 over 131072 keys; up to 128 tiles the test alone would cost 2 %).
constexpr int kCarry = 128;
constexpr int kSegs = 4;                 // row blocks' shares that the warps are told of ahead
// Some waits last as long as a whole share does (64 million keys a second): the one for room to hand out another, and those
// of warps that have nothing to do in it. A stall inside a share runs into one of its own waits and ends these as well.
constexpr long long kShareLimitNs = 60 * kWaitLimitNs;

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 consecutive columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
// 16 columns, waited for.
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// The wait for loads, and that nothing which uses the 32 registers at `r` is moved in front of it.
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_tie(uint32_t* r) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory descriptors with 128-byte swizzle (rows of 128 bytes, 8-row groups 1024 bytes apart): the low word has the
// address and the distance of 64-value column groups (used by the MN-major operand), the high word is the same for all.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return ((addr & 0x3FFFFu) >> 4) | (lbo >> 4 << 16); }
constexpr uint32_t kDescHi = 64u | (1u << 14) | (2u << 29);
// Instruction descriptor of kind::f16: fp32 accumulator, both operands fp16 (0) or bf16 (1), N columns, M = 128, the right
// operand MN-major if `mn`.
__host__ __device__ constexpr uint32_t mma_desc(int fmt, int n, bool mn) {
  return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((128u >> 4) << 24);
}
// Steps of 16 along the contraction, issued by one elected lane of a converged warp (without a branch: descriptors and
// predicates stay in uniform registers): left operand in shared memory (64 values of a 128-byte row) or in TMEM (8 columns
// a step), right operand K-major (the same) or MN-major (16 rows of 128 bytes a step). acc: add to the accumulator.
#define TFB_MMA2(LEFT, A_STEP, B_STEP)                                                                                  \
  "{\n\t.reg .pred e, p, t;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\t"                                                \
  "elect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, %3, %3;\n\t"                               \
  "mov.b32 x, %1;\n\tmov.b32 y, %2;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\t"                               \
  "@e tcgen05.mma.cta_group::1.kind::f16 [%0], " LEFT ", b, %3, p;\n\t"                                                \
  "add.u32 x, %1, " A_STEP ";\n\tadd.u32 y, %2, " B_STEP ";\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\t"        \
  "@e tcgen05.mma.cta_group::1.kind::f16 [%0], " LEFT ", b, %3, t;\n\t}"
__device__ __forceinline__ void mma2_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(TFB_MMA2("a", "2", "2")::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi) : "memory");
}
__device__ __forceinline__ void mma2_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(TFB_MMA2("[x]", "8", "128")::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi) : "memory");
}
#undef TFB_MMA2
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}
// One thread of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

// Shared memory by 32-bit addresses: through generic pointers the operand warps' stores and the softmax warps' exchange took
// twice the registers for addresses, and of 80 a thread there are none to spare. What the compiler put away and loaded again
// for every tile cost up to 20 % where one query tile's chain is all there is (64 rows x 16000 keys x 64: 144 us; 123 so),
// 6 % of the ragged prefill chunk.
__device__ __forceinline__ void store_shared(uint32_t dst, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// 2^x of a pair on the FMA pipes: the nearest integer n by the addition of 1.5 2^23 (whose low bits then hold n), a polynomial
// of degree 4 for 2^f on [-1/2, 1/2] (least relative error by iterated weighted least squares: 2.6e-6, a hundredth of
// the probabilities' rounding to fp16), and n added to the exponent. For the special function units' relief: they give 16
// powers a cycle and SM, 2048 cycles for a block's tile, as long as its two products take.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  x.x = fmaxf(x.x, -120.0f);             // (-inf too)
  x.y = fmaxf(x.y, -120.0f);
  const float2 big = make_float2(12582912.0f, 12582912.0f);
  const float2 t = __fadd2_rn(x, big);
  const float2 r = __fadd2_rn(t, make_float2(-12582912.0f, -12582912.0f));
  const float2 f = __fadd2_rn(x, make_float2(-r.x, -r.y));
  float2 y = make_float2(0.009570100344717503f, 0.009570100344717503f);
  y = __ffma2_rn(y, f, make_float2(0.05591785907745361f, 0.05591785907745361f));
  y = __ffma2_rn(y, f, make_float2(0.240247443318367f, 0.240247443318367f));
  y = __ffma2_rn(y, f, make_float2(0.6931217908859253f, 0.6931217908859253f));
  y = __ffma2_rn(y, f, make_float2(0.9999992847442627f, 0.9999992847442627f));
  return make_float2(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(t.x) << 23)),
                     __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(t.y) << 23)));
}

// A warp's arrival, one for all its lanes.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\t@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}"
               ::"r"(smem_u32(bar))
               : "memory");
}

// Byte offset of 16-byte chunk c (8 values) of row r in a tile of D-value rows.
template <int D>
__device__ __forceinline__ int tile_at(int r, int c) {
  return (c >> 3) * Smem<D>::kHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// ---------------------------------------------------------------------------------------------- shares of the work
// The work of a call is the list of its row blocks (cache head by cache head, in a head sequence by sequence, a
// sequence's last rows first), each with the tiles of keys that its rows see. It is shared out over the blocks of the
// grid (one for each SM) in one of two ways, whichever should end earlier:
//  - by units: a row block, or where there are fewer of them than SMs an even part of one, in turn;
//  - by tiles: equal runs of the list, which begin and end inside row blocks, so that all SMs end together whatever the
//    lengths are. Where all row blocks are equal, all but one or two rounds of them go by units first, in the list's
//    order: what is at work at a time then has few heads, whose keys and values stay in L2 (24 heads x 16384 tokens).
// A second kernel joins the parts of the row blocks that were cut (image step: 38 MB of them, about 9 us; their layout lets
// neighbouring lanes, which hold neighbouring rows, store next to one another: row by row the parts took 8 us each).
// Against a grid block for each row block (us, when the shares were built): a ragged causal chunk, 240 row blocks of 16 to 71 tiles, 209 / 270; 256
// short sequences 128 / 210; 140 row blocks of 8 tiles 37 / 55; 148 of them 37 / 33 (the join finds nothing to do);
// 4096 rows x 24 heads 265 / 272 (the SMs' clock falls from 1.89 to 1.8 GHz with their idle time gone).
struct Seg {                 // what a grid block does of a row block
  int64_t lo;                // first row of the sequence
  int h, b, nq, len;         // cache head (-1: nothing more), sequence, its rows and cached keys
  int row0, rows;            // first row of the row block, rows (query, head) of the sequence
  int tile0, nc, nf, f0;     // first cached tile, cached tiles, new tiles, first new tile
  int slot;                  // of the partial result, or -1: the row block is whole
};
struct Shares {
  int cut;                   // units: tiles of one (kWhole: row blocks); 0: by tiles
  int rounds;                // of units
  int64_t blocks;            // row blocks of a head
  int64_t total;             // units or tiles of a head
  int64_t base, run;         // by tiles: the first tile behind the rounds, tiles of a grid block
};
constexpr int kWhole = 1 << 30;
struct alignas(8) Joint {    // a row block to join: its sequence's first row, its parts (0: none), head, first row and rows
  int64_t lo;
  int parts, h, row0, rows;
};
__device__ __forceinline__ Joint* joints(const AttnParams& p, int dim) {       // of each grid block, behind the parts
  return reinterpret_cast<Joint*>(p.part + 2LL * p.items * kRows * (dim + 2));
}

// Tiles that the rows of row block rt see: cached ones, then new ones.
__device__ __forceinline__ void seen_tiles(const AttnParams& p, int nq, int len, int rt, int& tc, int& tf) {
  int see_c = len, see_f = p.kn ? nq : 0;
  if (p.causal) {
    const int last = (min((rt + 1) * kRows, nq * p.group) - 1) / p.group;    // the block's last query
    if (p.kn) see_f = last + 1;
    else see_c = max(0, min(len, len - nq + last + 1));
  }
  tc = (see_c + kKeys - 1) / kKeys;
  tf = (see_f + kKeys - 1) / kKeys;
}
// Tiles of a row block: with kLead for what its beginning and its end cost (cut 0), or as units.
constexpr int kLead = 4;
__device__ __forceinline__ int weight(const AttnParams& p, int nq, int len, int rt, int cut) {
  if (cut == kWhole) return 1;
  int tc, tf;
  seen_tiles(p, nq, len, rt, tc, tf);
  const int t = max(1, tc + tf);                            // (rows that see nothing are written too)
  return cut ? (t + cut - 1) / cut : t + kLead;
}
// Of values in [0, 2^50): sums, and quotients (32-bit division where it does: a 64-bit one takes a quarter of a microsecond,
// and nothing else of the block can begin before its first share is known).
__device__ __forceinline__ int64_t warp_sum(int64_t x) {
  const unsigned lo = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(x) & 0xFFFFFFu);
  return lo + (static_cast<int64_t>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(x >> 24))) << 24);
}
__device__ __forceinline__ int64_t quot(int64_t a, int64_t b) {
  return (a | b) >> 32 ? a / b : static_cast<unsigned>(a) / static_cast<unsigned>(b);
}
struct Seq {                 // a lane's sequence: rows, cached keys, row blocks, the last (largest) one's weight, all of them
  int64_t lo, sum;
  int nq, len, rts, top;
};
// Sequences b0 to b0 + 31, by a warp. The weights of a causal sequence's row blocks are added up lane by lane, or
// sequence by sequence with a lane a row block, whichever takes fewer turns.
__device__ Seq sequences(const AttnParams& p, int b0, int cut) {
  const int lane = threadIdx.x & 31;
  Seq s = {};
  if (b0 + lane < p.a.B) {
    seq_sizes(p, b0 + lane, s.nq, s.len, s.lo);
    s.rts = (s.nq * p.group + kRows - 1) / kRows;
    s.top = s.rts ? weight(p, s.nq, s.len, s.rts - 1, cut) : 0;
  }
  s.sum = (int64_t)s.rts * s.top;
  if (!p.causal || cut == kWhole) return s;
  const int most = __reduce_max_sync(0xffffffffu, s.rts);
  const int turns = __reduce_add_sync(0xffffffffu, min((s.rts + 31) >> 5, 1 << 25));
  if (most <= 2 * turns) {
    s.sum = 0;
    for (int rt = 0; rt < s.rts; ++rt) s.sum += weight(p, s.nq, s.len, rt, cut);
    return s;
  }
  for (unsigned left = __ballot_sync(0xffffffffu, s.rts > 0); left; left &= left - 1) {
    const int of = __ffs(left) - 1;
    const int nq = __shfl_sync(0xffffffffu, s.nq, of), len = __shfl_sync(0xffffffffu, s.len, of);
    const int rts = __shfl_sync(0xffffffffu, s.rts, of);
    int64_t sum = 0;
    for (int rt = lane; rt < rts; rt += 32) sum += weight(p, nq, len, rt, cut);
    sum = warp_sum(sum);
    if (lane == of) s.sum = sum;
  }
  return s;
}
__device__ Shares shares_of(const AttnParams& p) {           // a warp's work
  const int G = p.items;
  int64_t tiles = 0, blocks = 0;
  int longest = 0;
  for (int b0 = 0; b0 < p.a.B; b0 += 32) {
    const Seq q = sequences(p, b0, 0);
    tiles += warp_sum(q.sum);
    blocks += warp_sum(q.rts);
    longest = max(longest, __reduce_max_sync(0xffffffffu, q.top));
  }
  const int64_t all = tiles * p.a.heads, count = blocks * p.a.heads;
  // a part of a row block costs kLead tiles as well, the join 3
  const int64_t rounds = quot(count + G - 1, G), even = max(quot(all + G - 1, G), (int64_t)p.min_tiles + kLead);
  const int64_t by_tiles = even + kLead + 3, by_blocks = rounds * longest;
  const int64_t part = count < G ? max(quot(all - kLead * count + G - count - 1, G - count), (int64_t)p.min_tiles) : kWhole;
  const int64_t by_parts = part < longest - kLead ? part + kLead + 3 : by_blocks;
  Shares s = {};
  s.blocks = blocks;
  if (min(by_blocks, by_parts) <= by_tiles) {
    s.cut = by_parts < by_blocks ? static_cast<int>(part) : kWhole;
    s.rounds = static_cast<int>(rounds);
    return s;
  }
  if (tiles == blocks * longest) s.rounds = max(0, static_cast<int>(quot(count, G)) - 1);
  s.total = tiles;
  s.base = (int64_t)s.rounds * G * longest;
  s.run = max(quot(all - s.base + G - 1, G), (int64_t)p.min_tiles + kLead);
  return s;
}
struct Place {               // in the list of a head's row blocks
  int b, rt, nq, len;
  int64_t lo, off;           // tiles or units of the row block in front of it
};
// Position x of a head, by a warp; false: behind its end.
__device__ bool find_place(const AttnParams& p, int cut, int64_t x, Place& w) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  for (int b0 = 0; b0 < p.a.B; b0 += 32) {
    const Seq q = sequences(p, b0, cut);
    int64_t upto = q.sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > x);
    if (!hit) {
      before += __shfl_sync(0xffffffffu, upto, 31);
      continue;
    }
    const int src = __ffs(hit) - 1;
    w.b = b0 + src;
    w.nq = __shfl_sync(0xffffffffu, q.nq, src);
    w.len = __shfl_sync(0xffffffffu, q.len, src);
    w.lo = __shfl_sync(0xffffffffu, q.lo, src);
    const int rts = __shfl_sync(0xffffffffu, q.rts, src), each = __shfl_sync(0xffffffffu, q.top, src);
    int64_t rest = x - before - __shfl_sync(0xffffffffu, upto - q.sum, src);
    if (!p.causal || cut == kWhole) {    // equal row blocks
      const int64_t block = quot(rest, each);
      w.rt = rts - 1 - static_cast<int>(block);
      w.off = rest - block * each;
      return true;
    }
    for (int top = rts - 1; top >= 0; top -= 32) {
      const int t = top - lane >= 0 ? weight(p, w.nq, w.len, top - lane, cut) : 0;
      int64_t sum = t;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const unsigned in = __ballot_sync(0xffffffffu, sum > rest);
      if (in) {
        const int at = __ffs(in) - 1;
        w.rt = top - at;
        w.off = rest - __shfl_sync(0xffffffffu, sum - t, at);
        return true;
      }
      rest -= __shfl_sync(0xffffffffu, sum, 31);
    }
    return false;
  }
  return false;
}

template <typename T, int D, bool CARRY>
__global__ void __launch_bounds__(kThreadsP, 1) attn_many_kernel(const __grid_constant__ AttnParams p,
                                                               const __grid_constant__ CUtensorMap k_map,
                                                               const __grid_constant__ CUtensorMap v_map,
                                                               bool mapped) {
  using S = Smem<D>;
  constexpr bool kHalfQ = __is_same(T, __half);
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + S::kBar);
  Seg* seg = reinterpret_cast<Seg*>(smem + S::kSeg);
  static_assert(sizeof(Seg) <= 64, "");
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + S::kSeg + kSegs * 64);
  const int warp = threadIdx.x >> 5;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(bar + KFULL + i, 2);      // one arrival a warp: a barrier takes arrivals one after another
      bar_init(bar + VFULL + i, 2);
      bar_init(bar + QFULL + i, 8);
      bar_init(bar + PFULL + 2 * i, 8);
      bar_init(bar + PFULL + 2 * i + 1, 8);
      bar_init(bar + KEMPTY + i, 1);
      bar_init(bar + VEMPTY + i, 1);
      bar_init(bar + SFULL + i, 1);
      bar_init(bar + ODONE + i, 1);
    }
    bar_init(bar + IDLE, 1);
    for (int i = 0; i < kSegs; ++i) {
      bar_init(bar + GFULL + i, 1);
      bar_init(bar + GEMPTY + i, 21);    // the warps in front of the one that hands out the shares
    }
    bar_init_fence();
  }
  if (warp == 20) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  constexpr uint32_t tmem = 0;           // all 512 columns are this block's: the allocation starts at column 0
  pdl_trigger();
  pdl_wait();

  // share s of this block's, or null behind the last one (or after an error); each of 21 warps says when it is done with it
  auto share = [&](int s) -> const Seg* {
    if (!warp_wait(bar + GFULL + s % kSegs, (s / kSegs) & 1, p.err, kErrPrefill + 9, kShareLimitNs)) return nullptr;
    const Seg* g = seg + s % kSegs;
    return *reinterpret_cast<const volatile int*>(&g->h) < 0 ? nullptr : g;
  };
  auto share_done = [&](int s) { warp_arrive(bar + GEMPTY + s % kSegs); };

  if (warp == 21) {
    // ---------------------------------------------------------------------------------------- this block's share
    const Shares sh = shares_of(p);
    const int G = p.items, me = blockIdx.x;
    Joint joint = {};
    int s = 0;
    bool ok = true;
    // tiles [t0, t1) of a row block, t1 cut to its end; the end of the block's share for at == null
    auto hand_out = [&](const Place* at, int h, int t0, int t1) {
      if (s >= kSegs)
        ok = ok && warp_wait(bar + GEMPTY + s % kSegs, ((s / kSegs) & 1) ^ 1, p.err, kErrPrefill + 13, kShareLimitNs);
      if (!ok) return;
      Seg g;
      g.h = -1;
      if (at) {
        int tc, tf;
        seen_tiles(p, at->nq, at->len, at->rt, tc, tf);
        g.h = h, g.lo = at->lo, g.b = at->b, g.nq = at->nq, g.len = at->len;
        g.row0 = at->rt * kRows, g.rows = at->nq * p.group;
        g.tile0 = t0;
        g.nc = max(0, min(t1, tc) - t0);
        g.f0 = max(t0 - tc, 0);
        g.nf = max(0, min(t1, tc + tf) - tc - g.f0);
        g.slot = t0 > 0 ? me : t1 < tc + tf ? G + me : -1;
      }
      if (elect_one()) seg[s % kSegs] = g;
      warp_arrive(bar + GFULL + s % kSegs);
      ++s;
    };
    auto join_from_here = [&](const Place& at, int h, int parts) {
      joint.lo = at.lo, joint.parts = parts, joint.h = h, joint.row0 = at.rt * kRows;
      joint.rows = min(kRows, at.nq * p.group - joint.row0);
    };
    Place at;
    if (sh.cut && sh.cut != kWhole) {                       // one part of a row block
      int64_t units = 0;
      for (int b0 = 0; b0 < p.a.B; b0 += 32) units += warp_sum(sequences(p, b0, sh.cut).sum);
      if (me < units * p.a.heads) {
        const int h = static_cast<int>(quot(me, units));
        if (find_place(p, sh.cut, me - h * units, at)) {
          const int64_t t = weight(p, at.nq, at.len, at.rt, 0) - kLead, n = weight(p, at.nq, at.len, at.rt, sh.cut);
          if (at.off == 0 && n > 1) join_from_here(at, h, static_cast<int>(n));
          hand_out(&at, h, static_cast<int>(quot(t * at.off, n)), static_cast<int>(quot(t * (at.off + 1), n)));
        }
      }
    } else {
      for (int r = 0; r < sh.rounds && ok; ++r) {           // whole row blocks
        const int64_t x = (int64_t)r * G + me;
        if (x >= sh.blocks * p.a.heads) break;
        const int h = static_cast<int>(quot(x, sh.blocks));
        if (!find_place(p, kWhole, x - h * sh.blocks, at)) break;
        hand_out(&at, h, 0, weight(p, at.nq, at.len, at.rt, 0) - kLead);
      }
      int64_t x = sh.base + me * sh.run, left = sh.cut ? 0 : min(sh.run, sh.total * p.a.heads - x);
      int h = left > 0 ? static_cast<int>(quot(x, sh.total)) : 0;
      if (left > 0 && find_place(p, 0, x - h * sh.total, at)) {
        while (ok) {
          const int t = weight(p, at.nq, at.len, at.rt, 0), t0 = static_cast<int>(at.off);
          const int t1 = static_cast<int>(min((int64_t)t, t0 + left));
          const int first = max(t0 - kLead, 0), end = max(t1 - kLead, 0);   // a cut through the lead is none
          // (the row block ends t - t0 behind x)
          if (first == 0 && end > 0 && t1 < t)
            join_from_here(at, h, static_cast<int>(quot(x + t - t0 - 1 - sh.base, sh.run)) - me + 1);
          if (end > first) hand_out(&at, h, first, end);
          x += t1 - t0;
          left -= t1 - t0;
          if (left <= 0) break;
          at.off = 0;
          while (--at.rt < 0) {                             // the next sequence with rows
            if (++at.b == p.a.B) {
              at.b = 0;
              if (++h == p.a.heads) break;                  // (only if the lengths change under the call)
            }
            seq_sizes(p, at.b, at.nq, at.len, at.lo);
            at.rt = (at.nq * p.group + kRows - 1) / kRows;
          }
          if (h == p.a.heads) break;
        }
      }
    }
    hand_out(nullptr, 0, 0, 0);
    if (elect_one()) joints(p, D)[me] = joint;
  } else if (warp >= 16 && warp < 20) {
    // ------------------------------------------------------------------------------------------- keys and values
    const bool val = warp >= 18;
    const int t = threadIdx.x & 63;                         // rows t and t + 64 of a cached tile
    const int full = val ? VFULL : KFULL, empty = val ? VEMPTY : KEMPTY;
    const uint32_t ring = smem_u32(smem) + (val ? S::kV : S::kK);
    const uint8_t* codes = val ? p.c.v_codes : p.c.k_codes;
    const uint8_t* scales = val ? p.c.v_sf : p.c.k_sf;
    constexpr int CW = D / 32;           // 16-byte pieces of a row's codes
    bool ok = true;
    int sent = -1, done = 0;             // the last tile that TMA was asked for; tiles of the shares so far
    // Copies in flight land before the block's shared memory goes away, also where an error elsewhere ended the shares or the
    // products. (Of the last two of `made` tiles: a stage that has been filled again was empty before. No wait without an error.)
    auto land = [&](int made) {
      for (int j = max(max(sent - 1, made - 2), 0); j <= sent; ++j) bar_drain(bar + full + (j & 1), (j >> 1) & 1);
    };
    const Seg* g;
    for (int s = 0; ok && (g = share(s)); ++s) {
      const int nc = g->nc, n = nc + g->nf, f0 = g->f0, tile0 = g->tile0, len = g->len, nq = g->nq, h = g->h;
      const int64_t lo = g->lo;
      const int32_t* table = p.a.table + g->b * p.a.table_ld;
      share_done(s);
      int page[2];                         // of this thread's rows of the next cached tile, or -1 behind the length
      auto look = [&](int j) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int key = (tile0 + j) * kKeys + x * 64 + t;
          page[x] = j < nc && key < len
                        ? min(max(__ldg(table + (key >> p.a.page_shift)), 0), static_cast<int>(p.a.pages - 1)) : -1;
        }
      };
      uint4 cw[2][CW];
      uint2 sc[2];
      auto fetch = [&](int j) {            // zeros behind the length
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          sc[x] = make_uint2(0, 0);
#pragma unroll
          for (int i = 0; i < CW; ++i) cw[x][i] = make_uint4(0, 0, 0, 0);
          if (page[x] < 0) continue;
          const int key = (tile0 + j) * kKeys + x * 64 + t;
          const int64_t row = (((int64_t)page[x] * p.a.heads + h) << p.a.page_shift) + (key & ((1 << p.a.page_shift) - 1));
#pragma unroll
          for (int i = 0; i < CW; ++i) cw[x][i] = __ldg(reinterpret_cast<const uint4*>(codes + row * (D / 2)) + i);
          if (D == 128) sc[x] = __ldg(reinterpret_cast<const uint2*>(scales + row * (D / 16)));
          else sc[x].x = __ldg(reinterpret_cast<const uint32_t*>(scales + row * (D / 16)));
        }
      };
      if (nc > 0) {
        look(0);
        fetch(0);
        look(1);
      }
      for (int j = 0; j < nc && ok; ++j) {
        const int jj = done + j, st = jj & 1;
        if (jj >= 2) ok = warp_wait(bar + empty + st, ((jj >> 1) & 1) ^ 1, p.err, kErrPrefill + 1);
        if (!ok) {
          land(jj);
          break;
        }
        const uint32_t tile = ring + st * S::kTileB;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          uint32_t sp[D / 32];             // scale pairs
          sp[0] = e4m3x2_to_f16x2(sc[x].x & 0xFFFFu);
          sp[1] = e4m3x2_to_f16x2(sc[x].x >> 16);
          if (D == 128) {
            sp[D / 32 - 2] = e4m3x2_to_f16x2(sc[x].y & 0xFFFFu);
            sp[D / 32 - 1] = e4m3x2_to_f16x2(sc[x].y >> 16);
          }
#pragma unroll
          for (int i = 0; i < CW; ++i) {
            const uint32_t words[4] = {cw[x][i].x, cw[x][i].y, cw[x][i].z, cw[x][i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // word: 8 values, chunk 4 i + k; two chunks a scale
              uint32_t o[4];
              e2m1x8_scaled(words[k], __byte_perm(sp[i], 0, k < 2 ? 0x1010 : 0x3232), o);
              store_shared(tile + tile_at<D>(x * 64 + t, 4 * i + k), o[0], o[1], o[2], o[3]);
            }
          }
        }
        fetch(j + 1);
        look(j + 2);
        async_fence();
        warp_arrive(bar + full + st);
      }
      if (n > nc && ok) {
        const T* src = static_cast<const T*>(val ? p.vn : p.kn) + lo * (val ? p.vn_st : p.kn_st) +
                       h * (val ? p.vn_sh : p.kn_sh);
        const int64_t ld = val ? p.vn_st : p.kn_st;
        constexpr int CH = D / 8;          // 16-byte chunks of a row
        const int c = t % CH, r0 = t / CH;
        for (int j = nc; j < n && ok; ++j) {
          const int jj = done + j, st = jj & 1;
          if (jj >= 2) ok = warp_wait(bar + empty + st, ((jj >> 1) & 1) ^ 1, p.err, kErrPrefill + 4);
          if (!ok) {
            land(jj);
            break;
          }
          const int first = (f0 + j - nc) * kKeys;
          if (mapped && first + kKeys <= nq) {              // whole tiles by TMA: one thread's work
            if (warp & 1) {
              warp_arrive(bar + full + st);
            } else if (elect_one()) {
              bar_arrive_tx(bar + full + st, S::kTileB);
#pragma unroll
              for (int x = 0; x < D / 64; ++x)
                copy_tensor_3d(smem + (val ? S::kV : S::kK) + st * S::kTileB + x * S::kHalf, val ? &v_map : &k_map, bar + full + st, x * 64, h,
                               static_cast<int>(lo) + first);
            }
            __syncwarp();
            sent = jj;
            continue;
          }
          // the sequence's last rows, zeros behind them (what lies there may be anything)
          const uint32_t tile = ring + st * S::kTileB;
          const int key0 = first + r0;
          const T* from = src + key0 * ld + c * 8;
#pragma unroll 8
          for (int k = 0; k < 2 * CH; ++k) {
            const bool live = key0 + k * (64 / CH) < nq;
            copy16(tile + tile_at<D>(k * (64 / CH) + r0, c), live ? from + k * (64 / CH) * ld : src, live);
          }
          // waited for at once: the other stage's tile is what the products are at
          asm volatile("cp.async.wait_all;" ::: "memory");
          async_fence();
          warp_arrive(bar + full + st);
        }
      }
      done += n;
    }
    if (ok) land(done);
  } else if (warp == 20) {
    // ------------------------------------------------------------------------------------------------- products
    const uint32_t qb = smem_u32(smem + S::kQ), kb = smem_u32(smem + S::kK), vb = smem_u32(smem + S::kV);
    constexpr int fmt = kHalfQ ? 0 : 1;
    auto qk = [&](int i, int st, bool cached) {
      const uint32_t id = mma_desc(cached ? 0 : fmt, kKeys, false);
      const uint32_t a = desc_lo(qb + i * S::kTileB, 16), b = desc_lo(kb + st * S::kTileB, 16);
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        const uint32_t off = (k >> 1) * (S::kHalf >> 4) + (k & 1) * 4;
        mma2_ss(i * 128, a + off, b + off, id, k);
      }
      mma_commit(bar + SFULL + i);
    };
    auto pv = [&](int i, int st, bool cached, int part, uint32_t acc) {   // keys [32 part, +32) of both halves
      const uint32_t id = mma_desc(cached ? 0 : fmt, D, true);
      const uint32_t b = desc_lo(vb + st * S::kTileB, S::kHalf) + part * 2 * 128;
      mma2_ts(kColO + i * 128, i * 128 + part * 16, b, id, acc);
      mma2_ts(kColO + i * 128, i * 128 + 64 + part * 16, b + 4 * 128, id, 1);
    };
    int s = 0, n = 0, nc = 0, both = 0;  // shares so far; the last one's tiles, cached tiles, and if its tile 1 has rows
    auto take = [&]() -> bool {          // the next share, which may have no tiles; false: none is left
      const Seg* g = share(s);
      if (!g) return false;
      nc = g->nc, n = nc + g->nf, both = g->row0 + 128 < g->rows;
      share_done(s++);
      return true;
    };
    auto advance = [&]() -> bool {       // to the next share with tiles; only while no results are owed (see below)
      do {
        if (!take()) return false;
      } while (n == 0);
      return true;
    };
    int qs[2] = {0, 0}, ps[2] = {0, 0};  // phases waited for: query rows, probabilities
    bool ok = true;
    auto scores = [&](int i, int jj, int j) {               // of tile j of the share, jj of all
      if (j == 0 || (j == nc && !kHalfQ)) ok = warp_wait<true>(bar + QFULL + i, qs[i]++ & 1, p.err, kErrPrefill + 2);
      if (!ok) return;
      tc_after();
      qk(i, jj & 1, j < nc);
    };
    // tile jj of all, the first one of a share, whose keys are waited for here: nothing else is under way
    auto begin = [&](int jj) {
      ok = warp_wait<true>(bar + KFULL + (jj & 1), (jj >> 1) & 1, p.err, kErrPrefill + 5);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (ok && i <= both) scores(i, jj, 0);
      if (ok) mma_commit(bar + KEMPTY + (jj & 1));
    };
    if (advance()) {
      begin(0);
      for (int jj = 0, j = 0; ok; ++jj) {
        const bool last = j + 1 == n, cached = j < nc, add = CARRY ? (j & (kCarry - 1)) != 0 : j > 0;
        const int rows2 = both;
        // The next tile is looked for ahead of this one's last product, but only one share ahead: shares without tiles are
        // handed out behind this share's results (of four shares the block knows at a time), which wait for that product.
        const bool got = !last || take(), more = got && n > 0;   // n, nc and both are the next tile's from here on
        j = last ? 0 : j + 1;
        ok = warp_wait<true>(bar + VFULL + (jj & 1), (jj >> 1) & 1, p.err, kErrPrefill + 6);
        if (more) ok = ok && warp_wait<true>(bar + KFULL + ((jj + 1) & 1), ((jj + 1) >> 1) & 1, p.err, kErrPrefill + 8);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i <= rows2) {
            ok = warp_wait<true>(bar + PFULL + 2 * i, ps[i] & 1, p.err, kErrPrefill + 7);
            if (!ok) break;
            tc_after();
            pv(i, jj & 1, cached, 0, add);
            ok = warp_wait<true>(bar + PFULL + 2 * i + 1, ps[i]++ & 1, p.err, kErrPrefill + 7);
            if (!ok) break;
            tc_after();
            pv(i, jj & 1, cached, 1, 1);
            if (last) mma_commit(bar + ODONE + i);
          }
          if (more && i <= both) scores(i, jj + 1, j);
          if (!ok) break;
        }
        if (!ok) break;
        mma_commit(bar + VEMPTY + (jj & 1));
        if (more) {
          mma_commit(bar + KEMPTY + ((jj + 1) & 1));
        } else {
          if (!got || !advance()) break;
          begin(jj + 1);
        }
      }
    }
    mma_commit(bar + IDLE);
    bar_drain(bar + IDLE, 0);            // nothing of the tensor core is in flight from here on
  } else if (warp < 16) {
    // -------------------------------------------------------------------------------------------------- softmax
    const int i = warp >> 3, half = (warp >> 2) & 1, r = threadIdx.x & 127;
    const uint32_t lane = (uint32_t)(warp & 3) << 21;       // this warp's 32 TMEM lanes
    const uint32_t ts = tmem + lane + i * 128, to = tmem + lane + kColO + i * 128 + half * (D / 2);
    const uint32_t pair = smem_u32(smem) + S::kPair + (i * 256 + r) * 4;
    // this thread's sums in memory, 4 columns kRows apart, and their base and row sum (seldom used: addresses found there)
    auto carry_sums = [&]() {
      return reinterpret_cast<float4*>(p.carry) + (blockIdx.x * (D / 4) + half * (D / 8)) * kRows + i * 128 + r;
    };
    auto carry_row = [&]() {
      return reinterpret_cast<float2*>(p.carry + (int64_t)p.items * kRows * D) + (blockIdx.x * 2 + half) * kRows + i * 128 + r;
    };
    bool ok = true;
    int turn = 0, sp = 0, op = 0;        // phases waited for: scores, accumulators
    // what this thread tells the row's other one, for what that one tells (two buffers in turn: one barrier is enough; both
    // warps come here equally often, also where a wait has run out)
    auto tell = [&](float x) -> float {
      const uint32_t p2 = pair + (turn & 1) * 2048;
      ++turn;
      float y;
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(p2 + half * 512), "f"(x) : "memory");
      asm volatile("bar.sync %0, 64;" ::"r"(1 + i * 4 + (warp & 3)) : "memory");
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(y) : "r"(p2 + (half ^ 1) * 512) : "memory");
      return y;
    };
    const float plain = fmaxf(fabsf(p.scale_log2), 1e-30f); // a scale of 0: any small one (-inf * 0 would be NaN)
    // In front of tile j: the sums so far to those in memory, in plain values. The accumulator begins again with this tile's
    // products (until then it may still be rescaled).
    auto carry = [&](int j, int nc, float m, float& l) {
      ok = ok && warp_wait(bar + SFULL + i, sp & 1, p.err, kErrPrefill + 10);    // behind all products of the tiles so far
      if (!ok) return;
      tc_after();
      float2* row_at = carry_row();
      const float2 old = j > kCarry ? *row_at : make_float2(m, 0.0f);
      const float keep = exp2_fast(old.x - m), unit = j <= nc ? p.c.v_global : 1.0f;
      *row_at = make_float2(m, old.y * keep + l);
      l = 0.0f;
#pragma unroll 1
      for (int k = 0; k < D / 2; k += 16) {
        uint32_t o[16];
        tmem_ld16(to + k, o);
#pragma unroll
        for (int x = 0; x < 16; x += 4) {
          float4* at4 = carry_sums() + (k + x) / 4 * kRows;
          const float4 y = j > kCarry ? *at4 : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          *at4 = make_float4(y.x * keep + __uint_as_float(o[x]) * unit, y.y * keep + __uint_as_float(o[x + 1]) * unit,
                             y.z * keep + __uint_as_float(o[x + 2]) * unit, y.w * keep + __uint_as_float(o[x + 3]) * unit);
        }
      }
    };
    // The next share. Both warps of a row go on or neither does.
    int at = 0;
    auto next_share = [&]() -> const Seg* {
      const Seg* g = share(at);
      const bool got = g != nullptr;
      return tell(got ? 1.0f : 0.0f) != 0.0f && got ? g : nullptr;
    };
    auto is_live = [&](const Seg* g) { return g->nc + g->nf > 0 && (i == 0 || g->row0 + 128 < g->rows); };
    // this thread's half of the query row into shared memory, as fp16 over a power of two (`norm`, the result) or as it is;
    // negated for a negative scale. The result is NaN if a value of it is not finite.
    auto put_query = [&](const Seg* g, bool norm) -> float {
      const int row = g->row0 + i * 128 + r, rows = g->rows;
      const T* src = static_cast<const T*>(p.q) + (g->lo + row / p.group) * p.q_st +
                     (g->h * p.group + row % p.group) * p.q_sh + half * (D / 2);
      const uint32_t flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
      uint4 v[D / 16];
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
        v[c] = row < rows ? __ldg(reinterpret_cast<const uint4*>(src) + c) : make_uint4(0u, 0u, 0u, 0u);
      using T2 = std::conditional_t<kHalfQ, __half2, __nv_bfloat162>;
      T2 top2 = __habs2(reinterpret_cast<const T2&>(v[0].x));
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) top2 = __hmax2_nan(top2, __habs2(reinterpret_cast<const T2&>(w[k])));
      }
      const float lo = __low2float(top2), hi = __high2float(top2), amax = fmaxf(lo, hi);
      const bool bad = !(lo < INFINITY && hi < INFINITY);
      float e = 1.0f;
      if (norm && !kHalfQ) {
        e = pow2i(row_exponent(fmaxf(amax, tell(amax))));
        const float f = 1.0f / e;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          float x[8];
          unpack_bf16x8(v[c], x);
          v[c] = make_uint4(pack_f16x2(x[0] * f, x[1] * f), pack_f16x2(x[2] * f, x[3] * f),
                            pack_f16x2(x[4] * f, x[5] * f), pack_f16x2(x[6] * f, x[7] * f));
        }
      }
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
        *reinterpret_cast<uint4*>(smem + S::kQ + i * S::kTileB + tile_at<D>(r, half * (D / 16) + c)) =
            make_uint4(v[c].x ^ flip, v[c].y ^ flip, v[c].z ^ flip, v[c].w ^ flip);
      async_fence();
      warp_arrive(bar + QFULL + i);
      return bad ? bad_row() : e;
    };
    const Seg* g = next_share();
    float e = g && is_live(g) ? put_query(g, g->nc > 0) : 1.0f;
    while (g) {
      const int row = g->row0 + i * 128 + r, rows = g->rows;
      const int nc = g->nc, nf = g->nf, n = nc + nf;
      const bool live = is_live(g);
      const int q_at = row < rows ? row / p.group : g->nq - 1;
      int see_c = p.causal && !p.kn ? min(g->len, g->len - g->nq + q_at + 1) : g->len;
      float m = kNoMax, l = 0.0f;                           // base of the powers, their sum
      if (live && isnan(e)) l = see_c > 0 || p.kn ? e : 0.0f, e = 1.0f;
      float mul = nc > 0 ? plain * p.c.k_global * e : plain;
      see_c -= g->tile0 * kKeys + half * 64;
      const int see_f = (p.causal ? q_at + 1 : g->nq) - (g->f0 - nc) * kKeys - half * 64;
      // (a share's first scores, where this query tile had no rows in the one before)
      if (live) ok = ok && warp_wait(bar + SFULL + i, sp & 1, p.err, kErrPrefill + 10, kShareLimitNs);
      for (int j = 0; live && j < n; ++j) {
        if (CARRY && (j & (kCarry - 1)) == 0 && j > 0) carry(j, nc, m, l);
        ok = ok && warp_wait(bar + SFULL + i, sp++ & 1, p.err, kErrPrefill + 10);
        if (!ok) {
          tell(0.0f);
          continue;
        }
        tc_after();
        const bool cached = j < nc;
        if (j == nc) mul = plain;
        // the scores 32 at a time, the far ones twice (all 64 at once did not fit the registers)
        uint32_t s[32];
        const uint32_t th = ts + half * 64;
        const int left = (cached ? see_c : see_f) - j * kKeys;   // keys seen
        const bool masked = __any_sync(0xffffffffu, left < 64);
        auto get = [&](int k0) {
          tmem_ld32(th + k0, s);
          tmem_ld_wait();
          tmem_tie(s);
          if (masked) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (k0 + k >= left) s[k] = 0xFF800000u;       // -inf
          }
        };
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k0 = 32; k0 >= 0; k0 -= 32) {
          get(k0);
#pragma unroll
          for (int k = 0; k < 32; k += 8)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              top[x] = max3(top[x], __uint_as_float(s[k + 2 * x]), __uint_as_float(s[k + 2 * x + 1]));
        }
        float mt = fmaxf(max3(top[0], top[1], top[2]), top[3]);
        mt = fmaxf(mt, tell(mt)) * mul;
        const bool switched = j == nc && j > 0;             // from the cache's value scale to plain values
        if (switched || __any_sync(0xffffffffu, mt > m + kLazy)) {   // (the same in both warps of a row)
          const float mn = fmaxf(m, mt - kHead);
          float c = exp2_fast(m - mn);
          m = mn;
          l *= c;
          if (switched) c *= p.c.v_global;
          if (j > 0) {                                      // this tile's first product is behind the last P V
#pragma unroll 1
            for (int k = 0; k < D / 2; k += 16) {
              uint32_t o[16];
              tmem_ld16(to + k, o);
#pragma unroll
              for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * c);
              tmem_st16(to + k, o);
            }
          }
        }
        const float2 mul2 = make_float2(mul, mul), neg2 = make_float2(-m, -m);
        float2 sum2 = make_float2(0.0f, 0.0f);
        auto powers = [&](auto pack, auto poly) {
#pragma unroll
          for (int k0 = 0; k0 < 64; k0 += 32) {
            if (k0) get(k0);
            uint32_t pk[16];
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              float2 z = __ffma2_rn(make_float2(__uint_as_float(s[x]), __uint_as_float(s[x + 1])), mul2, neg2);
              z = (x >> 1) % 4 < decltype(poly)::value ? exp2_poly(z) : make_float2(exp2_fast(z.x), exp2_fast(z.y));
              sum2 = __fadd2_rn(sum2, z);
              pk[x >> 1] = pack(z.x, z.y);
            }
            tmem_st16(th + (k0 >> 1), pk);                  // keys k, k + 1 in column k / 2 of the half's own
            tmem_st_wait();
            tc_before();
            warp_arrive(bar + PFULL + 2 * i + (k0 >> 5));
          }
        };
        // a quarter of the powers on the FMA pipes beside TMA tiles (image step 264 -> 258 us at the time); none where the operand
        // warps' conversions need those pipes (ragged prefill 275 -> 262 us)
        using std::integral_constant;
        if (cached)
          powers([](float a, float b) { return pack_f16x2(a, b); }, integral_constant<int, 0>());
        else if (kHalfQ)
          powers([](float a, float b) { return pack_f16x2(a, b); }, integral_constant<int, 1>());
        else
          powers([](float a, float b) { return pack_bf16x2(a, b); }, integral_constant<int, 1>());
        l += sum2.x + sum2.y;
        // the last cached tile's scores are there: the query row in q's type, for the next tile
        if (j + 1 == nc && nf > 0 && !kHalfQ) put_query(g, false);
      }
      // the next share's query rows, so that its first scores come while these rows' results are written
      ++at;
      const Seg* next = next_share();
      if (next && is_live(next)) e = put_query(next, next->nc > 0);
      const bool carried = CARRY && live && n > kCarry;
      float keep = 0.0f;
      if (carried) {
        const float2 old = *carry_row();
        keep = exp2_fast(old.x - m);
        l += old.y * keep;
      }
      if (live) {
        ok = ok && warp_wait(bar + ODONE + i, op++ & 1, p.err, kErrPrefill + 12);
        tc_after();
        l += tell(l);
      }
      // ----------------------------------------------------------------------------------------------- results
      const float unit = nf > 0 ? 1.0f : p.c.v_global;      // of the accumulator
      if (m == kNoMax && !isnan(l)) l = 0.0f;               // no key seen (a hidden one's power is 2^-120, not 0)
      const bool part = g->slot >= 0;
      const int64_t tok = g->lo + row / p.group;
      const int hq = g->h * p.group + row % p.group;
      const int64_t to_row = (int64_t)g->slot * kRows + i * 128 + r;
      const float f = l == 0.0f ? 0.0f : part ? unit : unit / l;
      keep *= f / unit;
#pragma unroll 1
      for (int k = 0; k < D / 2; k += 16) {
        uint32_t o[16];
        if (live && ok) {                                   // uniform over the warp
          tmem_ld16(to + k, o);
        } else {
#pragma unroll
          for (int x = 0; x < 16; ++x) o[x] = 0u;
        }
        if (row < rows) {
          const int col = half * (D / 2) + k;
#pragma unroll
          for (int x = 0; x < 16; x += 8) {
            float y[8];
#pragma unroll
            for (int z = 0; z < 8; ++z) y[z] = __uint_as_float(o[x + z]) * f;
            if (carried) {
              const float4 a = carry_sums()[(k + x) / 4 * kRows], b = carry_sums()[((k + x) / 4 + 1) * kRows];
              y[0] += a.x * keep, y[1] += a.y * keep, y[2] += a.z * keep, y[3] += a.w * keep;
              y[4] += b.x * keep, y[5] += b.y * keep, y[6] += b.z * keep, y[7] += b.w * keep;
            }
            if (part) {
              float4* to4 = reinterpret_cast<float4*>(p.part) +
                            ((int64_t)g->slot * (D / 4) + (col + x) / 4) * kRows + i * 128 + r;
              to4[0] = make_float4(y[0], y[1], y[2], y[3]);
              to4[kRows] = make_float4(y[4], y[5], y[6], y[7]);
            } else
              store8(static_cast<T*>(p.out) + tok * p.o_st + hq * p.o_sh + col + x, y);
          }
        }
      }
      if (row < rows && half == 0) {
        if (part) {
          float* ml = p.part + 2LL * p.items * kRows * D + to_row * 2;
          ml[0] = m;
          ml[1] = l;
        } else if (p.lse) {
          p.lse[tok * p.Hq + hq] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718056f;
        }
      }
      tc_before();
      share_done(at - 1);
      g = next;
    }
  }
  tc_before();
  __syncthreads();
  if (warp == 20) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// Joins the parts of row blocks: each of the grid's blocks a share of the rows of one of them.
template <typename T, int D>
__global__ void __launch_bounds__(256, 4) join_many_kernel(const __grid_constant__ AttnParams p) {
  __shared__ unsigned some[8];           // which grid blocks hold a row block's first part
  pdl_trigger();
  pdl_wait();
  const Joint* all = joints(p, D);
  const unsigned mine = __ballot_sync(0xffffffffu, threadIdx.x < p.items && all[threadIdx.x].parts > 0);
  if (threadIdx.x % 32 == 0) some[threadIdx.x / 32] = mine;
  __syncthreads();
  int found = 0, of = 0;                 // row blocks to join; this block's: number blockIdx.x % found
#pragma unroll
  for (int w = 0; w < 8; ++w) found += __popc(some[w]);
  if (!found) return;
  int left = static_cast<int>(blockIdx.x) % found;
  for (; left >= __popc(some[of / 32]); of += 32) left -= __popc(some[of / 32]);
  of += static_cast<int>(__fns(some[of / 32], 0u, left + 1));
  const int share = blockIdx.x / found, shares = gridDim.x / found;
  if (share >= shares) return;
  const Joint j = all[of];
  // a warp takes 4 rows, a lane an eighth of one; where there are many parts, four or eight warps share them
  constexpr int V = D / 32;              // its float4
  __shared__ float4 acc_s[8][V][32];
  __shared__ float2 ml_s[8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, eighth = lane >> 2;
  const int warps = j.parts > 32 ? 8 : j.parts > 8 ? 4 : 1, of4 = warp & (warps - 1);
  const float4* acc_g = reinterpret_cast<const float4*>(p.part);
  const float2* ml_g = reinterpret_cast<const float2*>(p.part + 2LL * p.items * kRows * D);
  for (int r0 = share * (32 / warps); r0 < j.rows; r0 += shares * (32 / warps)) {
    const int r = r0 + warp / warps * 4 + (lane & 3);       // below kRows; behind the last row: read, not written
    float4 acc[V];
    float m = kNoMax, l = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float pm, float pl, const float4* y) {
      const float top = fmaxf(m, pm), a = exp2_fast(m - top), b = exp2_fast(pm - top);
      m = top;
      l = l * a + pl * b;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        acc[v].x = acc[v].x * a + y[v].x * b;
        acc[v].y = acc[v].y * a + y[v].y * b;
        acc[v].z = acc[v].z * a + y[v].z * b;
        acc[v].w = acc[v].w * a + y[v].w * b;
      }
    };
#pragma unroll 2
    for (int i = of4; i < j.parts; i += warps) {
      const int64_t slot = i ? of + i : p.items + of;
      const float2 s = ml_g[slot * kRows + r];
      float4 y[V];
#pragma unroll
      for (int v = 0; v < V; ++v) y[v] = acc_g[(slot * (D / 4) + eighth * V + v) * kRows + r];
      add(s.x, s.y, y);
    }
    if (warps > 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) acc_s[warp][v][lane] = acc[v];
      ml_s[warp][lane] = make_float2(m, l);
      __syncthreads();
      if (of4 == 0) {
        for (int x = 1; x < warps; ++x) {
          float4 y[V];
#pragma unroll
          for (int v = 0; v < V; ++v) y[v] = acc_s[warp + x][v][lane];
          add(ml_s[warp + x][lane].x, ml_s[warp + x][lane].y, y);
        }
      }
      __syncthreads();
    }
    if (of4 == 0 && r < j.rows) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int64_t tok = j.lo + (j.row0 + r) / p.group;
      const int hq = j.h * p.group + (j.row0 + r) % p.group;
      T* dst = static_cast<T*>(p.out) + tok * p.o_st + hq * p.o_sh + eighth * V * 4;
#pragma unroll
      for (int v = 0; v < V; v += 2)
        *reinterpret_cast<uint4*>(dst + v * 4) =
            make_uint4(pack2<T>(acc[v].x * inv, acc[v].y * inv), pack2<T>(acc[v].z * inv, acc[v].w * inv),
                       pack2<T>(acc[v + 1].x * inv, acc[v + 1].y * inv), pack2<T>(acc[v + 1].z * inv, acc[v + 1].w * inv));
      if (p.lse && eighth == 0) p.lse[tok * p.Hq + hq] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718056f;
    }
  }
}

struct ManyPlan {
  int blocks, min_tiles, join_blocks;    // blocks: 256 at most (a thread each of a join block)
  int64_t ws, carry;                     // carry: its place in the workspace, or 0
};
ManyPlan many_plan(int64_t dim, int64_t heads, int64_t B, int64_t max_keys, int64_t T, int64_t group, int sms) {
  ManyPlan f;
  f.min_tiles = 4;
  const int64_t tiles = (max_keys + kKeys - 1) / kKeys + (T + kKeys - 1) / kKeys + kLead;
  const int64_t most = std::max<int64_t>(1, tiles) * (T * group / kRows + B) * heads;      // never fewer than there are
  f.blocks = static_cast<int>(std::min<int64_t>(std::min(sms, 256), std::max(heads * B, (most + f.min_tiles - 1) / f.min_tiles)));
  f.join_blocks = static_cast<int>(std::min<int64_t>(4 * f.blocks, 64 * heads * (T * group / kRows + B)));
  f.ws = (2LL * f.blocks * kRows * (dim + 2) * 4 + f.blocks * (int64_t)sizeof(Joint) + 15) / 16 * 16;
  f.carry = tiles - kLead > kCarry ? f.ws : 0;
  if (f.carry) f.ws += (int64_t)f.blocks * kRows * (dim + 4) * 4;
  return f;
}

template <typename T, int D, bool CARRY>
tfb_status launch_many(AttnParams& p, const ManyPlan& f, const DeviceInfo* di, cudaStream_t s) {
  static std::atomic<bool> ready[64];
  const auto kernel = attn_many_kernel<T, D, CARRY>;
  if (!ready[di->device].load(std::memory_order_acquire)) {
    TFB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::kBytes));
    ready[di->device].store(true, std::memory_order_release);
  }
  // maps of the new keys and values; rows or heads without a stride of their own (expanded ones) are copied by hand
  alignas(64) CUtensorMap maps[2] = {};
  const int64_t hk = p.a.heads, ks = hk > 1 ? p.kn_sh : D, vs = hk > 1 ? p.vn_sh : D;
  const bool mapped = p.kn && p.a.T >= kKeys && ks > 0 && vs > 0 && p.kn_st > 0 && p.vn_st > 0;
  if (mapped) {
    tfb_status st = make_tmap_rows16(&maps[0], p.kn, D, hk, ks * 2, p.a.T, p.kn_st * 2, 64, kKeys);
    if (st == TFB_OK) st = make_tmap_rows16(&maps[1], p.vn, D, hk, vs * 2, p.a.T, p.vn_st * 2, 64, kKeys);
    if (st != TFB_OK) return st;
  }
  TFB_CUDA(launch_pdl(kernel, dim3(f.blocks), dim3(kThreadsP), Smem<D>::kBytes, s, p, maps[0], maps[1], mapped));
  if (f.blocks > 1)
    TFB_CUDA(launch_pdl(join_many_kernel<T, D>, dim3(f.join_blocks), dim3(256), 0, s, p));
  return TFB_OK;
}
template <typename T>
tfb_status launch_many_t(AttnParams& p, const ManyPlan& f, int64_t dim, const DeviceInfo* di, cudaStream_t s) {
  if (dim == 128) return f.carry ? launch_many<T, 128, true>(p, f, di, s) : launch_many<T, 128, false>(p, f, di, s);
  return f.carry ? launch_many<T, 64, true>(p, f, di, s) : launch_many<T, 64, false>(p, f, di, s);
}

}  // namespace

int64_t attn_many_ws(int64_t dim, int64_t heads, int64_t B, int64_t max_keys, int64_t T, int64_t group) {
  const DeviceInfo* di;
  if (device_info(&di) != TFB_OK) return -1;
  return many_plan(dim, heads, B, max_keys, T, group, di->sm_count).ws;
}

tfb_status attn_many(AttnParams& p, int dtype, int64_t dim, const DeviceInfo* di, void* ws, int64_t ws_bytes, cudaStream_t s) {
  const ManyPlan f = many_plan(dim, p.a.heads, p.a.B, (int64_t)p.a.max_pages << p.a.page_shift, p.a.T, p.group,
                               di->sm_count);
  if (f.ws > 0 && (!ws || ws_bytes < f.ws || !aligned(ws, 16)))
    return fail(TFB_BAD_ARG, "kv4_attention: needs a 16-byte aligned workspace of %lld bytes", (long long)f.ws);
  p.items = f.blocks;
  p.min_tiles = f.min_tiles;
  p.part = static_cast<float*>(ws);
  p.carry = f.carry ? p.part + f.carry / 4 : nullptr;
  return dtype == TFB_DT_F16 ? launch_many_t<__half>(p, f, dim, di, s) : launch_many_t<__nv_bfloat16>(p, f, dim, di, s);
}

}  // namespace tfb

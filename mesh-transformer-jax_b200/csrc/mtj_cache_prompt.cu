// Attention of many new tokens over a paged cache (prompts and portions of prompts of mtj_k_cache_attn), on the tensor cores.
//
// A job is 256 query rows: two tiles of 128, two heads of one group at the same tokens, or where groups are odd 256 tokens of one
// head.  Keys come in blocks of 128 (two pages): first those of the first tokens, then those of the window; a block of keys serves
// both tiles, so K and V cross from L2 once for 256 rows.  With d_head 64 and 128 one block has both tiles.  With d_head 256 an
// accumulator fills tensor memory, and two blocks, a cluster of 2, have a tile each: their products are cta_group::2 ones, each holds
// one page of K and half the columns of V, so that an SM reads 32 bytes a cycle (with a tile of its own 64, which is more than L2
// gives 148 of them: 3900 cycles a block of keys instead of 2048 of products).  A unit of work is one tile (d_head 256: both) on one
// key block,
//     S[128, 128] = Q K^T        tcgen05, operands in shared memory by TMA (128-byte swizzle), fp32 in tensor memory
//     P = 2^(S c - m)            a thread a row (d_head 256: two threads a row, 64 keys each), written over S as bf16
//     O[128, d] += P V           P from tensor memory, V as MN-major operand straight from the pages
// and units go round two score buffers: one thread issues S0 S1 | PV0 S2 | PV1 S3 | ..., so that while one warp group works out the
// weights of a unit, the tensor cores have the other unit's products.  For d_head 128 a unit is 1024 cycles of products and, at 16
// exponentials a cycle less the quarter that the multiply-add units take, 768 of exponentials; the chain of a tile (scores, maximum,
// weights, products, next scores) is what is left in the open.  32 heads of 128, 8 key heads, 8191 tokens, window 4096: 0.40 ms, 1040
// TFLOP/s of visible pairs, 0.445 ms (925) in a row of calls, where the SMs run at 1.6 GHz; tensor pipe 54 % active.  16 heads of 256, 2047
// tokens, window 1024: 49 us, 41 %.  Built and measured at the first of these, none ahead by more than 2 %: score buffers of 64 keys, two a tile, so that
// no tile waits for its scores (386 us from a warp of products a tile, 528 from one for both); two threads a row for 128-wide heads (407);
// pairs of blocks for them (414); a warp of products a tile with buffers of 128 (460: the tiles' products get in each other's way).
//
// A job is a sequence, a head (pair) and the tokens of a block.  148 blocks, one an SM, take whole jobs, longest first, in turns that
// go forth and back; where that would leave SMs idle for longer than a join takes, the line of all jobs' key blocks is cut into equal
// pieces instead, and where jobs are few, every job into pieces of its own (at least kLeastBlocks).  cache_begin_kernel plans that; jobs in
// several pieces are joined by cache_part_kernel from their parts' (maximum, sum, weighted values).
//
// The new tokens' keys and values are read where the caller has them: key blocks are those of the cached slots, the last one filled up,
// then 128 new tokens each.  Where new tokens begin a page, the block that has 64 of them in shared memory as keys of their own job
// stores them from there, by TMA; a warp of every block, and whoever has run out of jobs, stores the others row by row.  (16 x 256, 2047
// tokens: storing in a kernel before took 16 us, row by row beside the products it was longer than they were.)
//
// Scores, maxima, sums and O are 32-bit; P is rounded to bf16, half a step on average as large as the rounding of the output (a second
// term would be half as many products again).  O is rescaled when a row's scores have outgrown its reference, which waits for the
// products before.  The rows of V behind the sequence, of a page that does not exist, or that no token of the job sees, are zeroed in
// shared memory before they meet their zero weights.
// Every wait is bounded; where one runs out, what is in flight has landed and ended before a block leaves.
#include <cuda.h>
#include <math.h>

#include <algorithm>

#include "mtj_cache_kernels.h"

namespace mtj {
namespace {

constexpr int kRowsT = 128;                // rows of a tile
constexpr int kKeysB = 128;                // keys of a block: two pages
constexpr int kSoftThreads = 256;
constexpr int kCopyThreads = 64;
constexpr int kPromptThreads = kSoftThreads + 64 + kCopyThreads;      // and the warps of TMA and of the products
constexpr int kBlockNotes = 8;
constexpr int kBlocks = 148;               // one on each of a B200's SMs
constexpr int kMostPieces = kBlocks;       // pieces: one a block, or one a pair of blocks
constexpr int kLeastBlocks = 4;            // of a piece that a job is cut into: the join costs about as much as three
constexpr int kMostEntries = 8192;         // (sequence, token range) pairs of a launch
constexpr int kJoinCost = 8;               // what cutting and joining costs, in key blocks of every piece
constexpr int kPlanHead = 8, kPlanList = kPlanHead + kMostPieces * 8;      // places in the plan
constexpr int kSizeBins = 1024;
constexpr int kPolyOf = 4;                 // of this many pairs of weights one is worked out on the multiply-add units
constexpr float kExp0 = 0.99992806f, kExp1 = 0.69326097f, kExp2 = 0.24261114f, kExp3 = 0.05517167f;

constexpr int kJobTiles = 2;
template <int DH>
struct PromptCfg {
  static constexpr bool kPair = DH == 256;
  static constexpr int kTiles = kPair ? 1 : kJobTiles;           // of a block
  static constexpr int kKeysThread = kTiles == 2 ? 128 : 64;
  static constexpr int kChunks = DH / 64;                        // 64-column parts of a row
  static constexpr int kHalves = kTiles;                         // in which a thread announces its weights
  static constexpr int kKPages = kPair ? 1 : 2;                  // of a block's keys that this block holds
  static constexpr int kVChunks = kPair ? kChunks / 2 : kChunks;
  static constexpr uint32_t kQBytes = kTiles * kRowsT * DH * 2;
  static constexpr uint32_t kKBytes = kKPages * kPageTokens * DH * 2;
  static constexpr uint32_t kVBytes = kKeysB * kVChunks * 128;
  static constexpr int kKSlots = DH == 64 ? 4 : 2, kVSlots = DH == 64 ? 4 : DH == 128 ? 2 : 3;
  static constexpr uint32_t kSmem = kQBytes + kKSlots * kKBytes + kVSlots * kVBytes;
  static constexpr uint32_t kColS = 0, kColO = 256;    // tensor memory: S0 | S1 | O
  static constexpr uint32_t kTmemCols = 512;
  static_assert(kSmem <= 224 * 1024, "shared memory");
};

__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, int c0, int c1, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The warp of the products runs as one, with the same values in all lanes, and one lane issues: descriptors then come from uniform
// registers.  (In a branch of one lane, every product cost 90 cycles of moves: 720 for the eight of P V whatever their size.)
__device__ __forceinline__ uint32_t elected() {
  uint32_t x;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(x));
  return x;
}
__device__ __forceinline__ void commit_to(uint32_t bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(bar), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
      : "memory");
}
// the forms of a pair of blocks: arrivals in both, products over both blocks' operands and accumulators
__device__ __forceinline__ void commit_pair(uint32_t bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}"
      ::"r"(bar), "h"(static_cast<uint16_t>(3)), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ss_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts_pair(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
      : "memory");
}
__device__ __forceinline__ uint32_t pair_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void pair_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// on the first block's barrier
__device__ __forceinline__ void arrive_first(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .b32 x;\n\tmapa.shared::cluster.u32 x, %0, 0;\n\t"
      "mbarrier.arrive.shared::cluster.b64 _, [x];\n\t}"
      ::"r"(bar)
      : "memory");
}
// 1 into a word of the other block of the pair
__device__ __forceinline__ void set_in_other(uint32_t word, uint32_t rank) {
  asm volatile(
      "{\n\t.reg .b32 x;\n\t"
      "mapa.shared::cluster.u32 x, %0, %1;\n\t"
      "st.shared::cluster.u32 [x], 1;\n\t}"
      ::"r"(word), "r"(rank ^ 1u)
      : "memory");
}
// shared-memory matrix descriptor, 128-byte swizzle; lbo / sbo in bytes
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFF) | static_cast<uint64_t>((lbo >> 4) & 0x3FFF) << 16 |
         static_cast<uint64_t>((sbo >> 4) & 0x3FFF) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}
__device__ __forceinline__ float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two numbers in a register pair
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) { return pair_of(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ void unpair(uint64_t d, float* lo, float* hi) {
  uint32_t x, y;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(x), "=r"(y) : "l"(d));
  *lo = __uint_as_float(x);
  *hi = __uint_as_float(y);
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// NaN if one of them is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^x of a pair on the multiply-add units, for x in [-126, 9]: x = n + f with |f| <= 1/2 by adding and taking away 1.5 * 2^23 (the
// reduction of Cody and Waite), a polynomial of degree 3 in f (fitted here to the relative error, 8e-5 at most: a twentieth of the rounding to bf16 that follows),
// n added to its exponent
__device__ __forceinline__ void exp2_pair(uint64_t x, float* y0, float* y1) {
  const uint64_t magic = pair_of(12582912.f, 12582912.f);
  const uint64_t n = add_pair(x, magic);
  const uint64_t f = add_pair(x, fma_pair(n, pair_of(-1.f, -1.f), magic));
  uint64_t p = fma_pair(pair_of(kExp3, kExp3), f, pair_of(kExp2, kExp2));
  p = fma_pair(p, f, pair_of(kExp1, kExp1));
  p = fma_pair(p, f, pair_of(kExp0, kExp0));
  float p0, p1, n0, n1;
  unpair(p, &p0, &p1);
  unpair(n, &n0, &n1);
  *y0 = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(n0) << 23));
  *y1 = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(n1) << 23));
}
// 32 bytes in one store: a thread's part of a row fills whole sectors
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
// bits 0 .. n - 1
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
// 32 columns of this warp's lanes, on their way until tmem_wait()
__device__ __forceinline__ void tmem_fetch32(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// nothing that uses r comes before this place
__device__ __forceinline__ void pin32(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

struct PromptArgs {
  mtj_cache_attn_args c;                   // pointers from the launch's first sequence on
  float scale_log2;
  int by_heads, span, pieces;              // a job's tiles are two heads; tokens of a job; pieces
  int head_jobs, token_jobs;               // jobs of a token range, token ranges of a sequence
  int* plan;                               // whole jobs or not, jobs | [pieces][8]: sequence, head job, token job, first key
                                           // block, key blocks | entries by size
  float2* part_ml;                         // [pieces][2][kJobTiles * 128]
  float* part_o;                           // [pieces][2][kJobTiles * 128][d_head]
};

// The key blocks of a job: those with first tokens, then those of the window.  Places of keys: cached slots, up to a multiple of
// kKeysB, then the call's tokens (where it brings their keys).
struct JobKeys {
  int t_first, t_end;                      // its tokens
  int fresh, first;                        // new tokens, slot of the first of them
  int cached, tail;                        // slots that are read from pages; the first place of the call's tokens
  int low, sinks;                          // slots from sinks on and below low are seen by none of its tokens
  int low_block, sink_blocks, blocks;
  __device__ __forceinline__ int place(int j) const { return (j < sink_blocks ? j : low_block + j - sink_blocks) * kKeysB; }
  __device__ __forceinline__ int slot_of(int place) const { return place < tail ? place : place - tail + cached; }
  __device__ __forceinline__ int place_of(int slot) const { return slot < cached ? slot : slot - cached + tail; }
};
__device__ __forceinline__ JobKeys job_keys(const PromptArgs& a, const CacheSeq& s, int token_job) {
  JobKeys k;
  k.fresh = s.fresh;
  k.first = s.length - s.fresh;
  k.cached = a.c.k_new_dev ? k.first : s.length;
  k.tail = (k.cached + kKeysB - 1) / kKeysB * kKeysB;
  k.t_first = token_job * a.span;
  k.t_end = min(s.fresh, k.t_first + a.span);
  k.low = cache_window_low(k.first + k.t_first, a.c.window);
  k.sinks = min(a.c.sinks, k.low);
  k.low_block = k.place_of(k.low) / kKeysB;
  k.sink_blocks = k.sinks > 0 ? min(k.place_of(k.sinks - 1) / kKeysB + 1, k.low_block) : 0;
  k.blocks = k.t_end > k.t_first ? k.sink_blocks + k.place_of(k.first + k.t_end - 1) / kKeysB - k.low_block + 1 : 0;
  return k;
}
__device__ __forceinline__ CacheSeq prompt_seq(const PromptArgs& a, int b) {
  return cache_seq(a.c.lengths_dev, a.c.new_tokens_dev, b, a.c.tokens, a.c.pages);
}

// Block 0 plans; the others put zeros into the rows of the output that no token has, a warp a row.
constexpr int kBeginThreads = 256, kZeroRows = 64;
__device__ __forceinline__ int begin_scan(int v, int* sums, int* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  int before = x - v, total = 0;
  for (int w = 0; w < kBeginThreads / 32; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  *all = total;
  return before;
}
__global__ void __launch_bounds__(kBeginThreads) cache_begin_kernel(const PromptArgs a) {
  pdl_launch_dependents();
  const mtj_cache_attn_args& c = a.c;
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    const int64_t rows = static_cast<int64_t>(c.batch) * c.tokens, r0 = static_cast<int64_t>(blockIdx.x - 1) * kZeroRows;
    for (int64_t row = r0 + (tid >> 5); row < min(rows, r0 + kZeroRows); row += kBeginThreads / 32) {
      const int b = static_cast<int>(row / c.tokens), t = static_cast<int>(row - static_cast<int64_t>(b) * c.tokens);
      if (t < prompt_seq(a, b).fresh) continue;
      uint4* out = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(c.out_dev) + row * c.ld_out);
      for (int v = tid & 31; v < c.heads * (c.d_head / 8); v += 32) out[v] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  // before[e]: key blocks, later pieces, of a head job before entry e = (sequence, token job)
  __shared__ int before[kMostEntries + 1], sums[kBeginThreads / 32], bins[kSizeBins], s_most;
  const int entries = c.batch * a.token_jobs, per = (entries + kBeginThreads - 1) / kBeginThreads;
  const int e0 = min(entries, tid * per), e1 = min(entries, e0 + per);
  int mine = 0, jobs = 0, most = 0, total, all_jobs;
  if (tid == 0) s_most = 0;
  for (int e = e0; e < e1; ++e) {
    const int b = e / a.token_jobs;
    const CacheSeq s = prompt_seq(a, b);
    if (s.bad && e == b * a.token_jobs && c.status_dev) atomicOr(c.status_dev, kDevErrBadIndex);
    const int n = job_keys(a, s, e - b * a.token_jobs).blocks;
    before[e] = n;
    mine += n;
    jobs += n > 0;
    most = max(most, n);
  }
  int x = begin_scan(mine, sums, &total);
  begin_scan(jobs, sums, &all_jobs);
  atomicMax(&s_most, most);
  __syncthreads();
  most = s_most;
  const int64_t line = static_cast<int64_t>(total) * a.head_jobs;
  const int64_t job_count = static_cast<int64_t>(all_jobs) * a.head_jobs;
  const int64_t turns = (job_count + a.pieces - 1) / a.pieces;
  const bool whole = job_count == 0 || max(static_cast<int64_t>(most), turns * line / job_count) <= line / a.pieces + kJoinCost;
  const bool cut_jobs = !whole && job_count <= a.pieces / 2;
  if (tid == 0) {
    a.plan[0] = whole ? 1 : 0;
    a.plan[1] = static_cast<int>(job_count);
  }
  if (whole) {
    // entries by size, the largest first; the order among equals is of no consequence
    for (int i = tid; i < kSizeBins; i += kBeginThreads) bins[i] = 0;
    __syncthreads();
    for (int e = e0; e < e1; ++e)
      if (before[e] > 0) atomicAdd(&bins[kSizeBins - min(before[e], kSizeBins)], 1);
    __syncthreads();
    constexpr int kBinsEach = kSizeBins / kBeginThreads;
    int n = 0, counts[kBinsEach];
#pragma unroll
    for (int i = 0; i < kBinsEach; ++i) n += counts[i] = bins[tid * kBinsEach + i];
    x = begin_scan(n, sums, &total);
#pragma unroll
    for (int i = 0; i < kBinsEach; ++i) {
      bins[tid * kBinsEach + i] = x;
      x += counts[i];
    }
    __syncthreads();
    for (int e = e0; e < e1; ++e)
      if (before[e] > 0) a.plan[kPlanList + atomicAdd(&bins[kSizeBins - min(before[e], kSizeBins)], 1)] = e;
    if (tid < a.pieces) a.plan[kPlanHead + tid * 8 + 4] = 0;
    return;
  }
  // with pieces this wide they are at most a.pieces
  const int width = cut_jobs ? max(kLeastBlocks, static_cast<int>((line + a.pieces - job_count - 1) / (a.pieces - job_count))) : 0;
  if (cut_jobs) {
    mine = 0;
    for (int e = e0; e < e1; ++e) mine += before[e] = (before[e] + width - 1) / width;
    x = begin_scan(mine, sums, &total);
  }
  for (int e = e0; e < e1; ++e) {
    const int n = before[e];
    before[e] = x;
    x += n;
  }
  if (tid == 0) before[entries] = total;
  __syncthreads();
  const int64_t pieces_line = cut_jobs ? static_cast<int64_t>(total) * a.head_jobs : line;
  if (tid < a.pieces) {
    const int64_t used = min(pieces_line, static_cast<int64_t>(a.pieces));      // no piece before the last one is empty
    const int64_t at = cut_jobs || tid >= used ? tid : line * tid / used;
    int n = tid >= used ? 0 : cut_jobs ? 1 : static_cast<int>(line * (tid + 1) / used - at);
    int b = 0, head_job = 0, token_job = 0, j = 0;
    if (n > 0) {
      int lo = 0, hi = c.batch - 1;                      // the last sequence that begins at or before this place
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (static_cast<int64_t>(before[mid * a.token_jobs]) * a.head_jobs <= at) lo = mid;
        else hi = mid - 1;
      }
      b = lo;
      const int base = before[b * a.token_jobs], of_head = before[(b + 1) * a.token_jobs] - base;
      const int64_t rest = at - static_cast<int64_t>(base) * a.head_jobs;
      head_job = static_cast<int>(rest / of_head);
      const int within = static_cast<int>(rest - static_cast<int64_t>(head_job) * of_head);
      lo = 0;
      hi = a.token_jobs - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (before[b * a.token_jobs + mid] - base <= within) lo = mid;
        else hi = mid - 1;
      }
      token_job = lo;
      j = within - (before[b * a.token_jobs + token_job] - base);
      if (cut_jobs) {
        const int blocks = job_keys(a, prompt_seq(a, b), token_job).blocks, parts = (blocks + width - 1) / width, k = j;
        j = blocks * k / parts;
        n = blocks * (k + 1) / parts - j;
      }
    }
    int* p = a.plan + kPlanHead + tid * 8;
    p[0] = b;
    p[1] = head_job;
    p[2] = token_job;
    p[3] = j;
    p[4] = n;
  }
}

// A block's (or pair's) way through its jobs; every role goes it on its own.
struct Walk {
  int b, head_job, token_job, j, left, turn, jobs, piece;
  JobKeys k;
  int n;                                   // key blocks of the current job that belong to the block
  __device__ __forceinline__ bool begin(const PromptArgs& a, int which) {
    piece = which;
    turn = a.plan[0] ? 0 : -1;
    jobs = a.plan[1];
    if (turn >= 0) return take(a);
    const int* p = a.plan + kPlanHead + piece * 8;
    b = p[0];
    head_job = p[1];
    token_job = p[2];
    j = p[3];
    left = p[4];
    if (left > 0) enter(a);
    return left > 0;
  }
  // whole jobs: turn by turn, every other turn from the last block to the first
  __device__ __forceinline__ bool take(const PromptArgs& a) {
    const int64_t at = static_cast<int64_t>(turn) * a.pieces + (turn & 1 ? a.pieces - 1 - piece : piece);
    if (at >= jobs) return false;
    const int e = a.plan[kPlanList + at / a.head_jobs];
    b = e / a.token_jobs;
    token_job = e - b * a.token_jobs;
    head_job = static_cast<int>(at % a.head_jobs);
    j = 0;
    left = 0x7fffffff;
    enter(a);
    return true;
  }
  __device__ __forceinline__ void enter(const PromptArgs& a) {
    k = job_keys(a, prompt_seq(a, b), token_job);
    n = min(left, k.blocks - j);
  }
  __device__ __forceinline__ bool next(const PromptArgs& a) {
    if (turn >= 0) {
      ++turn;
      return take(a);
    }
    left -= n;
    if (left <= 0) return false;
    j = 0;
    ++token_job;
    for (;;) {
      if (token_job < a.token_jobs) {
        enter(a);
        if (k.blocks > 0) return true;
      }
      token_job = 0;                       // a sequence's token jobs without tokens are its last ones
      if (++head_job == a.head_jobs) {
        head_job = 0;
        if (++b >= a.c.batch) return false;      // cannot happen: the pieces end with the line
      }
      enter(a);
      if (k.blocks > 0) return true;
    }
  }
  __device__ __forceinline__ bool whole() const { return j == 0 && n == k.blocks; }
};

// Whether the 64 new tokens from t on fill a page of their own and are stored from shared memory.
__device__ __forceinline__ bool stored_by_page(const JobKeys& k, int t) {
  return k.first % kPageTokens == 0 && t / kPageTokens * kPageTokens + kPageTokens <= k.fresh;
}

// The other new rows into their slots, a warp a row, dealt out to all warps but those of TMA and products: the two that do nothing else
// begin at once, the softmax warps when they have run out of jobs.
constexpr int kStoreWarps = (kPromptThreads - 64) / 32;
template <int DH>
__device__ __forceinline__ void store_rows(const PromptArgs& a, int worker) {
  const int lane = threadIdx.x & 31;
  const int vecs = a.c.kv_heads * (DH / 8), stride = a.c.kv_heads * kPageTokens * (DH / 8);
  const int rows = a.c.batch * a.c.tokens;
  for (int row = blockIdx.x * kStoreWarps + worker; row < rows; row += kBlocks * kStoreWarps) {
    const int b = row / a.c.tokens, t = row - b * a.c.tokens;
    const CacheSeq s = prompt_seq(a, b);
    JobKeys k;
    k.fresh = s.fresh;
    k.first = s.length - s.fresh;
    if (t >= s.fresh || stored_by_page(k, t)) continue;
    const int slot = k.first + t, page = a.c.page_table_dev[static_cast<size_t>(b) * a.c.pages + slot / kPageTokens];
    if (!cache_page_ok(page, a.c.n_pages)) {
      if (lane == 0 && a.c.status_dev) atomicOr(a.c.status_dev, kDevErrBadIndex);
      continue;
    }
    const __nv_bfloat16* kn = static_cast<const __nv_bfloat16*>(a.c.k_new_dev) + static_cast<size_t>(row) * a.c.ld_k;
    const __nv_bfloat16* vn = static_cast<const __nv_bfloat16*>(a.c.v_new_dev) + static_cast<size_t>(row) * a.c.ld_v;
    const size_t at = static_cast<size_t>(page) * stride + slot % kPageTokens * (DH / 8);
    constexpr int kFlight = 4;
    for (int i = lane; i < vecs; i += 32 * kFlight) {
      uint4 xk[kFlight], xv[kFlight];
#pragma unroll
      for (int f = 0; f < kFlight; ++f)
        if (i + 32 * f < vecs) {
          xk[f] = load8_bf16(kn + (i + 32 * f) * 8);
          xv[f] = load8_bf16(vn + (i + 32 * f) * 8);
        }
#pragma unroll
      for (int f = 0; f < kFlight; ++f)
        if (i + 32 * f < vecs) {
          const int e = i + 32 * f;
          const size_t to = at + static_cast<size_t>(e / (DH / 8)) * (kPageTokens * (DH / 8)) + e % (DH / 8);
          static_cast<uint4*>(a.c.kpool_dev)[to] = xk[f];
          static_cast<uint4*>(a.c.vpool_dev)[to] = xv[f];
        }
    }
  }
}

template <int DH>
__global__ void __launch_bounds__(kPromptThreads, 1) cache_prompt_kernel(const __grid_constant__ CUtensorMap map_q,
                                                                      const __grid_constant__ CUtensorMap map_k,
                                                                      const __grid_constant__ CUtensorMap map_v,
                                                                      const __grid_constant__ CUtensorMap map_k_new,
                                                                      const __grid_constant__ CUtensorMap map_v_new, const PromptArgs a) {
  using C = PromptCfg<DH>;
  constexpr int kTiles = C::kTiles, kKeysThread = C::kKeysThread, kHalves = C::kHalves;
  constexpr bool kPair = C::kPair;
  constexpr int kBars = 2 + 2 * C::kKSlots + 2 * C::kVSlots + 11, kPeerBars = kPair ? 1 + C::kKSlots + C::kVSlots : 0;
  extern __shared__ __align__(1024) unsigned char prompt_smem[];
  __shared__ __align__(8) uint64_t bars[kBars + kPeerBars];
  __shared__ uint32_t tmem_slot, failed;
  __shared__ int to_store[C::kKSlots + C::kVSlots][2];      // rows of the pools that a slot's pages of new rows go to
  __shared__ int notes[kBlockNotes];                   // valid rows of a key block's pages: first | second << 8
  __shared__ float part_max[2][kRowsT];                // d_head 256: of the two threads of a row
  const uint32_t base = smem_u32(prompt_smem);
  const uint32_t sQ = base, sK = base + C::kQBytes, sV = sK + C::kKSlots * C::kKBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t q_full = bar0, q_empty = bar0 + 8, k_full = bar0 + 16, k_empty = k_full + 8 * C::kKSlots, v_full = k_empty + 8 * C::kKSlots,
                 v_empty = v_full + 8 * C::kVSlots, s_full = v_empty + 8 * C::kVSlots, p_full = s_full + 16, p_half = p_full + 16,
                 o_done = p_half + 16, o_free = o_done + 16, settled = o_free + 16;
  // the first block of a pair: the other one has its part
  const uint32_t q_peer = bar0 + 8 * kBars, k_peer = q_peer + 8, v_peer = k_peer + 8 * C::kKSlots;
  const uint32_t rank = kPair ? pair_rank() : 0;
  const int piece = kPair ? blockIdx.x >> 1 : blockIdx.x;
  auto give_up = [&]() {                               // a wait of this thread ran out: known to the block, or both of the pair
    atomicOr(&failed, 1u);
    if constexpr (kPair) set_in_other(smem_u32(&failed), rank);
  };
  if (threadIdx.x == 0) {
    for (int i = 0; i < kBars + kPeerBars; ++i) mbar_init(bar0 + 8u * i, 1);
    for (int i = 0; i < 2; ++i) {
      constexpr int kArrivals = (kPair ? 2 : 1) * kSoftThreads / 32 / kTiles;      // a warp each, of a pair both blocks'
      mbar_init(p_full + 8u * i, kArrivals);
      mbar_init(p_half + 8u * i, kArrivals);
      mbar_init(o_free + 8u * i, kArrivals);
    }
    mbar_fence_init();
    failed = 0;
  }
  if (warp == 9) {
    if constexpr (kPair) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(C::kTmemCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(C::kTmemCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  fence_before();
  if constexpr (kPair) pair_sync();                    // both blocks' barriers exist before either is signalled
  else __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_wait();
  pdl_launch_dependents();                             // behind the allocation of tensor memory
  const int group = a.c.heads / a.c.kv_heads;

  if (warp >= 8) {
    // registers: 8 warps of 200 and 4 of 88 are 62464 of the 64512 that the block is launched with
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    Walk w;
    const bool work = w.begin(a, piece);
    if (warp == 8) {
      // ---- TMA ----
      if (lane == 0 && work) {
        int kc = 0, vc = 0, seg = 0;                         // key blocks, value slots and jobs so far, as they have been asked for
        constexpr int kKChunk = C::kKPages * kPageTokens * 128;      // bytes of 64 columns of a slot of keys
        const int v_chunk0 = kPair ? rank * C::kVChunks : 0;
        uint32_t storing_k = 0, storing_v = 0;               // slots with rows to store
        bool ok = true;
        // a slot's new rows go to their pages when the products have read it, before it is filled again
        auto store_k = [&](int st) {
          const int* rows = to_store[st];
          storing_k &= ~(1u << st);
#pragma unroll
          for (int h = 0; h < C::kKPages; ++h)
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c)
              if (rows[h] >= 0) tma_store(&map_k, c * 64, rows[h], sK + st * C::kKBytes + c * kKChunk + h * (kPageTokens * 128));
          asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
        };
        auto store_v = [&](int st) {
          const int* rows = to_store[C::kKSlots + st];
          storing_v &= ~(1u << st);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < C::kVChunks; ++c)
              if (rows[h] >= 0)
                tma_store(&map_v, (v_chunk0 + c) * 64, rows[h], sV + st * C::kVBytes + c * (kKeysB * 128) + h * (kPageTokens * 128));
          asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
        };
        do {
          const int head0 = w.head_job * (a.by_heads ? 2 : 1), kvh = head0 / group;
          if (seg > 0) ok = mbar_wait(q_empty, (seg - 1) & 1);
          if (!ok) break;
          mbar_expect_tx(q_full, C::kQBytes);
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c)
              tma_box(sQ + (t * C::kChunks + c) * (kRowsT * 128), &map_q, (head0 + (a.by_heads ? t + rank : 0)) * DH + c * 64,
                      w.b * a.c.tokens + w.k.t_first + (a.by_heads ? 0 : (t + rank) * kRowsT), q_full);
          ++seg;
          const int32_t* table = a.c.page_table_dev + static_cast<size_t>(w.b) * a.c.pages;
          // a key block's pages, or its rows of new tokens: the row where each 64 begin, how many hold something, the page they are stored
          // to; looked up before the slot is waited for, because the products wait for what comes behind that
          struct Block {
            int row[2], valid[2], target[2];
            bool cached;
          };
          auto look_up = [&](int j) {
            Block x;
            const int place = w.k.place(w.j + j);
            x.cached = place < w.k.tail;
            // a key head's new rows are stored by the job that has these tokens and the group's first head
            const bool mine = !x.cached && place - w.k.tail >= w.k.t_first && place - w.k.tail < w.k.t_end && head0 % group == 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              x.target[h] = -1;
              if (!x.cached) {
                const int t = place - w.k.tail + h * kPageTokens;
                x.valid[h] = min(kPageTokens, max(0, w.k.fresh - t));
                x.row[h] = w.b * a.c.tokens + t;
                if (mine && x.valid[h] > 0 && stored_by_page(w.k, t)) {
                  const int page = table[(w.k.first + t) / kPageTokens];
                  if (cache_page_ok(page, a.c.n_pages)) x.target[h] = (page * a.c.kv_heads + kvh) * kPageTokens;
                  else if (a.c.status_dev) atomicOr(a.c.status_dev, kDevErrBadIndex);
                }
                continue;
              }
              const int at = place / kPageTokens + h;
              const bool seen = at * kPageTokens < w.k.sinks || (at + 1) * kPageTokens > w.k.low;
              x.valid[h] = seen ? min(kPageTokens, max(0, w.k.cached - at * kPageTokens)) : 0;
              int page = x.valid[h] > 0 ? table[at] : 0;
              if (!cache_page_ok(page, a.c.n_pages)) {
                // not read: page 0 stands in, nobody sees its scores
                x.valid[h] = page = 0;
                if (a.c.status_dev) atomicOr(a.c.status_dev, kDevErrBadIndex);
              }
              x.row[h] = (page * a.c.kv_heads + kvh) * kPageTokens;
            }
            return x;
          };
          auto load_k = [&](const Block& x) {
            const int st = kc % C::kKSlots;
            const CUtensorMap* map = x.cached ? &map_k : &map_k_new;
            const int col = x.cached ? 0 : kvh * DH;
            if (kc >= C::kKSlots && !mbar_wait(k_empty + 8 * st, (kc / C::kKSlots - 1) & 1)) return false;
            if (storing_k >> st & 1u) store_k(st);
            mbar_expect_tx(k_full + 8 * st, C::kKBytes);
#pragma unroll
            for (int h = 0; h < C::kKPages; ++h)
#pragma unroll
              for (int c = 0; c < C::kChunks; ++c)
                tma_box(sK + st * C::kKBytes + c * kKChunk + h * (kPageTokens * 128), map, col + c * 64, kPair && rank ? x.row[1] : x.row[h],
                        k_full + 8 * st);
            const int t0 = kPair && rank ? x.target[1] : x.target[0], t1 = kPair ? -1 : x.target[1];
            if (t0 >= 0 || t1 >= 0) {
              storing_k |= 1u << st;
              to_store[st][0] = t0;
              to_store[st][1] = t1;
            }
            ++kc;
            return true;
          };
          auto load_v = [&](const Block& x) {
            const CUtensorMap* map = x.cached ? &map_v : &map_v_new;
            const int col = x.cached ? 0 : kvh * DH;
            const int st = vc % C::kVSlots;
            if (vc >= C::kVSlots && !mbar_wait(v_empty + 8 * st, (vc / C::kVSlots - 1) & 1)) return false;
            if (storing_v >> st & 1u) store_v(st);
            mbar_expect_tx(v_full + 8 * st, C::kVBytes);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int c = 0; c < C::kVChunks; ++c)
                tma_box(sV + st * C::kVBytes + c * (kKeysB * 128) + h * (kPageTokens * 128), map, col + (v_chunk0 + c) * 64, x.row[h],
                        v_full + 8 * st);
            if (x.target[0] >= 0 || x.target[1] >= 0) {
              storing_v |= 1u << st;
              to_store[C::kKSlots + st][0] = x.target[0];
              to_store[C::kKSlots + st][1] = x.target[1];
            }
            ++vc;
            return true;
          };
          // in the order in which the products want them: S0 (S1) | PV0 S2 | PV1 S3 ...; the softmax warps' note of a block is written
          // before the arrival that its products wait for
          Block now = look_up(0), then;
          notes[kc % kBlockNotes] = now.valid[0] | now.valid[1] << 8;
          ok = load_k(now);
          for (int j = 0; ok && j < w.n; ++j) {
            if (j + 1 < w.n) {
              then = look_up(j + 1);
              notes[kc % kBlockNotes] = then.valid[0] | then.valid[1] << 8;
              ok = load_k(then);
            }
            if (ok) ok = load_v(now);
            now = then;
          }
        } while (ok && w.next(a));
        // what the last round of slots holds
        for (int n = max(0, kc - C::kKSlots); ok && n < kc; ++n) {
          ok = mbar_wait(k_empty + 8 * (n % C::kKSlots), (n / C::kKSlots) & 1);
          if (ok && (storing_k >> (n % C::kKSlots) & 1u)) store_k(n % C::kKSlots);
        }
        for (int n = max(0, vc - C::kVSlots); ok && n < vc; ++n) {
          ok = mbar_wait(v_empty + 8 * (n % C::kVSlots), (n / C::kVSlots) & 1);
          if (ok && (storing_v >> (n % C::kVSlots) & 1u)) store_v(n % C::kVSlots);
        }
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        if (!ok) {
          // what was asked for lands before the block leaves
          for (int n = max(0, kc - C::kKSlots); n < kc; ++n) mbar_settle(k_full + 8 * (n % C::kKSlots), (n / C::kKSlots) & 1);
          for (int n = max(0, vc - C::kVSlots); n < vc; ++n) mbar_settle(v_full + 8 * (n % C::kVSlots), (n / C::kVSlots) & 1);
          if (seg > 0) mbar_settle(q_full, (seg - 1) & 1);
          give_up();
        }
      }
    } else if (warp == 9) {
      // ---- products ----
      if (kPair && rank != 0) {
        // the second block of a pair tells the first what has landed, in the order in which the products want it
        if (lane == 0 && work) {
          int kc = 0, vc = 0, seg = 0;
          bool ok = true;
          auto tell = [&](uint32_t full, uint32_t peer, int n, int slots) {
            ok = ok && mbar_wait(full + 8 * (n % slots), (n / slots) & 1);
            if (ok) arrive_first(peer + 8 * (n % slots));
          };
          do {
            tell(q_full, q_peer, seg++, 1);
            tell(k_full, k_peer, kc++, C::kKSlots);
            for (int j = 0; ok && j < w.n; ++j) {
              if (j + 1 < w.n) tell(k_full, k_peer, kc++, C::kKSlots);
              tell(v_full, v_peer, vc++, C::kVSlots);
            }
          } while (ok && w.next(a));
          if (!ok) give_up();
        }
      } else if (work) {
        const uint32_t leader = elected();
        auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0; };
        auto commit = [&](uint32_t bar) {
          if constexpr (kPair) commit_pair(bar, leader);
          else commit_to(bar, leader);
        };
        constexpr uint32_t kM = kPair ? 2 * kRowsT : kRowsT;
        constexpr uint32_t kIdS = (1u << 4) | (1u << 7) | (1u << 10) | ((kKeysB >> 3) << 17) | ((kM >> 4) << 24);
        constexpr uint32_t kIdO = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((DH >> 3) << 17) | ((kM >> 4) << 24);
        int k0 = 0, u0 = 0, seg = 0;                         // key blocks, units and jobs before the current job
        bool ok = true;
        do {
          // the same in all lanes, and known to be: what hangs on it stays in uniform registers
          const int blocks = __reduce_max_sync(0xffffffffu, w.n), units = blocks * kTiles;
          auto keys_there = [&](int u) {
            const int j = k0 + u / kTiles, st = j % C::kKSlots;
            const uint32_t parity = (j / C::kKSlots) & 1;
            return (u % kTiles != 0 || wait(k_full + 8 * st, parity)) && (!kPair || wait(k_peer + 8 * st, parity));
          };
          auto issue_s = [&](int u) {
            const int j = k0 + u / kTiles, t = u % kTiles, st = j % C::kKSlots, buf = (u0 + u) & 1;
            fence_after();
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c) {
              const uint64_t qd = smem_desc(sQ + (t * C::kChunks + c) * (kRowsT * 128), 16, 1024);
              const uint64_t kd = smem_desc(sK + st * C::kKBytes + c * (C::kKPages * kPageTokens * 128), 16, 1024);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if constexpr (kPair) mma_ss_pair(tmem + C::kColS + buf * kKeysB, qd + 2 * k, kd + 2 * k, kIdS, (c | k) ? 1u : 0u, leader);
                else mma_ss(tmem + C::kColS + buf * kKeysB, qd + 2 * k, kd + 2 * k, kIdS, (c | k) ? 1u : 0u, leader);
              }
            }
            commit(s_full + 8 * buf);
            if (t == kTiles - 1) commit(k_empty + 8 * st);
            if (u == units - 1) commit(q_empty);
          };
          auto issue_pv = [&](int u) {
            const int j = u / kTiles, t = u % kTiles, buf = (u0 + u) & 1, n = k0 + j, st = n % C::kVSlots;
            const uint32_t parity = ((u0 + u) >> 1) & 1, landed = (n / C::kVSlots) & 1;
            // the accumulator's last job has been read
            if (seg > 0 && u < kTiles && !wait(o_free + 8 * t, (seg - 1) & 1)) return false;
            // a wait costs 60 ns even where there is nothing to wait for: those that are likely over come before those for the weights,
            // the next unit's keys among them
            if (t == 0 && !wait(v_full + 8 * st, landed)) return false;
            if (kPair && !wait(v_peer + 8 * st, landed)) return false;
            const bool more = u + 2 < units;
            if (C::kHalves == 1 && more && !keys_there(u + 2)) return false;
            if (!wait((C::kHalves == 2 ? p_half : p_full) + 8 * buf, parity)) return false;
            const uint64_t vd = smem_desc(sV + st * C::kVBytes, kKeysB * 128, 1024);
            const uint32_t pa = tmem + C::kColS + buf * kKeysB;
#pragma unroll
            for (int h = 0; h < 2; ++h) {                    // by the page: the second half of the weights comes later
              if (C::kHalves == 2 && h == 1) {
                if (more && !keys_there(u + 2)) return false;
                if (!wait(p_full + 8 * buf, parity)) return false;
              }
              fence_after();
#pragma unroll
              for (int k = 4 * h; k < 4 * h + 4; ++k) {
                const uint64_t rows16 = vd + static_cast<uint64_t>((k * 2048) >> 4);
                if constexpr (kPair) mma_ts_pair(tmem + C::kColO, pa + 8 * k, rows16, kIdO, (j | k) ? 1u : 0u, leader);
                else mma_ts(tmem + C::kColO + t * DH, pa + 8 * k, rows16, kIdO, (j | k) ? 1u : 0u, leader);
              }
            }
            if (t == kTiles - 1) commit(v_empty + 8 * st);
            commit(o_done + 8 * buf);
            if (more) issue_s(u + 2);
            return true;
          };
          ok = wait(q_full, seg & 1) && (!kPair || wait(q_peer, seg & 1));
          for (int u = 0; ok && u < min(units, 2); ++u) {
            ok = keys_there(u);
            if (ok) issue_s(u);
          }
          for (int u = 0; ok && u < units; ++u) ok = issue_pv(u);
          k0 += blocks;
          u0 += units;
          ++seg;
        } while (__any_sync(0xffffffffu, ok && w.next(a)));
        if (!ok && leader) give_up();
      }
    } else if (warp >= 10) {
      // ---- the new rows into their slots ----
      if (a.c.k_new_dev) store_rows<DH>(a, warp - 10);
    }
  } else {
    // ---- weights ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    Walk w;
    if (w.begin(a, piece)) {
      const int wg = warp >> 2, quad = warp & 3;
      const int tile = kTiles == 2 ? wg : 0, part = kTiles == 2 ? 0 : wg;      // of this block; of the keys of a block
      const int job_tile = kPair ? rank : tile;
      auto announce = [&](uint32_t bar) {
        fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (kPair) arrive_first(bar);
          else arrive_at(bar);
        }
      };
      const int r = quad * 32 + lane;                        // row of the tile = lane of tensor memory
      const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
      int block = 0;                                         // key blocks so far
      bool ok = true;
      do {
        const int head = w.head_job * (a.by_heads ? 2 : 1) + (a.by_heads ? job_tile : 0);
        const int t0 = w.k.t_first + (a.by_heads ? 0 : job_tile * kRowsT), t = t0 + r;
        const int p = t < w.k.fresh ? w.k.first + t : -1;
        const int p_last = w.k.first + w.k.t_end - 1;
        const int warp_first = w.k.first + t0 + quad * 32;   // slots of the warp's rows: warp_first .. + 31
        float m_ref = -INFINITY, l = 0.f;
        for (int j = 0; j < w.n; ++j, ++block) {
          const int u = kTiles == 2 ? 2 * block + wg : block;
          // slots of the block's and of this thread's first key
          const int slot0 = w.k.slot_of(w.k.place(w.j + j)), key = slot0 + part * kKeysThread;
          const int warp_last = min(warp_first + 31, p_last);
          const bool inside = key + kKeysThread - 1 <= warp_first && warp_last >= warp_first &&
                              (key + kKeysThread - 1 < a.c.sinks || warp_last - key < a.c.window);
          const bool unseen = slot0 < w.k.low && slot0 + kKeysB > w.k.sinks;         // some of them, by all tokens
          if (ok) ok = mbar_wait(s_full + 8 * (u & 1), (u >> 1) & 1);
          fence_after();
          const int note = notes[block % kBlockNotes];
          const uint32_t at_s = tmem + lanes + C::kColS + (u & 1) * kKeysB + part * kKeysThread;
          uint32_t x[kKeysThread];
#pragma unroll
          for (int i = 0; i < kKeysThread; i += 32) tmem_fetch32(at_s + i, x + i);
          tmem_wait();
#pragma unroll
          for (int i = 0; i < kKeysThread; i += 32) pin32(x + i);
          constexpr int kFullNote = kPageTokens | kPageTokens << 8;
          // V's rows that hold nothing, or nothing that a token of the job sees: zeroed before anybody's weights are announced
          if (note != kFullNote || unseen) {
            const int st = block % C::kVSlots;
            if (ok) ok = mbar_wait(v_full + 8 * st, (block / C::kVSlots) & 1);
            if (tile == 0) {
              // [64-column part][page][64 rows][128 bytes]: a thread has a row of some parts, its pieces in an order that meets all banks
              const int h = r / kPageTokens, row = r % kPageTokens, slot = slot0 + r;
              if (row >= ((note >> (8 * h)) & 255) || (slot >= w.k.sinks && slot < w.k.low)) {
                unsigned char* at = prompt_smem + (sV - base) + st * C::kVBytes + r * 128;
                for (int c = kTiles == 1 ? wg : 0; c < C::kVChunks; c += 3 - kTiles)
#pragma unroll
                  for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(at + c * (kKeysB * 128) + ((i + lane) & 7) * 16) = make_uint4(0, 0, 0, 0);
              }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
          if (note != kFullNote || !inside) {
            // the row's visible keys as bits: up to its own slot, in the window or among the first tokens, in a page that holds something
            const int hi = p - key, lo = p - a.c.window + 1 - key, sk = a.c.sinks - key;
#pragma unroll
            for (int i = 0; i < kKeysThread / 32; ++i) {
              const int within = part * kKeysThread + 32 * i;
              const int held = (within < kPageTokens ? note & 255 : note >> 8) - within % kPageTokens;
              const uint32_t see = low_bits(min(hi + 1, held + 32 * i) - 32 * i) & (~low_bits(lo - 32 * i) | low_bits(sk - 32 * i));
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(see >> e & 1u)) x[32 * i + e] = 0xff800000u;
            }
          }
          float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < kKeysThread; i += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) tops[e] = max3(tops[e], __uint_as_float(x[i + 2 * e]), __uint_as_float(x[i + 2 * e + 1]));
          float top = max3(max3(tops[0], tops[1], tops[2]), tops[3], tops[3]) * a.scale_log2;      // scale > 0
          if constexpr (kTiles == 1) {
            part_max[part][r] = top;
            asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory");
            top = max3(top, part_max[part ^ 1][r], top);
            asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory");
          }
          // the reference stays until a score is 2^8 above it, and is then put 2^8 above that score: weights are below 2^8, and a row whose
          // first keys are poor ones (a few first tokens, the edge of its window) does not have O rescaled for its next ones
          float m_new = m_ref;
          if (!(top <= m_ref + 8.0f)) m_new = top + 8.0f;     // a score that is NaN makes the row NaN: the reference, and with it the sum
          if (__any_sync(0xffffffffu, m_new != m_ref && m_ref != -INFINITY)) {
            const float corr = m_new == m_ref || m_ref == -INFINITY ? 1.0f : exp2_ftz(m_ref - m_new);
            l *= corr;
            // O changes scale: the tile's products so far must have landed
            const int before = u - kTiles;
            if (ok) ok = mbar_wait(o_done + 8 * (before & 1), (before >> 1) & 1);
            fence_after();
#pragma unroll 1
            for (int c0 = 0; c0 < DH / (3 - kTiles); c0 += 16) {
              const uint32_t at = tmem + lanes + C::kColO + tile * DH + part * (DH / 2) + c0;
              uint32_t o[16];
              tmem_load16(at, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
              tmem_store16(at, o);
            }
          }
          const float neg = m_new == -INFINITY ? 0.f : -m_new;
          const uint64_t scale2 = pair_of(a.scale_log2, a.scale_log2), neg2 = pair_of(neg, neg);
          const uint32_t at_p = tmem + lanes + C::kColS + (u & 1) * kKeysB + part * (kKeysThread / 2);
          uint64_t sums[2] = {0, 0};
#pragma unroll
          for (int half = 0; half < kHalves; ++half) {
#pragma unroll
            for (int i = half * (kKeysThread / kHalves); i < (half + 1) * (kKeysThread / kHalves); i += 2) {
              const uint64_t e2 = fma_pair(pair_of(x[i], x[i + 1]), scale2, neg2);
              float y0, y1;
              if (kPolyOf > 0 && (i / 2) % kPolyOf == kPolyOf - 1) {
                float e0, e1;
                unpair(e2, &e0, &e1);
                exp2_pair(pair_of(fmaxf(e0, -126.f), fmaxf(e1, -126.f)), &y0, &y1);
              } else {
                unpair(e2, &y0, &y1);
                y0 = exp2_ftz(y0);
                y1 = exp2_ftz(y1);
              }
              sums[(i / 2) & 1] = add_pair(sums[(i / 2) & 1], pair_of(y0, y1));
              x[i / 2] = pack_bf16x2(y0, y1);
            }
#pragma unroll
            for (int i = half * (kKeysThread / kHalves / 2); i < (half + 1) * (kKeysThread / kHalves / 2); i += 32) tmem_store32(at_p + i, x + i);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            announce((half < kHalves - 1 ? p_half : p_full) + 8 * (u & 1));
          }
          float sum0, sum1;
          unpair(add_pair(sums[0], sums[1]), &sum0, &sum1);
          l += sum0 + sum1;
          m_ref = m_new;
        }
        // the job's result, or the piece's part of it
        const int u = kTiles == 2 ? 2 * (block - 1) + wg : block - 1;
        if (ok) ok = mbar_wait(o_done + 8 * (u & 1), (u >> 1) & 1);
        fence_after();
        if constexpr (kTiles == 1) {
          asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory");
          part_max[part][r] = l;
          asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory");
          l = part_max[0][r] + part_max[1][r];
        }
        const bool whole = w.whole();
        const float inv = m_ref == -INFINITY ? 0.f : 1.0f / l;
        const bool wide_out = ((reinterpret_cast<uintptr_t>(a.c.out_dev) & 31) | (a.c.ld_out & 15)) == 0;
        const size_t part_row = (static_cast<size_t>(piece) * 2 + (w.j == 0 ? 1 : 0)) * (kJobTiles * kRowsT) + job_tile * kRowsT + r;
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.c.out_dev) +
                             (static_cast<size_t>(w.b) * a.c.tokens + min(t, a.c.tokens - 1)) * a.c.ld_out + head * DH;
#pragma unroll 1
        for (int c0 = part * (DH / 2); c0 < (kTiles == 2 ? DH : (part + 1) * (DH / 2)); c0 += 32) {
          uint32_t o[32];
          tmem_load32(tmem + lanes + C::kColO + tile * DH + c0, o);
          if (whole && p >= 0) {
            uint32_t y[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = pack_bf16x2(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
            if (wide_out) {
              store32(out + c0, y);
              store32(out + c0 + 16, y + 8);
            } else {
#pragma unroll
              for (int i = 0; i < 16; i += 4) *reinterpret_cast<uint4*>(out + c0 + 2 * i) = make_uint4(y[i], y[i + 1], y[i + 2], y[i + 3]);
            }
          } else if (!whole) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) store32(a.part_o + part_row * DH + c0 + i, o + i);
          }
        }
        if (!whole && part == 0) a.part_ml[part_row] = make_float2(m_ref, l);
        announce(o_free + 8 * tile);
      } while (w.next(a));
      if (!ok) give_up();
    }
    if (a.c.k_new_dev) store_rows<DH>(a, 2 + warp);
  }
  fence_before();
  if constexpr (kPair) pair_sync();                    // neither block leaves, or frees, while the other may still signal it
  else __syncthreads();
  if (failed) {
    // products may still be reading shared memory and tensor memory, which nobody has waited for: they end before either is given back
    if (warp == 9 && rank == 0) {
      const uint32_t leader = elected();
      if constexpr (kPair) commit_pair(settled, leader);
      else commit_to(settled, leader);
      mbar_settle(settled, 0);
    }
    if constexpr (kPair) pair_sync();
    else __syncthreads();
  }
  if (warp == 9) {
    fence_after();
    if constexpr (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmemCols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmemCols) : "memory");
  }
  if (threadIdx.x == 0 && failed && a.c.status_dev) atomicOr(a.c.status_dev, kDevErrTimeout);
}

// Joins jobs that lie in several pieces.  blockIdx.y is a piece that begins inside a job, the first such of the job; a block has 8 rows,
// a warp a row.
constexpr int kPartRows = 8;
template <int DH>
__global__ void __launch_bounds__(32 * kPartRows) cache_part_kernel(const PromptArgs a) {
  constexpr int kRows = kJobTiles * kRowsT, kVecs = DH / 128 > 0 ? DH / 128 : 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  const int piece = blockIdx.y + 1;
  const int* plan = a.plan + kPlanHead;
  auto same_job = [&](int i) {
    const int *p = plan + piece * 8, *q = plan + i * 8;
    return q[4] > 0 && q[0] == p[0] && q[1] == p[1] && q[2] == p[2];
  };
  const int* p = plan + piece * 8;
  if (p[4] <= 0 || p[3] == 0) return;                                  // no piece, or one that begins a job
  if (same_job(piece - 1) && plan[(piece - 1) * 8 + 3] != 0) return;     // not the first inside its job
  int n = 2;
  while (piece + n - 1 < a.pieces && same_job(piece + n - 1) && plan[(piece + n - 1) * 8 + 3] != 0) ++n;
  const int r = blockIdx.x * kPartRows + warp, tile = r / kRowsT;
  const CacheSeq s = prompt_seq(a, p[0]);
  const int t = p[2] * a.span + (a.by_heads ? r % kRowsT : r);
  const int head = p[1] * (a.by_heads ? 2 : 1) + (a.by_heads ? tile : 0);
  if (t >= s.fresh) return;
  // the job's first part ends the piece before, the others begin theirs
  auto row_of = [&](int k) { return (static_cast<size_t>(piece - 1 + k) * 2 + (k == 0 ? 1 : 0)) * kRows + r; };
  float top = -INFINITY;
  for (int k = lane; k < n; k += 32) top = fmaxf(top, a.part_ml[row_of(k)].x);
  top = warp_max(top);
  float l = 0.f, o[kVecs * 4] = {};
  for (int k = 0; k < n; ++k) {
    const float2 ml = a.part_ml[row_of(k)];
    const float f = ml.x == -INFINITY ? 0.f : exp2_ftz(ml.x - top);
    l = fmaf(ml.y, f, l);
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      if (DH == 64 && lane >= 16) break;
      const float4 y = *reinterpret_cast<const float4*>(a.part_o + row_of(k) * DH + v * 128 + lane * 4);
      o[4 * v] = fmaf(y.x, f, o[4 * v]);
      o[4 * v + 1] = fmaf(y.y, f, o[4 * v + 1]);
      o[4 * v + 2] = fmaf(y.z, f, o[4 * v + 2]);
      o[4 * v + 3] = fmaf(y.w, f, o[4 * v + 3]);
    }
  }
  const float inv = top == -INFINITY ? 0.f : 1.f / l;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.c.out_dev) + (static_cast<size_t>(p[0]) * a.c.tokens + t) * a.c.ld_out + head * DH;
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    if (DH == 64 && lane >= 16) break;
    *reinterpret_cast<uint2*>(out + v * 128 + lane * 4) =
        make_uint2(pack_bf16x2(o[4 * v] * inv, o[4 * v + 1] * inv), pack_bf16x2(o[4 * v + 2] * inv, o[4 * v + 3] * inv));
  }
}

template <int DH>
cudaError_t launch(PromptArgs a, bool join, cudaStream_t s) {
  using C = PromptCfg<DH>;
  const mtj_cache_attn_args& c = a.c;
  CUtensorMap mq, mk, mv, mkn, mvn;
  const int64_t pool_rows = static_cast<int64_t>(c.n_pages) * c.kv_heads * kPageTokens, rows = static_cast<int64_t>(c.batch) * c.tokens;
  cudaError_t e = make_tensor_map_bf16(&mq, c.q_dev, rows, static_cast<int64_t>(c.heads) * DH, kRowsT, c.ld_q);
  if (e == cudaSuccess) e = make_tensor_map_bf16(&mk, c.kpool_dev, pool_rows, DH, kPageTokens);
  if (e == cudaSuccess) e = make_tensor_map_bf16(&mv, c.vpool_dev, pool_rows, DH, kPageTokens);
  mkn = mk;
  mvn = mv;
  if (e == cudaSuccess && c.k_new_dev) {
    e = make_tensor_map_bf16(&mkn, c.k_new_dev, rows, static_cast<int64_t>(c.kv_heads) * DH, kPageTokens, c.ld_k);
    if (e == cudaSuccess) e = make_tensor_map_bf16(&mvn, c.v_new_dev, rows, static_cast<int64_t>(c.kv_heads) * DH, kPageTokens, c.ld_v);
  }
  static DeviceOnce once;
  if (e == cudaSuccess)
    e = once.run([&] { return cudaFuncSetAttribute(cache_prompt_kernel<DH>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(C::kSmem)); });
  if (e != cudaSuccess) return e;
  e = launch_pdl(cache_begin_kernel, dim3(1 + static_cast<unsigned>((rows + kZeroRows - 1) / kZeroRows)), dim3(kBeginThreads), 0, s, false, a);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kBlocks);
  cfg.blockDim = dim3(kPromptThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {2, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = C::kPair ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, cache_prompt_kernel<DH>, mq, mk, mv, mkn, mvn, a);
  if (e == cudaSuccess && join)
    e = launch_pdl(cache_part_kernel<DH>, dim3(kJobTiles * kRowsT / kPartRows, a.pieces - 1), dim3(32 * kPartRows), 0, s, true, a);
  return e;
}

bool pairs_heads(const mtj_cache_attn_args& c) { return (c.heads / c.kv_heads) % 2 == 0; }
int job_span(const mtj_cache_attn_args& c) { return pairs_heads(c) ? kRowsT : kJobTiles * kRowsT; }
int pieces_for(const mtj_cache_attn_args& c) { return c.d_head == 256 ? kBlocks / 2 : kBlocks; }      // pairs of blocks, blocks
constexpr int64_t kPlanBytes = ((kPlanList + kMostEntries) * 4 + 255) / 256 * 256;
int64_t part_rows(const mtj_cache_attn_args& c) { return static_cast<int64_t>(pieces_for(c)) * 2 * kJobTiles * kRowsT; }

// most key blocks of a job
int64_t most_blocks(const mtj_cache_attn_args& c) {
  const int64_t slots = (static_cast<int64_t>(c.pages) * kPageTokens + kKeysB - 1) / kKeysB + 1;      // and the block between cached and new
  const int64_t seen = (static_cast<int64_t>(c.window) + job_span(c)) / kKeysB + 3 + (static_cast<int64_t>(c.sinks) + kKeysB - 1) / kKeysB + 1;
  return std::min(slots, seen);
}
// whether no job can lie in several pieces: jobs of few blocks are taken whole
bool all_whole(const mtj_cache_attn_args& c) { return most_blocks(c) <= kJoinCost; }
// sequences of a launch: as many as the plan has entries for, and as have their key blocks counted in 32 bits
int64_t most_sequences(const mtj_cache_attn_args& c) {
  const int64_t token_jobs = (static_cast<int64_t>(c.tokens) + job_span(c) - 1) / job_span(c);
  return std::min(kMostEntries / token_jobs, 0x7fffffff / (token_jobs * most_blocks(c)));
}

}  // namespace

int64_t cache_prompt_scratch(const mtj_cache_attn_args& c) { return kPlanBytes + part_rows(c) * (8 + c.d_head * 4); }

bool cache_prompt_fits(const mtj_cache_attn_args& c) { return most_sequences(c) > 0; }

cudaError_t run_cache_prompt(const mtj_cache_attn_args& c, char* scratch, cudaStream_t s) {
  PromptArgs a = {};
  a.c = c;
  a.scale_log2 = c.scale * 1.4426950408889634f;
  a.by_heads = pairs_heads(c);
  a.span = job_span(c);
  a.pieces = pieces_for(c);
  a.head_jobs = c.heads / (a.by_heads ? 2 : 1);
  a.token_jobs = (c.tokens + a.span - 1) / a.span;
  a.plan = reinterpret_cast<int*>(scratch);
  a.part_ml = reinterpret_cast<float2*>(scratch + kPlanBytes);
  a.part_o = reinterpret_cast<float*>(scratch + kPlanBytes + part_rows(c) * 8);
  const int most = static_cast<int>(most_sequences(c));
  for (int b0 = 0; b0 < c.batch; b0 += most) {
    a.c.batch = std::min(most, c.batch - b0);
    const bool join = !all_whole(c);
    const cudaError_t e = c.d_head == 64 ? launch<64>(a, join, s) : c.d_head == 128 ? launch<128>(a, join, s) : launch<256>(a, join, s);
    if (e != cudaSuccess) return e;
    const size_t rows = static_cast<size_t>(a.c.batch) * c.tokens;
    auto step = [&](const void* p, int64_t ld) { return p ? static_cast<const __nv_bfloat16*>(p) + rows * ld : nullptr; };
    a.c.q_dev = step(a.c.q_dev, c.ld_q);
    a.c.k_new_dev = step(a.c.k_new_dev, c.ld_k);
    a.c.v_new_dev = step(a.c.v_new_dev, c.ld_v);
    a.c.out_dev = static_cast<__nv_bfloat16*>(a.c.out_dev) + rows * c.ld_out;
    a.c.page_table_dev += static_cast<size_t>(a.c.batch) * c.pages;
    a.c.lengths_dev += a.c.batch;
    if (a.c.new_tokens_dev) a.c.new_tokens_dev += a.c.batch;
  }
  return cudaSuccess;
}

}  // namespace mtj

// Attention of many new tokens over a paged cache (prompts and portions of prompts of mtj_k_cache_attn), on the tensor cores.
//
// A block has 256 query rows: two tiles of 128, two heads of one group at the same tokens, or where groups are odd 256 tokens of one
// head (d_head 64 and 128), or one tile of 128 (d_head 256, whose accumulator fills tensor memory).  Keys come in blocks of 128 (two pages):
// first those of the first tokens, then those of the window; a block of keys serves both tiles, so K and V cross from L2 once
// for 256 rows.  A unit of work is one tile on one key block,
//     S[128, 128] = Q K^T        tcgen05, operands in shared memory by TMA (128-byte swizzle), fp32 in tensor memory
//     P = 2^(S c - m)            a thread a row (d_head 256: two threads a row, 64 keys each), written over S as bf16
//     O[128, d] += P V           P from tensor memory, V as MN-major operand straight from the pages
// and units go round two score buffers: one thread issues S0 S1 | PV0 S2 | PV1 S3 | ..., so that while one warp group works out the
// weights of a unit, the tensor cores have the other unit's products.  The bound for d_head 128 is shared by the tensor cores (1024
// cycles a unit) and the exponentials (16 a cycle: 1024).
//
// Scores, maxima, sums and O are 32-bit; P is rounded to bf16, half a step on average as large as the rounding of the output (a second
// term would be half as many products again).  O is rescaled when a row's maximum has grown by more than 2^8.  The rows of V
// behind the sequence, or of a page that does not exist, are zeroed in shared memory before they meet their zero weights.
// Every wait is bounded.
#include <cuda.h>
#include <math.h>

#include "mtj_cache_kernels.h"

namespace mtj {
namespace {

constexpr int kRowsT = 128;                // rows of a tile
constexpr int kKeysB = 128;                // keys of a block: two pages
constexpr int kSoftThreads = 256;
constexpr int kPromptThreads = kSoftThreads + 64;      // and the warps of TMA and of the products
constexpr int kBlockNotes = 8;
constexpr int kPolyOf = 4;                 // of this many pairs of weights one is worked out on the multiply-add units
constexpr float kExp0 = 0.99992806f, kExp1 = 0.69326097f, kExp2 = 0.24261114f, kExp3 = 0.05517167f;

template <int DH>
struct PromptCfg {
  static constexpr int kTiles = DH == 256 ? 1 : 2;
  static constexpr int kKeysThread = kTiles == 2 ? 128 : 64;
  static constexpr int kChunks = DH / 64;              // 64-column parts of a row
  static constexpr uint32_t kQBytes = kTiles * kRowsT * DH * 2;
  static constexpr uint32_t kKBytes = kKeysB * DH * 2;
  // d_head 256: one block of keys, and values by the page
  static constexpr int kKSlots = DH == 256 ? 1 : DH == 128 ? 2 : 4, kVSlots = DH == 256 ? 3 : DH == 128 ? 3 : 4;
  static constexpr int kVPages = DH == 256 ? 1 : 2;    // of a slot
  static constexpr uint32_t kVBytes = kVPages * kPageTokens * DH * 2;
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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^x of a pair on the multiply-add units, for x in [-126, 9]: x = n + f with |f| <= 1/2 by adding and taking away 1.5 * 2^23, a
// polynomial of degree 3 in f (fitted to the relative error, 8e-5 at most: a twentieth of the rounding to bf16 that follows),
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

// The new tokens' keys and values into their slots: a warp a (token, sequence) and key head, 16 bytes a lane.
__global__ void __launch_bounds__(256) cache_append_kernel(const mtj_cache_attn_args a) {
  pdl_launch_dependents();
  const int vecs = a.kv_heads * (a.d_head / 8);
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = i / vecs;
  if (row >= static_cast<int64_t>(a.batch) * a.tokens) return;
  const int piece = static_cast<int>(i - row * vecs), t = static_cast<int>(row % a.tokens), b = static_cast<int>(row / a.tokens);
  const CacheSeq s = cache_seq(a.lengths_dev, a.new_tokens_dev, b, a.tokens, a.pages);
  if (t >= s.fresh) return;
  const int slot = s.length - s.fresh + t;
  const int page = a.page_table_dev[static_cast<size_t>(b) * a.pages + slot / kPageTokens];
  if (!cache_page_ok(page, a.n_pages)) return;         // reported by the attention, which reads the same table
  const int h = piece / (a.d_head / 8), e = piece % (a.d_head / 8);
  const size_t at = ((static_cast<size_t>(page) * a.kv_heads + h) * kPageTokens + slot % kPageTokens) * (a.d_head / 8) + e;
  static_cast<uint4*>(a.kpool_dev)[at] = load8_bf16(static_cast<const __nv_bfloat16*>(a.k_new_dev) + row * a.ld_k + piece * 8);
  static_cast<uint4*>(a.vpool_dev)[at] = load8_bf16(static_cast<const __nv_bfloat16*>(a.v_new_dev) + row * a.ld_v + piece * 8);
}

// by_heads: a block's two tiles are heads 2i and 2i + 1 at the same tokens, otherwise 256 tokens of one head
template <int DH>
__global__ void __launch_bounds__(kPromptThreads, 1) cache_prompt_kernel(const __grid_constant__ CUtensorMap map_q,
                                                                      const __grid_constant__ CUtensorMap map_k,
                                                                      const __grid_constant__ CUtensorMap map_v,
                                                                      const mtj_cache_attn_args a, float scale_log2, int by_heads,
                                                                      int token_tiles) {
  using C = PromptCfg<DH>;
  constexpr int kTiles = C::kTiles, kKeysThread = C::kKeysThread;
  extern __shared__ __align__(1024) unsigned char prompt_smem[];
  __shared__ __align__(8) uint64_t bars[1 + 2 * C::kKSlots + 2 * C::kVSlots + 6];
  __shared__ uint32_t tmem_slot, failed;
  __shared__ int notes[kBlockNotes];                   // valid rows of a key block's pages: first | second << 8
  __shared__ float part_max[2][kRowsT];                // d_head 256: of the two threads of a row
  const uint32_t base = smem_u32(prompt_smem);
  const uint32_t sQ = base, sK = base + C::kQBytes, sV = sK + C::kKSlots * C::kKBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t q_full = bar0, k_full = bar0 + 8, k_empty = k_full + 8 * C::kKSlots, v_full = k_empty + 8 * C::kKSlots,
                 v_empty = v_full + 8 * C::kVSlots, s_full = v_empty + 8 * C::kVSlots, p_full = s_full + 16, o_done = p_full + 16;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 1 + 2 * C::kKSlots + 2 * C::kVSlots + 6; ++i) mbar_init(bar0 + 8u * i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(p_full + 8u * i, kTiles == 2 ? 128 : 256);
    mbar_fence_init();
    failed = 0;
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(C::kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;

  // what this block has: sequence b, the tiles' first head and token; later tokens, which see more, first
  const int b = blockIdx.z, group = a.heads / a.kv_heads;
  const int tile0 = (token_tiles - 1 - static_cast<int>(blockIdx.y)) * (kTiles == 2 && !by_heads ? 2 : 1);
  const int head0 = blockIdx.x * (by_heads ? 2 : 1), kvh = head0 / group;
  const CacheSeq s = cache_seq(a.lengths_dev, a.new_tokens_dev, b, a.tokens, a.pages);
  if (s.bad && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0 && a.status_dev) atomicOr(a.status_dev, kDevErrBadIndex);
  const int t_first = tile0 * kRowsT, t_end = min(s.fresh, t_first + (kTiles == 2 && !by_heads ? 2 : 1) * kRowsT);
  const int p_first = s.length - s.fresh + t_first, p_last = s.length - s.fresh + t_end - 1;
  const int low = cache_window_low(p_first, a.window);
  const int low_block = low / kKeysB, sink_blocks = min((min(a.sinks, low) + kKeysB - 1) / kKeysB, low_block);
  const int nb = t_end > t_first ? sink_blocks + p_last / kKeysB - low_block + 1 : 0;
  const int units = nb * kTiles;
  auto first_key = [&](int j) { return (j < sink_blocks ? j : low_block + j - sink_blocks) * kKeysB; };
  pdl_wait();

  if (warp == 8) {
    // ---- TMA ----
    if (lane == 0 && nb > 0) {
      asm volatile("fence.proxy.async;" ::: "memory");     // the slots' newest rows were stored by the kernel before
      mbar_expect_tx(q_full, C::kQBytes);
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c)
          tma_box(sQ + (t * C::kChunks + c) * (kRowsT * 128), &map_q, (head0 + (by_heads ? t : 0)) * DH + c * 64,
                  b * a.tokens + t_first + (by_heads ? 0 : t * kRowsT), q_full);
      const int32_t* table = a.page_table_dev + static_cast<size_t>(b) * a.pages;
      int page[2], valid[2];
      auto look_up = [&](int j) {
        const int key = first_key(j);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = key / kPageTokens + h;
          valid[h] = min(kPageTokens, max(0, s.length - at * kPageTokens));
          page[h] = valid[h] > 0 ? table[at] : 0;
          if (!cache_page_ok(page[h], a.n_pages)) {
            valid[h] = page[h] = 0;
            if (a.status_dev) atomicOr(a.status_dev, kDevErrBadIndex);
          }
        }
      };
      auto load_k = [&](int j) {
        const int st = j % C::kKSlots;
        if (j >= C::kKSlots && !mbar_wait(k_empty + 8 * st, (j / C::kKSlots - 1) & 1)) return false;
        look_up(j);
        notes[j % kBlockNotes] = valid[0] | valid[1] << 8;
        // a page without valid rows is not read: page 0 stands in, nobody sees its scores
        mbar_expect_tx(k_full + 8 * st, C::kKBytes);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < C::kChunks; ++c)
            tma_box(sK + st * C::kKBytes + c * (kKeysB * 128) + h * (kPageTokens * 128), &map_k, c * 64,
                    (page[h] * a.kv_heads + kvh) * kPageTokens, k_full + 8 * st);
        return true;
      };
      auto load_v = [&](int j) {
        look_up(j);
        for (int i = 0; i < 2 / C::kVPages; ++i) {
          const int n = j * (2 / C::kVPages) + i, st = n % C::kVSlots;
          if (n >= C::kVSlots && !mbar_wait(v_empty + 8 * st, (n / C::kVSlots - 1) & 1)) return false;
          mbar_expect_tx(v_full + 8 * st, C::kVBytes);
#pragma unroll
          for (int h = 0; h < C::kVPages; ++h)
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c)
              tma_box(sV + st * C::kVBytes + c * (C::kVPages * kPageTokens * 128) + h * (kPageTokens * 128), &map_v, c * 64,
                      (page[C::kVPages == 2 ? h : i] * a.kv_heads + kvh) * kPageTokens, v_full + 8 * st);
        }
        return true;
      };
      // in the order in which the products want them: S0 (S1) | PV0 S2 | PV1 S3 ...
      bool ok = load_k(0);
      for (int j = 0; ok && j < nb; ++j) {
        if (j + 1 < nb) ok = load_k(j + 1);
        if (ok) ok = load_v(j);
      }
      if (!ok) atomicOr(&failed, 1u);
    }
  } else if (warp == 9) {
    // ---- products ----
    if (nb > 0) {
      const uint32_t leader = elected();
      auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0; };
      constexpr uint32_t kIdS = (1u << 4) | (1u << 7) | (1u << 10) | ((kKeysB >> 3) << 17) | ((kRowsT >> 4) << 24);
      constexpr uint32_t kIdO = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((DH >> 3) << 17) | ((kRowsT >> 4) << 24);
      auto issue_s = [&](int u) {
        const int j = u / kTiles, t = u % kTiles, st = j % C::kKSlots;
        if (t == 0 && !wait(k_full + 8 * st, (j / C::kKSlots) & 1)) return false;
        fence_after();
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) {
          const uint64_t qd = smem_desc(sQ + (t * C::kChunks + c) * (kRowsT * 128), 16, 1024);
          const uint64_t kd = smem_desc(sK + st * C::kKBytes + c * (kKeysB * 128), 16, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_ss(tmem + C::kColS + (u & 1) * kKeysB, qd + 2 * k, kd + 2 * k, kIdS, (c | k) ? 1u : 0u, leader);
        }
        commit_to(s_full + 8 * (u & 1), leader);
        if (t == kTiles - 1) commit_to(k_empty + 8 * st, leader);
        return true;
      };
      auto issue_pv = [&](int u) {
        const int j = u / kTiles, t = u % kTiles;
        if (!wait(p_full + 8 * (u & 1), (u >> 1) & 1)) return false;
#pragma unroll
        for (int i = 0; i < 2 / C::kVPages; ++i) {
          const int n = j * (2 / C::kVPages) + i, st = n % C::kVSlots;
          if (t == 0 && !wait(v_full + 8 * st, (n / C::kVSlots) & 1)) return false;
          fence_after();
          const uint64_t vd = smem_desc(sV + st * C::kVBytes, C::kVPages * kPageTokens * 128, 1024);
          const uint32_t pa = tmem + C::kColS + (u & 1) * kKeysB + i * (kPageTokens / 2);
#pragma unroll
          for (int k = 0; k < C::kVPages * 4; ++k)
            mma_ts(tmem + C::kColO + t * DH, pa + 8 * k, vd + static_cast<uint64_t>((k * 2048) >> 4), kIdO, (j | i | k) ? 1u : 0u, leader);
          if (t == kTiles - 1) commit_to(v_empty + 8 * st, leader);
        }
        commit_to(o_done + 8 * (u & 1), leader);
        return true;
      };
      bool ok = wait(q_full, 0) && issue_s(0);
      if (ok && units > 1) ok = issue_s(1);
      for (int u = 0; ok && u < units; ++u) {
        ok = issue_pv(u);
        if (ok && u + 2 < units) ok = issue_s(u + 2);
      }
      if (!ok && leader) atomicOr(&failed, 1u);
    }
  } else {
    // ---- weights ----
    const int wg = warp >> 2, quad = warp & 3;
    const int tile = kTiles == 2 ? wg : 0, part = kTiles == 2 ? 0 : wg;      // of the keys of a block
    const int r = quad * 32 + lane;                        // row of the tile = lane of tensor memory
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const int head = head0 + (by_heads ? tile : 0), t0 = t_first + (by_heads ? 0 : tile * kRowsT);
    const int t = t0 + r;
    const int p = t < s.fresh ? s.length - s.fresh + t : -1;
    const int warp_first = s.length - s.fresh + t0 + quad * 32;      // slots of the warp's rows: warp_first .. + 31
    float m_ref = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < nb; ++j) {
      const int u = kTiles == 2 ? 2 * j + wg : j;
      if (ok) ok = mbar_wait(s_full + 8 * (u & 1), (u >> 1) & 1);
      fence_after();
      const int key = first_key(j) + part * kKeysThread;
      const int note = notes[j % kBlockNotes];
      const uint32_t at_s = tmem + lanes + C::kColS + (u & 1) * kKeysB + part * kKeysThread;
      uint32_t x[kKeysThread];
#pragma unroll
      for (int i = 0; i < kKeysThread; i += 32) tmem_fetch32(at_s + i, x + i);
      tmem_wait();
#pragma unroll
      for (int i = 0; i < kKeysThread; i += 32) pin32(x + i);
      // V's rows that hold nothing: zeroed before anybody's weights are announced
      if (note != (kPageTokens | kPageTokens << 8)) {
#pragma unroll
        for (int i = 0; i < 2 / C::kVPages; ++i) {
          const int n = j * (2 / C::kVPages) + i, st = n % C::kVSlots;
          if (ok) ok = mbar_wait(v_full + 8 * st, (n / C::kVSlots) & 1);
          if (tile == 0) {
            // [64-column part][page][64 rows][128 bytes]
            for (int e = threadIdx.x; e < static_cast<int>(C::kVBytes / 16); e += kTiles == 2 ? 128 : 256) {
              const int row = e / 8 % kPageTokens, h = C::kVPages == 2 ? e / 8 / kPageTokens % 2 : i;
              if (row >= ((note >> (8 * h)) & 255))
                *reinterpret_cast<uint4*>(prompt_smem + (sV - base) + st * C::kVBytes + e * 16) = make_uint4(0, 0, 0, 0);
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      const int warp_last = min(warp_first + 31, p_last);
      const bool whole = note == (kPageTokens | kPageTokens << 8) && key + kKeysThread - 1 <= warp_first &&
                         (key + kKeysThread - 1 < a.sinks || warp_last - key < a.window) && warp_last >= warp_first;
      if (!whole) {
        // the row's visible keys as bits: up to its own slot, in the window or among the first tokens, in a page that holds something
        const int hi = p - key, lo = p - a.window + 1 - key, sk = a.sinks - key;
#pragma unroll
        for (int w = 0; w < kKeysThread / 32; ++w) {
          const int within = part * kKeysThread + 32 * w;
          const int held = (within < kPageTokens ? note & 255 : note >> 8) - within % kPageTokens;
          const uint32_t see = low_bits(min(hi + 1, held + 32 * w) - 32 * w) & (~low_bits(lo - 32 * w) | low_bits(sk - 32 * w));
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(see >> i & 1u)) x[32 * w + i] = 0xff800000u;
        }
      }
      float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < kKeysThread; i += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) tops[e] = max3(tops[e], __uint_as_float(x[i + 2 * e]), __uint_as_float(x[i + 2 * e + 1]));
      float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * scale_log2;      // scale > 0
      if constexpr (kTiles == 1) {
        part_max[part][r] = top;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory");
        top = fmaxf(top, part_max[part ^ 1][r]);
        asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory");
      }
      float m_new = m_ref;
      if (top > m_ref + 8.0f || (m_ref == -INFINITY && top > -INFINITY)) m_new = top;
      const float corr = (m_new == m_ref || m_ref == -INFINITY) ? 1.0f : exp2_ftz(m_ref - m_new);
      const float neg = m_new == -INFINITY ? 0.f : -m_new;
      const uint64_t scale2 = pair_of(scale_log2, scale_log2), neg2 = pair_of(neg, neg);
      uint64_t sums[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < kKeysThread; i += 2) {
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
      float sum0, sum1;
      unpair(add_pair(sums[0], sums[1]), &sum0, &sum1);
      l = fmaf(l, corr, sum0 + sum1);
      if (__any_sync(0xffffffffu, corr != 1.0f)) {
        // O changes scale: the tile's products so far must have landed
        const int before = u - kTiles;
        if (ok) ok = mbar_wait(o_done + 8 * (before & 1), (before >> 1) & 1);
        fence_after();
#pragma unroll 1
        for (int c0 = 0; c0 < DH / (3 - kTiles); c0 += 32) {
          const uint32_t at = tmem + lanes + C::kColO + tile * DH + part * (DH / 2) + c0;
          uint32_t o[32];
          tmem_load32(at, o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
          tmem_store32(at, o);
        }
      }
#pragma unroll
      for (int i = 0; i < kKeysThread / 2; i += 32)
        tmem_store32(tmem + lanes + C::kColS + (u & 1) * kKeysB + part * (kKeysThread / 2) + i, x + i);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      fence_before();
      arrive_at(p_full + 8 * (u & 1));
      m_ref = m_new;
    }
    if (nb > 0) {
      const int u = kTiles == 2 ? 2 * (nb - 1) + wg : nb - 1;
      if (ok) ok = mbar_wait(o_done + 8 * (u & 1), (u >> 1) & 1);
      if (!ok) atomicOr(&failed, 1u);
    }
    fence_after();
    if constexpr (kTiles == 1) {
      asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory");
      part_max[part][r] = l;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory");
      l = part_max[0][r] + part_max[1][r];
    }
    const float inv = nb > 0 && l > 0.f ? 1.0f / l : 0.f;
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out_dev) + (static_cast<size_t>(b) * a.tokens + min(t, a.tokens - 1)) * a.ld_out + head * DH;
#pragma unroll 1
    for (int c0 = part * (DH / 2); c0 < (kTiles == 2 ? DH : (part + 1) * (DH / 2)); c0 += 32) {
      uint32_t o[32];
      if (nb > 0) {
        tmem_load32(tmem + lanes + C::kColO + tile * DH + c0, o);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0u;
      }
      if (t < a.tokens) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = p < 0 ? 0.f : __uint_as_float(o[i + e]);
          store8(out + c0 + i, v, inv);
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 9) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmemCols) : "memory");
  }
  if (threadIdx.x == 0 && failed && a.status_dev) atomicOr(a.status_dev, kDevErrTimeout);
}

template <int DH>
cudaError_t launch(const mtj_cache_attn_args& a, cudaStream_t s) {
  using C = PromptCfg<DH>;
  CUtensorMap mq, mk, mv;
  const int64_t pool_rows = static_cast<int64_t>(a.n_pages) * a.kv_heads * kPageTokens;
  cudaError_t e = make_tensor_map_bf16(&mq, a.q_dev, static_cast<int64_t>(a.batch) * a.tokens, static_cast<int64_t>(a.heads) * DH, kRowsT, a.ld_q);
  if (e == cudaSuccess) e = make_tensor_map_bf16(&mk, a.kpool_dev, pool_rows, DH, kPageTokens);
  if (e == cudaSuccess) e = make_tensor_map_bf16(&mv, a.vpool_dev, pool_rows, DH, kPageTokens);
  static DeviceOnce once;
  if (e == cudaSuccess)
    e = once.run([&] { return cudaFuncSetAttribute(cache_prompt_kernel<DH>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(C::kSmem)); });
  if (e != cudaSuccess) return e;
  if (a.k_new_dev) {
    const int64_t vecs = static_cast<int64_t>(a.batch) * a.tokens * a.kv_heads * (DH / 8);
    e = launch_pdl(cache_append_kernel, dim3(static_cast<unsigned>((vecs + 255) / 256)), dim3(256), 0, s, false, a);
    if (e != cudaSuccess) return e;
  }
  const bool by_heads = C::kTiles == 2 && (a.heads / a.kv_heads) % 2 == 0;
  const int span = C::kTiles == 2 && !by_heads ? 2 * kRowsT : kRowsT;
  const int tiles = (a.tokens + span - 1) / span;
  return launch_pdl(cache_prompt_kernel<DH>, dim3(a.heads / (by_heads ? 2 : 1), tiles, a.batch), dim3(kPromptThreads), C::kSmem, s,
                    a.k_new_dev != nullptr, mq, mk, mv, a, a.scale * 1.4426950408889634f, by_heads ? 1 : 0, tiles);
}

}  // namespace

cudaError_t run_cache_prompt(const mtj_cache_attn_args& a, cudaStream_t s) {
  return a.d_head == 64 ? launch<64>(a, s) : a.d_head == 128 ? launch<128>(a, s) : launch<256>(a, s);
}

}  // namespace mtj

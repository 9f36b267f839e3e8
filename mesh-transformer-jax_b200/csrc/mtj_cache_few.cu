// Attention of a few new tokens over a paged cache (mtj_k_cache_attn), bound by the bytes of the cached keys and values.
//
// A unit of work is (sequence, key head, tile of 8 NT query rows); the rows are the tokens and the query heads of the group, so
// every cached byte is read once for all of them.  The visible slots of a unit are tiles of 16 KB (16, 32 or 64 keys with their
// values): those of the first tokens, then those of the window.  All tiles of all units stand in one line, which is cut into equal
// pieces, one a block, two blocks an SM: sequences of any lengths load every SM alike, and one sequence uses all of them.  A unit
// that lies in several pieces is joined by a second kernel from its parts' (maximum, sum, weighted values); two launches, no
// counters and no order of arrival, so a call gives the same bits every time.
//
// A producer warp keeps a ring of tiles full by TMA (its lanes look up 32 pages at a time); four warps work, each on 16 keys of its
// own with its own running maximum and sum:
//     S^T[16 keys, rows] = K Q^T     keys are the M dimension of mma.sync, so that one query row wastes 7/8 of a small N and not
//     O^T[16 d, rows]   += V^T P^T   15/16 of M; K by ldmatrix, V by ldmatrix.trans, P transposed between the two by movmatrix
// tcgen05 takes keys as M too (64 or 128, with N from 8 rows on) and would be no emptier.  It has the scores and the weights a trip through
// tensor and shared memory away, which one token, bound by traffic, gains nothing from; for drafted tokens, where the chain of a tile
// counts and not the bytes, that form has not been built or measured.  Queries in 32 bits are the exact sum of three bf16 numbers, three products each.  The weights P go into the
// product as two bf16 numbers (three for 32-bit queries), an error of 2^-16 (2^-24): one would cost as much as the rounding of
// the output (and save 6 of 44 us with 5 drafts, 4 heads a key head and 8 sequences of up to 8191 slots).  Scores, maxima, sums and
// outputs are 32-bit.
//
// New keys and values are laid over the rows of the tile that has just arrived, and stored to their slots by the blocks of the
// first row tile: nobody reads in this launch what it stores.  Values behind the sequence, and between the first tokens and the
// window, are zeroed in the tile, since weight zero times whatever stands there must be zero.
//
// 8 key heads of 128 with 4 query heads each: one token of 32 sequences of 2000 to 16383 slots 197 us, 1.21 GB at 6.1 TB/s, and 31 us for
// the join that adds up the weights; five tokens of 8 sequences, window 4096, 39 us for 107 MB: there the chain of a tile (two products
// with a softmax between them, 20 rows) and the ragged ends of 64 units count, not the bytes.
#include <cuda.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "mtj_cache_kernels.h"

namespace mtj {
namespace {

constexpr int kWorkers = 4;                          // warps
constexpr int kPieces = 2 * 148;                     // two blocks on each of a B200's SMs
constexpr int kFewThreads = 32 * kWorkers + 32;
constexpr uint32_t kTileBytes = 16384;               // keys and values
constexpr int kJoinThreads = 256;
constexpr float kGrowth = 8.f;                       // weights stay below 2^8
constexpr int kWeightSlots = 1024;                   // slots of one key head that a block of the second kernel adds weights to

// n tiles of rows that a warp takes: its accumulators are DH / 4 registers each
constexpr int few_n_tiles(int dh, int nt) { return dh == 256 ? 1 : dh == 128 && nt == 4 ? 2 : nt; }
// times 16 keys that a warp works on side by side (64-wide heads and 24 rows: two times are 7 % ahead with 8000 slots, one time 10 % with 500)
constexpr int few_sub(int dh, int nt) { return dh == 256 || nt == 3 || few_n_tiles(dh, nt) == 4 ? 1 : 2; }

template <int DH, int NT, typename T>
struct FewCfg {
  static constexpr int kKeys = 4096 / DH;            // of a tile: 16, 32, 64
  static constexpr int kNt = few_n_tiles(DH, NT), kRowWarps = NT / kNt;      // warps beside each other on the same keys
  static constexpr int kSub = few_sub(DH, NT);
  static constexpr int kKeyWarps = kKeys / (16 * kSub);
  static constexpr int kTeam = kKeyWarps * kRowWarps;      // warps that share a tile
  static constexpr int kTeams = kWorkers / kTeam;
  static constexpr int kParts = kWorkers / kRowWarps;      // warps with results for one row
  static constexpr int kChains = kSub * kNt >= 4 ? 1 : 2;  // of sums for a score
  static constexpr int kRows = 8 * NT;
  static constexpr int kQTerms = sizeof(T) == 2 ? 1 : 3, kPTerms = sizeof(T) == 4 ? 3 : 2;
  // 32-bit queries: the product adds 16 terms at a time, what it adds them to is rounded towards zero, so the sums over steps and
  // keys are taken with additions that round to the nearest (a token behind 2052 keys: 1.1e-6 off without)
  static constexpr bool kExactSums = sizeof(T) == 4;
  static constexpr int kSteps = DH / 16;
  static constexpr uint32_t kQBytes = kQTerms * NT * kSteps * 32 * 8;
  static constexpr int kLdO = DH + 4;                // words: rows two apart fall into other banks
  static constexpr uint32_t kOBytes = 2 * kRows * kLdO * 4;
  // two blocks an SM: 227 KB less 1 KB a block, the alignment of the ring and the statically allocated part
  static constexpr uint32_t kRoom = 111 * 1024 - 1024 - kQBytes - kOBytes - 4 * 1024;
  // a stage always belongs to the same team, which meets its phases one after the other: with a stage that teams take in turn, the
  // parity that a team waits for is also that of the phase before the one another team still waits for
  static constexpr int kStages = static_cast<int>(kRoom / kTileBytes < 6 ? kRoom / kTileBytes : 6) / kTeams * kTeams;
  static constexpr uint32_t kSmem = 1024 + kStages * kTileBytes + kQBytes + kOBytes;
  static_assert(kTeams * kTeam == kWorkers && kParts >= 2, "all warps work");
  static_assert(kStages >= 4 && kStages % kTeams == 0, "a ring");
};

__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void worker_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWorkers) : "memory"); }
// the same; whether any worker says so
__device__ __forceinline__ bool worker_any(bool x) {
  uint32_t y;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(y)
      : "r"(x ? 1u : 0u), "n"(32 * kWorkers)
      : "memory");
  return y != 0;
}
// byte of (row, 16-byte piece c of the row) in a tile that TMA stored with the 128-byte swizzle, 64 columns a box
template <int ROWS>
__device__ __forceinline__ uint32_t piece_at(int row, int c) {
  return static_cast<uint32_t>((c >> 3) * (ROWS * 128) + row * 128 + ((c ^ row) & 7) * 16);
}
// x = t[0] + t[1] + ..., each a bf16 number
template <int TERMS>
__device__ __forceinline__ void split2(float x, float y, uint32_t* t) {
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    t[i] = pack_bf16x2(x, y);
    x -= bf16_lo(t[i]);
    y -= bf16_hi(t[i]);
  }
}

// What one call's slice of tokens makes of a sequence: tokens t0 .. t0 + tokens - 1 of the call.
struct FewSeq {
  int length, fresh;       // slots up to the slice's last token, tokens of the slice
  int sink_tiles, low_tile, tiles;
};
template <int KEYS>
__device__ __forceinline__ FewSeq few_seq(const CacheFewArgs& a, int2 held) {
  FewSeq f;
  f.length = held.x;
  f.fresh = held.y;
  f.sink_tiles = f.low_tile = f.tiles = 0;
  if (f.fresh > 0) {
    const int low = cache_window_low(f.length - f.fresh, a.c.window);
    f.low_tile = low / KEYS;
    f.sink_tiles = min((min(a.c.sinks, low) + KEYS - 1) / KEYS, f.low_tile);
    f.tiles = f.sink_tiles + (f.length - 1) / KEYS - f.low_tile + 1;
  }
  return f;
}
// .x slots up to the slice's last token, .y tokens of the slice
__device__ __forceinline__ int2 few_held(const CacheFewArgs& a, int b, bool report) {
  const CacheSeq s = cache_seq(a.c.lengths_dev, a.c.new_tokens_dev, b, a.c.tokens, a.c.pages);
  if (s.bad && report && a.c.status_dev) atomicOr(a.c.status_dev, kDevErrBadIndex);
  const int fresh = min(max(s.fresh - a.t0, 0), a.tokens);
  return make_int2(s.length - s.fresh + min(s.fresh, a.t0) + fresh, fresh);
}

// Where units are few beside the blocks (aligned), no piece reaches over a unit's end: changing units costs a block about as much as
// two rounds of tiles (16 units of 129 tiles: 16 against 10.5 us).  With the pieces this wide they are at most as many as the blocks.
__device__ __forceinline__ int piece_width(const CacheFewArgs& a, int total, int units) {
  const int w = max(a.least, (total + kPieces - units - 1) / (kPieces - units));
  return (w + a.teams - 1) / a.teams * a.teams;
}
__device__ __forceinline__ int pieces_in(int tiles, int width) { return max(1, (tiles + width - 1) / width); }

// The line of tiles: prefix[b] tiles lie before sequence b, its units one after the other.  Called by all threads of a block.
static_assert(kFewBatch <= 2 * kFewThreads, "two sequences a thread");
template <int KEYS>
__device__ __forceinline__ void lay_out(const CacheFewArgs& a, int units, int2* held, int* prefix, int* first, int* scan) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = 2 * tid;
  if (a.c.batch <= 32) {
    // one warp, without the block's barriers
    if (warp == 0) {
      auto before = [&](int n, int* all) {
        int x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        *all = __shfl_sync(0xffffffffu, x, 31);
        return x - n;
      };
      auto put = [&](int* at, int* out, int x, int all) {
        if (lane < a.c.batch) at[lane] = x;
        if (lane == 0) at[a.c.batch] = all;
        if (out && blockIdx.x == 0 && lane < a.c.batch) out[lane] = x;
        if (out && blockIdx.x == 0 && lane == 0) out[a.c.batch] = all;
      };
      int tiles = 0, total, pieces;
      if (lane < a.c.batch) {
        held[lane] = few_held(a, lane, blockIdx.x == 0);
        tiles = few_seq<KEYS>(a, held[lane]).tiles;
      }
      const int tiles_before = before(tiles * units, &total);
      put(prefix, a.prefix, tiles_before, total);
      if (a.aligned) {
        const int n = lane < a.c.batch ? pieces_in(tiles, piece_width(a, total, a.c.batch * units)) * units : 0;
        const int x = before(n, &pieces);
        put(first, nullptr, x, pieces);
      }
    }
    __syncthreads();
    return;
  }
  int n0 = 0, n1 = 0;
  if (b < a.c.batch) {
    held[b] = few_held(a, b, blockIdx.x == 0);
    n0 = few_seq<KEYS>(a, held[b]).tiles * units;
  }
  if (b + 1 < a.c.batch) {
    held[b + 1] = few_held(a, b + 1, blockIdx.x == 0);
    n1 = few_seq<KEYS>(a, held[b + 1]).tiles * units;
  }
  int x = n0 + n1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) scan[warp] = x;
  __syncthreads();
  int before = x - n0 - n1, total = 0;
  for (int w = 0; w < kFewThreads / 32; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  if (b <= a.c.batch) prefix[b] = before;
  if (b + 1 <= a.c.batch) prefix[b + 1] = before + n0;
  if (blockIdx.x == 0) {                   // for the second kernel
    if (b <= a.c.batch) a.prefix[b] = before;
    if (b + 1 <= a.c.batch) a.prefix[b + 1] = before + n0;
  }
  if (a.aligned) {
    // pieces of sequence b: first[b] before it, its units' after one another
    const int width = piece_width(a, total, a.c.batch * units);
    n0 = b < a.c.batch ? pieces_in(n0 / units, width) * units : 0;
    n1 = b + 1 < a.c.batch ? pieces_in(n1 / units, width) * units : 0;
    x = n0 + n1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    before = x - n0 - n1;
    for (int w = 0; w < warp; ++w) before += scan[w];
    if (b <= a.c.batch) first[b] = before;
    if (b + 1 <= a.c.batch) first[b + 1] = before + n0;
  }
  __syncthreads();
}
__device__ __forceinline__ int sequence_of(const int* prefix, int batch, int x) {
  int lo = 0, hi = batch - 1;              // the last sequence that begins at or before x: one with tiles
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// no piece is empty
__device__ __forceinline__ int pieces_of(int64_t total, int most) { return static_cast<int>(min(total, static_cast<int64_t>(most))); }
__device__ __forceinline__ int piece_begin(int64_t total, int pieces, int i) { return static_cast<int>(total * i / pieces); }

template <int DH, int NT, typename T>
__global__ void __launch_bounds__(kFewThreads, 2) cache_few_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                const __grid_constant__ CUtensorMap map_v, const CacheFewArgs a) {
  using C = FewCfg<DH, NT, T>;
  constexpr int kKeys = C::kKeys, kRows = C::kRows, kSteps = C::kSteps, kStages = C::kStages;
  extern __shared__ unsigned char few_raw[];
  __shared__ __align__(8) uint64_t bars[2 * kStages];
  __shared__ int tile_slot[kStages];                 // first slot of the tile in this stage, -1: its page does not exist
  __shared__ int tile_page[kStages];
  __shared__ int scan[kFewThreads / 32];
  __shared__ int prefix[kFewBatch + 1], first_piece[kFewBatch + 1];
  __shared__ int2 held[kFewBatch];
  __shared__ float sm_m[C::kParts][kRows], sm_l[C::kParts][kRows];
  const uint32_t raw = smem_u32(few_raw), ring = (raw + 1023) & ~1023u;
  unsigned char* ring_ptr = few_raw + (ring - raw);
  uint2* q_frag = reinterpret_cast<uint2*>(ring_ptr + kStages * kTileBytes);
  float* o_buf = reinterpret_cast<float*>(ring_ptr + kStages * kTileBytes + C::kQBytes);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = a.c.heads / a.c.kv_heads, rows = a.tokens * group, row_tiles = (rows + kRows - 1) / kRows;
  const int units = a.c.kv_heads * row_tiles;
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int st) { return bar0 + 8u * st; };
  auto empty_bar = [&](int st) { return bar0 + 8u * (kStages + st); };
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full_bar(i), 1);
      mbar_init(empty_bar(i), C::kTeam);
    }
    mbar_fence_init();
  }
  pdl_launch_dependents();                           // the second kernel waits for this one's end
  lay_out<kKeys>(a, units, held, prefix, first_piece, scan);
  const int64_t total = prefix[a.c.batch];
  int begin, end;
  if (a.aligned) {
    if (static_cast<int>(blockIdx.x) >= first_piece[a.c.batch]) return;
    const int b = sequence_of(first_piece, a.c.batch, blockIdx.x);
    const FewSeq s = few_seq<kKeys>(a, held[b]);
    const int n = (first_piece[b + 1] - first_piece[b]) / units, rest = blockIdx.x - first_piece[b], unit = rest / n, k = rest - unit * n;
    begin = prefix[b] + unit * s.tiles + unit_piece_begin(s.tiles, n, k);
    end = prefix[b] + unit * s.tiles + unit_piece_begin(s.tiles, n, k + 1);
    if (s.tiles == 0) {                              // rows that see nothing
      const int kvh = unit / row_tiles, row0 = unit % row_tiles * kRows;
      const float zero[8] = {};
      for (int i = tid; i < min(kRows, rows - row0) * (DH / 8); i += kFewThreads) {
        const int r = row0 + i / (DH / 8), t = r / group;
        store8(static_cast<T*>(a.c.out_dev) + (static_cast<size_t>(b) * a.c.tokens + a.t0 + t) * a.c.ld_out +
                   (kvh * group + r - t * group) * DH + i % (DH / 8) * 8, zero, 0.f);
      }
      return;
    }
  } else {
    const int pieces = pieces_of(total, gridDim.x);
    if (static_cast<int>(blockIdx.x) >= pieces) return;
    begin = piece_begin(total, pieces, blockIdx.x);
    end = piece_begin(total, pieces, blockIdx.x + 1);
  }

  if (warp == kWorkers) {
    // ---- producer ----
    int st = 0, issued = 0;                          // stage, tiles so far
    uint32_t phase = 1;                              // a fresh barrier counts as having passed the phase before its first
    bool ok = true;
    for (int x0 = begin; ok && x0 < end; x0 += 32) {
      int page = -1, row = 0, slot = -1;
      const int x = x0 + lane;
      if (x < end) {
        const int b = sequence_of(prefix, a.c.batch, x);
        const FewSeq s = few_seq<kKeys>(a, held[b]);
        const int rest = x - prefix[b], unit = rest / s.tiles, tile = rest - unit * s.tiles;
        slot = (tile < s.sink_tiles ? tile : s.low_tile + tile - s.sink_tiles) * kKeys;
        page = a.c.page_table_dev[static_cast<size_t>(b) * a.c.pages + slot / kPageTokens];
        if (cache_page_ok(page, a.c.n_pages)) {
          row = (page * a.c.kv_heads + unit / row_tiles) * kPageTokens + slot % kPageTokens;
        } else {
          page = slot = -1;
          if (a.c.status_dev) atomicOr(a.c.status_dev, kDevErrBadIndex);
        }
      }
      const int n = min(32, end - x0);
      for (int i = 0; i < n; ++i) {
        const int r = __shfl_sync(0xffffffffu, row, i), sl = __shfl_sync(0xffffffffu, slot, i), pg = __shfl_sync(0xffffffffu, page, i);
        if (lane == 0) {
          ok = mbar_wait(empty_bar(st), phase);
          if (ok) {
            tile_slot[st] = sl;
            tile_page[st] = pg;
            if (sl < 0) {
              arrive(full_bar(st));
            } else {
              mbar_expect_tx(full_bar(st), kTileBytes);
              const uint32_t dst = ring + st * kTileBytes;
#pragma unroll
              for (int c = 0; c < DH / 64; ++c) {
                tma_rows(dst + c * (kKeys * 128), &map_k, c * 64, r, full_bar(st));
                tma_rows(dst + kTileBytes / 2 + c * (kKeys * 128), &map_v, c * 64, r, full_bar(st));
              }
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (!ok) break;
        ++issued;
        if (++st == kStages) {
          st = 0;
          phase ^= 1;
        }
      }
    }
    if (lane == 0) {
      if (!ok && a.c.status_dev) atomicOr(a.c.status_dev, kDevErrTimeout);
      // the last round of tiles has landed before the block leaves, also where the warps that should have waited for them gave up
      for (int i = max(0, issued - kStages); i < issued; ++i) mbar_settle(full_bar(i % kStages), (i / kStages) & 1);
    }
    return;
  }

  // ---- workers ----
  const int team = warp / C::kTeam, key0 = (warp % C::kKeyWarps) * (16 * C::kSub);   // this warp's keys of its team's tiles
  const int nt0 = C::kRowWarps == 1 ? 0 : warp / C::kKeyWarps % C::kRowWarps * C::kNt;     // and its rows' first n tile
  const int part_id = team * C::kKeyWarps + warp % C::kKeyWarps;
  const int g = lane >> 2, c = lane & 3;                                 // fragment coordinates
  constexpr int kNt = C::kNt;
  constexpr int kSub = C::kSub;
  constexpr int kBlock = kNt * kSub == 1 ? 4 : 2;    // steps whose products are issued side by side
  constexpr bool kQInRegisters = C::kQTerms * kNt * kSteps <= 16;
  uint2 qr[kQInRegisters ? C::kQTerms * kNt * kSteps : 1];
  bool arrived = true;
  int count = 0;                                                         // tiles of this block so far
  for (int x = begin; x < end;) {
    const int b = sequence_of(prefix, a.c.batch, x);
    const FewSeq s = few_seq<kKeys>(a, held[b]);
    const int rest = x - prefix[b], unit = rest / s.tiles, tile0 = rest - unit * s.tiles;
    const int n_tiles = min(s.tiles - tile0, end - x);
    const int kvh = unit / row_tiles, row0 = unit % row_tiles * kRows;
    const int first = s.length - s.fresh;                                // slot of the slice's first token
    const int low = cache_window_low(first, a.c.window);                 // and the first of its window

    // queries as the B operand: fragment (term, n tile, k step, lane); a thread brings 8 numbers of a row
    constexpr int kPieces = kRows * (DH / 8), kEach = (kPieces + 32 * kWorkers - 1) / (32 * kWorkers);
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int i = u * 32 * kWorkers + tid, r = i / (DH / 8), piece = i % (DH / 8);
      if (kPieces % (32 * kWorkers) != 0 && i >= kPieces) break;
      const int t = (row0 + r) / group;
      uint32_t w[C::kQTerms][4] = {};
      if (row0 + r < rows && t < s.fresh) {
        const T* q = static_cast<const T*>(a.c.q_dev) + (static_cast<size_t>(b) * a.c.tokens + a.t0 + t) * a.c.ld_q +
                     (kvh * group + row0 + r - t * group) * DH + piece * 8;
        if constexpr (sizeof(T) == 2) {
          const uint4 x = *reinterpret_cast<const uint4*>(q);
          w[0][0] = x.x;
          w[0][1] = x.y;
          w[0][2] = x.z;
          w[0][3] = x.w;
        } else {
          const float4 x = reinterpret_cast<const float4*>(q)[0], y = reinterpret_cast<const float4*>(q)[1];
          const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t part[C::kQTerms];
            split2<C::kQTerms>(v[2 * e], v[2 * e + 1], part);
#pragma unroll
            for (int m = 0; m < C::kQTerms; ++m) w[m][e] = part[m];
          }
        }
      }
#pragma unroll
      for (int m = 0; m < C::kQTerms; ++m) {
        uint32_t* at = reinterpret_cast<uint32_t*>(q_frag + ((m * NT + (r >> 3)) * kSteps + (piece >> 1)) * 32 + (r & 7) * 4) + (piece & 1);
#pragma unroll
        for (int e = 0; e < 4; ++e) at[2 * e] = w[m][e];
      }
    }
    worker_sync();
    if constexpr (kQInRegisters) {
#pragma unroll
      for (int m = 0; m < C::kQTerms; ++m)
#pragma unroll
        for (int i = 0; i < kNt * kSteps; ++i) qr[m * kNt * kSteps + i] = q_frag[((m * NT + nt0) * kSteps + i) * 32 + lane];
    }
    int place[kNt][2];                                                    // slot of the token of rows 2c, 2c + 1; -1: no such row
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = row0 + (nt0 + nt) * 8 + 2 * c + e, t = r / group;
        place[nt][e] = r < rows && t < s.fresh ? first + t : -1;
      }

    float o[kSteps][kNt][4], m[kNt][2], l[kNt][2];
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int d = 0; d < kSteps; ++d) o[d][nt][0] = o[d][nt][1] = o[d][nt][2] = o[d][nt][3] = 0.f;
    }

    for (int i = 0; i < n_tiles && arrived; ++i, ++count) {
      if (count % C::kTeams != team) continue;
      const int st = count % kStages;
      arrived = __all_sync(0xffffffffu, mbar_wait(full_bar(st), (count / kStages) & 1)) != 0;      // the warp goes on or ends as one
      if (!arrived) break;
      const int slot0 = tile_slot[st] + key0;
      if (tile_slot[st] >= 0) {
        const uint32_t sk = ring + st * kTileBytes, sv = sk + kTileBytes / 2;
        // slots of new tokens, and values that nobody sees: behind the sequence, or between the first tokens and the window
        if (slot0 + 16 * kSub > first || (slot0 < low && slot0 + 16 * kSub > a.c.sinks)) {
          unsigned char* pk = ring_ptr + st * kTileBytes;
          const size_t page = static_cast<size_t>(tile_page[st]) * a.c.kv_heads + kvh;
          for (int v = lane; v < 16 * kSub * (DH / 8); v += 32) {
            const int r = v / (DH / 8), piece = v % (DH / 8), j = slot0 + r, t = j - first;
            const uint32_t at = piece_at<kKeys>(key0 + r, piece);
            if (j >= s.length || (j >= a.c.sinks && j < low)) {
              *reinterpret_cast<uint4*>(pk + kTileBytes / 2 + at) = make_uint4(0, 0, 0, 0);
            } else if (t >= 0 && a.c.k_new_dev) {
              const size_t row = static_cast<size_t>(b) * a.c.tokens + a.t0 + t;
              const T* k = static_cast<const T*>(a.c.k_new_dev) + row * a.c.ld_k + kvh * DH + piece * 8;
              const T* w = static_cast<const T*>(a.c.v_new_dev) + row * a.c.ld_v + kvh * DH + piece * 8;
              const uint4 xk = load8_bf16(k), xv = load8_bf16(w);
              *reinterpret_cast<uint4*>(pk + at) = xk;
              *reinterpret_cast<uint4*>(pk + kTileBytes / 2 + at) = xv;
              if (row0 == 0) {
                const size_t dst = (page * kPageTokens + j % kPageTokens) * (DH / 8) + piece;
                static_cast<uint4*>(a.c.kpool_dev)[dst] = xk;
                static_cast<uint4*>(a.c.vpool_dev)[dst] = xv;
              }
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");    // these stores before the next tile's arrival here
          __syncwarp();
        }
        // S^T
        float sc[C::kChains][kSub][kNt][4];
#pragma unroll
        for (int ch = 0; ch < C::kChains; ++ch)
#pragma unroll
          for (int sb = 0; sb < kSub; ++sb)
#pragma unroll
            for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) sc[ch][sb][nt][e] = 0.f;
        const int krow = key0 + (lane & 15);
#pragma unroll
        for (int k0 = 0; k0 < kSteps; k0 += kBlock) {
          uint32_t ka[kBlock][kSub][4];
          float part[kBlock][kSub][kNt][4];
#pragma unroll
          for (int u = 0; u < kBlock; ++u)
#pragma unroll
            for (int sb = 0; sb < kSub; ++sb) {
              ldsm4(ka[u][sb], sk + piece_at<kKeys>(krow + 16 * sb, (k0 + u) * 2 + (lane >> 4)));
#pragma unroll
              for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) part[u][sb][nt][e] = 0.f;
            }
#pragma unroll
          for (int q = 0; q < C::kQTerms; ++q) {
            const int term = C::kQTerms - 1 - q;                         // smallest first
#pragma unroll
            for (int u = 0; u < kBlock; ++u)
#pragma unroll
              for (int nt = 0; nt < kNt; ++nt) {
                uint2 bq;
                if constexpr (kQInRegisters) bq = qr[(term * kNt + nt) * kSteps + k0 + u];
                else bq = q_frag[((term * NT + nt0 + nt) * kSteps + k0 + u) * 32 + lane];
#pragma unroll
                for (int sb = 0; sb < kSub; ++sb)
                  mma16(C::kExactSums ? part[u][sb][nt] : sc[u % C::kChains][sb][nt], ka[u][sb], bq.x, bq.y);
              }
          }
          if constexpr (C::kExactSums) {
#pragma unroll
            for (int u = 0; u < kBlock; ++u)
#pragma unroll
              for (int sb = 0; sb < kSub; ++sb)
#pragma unroll
                for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
                  for (int e = 0; e < 4; ++e) sc[u % C::kChains][sb][nt][e] += part[u][sb][nt][e];
          }
        }
        // weights
        const int last = slot0 + 16 * kSub - 1;
        const bool whole = last <= first && (last < a.c.sinks || s.length - 1 - slot0 < a.c.window);     // every row sees every key
        float v[kSub][kNt][4];
        bool grow = false;
#pragma unroll
        for (int sb = 0; sb < kSub; ++sb)
#pragma unroll
          for (int nt = 0; nt < kNt; ++nt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float y = sc[0][sb][nt][e];
              if (C::kChains == 2) y += sc[C::kChains - 1][sb][nt][e];
              y *= a.scale_log2;
              const int j = slot0 + sb * 16 + g + (e >> 1) * 8, p = place[nt][e & 1];
              if (whole ? p < 0 : (j > p || (j >= a.c.sinks && p - j >= a.c.window))) y = -INFINITY;
              grow |= y > m[nt][e & 1] + kGrowth;
              v[sb][nt][e] = y;
            }
            if (a.scores) {
              // [tile of the line][key][row]
              const size_t at = (static_cast<size_t>(x + i) * kKeys + key0 + sb * 16 + g) * a.score_rows;
              const int r = (nt0 + nt) * 8 + 2 * c;
              if (a.score_rows == 1) {
                if (r == 0) {
                  a.scores[at] = v[sb][nt][0];
                  a.scores[at + 8] = v[sb][nt][2];
                }
              } else if (r < a.score_rows) {
                *reinterpret_cast<float2*>(a.scores + at + r) = make_float2(v[sb][nt][0], v[sb][nt][1]);
                *reinterpret_cast<float2*>(a.scores + at + 8 * a.score_rows + r) = make_float2(v[sb][nt][2], v[sb][nt][3]);
              }
            }
          }
        // the maxima that weights refer to move when a score exceeds one by more than kGrowth
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int nt = 0; nt < kNt; ++nt) {
            float corr[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float top = m[nt][e];
#pragma unroll
              for (int sb = 0; sb < kSub; ++sb) top = fmaxf(top, fmaxf(v[sb][nt][e], v[sb][nt][e + 2]));
#pragma unroll
              for (int sh = 4; sh < 32; sh <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, sh));
              corr[e] = m[nt][e] == top ? 1.f : exp2_fast(m[nt][e] - top);
              m[nt][e] = top;
              l[nt][e] *= corr[e];
            }
#pragma unroll
            for (int d = 0; d < kSteps; ++d)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[d][nt][e] *= corr[e & 1];
          }
        }
        uint32_t pb[C::kPTerms][kSub][kNt][2];
#pragma unroll
        for (int sb = 0; sb < kSub; ++sb)
#pragma unroll
          for (int nt = 0; nt < kNt; ++nt) {
            float* y = v[sb][nt];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float base = m[nt][e] == -INFINITY ? 0.f : m[nt][e];
              y[e] = exp2_fast(y[e] - base);
              y[e + 2] = exp2_fast(y[e + 2] - base);
              l[nt][e] += y[e] + y[e + 2];
            }
            uint32_t lo[C::kPTerms], hi[C::kPTerms];
            split2<C::kPTerms>(y[0], y[1], lo);
            split2<C::kPTerms>(y[2], y[3], hi);
#pragma unroll
            for (int p = 0; p < C::kPTerms; ++p) {
              pb[p][sb][nt][0] = transposed(lo[p]);
              pb[p][sb][nt][1] = transposed(hi[p]);
            }
          }
        // O^T
        const int vrow = key0 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int d0 = 0; d0 < kSteps; d0 += kBlock) {
#pragma unroll
          for (int sb = 0; sb < kSub; ++sb) {
            uint32_t va[kBlock][4];
            float part[kBlock][kNt][4];
#pragma unroll
            for (int u = 0; u < kBlock; ++u) {
              ldsm4_trans(va[u], sv + piece_at<kKeys>(vrow + 16 * sb, (d0 + u) * 2 + ((lane >> 3) & 1)));
#pragma unroll
              for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) part[u][nt][e] = 0.f;
            }
#pragma unroll
            for (int p = C::kPTerms - 1; p >= 0; --p)
#pragma unroll
              for (int u = 0; u < kBlock; ++u)
#pragma unroll
                for (int nt = 0; nt < kNt; ++nt)
                  mma16(C::kExactSums ? part[u][nt] : o[d0 + u][nt], va[u], pb[p][sb][nt][0], pb[p][sb][nt][1]);
            if constexpr (C::kExactSums) {
#pragma unroll
              for (int u = 0; u < kBlock; ++u)
#pragma unroll
                for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
                  for (int e = 0; e < 4; ++e) o[d0 + u][nt][e] += part[u][nt][e];
            }
          }
        }
      }
      else if (a.scores) {
        // a page that does not exist: nobody sees its keys
        for (int v = lane; v < 16 * kSub * a.score_rows; v += 32)
          a.scores[(static_cast<size_t>(x + i) * kKeys + key0) * a.score_rows + v] = -INFINITY;
      }
      // every load of the tile has been used by a product that was issued: which lane hands it back hangs on the last one
      const int by = __any_sync(0xffffffffu, __float_as_uint(o[kSteps - 1][kNt - 1][0]) == 0x7fc0deadu) ? 1 : 0;
      if (lane == by) arrive(empty_bar(st));
    }

    // the warps' results: maxima, then two warps a row store what the others of the row, if any, add to
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[nt][e];
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, sh);
        if (g == 0) {
          sm_m[part_id][(nt0 + nt) * 8 + 2 * c + e] = m[nt][e];
          sm_l[part_id][(nt0 + nt) * 8 + 2 * c + e] = sum;
        }
      }
    worker_sync();
    float* mine = o_buf + (part_id & 1) * kRows * C::kLdO;
#pragma unroll
    for (int half = 0; half < C::kParts / 2; ++half) {
      if ((part_id >> 1) == half) {
#pragma unroll
        for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = (nt0 + nt) * 8 + 2 * c + e;
            float top = sm_m[0][r];
#pragma unroll
            for (int w = 1; w < C::kParts; ++w) top = fmaxf(top, sm_m[w][r]);
            const float f = m[nt][e] == -INFINITY ? 0.f : exp2_fast(m[nt][e] - top);
#pragma unroll
            for (int d = 0; d < kSteps; ++d) {
              float* at = mine + r * C::kLdO + d * 16 + g;
              at[0] = half ? fmaf(o[d][nt][e], f, at[0]) : o[d][nt][e] * f;
              at[8] = half ? fmaf(o[d][nt][e + 2], f, at[8]) : o[d][nt][e + 2] * f;
            }
          }
      }
      worker_sync();
    }
    const bool starts = tile0 == 0, whole_unit = starts && n_tiles == s.tiles;
    if (tid == 0 && starts) a.unit_blocks[2 * (b * units + unit)] = blockIdx.x;
    if (tid == 0 && tile0 + n_tiles == s.tiles) a.unit_blocks[2 * (b * units + unit) + 1] = blockIdx.x;
    const size_t part = static_cast<size_t>(blockIdx.x) * 2 + (starts ? 1 : 0);
    for (int i = tid; i < kRows * (DH / 8); i += 32 * kWorkers) {
      const int r = i / (DH / 8), d = i % (DH / 8) * 8, t = (row0 + r) / group;
      const float* p0 = o_buf + r * C::kLdO + d;
      const float* p1 = p0 + kRows * C::kLdO;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = p0[e] + p1[e];
      float top = sm_m[0][r], sum = 0.f;
#pragma unroll
      for (int w = 1; w < C::kParts; ++w) top = fmaxf(top, sm_m[w][r]);
#pragma unroll
      for (int w = 0; w < C::kParts; ++w) sum += sm_m[w][r] == -INFINITY ? 0.f : sm_l[w][r] * exp2_fast(sm_m[w][r] - top);
      if (whole_unit) {
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
        if (row0 + r < rows) {
          T* out = static_cast<T*>(a.c.out_dev) + (static_cast<size_t>(b) * a.c.tokens + a.t0 + t) * a.c.ld_out +
                   (kvh * group + row0 + r - t * group) * DH + d;
          store8(out, v, inv);
        }
      } else {
        float4* dst = reinterpret_cast<float4*>(a.part_o + (part * kRows + r) * DH + d);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
      if (d == 0) {
        if (!whole_unit) a.part_ml[part * kRows + r] = make_float2(top, sum);
        else if (a.lse) a.lse[(static_cast<size_t>(b) * units + unit) * kRows + r] = make_float2(top, sum);
      }
    }
    // the buffers and the queries may be overwritten; a wait that ran out in one warp ends the block's work in all
    if (worker_any(!arrived)) {
      if (tid == 0 && a.c.status_dev) atomicOr(a.c.status_dev, kDevErrTimeout);
      break;
    }
    x += n_tiles;
  }
}

// Second kernel, a sequence and key head by blockIdx.z and .y: the first join_rows blocks in x join a row's parts where several blocks
// worked on its unit, and write the zeros of rows that nobody worked on; the others add the attention weights of kWeightSlots slots.
template <int DH, typename T>
__global__ void __launch_bounds__(kJoinThreads, 4) cache_join_kernel(const CacheFewArgs a, int tile_rows, int join_rows) {
  constexpr int kKeys = 4096 / DH;
  constexpr int kLanes = DH / 4, kGroups = kJoinThreads / kLanes;
  __shared__ float4 sm_o[kGroups][kLanes];
  __shared__ float sm_l[kGroups];
  __shared__ float row_m[32], row_inv[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = a.c.heads / a.c.kv_heads, rows = a.tokens * group, row_tiles = (rows + tile_rows - 1) / tile_rows;
  const int units = a.c.kv_heads * row_tiles;
  const int slots = a.c.pages * kPageTokens;
  const int b = blockIdx.z, kvh = blockIdx.y;
  const bool joins = static_cast<int>(blockIdx.x) < join_rows;
  const int inner = joins ? blockIdx.x : blockIdx.x - join_rows;         // row, or part of the slots
  const FewSeq s = few_seq<kKeys>(a, few_held(a, b, false));
  pdl_wait();
  pdl_launch_dependents();
  // the blocks that worked on a unit: the first one and how many (0: a wait ran out, and which they were is not known)
  auto blocks_of = [&](int unit, int* n) {
    const int2 ends = *reinterpret_cast<const int2*>(a.unit_blocks + 2 * (b * units + unit));
    *n = unit_blocks_of(ends.x, ends.y, a.pieces);
    return ends.x;
  };

  // part k of the unit that lies at [u0, u1) in the line: the end of the first block's piece, then the beginnings of the next ones'
  if (joins) {
    const int row = inner, t = row / group;
    T* out = static_cast<T*>(a.c.out_dev) + (static_cast<size_t>(b) * a.c.tokens + a.t0 + t) * a.c.ld_out + (kvh * group + row - t * group) * DH;
    if (t >= s.fresh) {
      const float zero[8] = {};
      if (tid < DH / 8) store8(out + tid * 8, zero, 0.f);
      return;
    }
    const int unit = kvh * row_tiles + row / tile_rows, r = row % tile_rows;
    int n;
    const int fb = blocks_of(unit, &n);
    if (n == 1) return;                                                  // one block had it all
    if (n == 0) {
      const float zero[8] = {};
      if (tid < DH / 8) store8(out + tid * 8, zero, 0.f);
      if (tid == 0 && a.c.status_dev) atomicOr(a.c.status_dev, kDevErrTimeout);
      return;
    }
    auto part_of = [&](int k) { return (static_cast<size_t>(fb + k) * 2 + (k == 0 ? 1 : 0)) * tile_rows + r; };
    float top = -INFINITY;
    for (int k = lane; k < n; k += 32) top = fmaxf(top, a.part_ml[part_of(k)].x);
    top = warp_max(top);
    const int gl = tid % kLanes, gg = tid / kLanes;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    for (int k = gg; k < n; k += kGroups) {
      const float2 ml = a.part_ml[part_of(k)];
      const float f = ml.x == -INFINITY ? 0.f : exp2_fast(ml.x - top);
      const float4 v = *reinterpret_cast<const float4*>(a.part_o + part_of(k) * DH + gl * 4);
      l = fmaf(ml.y, f, l);
      o.x = fmaf(v.x, f, o.x);
      o.y = fmaf(v.y, f, o.y);
      o.z = fmaf(v.z, f, o.z);
      o.w = fmaf(v.w, f, o.w);
    }
    sm_o[gg][gl] = o;
    if (gl == 0) sm_l[gg] = l;
    __syncthreads();
    if (tid < DH / 8) {
      float v[8] = {};
      l = 0.f;
      for (int k = 0; k < kGroups; ++k) {
        const float4 x = sm_o[k][tid * 2], y = sm_o[k][tid * 2 + 1];
        v[0] += x.x;
        v[1] += x.y;
        v[2] += x.z;
        v[3] += x.w;
        v[4] += y.x;
        v[5] += y.y;
        v[6] += y.z;
        v[7] += y.w;
        l += sm_l[k];
      }
      store8(out + tid * 8, v, l != 0.f ? 1.f / l : 0.f);
    }
    return;
  }

  // attention weights
  if (inner * kWeightSlots >= s.length) return;
  const size_t base = (static_cast<size_t>(b) * a.c.kv_heads + kvh) * slots;
  constexpr int kEach = kWeightSlots / kJoinThreads;
  float sum[kEach], old[kEach];
  int at_key[kEach];                                                     // where the slot's scores stand in its units, in keys; -1: nobody sees it
  const int fresh0 = s.length - s.fresh;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = inner * kWeightSlots + i * kJoinThreads + tid, tl = j / kKeys;
    sum[i] = 0.f;
    old[i] = a.c.weights_in_dev && j < fresh0 ? a.c.weights_in_dev[base + j] : 0.f;
    const int tile = tl < s.sink_tiles ? tl : tl >= s.low_tile ? s.sink_tiles + tl - s.low_tile : -1;
    at_key[i] = j < s.length && s.tiles > 0 && tile >= 0 ? tile * kKeys + j % kKeys : -1;
  }
  const bool fours = (a.score_rows & 3) == 0;
  for (int rt = 0; rt < (s.tiles > 0 ? row_tiles : 0); ++rt) {
    const int unit = kvh * row_tiles + rt, live = min(tile_rows, rows - rt * tile_rows);
    const float* scores = a.scores + static_cast<size_t>(a.prefix[b] + unit * s.tiles) * kKeys * a.score_rows;
    // the first rows' scores are on their way while the rows' maxima and sums are put together
    float4 head[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (fours && at_key[i] >= 0) head[i] = *reinterpret_cast<const float4*>(scores + static_cast<size_t>(at_key[i]) * a.score_rows);
    int n;
    const int fb = blocks_of(unit, &n);
    if (n == 0) {
      if (tid == 0 && a.c.status_dev) atomicOr(a.c.status_dev, kDevErrTimeout);
      continue;
    }
    __syncthreads();                                                     // the tile before has been worked off
    for (int r = warp; r < live; r += kJoinThreads / 32) {
      float top = -INFINITY, l = 0.f;
      if (n == 1) {
        const float2 ml = a.lse[(static_cast<size_t>(b) * units + unit) * tile_rows + r];
        top = ml.x;
        l = ml.y;
      } else {
        auto part_of = [&](int k) { return (static_cast<size_t>(fb + k) * 2 + (k == 0 ? 1 : 0)) * tile_rows + r; };
        for (int k = lane; k < n; k += 32) top = fmaxf(top, a.part_ml[part_of(k)].x);
        top = warp_max(top);
        for (int k = lane; k < n; k += 32) {
          const float2 ml = a.part_ml[part_of(k)];
          if (ml.x > -INFINITY) l = fmaf(ml.y, exp2_fast(ml.x - top), l);
        }
        l = warp_sum(l);
      }
      if (lane == 0) {
        row_m[r] = top == -INFINITY ? 0.f : top;
        row_inv[r] = l != 0.f ? 1.f / l : 0.f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (at_key[i] < 0) continue;
      const float* sc = scores + static_cast<size_t>(at_key[i]) * a.score_rows;
      for (int r = 0; r < live; r += 4) {
        float4 x = head[i];
        if (!fours) {
          x.x = sc[r];
          x.y = r + 1 < live ? sc[r + 1] : -INFINITY;
          x.z = r + 2 < live ? sc[r + 2] : -INFINITY;
          x.w = r + 3 < live ? sc[r + 3] : -INFINITY;
        } else if (r > 0) {
          x = *reinterpret_cast<const float4*>(sc + r);
        }
        sum[i] = fmaf(exp2_fast(x.x - row_m[r]), row_inv[r], sum[i]);
        if (r + 1 < live) sum[i] = fmaf(exp2_fast(x.y - row_m[r + 1]), row_inv[r + 1], sum[i]);
        if (r + 2 < live) sum[i] = fmaf(exp2_fast(x.z - row_m[r + 2]), row_inv[r + 2], sum[i]);
        if (r + 3 < live) sum[i] = fmaf(exp2_fast(x.w - row_m[r + 3]), row_inv[r + 3], sum[i]);
      }
    }
  }
  const bool in_place = a.c.weights_in_dev == a.c.weights_out_dev;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = inner * kWeightSlots + i * kJoinThreads + tid;
    if (j < s.length && (at_key[i] >= 0 || !in_place || j >= fresh0)) a.c.weights_out_dev[base + j] = old[i] + sum[i];
  }
}

// Most rows of a tile: what the accumulators (d_head / 2 registers for 8 rows) and the 32-bit queries' three terms leave room for.
int widest_tile(const mtj_cache_attn_args& c) {
  const int rows = c.d_head == 256 ? 16 : 32;
  return c.dtype == MTJ_F32 && c.d_head > 64 ? rows / 2 : rows;
}
// as few tiles as can be, and those as narrow as hold the rows (24 rows of 8 x 8 heads behind 8000 slots, in tiles of 24 / 32: 64-wide
// 55 / 70 us, 128-wide 78 / 84)
int tile_rows_for(int rows, int widest) {
  const int tiles = (rows + widest - 1) / widest;
  return ((rows + tiles - 1) / tiles + 7) / 8 * 8;
}

// tiles that a sequence's slice can see at most
int64_t most_tiles(const mtj_cache_attn_args& c, int tokens) {
  const int64_t keys = 4096 / c.d_head, slots = static_cast<int64_t>(c.pages) * kPageTokens;
  const int64_t seen = std::min<int64_t>(slots, static_cast<int64_t>(c.window) + tokens + std::min<int64_t>(c.sinks, slots));
  return std::min(slots / keys, seen / keys + 3);
}

template <int DH, int NT, typename T>
cudaError_t launch(const CacheFewArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, int pieces, cudaStream_t s) {
  using C = FewCfg<DH, NT, T>;
  static DeviceOnce once;
  cudaError_t e = once.run([&] {
    return cudaFuncSetAttribute(cache_few_kernel<DH, NT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(C::kSmem));
  });
  if (e != cudaSuccess) return e;
  e = launch_pdl(cache_few_kernel<DH, NT, T>, dim3(pieces), dim3(kFewThreads), C::kSmem, s, false, mk, mv, a);
  if (e != cudaSuccess) return e;
  const int join = a.whole ? 0 : a.tokens * (a.c.heads / a.c.kv_heads);
  const int weigh = a.c.weights_out_dev ? (a.c.pages * kPageTokens + kWeightSlots - 1) / kWeightSlots : 0;
  if (join + weigh == 0) return cudaSuccess;
  return launch_pdl(cache_join_kernel<DH, T>, dim3(join + weigh, a.c.kv_heads, a.c.batch), dim3(kJoinThreads), 0, s, true, a, C::kRows, join);
}

template <int DH, typename T>
cudaError_t launch_rows(const CacheFewArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, int tile_rows, int pieces, cudaStream_t s) {
  if (tile_rows == 8) return launch<DH, 1, T>(a, mk, mv, pieces, s);
  constexpr bool kWide = sizeof(T) == 2 || DH == 64;       // as widest_tile()
  if constexpr (DH == 128 || kWide) {
    if (tile_rows == 16) return launch<DH, 2, T>(a, mk, mv, pieces, s);
  }
  if constexpr (DH < 256 && kWide) {
    if (tile_rows == 24) return launch<DH, 3, T>(a, mk, mv, pieces, s);
    if (tile_rows == 32) return launch<DH, 4, T>(a, mk, mv, pieces, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

CacheFewPlan plan_cache_few(const mtj_cache_attn_args& c) {
  CacheFewPlan p = {};
  const int group = c.heads / c.kv_heads, widest = widest_tile(c);
  // tokens of a slice: up to four row tiles (each reads the keys again, from L2)
  p.tokens = std::min(c.tokens, std::max(1, 4 * widest / group));
  const int rows = p.tokens * group;
  p.tile_rows = tile_rows_for(rows, widest);
  p.batch = std::min(c.batch, kFewBatch);
  const int64_t units = static_cast<int64_t>(p.batch) * c.kv_heads * ((rows + p.tile_rows - 1) / p.tile_rows);
  const int64_t tiles = units * most_tiles(c, p.tokens);
  p.aligned = units <= kPieces / 2;
  const int nt = p.tile_rows / 8;
  p.teams = kWorkers / (4096 / c.d_head / (16 * few_sub(c.d_head, nt)) * (nt / few_n_tiles(c.d_head, nt)));      // as FewCfg has them
  // up to four rounds of tiles the second kernel costs more than it gives
  p.whole = p.aligned && most_tiles(c, p.tokens) <= 4 * p.teams;
  p.least = p.whole ? 4 * p.teams : p.teams;
  p.pieces = static_cast<int>(p.aligned ? std::min<int64_t>(kPieces, units * ((most_tiles(c, p.tokens) + p.least - 1) / p.least))
                                        : std::min<int64_t>(kPieces, tiles));
  p.score_rows = rows == 1 ? 1 : std::min(p.tile_rows, (rows + 1) / 2 * 2);
  auto take = [&](int64_t bytes) {
    const int64_t at = p.total;
    p.total += (bytes + 255) / 256 * 256;
    return at;
  };
  p.prefix_off = take((kFewBatch + 1) * 4);
  p.units_off = take(units * 8);
  p.ml_off = take(static_cast<int64_t>(p.pieces) * 2 * p.tile_rows * 8);
  p.o_off = take(static_cast<int64_t>(p.pieces) * 2 * p.tile_rows * c.d_head * 4);
  p.lse_off = take(c.weights_out_dev ? units * p.tile_rows * 8 : 0);
  p.scores_off = take(c.weights_out_dev ? tiles * (4096 / c.d_head) * p.score_rows * 4 : 0);
  return p;
}

cudaError_t run_cache_few(const mtj_cache_attn_args& c, const CacheFewPlan& p, char* scratch, cudaStream_t s) {
  CUtensorMap mk, mv;
  const int64_t pool_rows = static_cast<int64_t>(c.n_pages) * c.kv_heads * kPageTokens;
  const int keys = 4096 / c.d_head;
  cudaError_t e = make_tensor_map_bf16(&mk, c.kpool_dev, pool_rows, c.d_head, keys);
  if (e == cudaSuccess) e = make_tensor_map_bf16(&mv, c.vpool_dev, pool_rows, c.d_head, keys);
  if (e != cudaSuccess) return e;
  const size_t type = c.dtype == MTJ_F32 ? 4 : 2;
  const int64_t slots = static_cast<int64_t>(c.pages) * kPageTokens;
  for (int b0 = 0; b0 < c.batch; b0 += p.batch)
    for (int t0 = 0; t0 < c.tokens; t0 += p.tokens) {
      CacheFewArgs a = {};
      a.c = c;
      a.t0 = t0;
      a.tokens = std::min(p.tokens, c.tokens - t0);
      a.c.batch = std::min(p.batch, c.batch - b0);
      a.c.page_table_dev += static_cast<size_t>(b0) * c.pages;
      a.c.lengths_dev += b0;
      if (c.new_tokens_dev) a.c.new_tokens_dev += b0;
      auto shift = [&](auto*& q, int64_t ld) {
        if (q) q = reinterpret_cast<std::remove_reference_t<decltype(q)>>(
                   reinterpret_cast<uintptr_t>(q) + static_cast<size_t>(b0) * c.tokens * ld * type);
      };
      shift(a.c.q_dev, c.ld_q);
      shift(a.c.k_new_dev, c.ld_k);
      shift(a.c.v_new_dev, c.ld_v);
      shift(a.c.out_dev, c.ld_out);
      if (c.weights_out_dev) {
        // later slices add to what the earlier ones left; their tokens' slots begin at zero in their turn
        if (t0 > 0) a.c.weights_in_dev = c.weights_out_dev;
        if (a.c.weights_in_dev) a.c.weights_in_dev += static_cast<size_t>(b0) * c.kv_heads * slots;
        a.c.weights_out_dev += static_cast<size_t>(b0) * c.kv_heads * slots;
        a.lse = reinterpret_cast<float2*>(scratch + p.lse_off);
        a.scores = reinterpret_cast<float*>(scratch + p.scores_off);
      }
      a.scale_log2 = c.scale * 1.4426950408889634f;
      a.score_rows = p.score_rows;
      a.aligned = p.aligned;
      a.whole = p.whole;
      a.least = p.least;
      a.teams = p.teams;
      a.pieces = p.pieces;
      a.prefix = reinterpret_cast<int32_t*>(scratch + p.prefix_off);
      a.unit_blocks = reinterpret_cast<int32_t*>(scratch + p.units_off);
      a.part_ml = reinterpret_cast<float2*>(scratch + p.ml_off);
      a.part_o = reinterpret_cast<float*>(scratch + p.o_off);
      const bool f32 = c.dtype == MTJ_F32;
      if (c.d_head == 64) e = f32 ? launch_rows<64, float>(a, mk, mv, p.tile_rows, p.pieces, s) : launch_rows<64, __nv_bfloat16>(a, mk, mv, p.tile_rows, p.pieces, s);
      else if (c.d_head == 128) e = f32 ? launch_rows<128, float>(a, mk, mv, p.tile_rows, p.pieces, s) : launch_rows<128, __nv_bfloat16>(a, mk, mv, p.tile_rows, p.pieces, s);
      else e = f32 ? launch_rows<256, float>(a, mk, mv, p.tile_rows, p.pieces, s) : launch_rows<256, __nv_bfloat16>(a, mk, mv, p.tile_rows, p.pieces, s);
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

}  // namespace mtj

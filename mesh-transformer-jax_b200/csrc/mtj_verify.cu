// Verification of drafted tokens against the target model's logits (mtj_verify_drafts).
//
// verify_rows_kernel: every row of logits that takes part is read once, kChunk entries a warp at a time: their maximum (greedy: and where it
//   first stands) and the sum of exp((l - maximum) / temp).  A lane holds its entries in registers, so the maximum is known before
//   the first exponential, and has the next ones on their way meanwhile.  The rows that take part stand in one line that is cut into
//   equal pieces, one a warp: rows behind a sequence's drafts cost nothing.
// verify_pick_kernel: a cluster of blocks a sequence.  Every block adds up the chunks of all rows, in 64 bits, and
//   decides alike how many drafts are taken; then the cluster shares out the one row that the next token comes from.
//   The race r_i / -log(noise_i) is run in 32 bits with a bound on the error of every entry; those that can win it are run
//   again in 64 bits, so that the token does not hang on the rounding of a near-tie.  What does
//   not hang on the rows kernel (noise, the drafts' own logits) is read and worked out while that one runs.
//
// What is 32-bit is the sum of a chunk's exponentials, about 1e-7 of itself off (2^-18 at most); sums over chunks, the drafts' shares, their
// comparison and the entries that decide the race are 64-bit.  Which side of u q < p and of p > q an entry is on thus holds for shares that
// are further apart than that; closer ones are decided by the rounding of their rows' sums.
// Bound by the bytes of the logits.  64 sequences of up to 7 drafts, 50400
// entries in 32 bits: 26 us for 103 MB of rows (4.0 TB/s) and 25 us for the race alone, 41 us together, since the race reads its noise and
// takes the logarithms while the rows are read.  (With logf and divisions instead of approximations and their bounds 29 and 45 us.)
#include <math.h>

#include <algorithm>
#include <string>

#include "mtj_cache.cuh"
#include "mtj_kernels.h"

namespace mtj {
namespace {

constexpr int kRowThreads = 768;
constexpr int kPerLane = 32;
constexpr int kChunk = 32 * kPerLane;
constexpr int kRowBlocks = 148;            // one an SM
constexpr int kRowBatch = 4096;            // sequences of a launch
constexpr int kMostDrafts = 1024;          // of a sequence
constexpr int kPickThreads = 512;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kPickCluster = 8;
constexpr int kHeld = 16;                  // entries of the race that a thread has at once
constexpr float kLowestTemp = 8.673617e-19f;      // 2^-60
constexpr float kLog2e = 1.442695041f;

struct ChunkStat {
  float top, sum;      // largest entry; sum of exp((l - top) / temp) over the chunk, NaN where an entry is
  int32_t at, pad;     // where it first stands (greedy)
};

__device__ __forceinline__ float value_at(const float* p, int i) { return p[i]; }
__device__ __forceinline__ float value_at(const __nv_bfloat16* p, int i) { return __bfloat162float(p[i]); }

__device__ __forceinline__ int drafts_of(const mtj_verify_args& a, int b) {
  return a.counts_dev ? min(max(a.counts_dev[b], 0), a.drafts) : a.drafts;
}
__device__ __forceinline__ float temp_of(const mtj_verify_args& a, int b) { return a.temp_dev ? a.temp_dev[b] : a.temp; }
// no temperature (nor one so low that scaled logits leave 32 bits): the largest logit has it all
__device__ __forceinline__ bool is_greedy(float temp) { return !(temp >= kLowestTemp); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t two(float x, float y) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
__device__ __forceinline__ void untwo(uint64_t d, float* x, float* y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(*x), "=f"(*y) : "l"(d)); }

// rows of one sequence: 0 .. drafts the target's, then the draft's
template <typename T>
__device__ __forceinline__ const T* row_of(const mtj_verify_args& a, int b, int r) {
  return r <= a.drafts ? static_cast<const T*>(a.target_dev) + b * a.batch_target + r * a.ld_target
                       : static_cast<const T*>(a.draft_dev) + b * a.batch_draft + (r - a.drafts - 1) * a.ld_draft;
}
// how many of them take part: the target's 0 .. n, the draft's 0 .. n - 1 where the target does not choose by itself
__device__ __forceinline__ int rows_in(const mtj_verify_args& a, int b) {
  const int n = drafts_of(a, b);
  return n + 1 + (a.draft_dev && !is_greedy(temp_of(a, b)) ? n : 0);
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads, 1) verify_rows_kernel(const mtj_verify_args a, ChunkStat* stats, int rows, int chunks) {
  constexpr int kVec = 16 / sizeof(T), kLoads = kPerLane / kVec;
  __shared__ int before[kRowBatch + 1], scan[kRowThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  // before[b]: rows of the line before sequence b
  {
    const int per = (a.batch + kRowThreads - 1) / kRowThreads, b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
    int sum = 0;
    for (int b = b0; b < b1; ++b) sum += before[b] = rows_in(a, b);
    int x = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    x -= sum;
    int all = 0;
    for (int w = 0; w < kRowThreads / 32; ++w) {
      if (w < warp) x += scan[w];
      all += scan[w];
    }
    for (int b = b0; b < b1; ++b) {
      const int n = before[b];
      before[b] = x;
      x += n;
    }
    if (tid == 0) before[a.batch] = all;
    __syncthreads();
  }
  const int64_t line = static_cast<int64_t>(before[a.batch]) * chunks;
  // pieces are dealt out block by block, so that a short line has all SMs
  const int64_t worker = static_cast<int64_t>(warp) * gridDim.x + blockIdx.x, workers = static_cast<int64_t>(gridDim.x) * (kRowThreads / 32);
  const int64_t begin = line * worker / workers, end = line * (worker + 1) / workers;

  // where this warp is in the line; the next chunk is looked up while the last one's entries are worked on
  struct Place {
    int b, k, c, n, rows;      // sequence, row and chunk of it; drafted tokens, rows that take part
  } at = {};
  struct Item {
    const T* row;
    ChunkStat* out;
    int i0;                    // first entry: chunks begin at 16-byte boundaries, up to a vector before the row's first entry
    float temp;
  };
  auto enter = [&]() {
    at.n = drafts_of(a, at.b);
    at.rows = before[at.b + 1] - before[at.b];
  };
  auto item = [&]() {
    const int r = at.k <= at.n ? at.k : a.drafts + at.k - at.n;
    Item it;
    it.row = row_of<T>(a, at.b, r);
    it.out = stats + (static_cast<int64_t>(at.b) * rows + r) * chunks + at.c;
    it.i0 = at.c * kChunk - static_cast<int>((reinterpret_cast<uintptr_t>(it.row) & 15) / sizeof(T));
    it.temp = temp_of(a, at.b);
    return it;
  };
  auto step = [&]() {
    if (++at.c < chunks) return;
    at.c = 0;
    if (++at.k < at.rows) return;
    at.k = 0;
    ++at.b;                    // every sequence has a row
    enter();
  };
  auto fetch = [&](const Item& it, uint4* x) {
    if (it.i0 >= 0 && it.i0 + kChunk <= a.vocab) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) x[u] = ld_cached16(it.row + it.i0 + (u * 32 + lane) * kVec);
      return;
    }
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      // a row's ends
      const int i = it.i0 + (u * 32 + lane) * kVec;
      float v[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = i + e >= 0 && i + e < a.vocab ? value_at(it.row, i + e) : -INFINITY;
      if constexpr (sizeof(T) == 4)
        x[u] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      else
        x[u] = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4 % kVec], v[5 % kVec]), pack_bf16x2(v[6 % kVec], v[7 % kVec]));
    }
  };
  auto entry = [&](const uint4* x, int u, int e) {
    const int word = e * static_cast<int>(sizeof(T)) >> 2;
    const uint32_t w = word == 0 ? x[u].x : word == 1 ? x[u].y : word == 2 ? x[u].z : x[u].w;
    if constexpr (sizeof(T) == 4) return __uint_as_float(w);
    else return e & 1 ? bf16_hi(w) : bf16_lo(w);
  };
  auto work = [&](const Item& it, const uint4* x) {
    float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
#pragma unroll
      for (int e = 0; e < kVec; e += 4) {
        asm("max.f32 %0, %0, %1, %2;" : "+f"(t0) : "f"(entry(x, u, e)), "f"(entry(x, u, e + 1)));
        asm("max.f32 %0, %0, %1, %2;" : "+f"(t1) : "f"(entry(x, u, e + 2)), "f"(entry(x, u, e + 3)));
      }
    const float top = warp_max(fmaxf(t0, t1));
    int where = 0x7fffffff;
    float sum = 0.f;
    if (is_greedy(it.temp)) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u)
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (entry(x, u, e) == top) where = min(where, it.i0 + (u * 32 + lane) * kVec + e);
      where = static_cast<int>(__reduce_min_sync(0xffffffffu, static_cast<unsigned>(where)));
    } else if (top > -INFINITY) {
      // 2^((l - top) scale): the largest entry is taken away first.  (l scale - top scale in one rounding has top scale's own rounding in
      // every exponent, 2^-24 of a number that has no bound: at temperatures below 1e-3 more than the shares have bits.)
      const float scale = kLog2e / it.temp;
      const uint64_t scale2 = two(scale, scale), top2 = two(-top, -top);
      uint64_t s0 = 0, s1 = 0;
#pragma unroll
      for (int u = 0; u < kLoads; ++u)
#pragma unroll
        for (int e = 0; e < kVec; e += 4) {
          uint64_t y0, y1;
          float f0, f1, f2, f3;
          asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y0) : "l"(two(entry(x, u, e), entry(x, u, e + 1))), "l"(top2));
          asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y1) : "l"(two(entry(x, u, e + 2), entry(x, u, e + 3))), "l"(top2));
          asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(y0) : "l"(scale2));
          asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(y1) : "l"(scale2));
          untwo(y0, &f0, &f1);
          untwo(y1, &f2, &f3);
          asm("add.rn.f32x2 %0, %0, %1;" : "+l"(s0) : "l"(two(ex2(f0), ex2(f1))));
          asm("add.rn.f32x2 %0, %0, %1;" : "+l"(s1) : "l"(two(ex2(f2), ex2(f3))));
        }
      float f0, f1, f2, f3;
      untwo(s0, &f0, &f1);
      untwo(s1, &f2, &f3);
      sum = warp_sum((f0 + f1) + (f2 + f3));
    } else {
      // nothing above -inf; the maximum has passed over NaN
      bool nan = false;
#pragma unroll
      for (int u = 0; u < kLoads; ++u)
#pragma unroll
        for (int e = 0; e < kVec; ++e) nan |= entry(x, u, e) != entry(x, u, e);
      if (__any_sync(0xffffffffu, nan)) sum = NAN;
    }
    if (lane == 0) *it.out = {top, sum, where, 0};
  };
  if (begin >= end) return;
  {
    const int64_t line_row = begin / chunks;
    at.c = static_cast<int>(begin - line_row * chunks);
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (before[mid] <= line_row) lo = mid;
      else hi = mid - 1;
    }
    at.b = lo;
    at.k = static_cast<int>(line_row) - before[lo];
    enter();
  }
  uint4 x[2][kLoads];
  Item it[2];
  it[0] = item();
  fetch(it[0], x[0]);
  for (int64_t i = begin; i < end; i += 2) {
    if (i + 1 < end) {
      step();
      it[1] = item();
      fetch(it[1], x[1]);
    }
    work(it[0], x[0]);
    if (i + 1 >= end) break;
    if (i + 2 < end) {
      step();
      it[0] = item();
      fetch(it[0], x[0]);
    }
    work(it[1], x[1]);
  }
}

struct RowShare {
  float top;           // largest logit of the row
  int at;              // its first place
  double sum;          // sum of exp((l - top) / temp); NaN: the row has no shares
  double log_sum;
};

// log of the share of logit l in a row
__device__ __forceinline__ double log_share(const RowShare& s, float l, double temp) {
  return (static_cast<double>(l) - static_cast<double>(s.top)) / temp - s.log_sum;
}
__device__ __forceinline__ double share(const RowShare& s, float l, double temp) {
  return l == s.top ? 1.0 / s.sum : exp((static_cast<double>(l) - static_cast<double>(s.top)) / temp) / s.sum;
}

struct Racer {
  double score;
  int at;
  float l;             // its logit
};
__device__ __forceinline__ void take_better(Racer& x, const Racer& y) {
  if (y.score > x.score || (y.score == x.score && y.at < x.at)) x = y;
}
__device__ __forceinline__ Racer from_lane(const Racer& x, int mask) {
  return {__shfl_xor_sync(0xffffffffu, x.score, mask), __shfl_xor_sync(0xffffffffu, x.at, mask), __shfl_xor_sync(0xffffffffu, x.l, mask)};
}

__device__ __forceinline__ uint32_t pick_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void pick_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void put_to_first(Racer* slot, const Racer& x) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_u32(slot)));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(x.score) : "memory");
  asm volatile("st.shared::cluster.u32 [%0 + 8], %1;" ::"r"(at), "r"(x.at) : "memory");
  asm volatile("st.shared::cluster.f32 [%0 + 12], %1;" ::"r"(at), "f"(x.l) : "memory");
}

// Blocks of a cluster a sequence: as many as keep two an SM, up to eight.
template <typename T>
__global__ void __launch_bounds__(kPickThreads, 2) verify_pick_kernel(const mtj_verify_args a, const ChunkStat* stats, int rows, int chunks,
                                                                   int cluster) {
  extern __shared__ RowShare row_share[];          // [rows]
  __shared__ float sm_best[kPickWarps];
  __shared__ Racer sm_win[kPickWarps], racers[kPickCluster];      // of the warps; in the first block, of the blocks
  __shared__ int s_taken;
  const int b = blockIdx.x / cluster, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = pick_rank();
  const int n = drafts_of(a, b), n_out = a.drafts + 1;
  const float temp = temp_of(a, b);
  const bool greedy = is_greedy(temp);
  const int32_t* tokens = a.draft_tokens_dev + static_cast<size_t>(b) * a.drafts;
  const float* noise = a.noise_dev + static_cast<size_t>(b) * a.vocab;
  const int per = (a.vocab + cluster - 1) / cluster;
  const int i0 = static_cast<int>(rank) * per, i1 = min(a.vocab, i0 + per);
  pick_sync();                                     // all blocks of the cluster are there: the first one's memory may be written

  // before the rows kernel has ended: the drafts' own entries (the first 32), the noise
  int x0 = -1;
  float p0 = 0.f, q0 = 0.f, u0 = 0.f, wait_of[kHeld];
  if (warp == 0 && lane < n) {
    x0 = tokens[lane];
    if (x0 < 0 || x0 >= a.vocab) x0 = -1;
    if (x0 >= 0 && !greedy) {
      p0 = value_at(row_of<T>(a, b, lane), x0);
      if (a.draft_dev) q0 = value_at(row_of<T>(a, b, a.drafts + 1 + lane), x0);
      u0 = a.accept_dev[static_cast<size_t>(b) * a.drafts + lane];
    }
  }
  // -log2 of the noise, off by at most 2^-22 (1 + itself); beyond [tiny, 1) nothing is waited for
  auto fetch_noise = [&](int first) {
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      const int i = first + h * kPickThreads + tid;
      wait_of[h] = i < i1 ? noise[i] : 1.f;
    }
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      if (first + h * kPickThreads >= i1) break;             // none of the block's
      wait_of[h] = wait_of[h] < 1.f ? -lg2(wait_of[h]) : INFINITY;
    }
  };
  if (!greedy) fetch_noise(i0);
  const float p0_first = p0;                       // of draft `lane`
  pdl_wait();
  const double t64 = greedy ? 1.0 : static_cast<double>(temp), inv_t64 = 1.0 / t64;
  for (int r = warp; r < rows; r += kPickWarps) {
    if (r <= a.drafts ? r > n : (r - a.drafts - 1 >= n || greedy)) continue;
    const ChunkStat* st = stats + (static_cast<int64_t>(b) * rows + r) * chunks;
    constexpr int kSeen = 2;                       // chunks that a lane keeps: vocabularies up to 65536 are read once
    ChunkStat seen[kSeen];
#pragma unroll
    for (int i = 0; i < kSeen; ++i) seen[i] = lane + 32 * i < chunks ? st[lane + 32 * i] : ChunkStat{-INFINITY, 0.f, 0x7fffffff, 0};
    float top = -INFINITY;
    int at = 0x7fffffff;
    auto larger = [&](const ChunkStat& s) {
      if (s.top > top) {
        top = s.top;
        at = s.at;
      }
    };
#pragma unroll
    for (int i = 0; i < kSeen; ++i) larger(seen[i]);
    for (int c = lane + 32 * kSeen; c < chunks; c += 32) larger(st[c]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float t2 = __shfl_xor_sync(0xffffffffu, top, o);
      const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
      if (t2 > top || (t2 == top && a2 < at)) {
        top = t2;
        at = a2;
      }
    }
    double sum = 0.0;
    if (!greedy) {
      auto add = [&](const ChunkStat& s) {
        if (s.top > -INFINITY)
          sum += static_cast<double>(s.sum) * (s.top == top ? 1.0 : exp((static_cast<double>(s.top) - static_cast<double>(top)) * inv_t64));
        else
          sum += static_cast<double>(s.sum);       // 0 or NaN
      };
#pragma unroll
      for (int i = 0; i < kSeen; ++i) add(seen[i]);
      for (int c = lane + 32 * kSeen; c < chunks; c += 32) add(st[c]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (!(sum > 0.0)) sum = NAN;                   // a row without shares: NaN or +inf in it, or nothing above -inf
    if (lane == 0) row_share[r] = {top, greedy && top > -INFINITY ? at : 0, sum, greedy ? 0.0 : log(sum)};
  }
  __syncthreads();
  if (warp == 0) {
    int taken = 0;
    for (int k0 = 0; k0 < n && taken == k0; k0 += 32) {
      const int k = k0 + lane;
      bool good = false;
      if (k < n) {
        if (k0 > 0) {
          x0 = tokens[k];
          if (x0 < 0 || x0 >= a.vocab) x0 = -1;
          if (x0 >= 0 && !greedy) {
            p0 = value_at(row_of<T>(a, b, k), x0);
            if (a.draft_dev) q0 = value_at(row_of<T>(a, b, a.drafts + 1 + k), x0);
            u0 = a.accept_dev[static_cast<size_t>(b) * a.drafts + k];
          }
        }
        if (x0 >= 0) {
          if (greedy) {
            good = x0 == row_share[k].at;
          } else {
            const double p = share(row_share[k], p0, t64);
            const double q = a.draft_dev ? share(row_share[a.drafts + 1 + k], q0, t64) : 1.0;
            good = static_cast<double>(u0) * q < p;
          }
        }
      }
      const uint32_t no = ~__ballot_sync(0xffffffffu, good);
      taken += min(no ? __ffs(no) - 1 : 32, n - k0);
    }
    if (lane == 0) s_taken = taken;
  }
  __syncthreads();
  const int taken = s_taken;
  // the taken tokens, while the next one is looked for
  int32_t* out = a.tokens_out_dev + static_cast<size_t>(b) * n_out;
  float* logs = a.logprobs_out_dev ? a.logprobs_out_dev + static_cast<size_t>(b) * n_out : nullptr;
  if (rank == 0 && warp == 0) {
    for (int k = lane; k < n_out; k += 32) {
      if (k == taken) continue;
      out[k] = k < taken ? tokens[k] : -1;
      if (logs) logs[k] = k >= taken || greedy ? 0.f : static_cast<float>(log_share(row_share[k], k < 32 ? p0_first : value_at(row_of<T>(a, b, k), tokens[k]), t64));
    }
    if (lane == 0) a.accepted_out_dev[b] = taken;
  }
  int next;
  float next_log = 0.f;
  if (greedy) {
    next = row_share[taken].at;
  } else {
    const T* prow = row_of<T>(a, b, taken);
    const RowShare ps = row_share[taken];
    const bool refused = taken < n;
    const bool known = refused && a.draft_dev;
    const T* qrow = known ? row_of<T>(a, b, a.drafts + 1 + taken) : prow;
    const RowShare qs = known ? row_share[a.drafts + 1 + taken] : ps;
    const int without = refused && !known ? tokens[taken] : -1;
    const float scale = kLog2e / temp;
    const float p_inv = static_cast<float>(1.0 / ps.sum), q_inv = known ? static_cast<float>(1.0 / qs.sum) : 0.f;
    // on a share: its argument, up to 126, has the roundings of the difference, of the scale's quotient and of the product and the error of the
    // scale's constant, 126 ln 2 (3 * 2^-24 + 2^-26) = 1.67e-5 at most; the exponential's 2^-22, the reciprocal sum's, the share's and
    // the difference's roundings make it 1.73e-5, half of what is allowed for
    constexpr float kSlack = 3.0517578125e-5f;                         // 2^-15
    constexpr float kLogSlack = 4.76837158e-7f;                        // 2^-21
    // two shares below 2^-126 count as zero in 32 bits: where no difference is larger, everything is run in 64 bits
    constexpr float kLeast = 2.35098870e-38f;                          // 2^-125
    Racer win = {0.0, 0x7fffffff, 0.f};
    auto run = [&](int i, bool difference) {
      const float l = value_at(prow, i);
      const double p = share(ps, l, t64);
      const double q = !difference ? 0.0 : known ? share(qs, value_at(qrow, i), t64) : i == without ? p : 0.0;
      const double r = p - q;
      if (r > 0.0) take_better(win, {r / -log(static_cast<double>(noise[i])), i, l});
    };
    // 32 bits: this block's entries, kHeld a thread at a time, their lower bounds, and whose upper bound reaches the best of them
    float best = 0.f;
    for (int first = i0; first < i1; first += kHeld * kPickThreads) {
      if (first > i0) fetch_noise(first);
      float lp[kHeld], upper[kHeld];
#pragma unroll
      for (int h = 0; h < kHeld; ++h) {
        const int i = first + h * kPickThreads + tid;
        lp[h] = i < i1 ? value_at(prow, i) : -INFINITY;
        upper[h] = i < i1 && known ? value_at(qrow, i) : -INFINITY;
      }
#pragma unroll
      for (int h = 0; h < kHeld; ++h) {
        if (first + h * kPickThreads >= i1) break;
        const float p = ex2((lp[h] - ps.top) * scale) * p_inv;
        const float q = known ? ex2((upper[h] - qs.top) * scale) * q_inv : 0.f;
        const bool out = first + h * kPickThreads + tid == without;
        const float r = out ? 0.f : p - q, slack = out ? 0.f : kSlack * (p + q);
        // the wait's bounds are its own error's twice over; quotients are within 2^-21
        const float late = fmaf(wait_of[h], 1.f + kLogSlack, kLogSlack), soon = fmaf(wait_of[h], 1.f - kLogSlack, -kLogSlack);
        best = fmaxf(best, (r - slack - kLeast) * (1.f - 4e-6f) * reciprocal(late));
        upper[h] = (r + slack + kLeast) * (1.f + 4e-6f) * (soon > 0.f ? reciprocal(soon) : INFINITY);
      }
      best = warp_max(best);
      if (lane == 0) sm_best[warp] = best;
      __syncthreads();
      best = warp_max(lane < kPickWarps ? sm_best[lane] : 0.f);
      __syncthreads();
      uint32_t can = 0;
#pragma unroll
      for (int h = 0; h < kHeld; ++h) {
        if (first + h * kPickThreads >= i1) break;
        if (upper[h] > 0.f && upper[h] >= best && first + h * kPickThreads + tid < i1) can |= 1u << h;
      }
      for (; can; can &= can - 1) run(first + (__ffs(can) - 1) * kPickThreads + tid, true);
    }
    auto block_best = [&]() {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) take_better(win, from_lane(win, o));
      if (lane == 0) sm_win[warp] = win;
      __syncthreads();
      win = sm_win[lane % kPickWarps];
#pragma unroll
      for (int o = kPickWarps / 2; o > 0; o >>= 1) take_better(win, from_lane(win, o));
    };
    block_best();
    if (tid == 0) put_to_first(&racers[rank], win);
    pick_sync();
    if (rank != 0) return;
    for (int r = 0; r < cluster; ++r) take_better(win, racers[r]);
    if (win.at >= a.vocab) {
      // the difference is zero everywhere: the target's own shares
      for (int i = tid; i < a.vocab; i += kPickThreads) run(i, false);
      __syncthreads();
      block_best();
    }
    next = win.at < a.vocab ? win.at : 0;
    next_log = static_cast<float>(log_share(ps, win.at < a.vocab ? win.l : value_at(prow, 0), t64));
  }
  if (rank == 0 && tid == 0) {
    out[taken] = next;
    if (logs) logs[taken] = next_log;
  }
}

int rows_of(const mtj_verify_args& a) { return a.drafts + 1 + (a.draft_dev ? a.drafts : 0); }
int chunks_of(const mtj_verify_args& a) { return (a.vocab + kChunk + 15) / kChunk; }      // room for the skew of a row's start
int64_t stats_bytes(const mtj_verify_args& a) {
  return static_cast<int64_t>(std::min(a.batch, kRowBatch)) * rows_of(a) * chunks_of(a) * static_cast<int64_t>(sizeof(ChunkStat));
}

int32_t check_args(const mtj_verify_args* a, std::string* err) {
  auto bad = [&](const char* what) {
    *err = what;
    return static_cast<int32_t>(MTJ_ERR_INVALID);
  };
  if (!a || !a->target_dev || !a->noise_dev || !a->tokens_out_dev || !a->accepted_out_dev) return bad("null argument");
  if (a->batch <= 0 || a->vocab <= 0 || a->drafts < 0) return bad("batch and vocab must be positive, drafts not negative");
  if (a->drafts > 0 && (!a->draft_tokens_dev || !a->accept_dev)) return bad("null argument");
  if (a->drafts > kMostDrafts) return bad("at most 1024 drafted tokens a sequence");
  if (a->dtype != MTJ_F32 && a->dtype != MTJ_BF16) {
    *err = "dtype must be MTJ_F32 or MTJ_BF16";
    return MTJ_ERR_UNSUPPORTED;
  }
  if (!a->temp_dev && a->temp == INFINITY) return bad("temp must be finite");
  const uintptr_t size = a->dtype == MTJ_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(a->target_dev) | reinterpret_cast<uintptr_t>(a->draft_dev)) & (size - 1))
    return bad("logits must be aligned to their type");
  if (a->ld_target < a->vocab || (a->draft_dev && a->ld_draft < a->vocab)) return bad("a row's stride is shorter than the vocabulary");
  if (a->batch_target < 0 || a->batch_draft < 0) return bad("strides must not be negative");
  if (a->vocab > 1 << 30) return bad("the vocabulary is too large");
  if (static_cast<int64_t>(a->batch) * rows_of(*a) > 0x7fffffff / chunks_of(*a)) return bad("batch * drafts * vocab is too large");
  return MTJ_OK;
}

template <typename T>
cudaError_t run(const mtj_verify_args& all, ChunkStat* stats, cudaStream_t s) {
  const int rows = rows_of(all), chunks = chunks_of(all);
  // the shares of 2049 rows are 48 KB and 24 bytes, more than a kernel has without asking
  static DeviceOnce once;
  cudaError_t e = once.run([&] {
    return cudaFuncSetAttribute(verify_pick_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>((2 * kMostDrafts + 1) * sizeof(RowShare)));
  });
  if (e != cudaSuccess) return e;
  for (int b0 = 0; b0 < all.batch; b0 += kRowBatch) {
    mtj_verify_args a = all;
    a.batch = std::min(kRowBatch, all.batch - b0);
    a.target_dev = static_cast<const T*>(all.target_dev) + b0 * all.batch_target;
    if (all.draft_dev) a.draft_dev = static_cast<const T*>(all.draft_dev) + b0 * all.batch_draft;
    const int64_t per = all.drafts;
    if (all.draft_tokens_dev) a.draft_tokens_dev += b0 * per;
    if (all.accept_dev) a.accept_dev += b0 * per;
    a.noise_dev += static_cast<int64_t>(b0) * all.vocab;
    if (all.counts_dev) a.counts_dev += b0;
    if (all.temp_dev) a.temp_dev += b0;
    a.tokens_out_dev += b0 * (per + 1);
    a.accepted_out_dev += b0;
    if (all.logprobs_out_dev) a.logprobs_out_dev += b0 * (per + 1);
    // as many blocks a sequence as leave two an SM, and no more than its entries are worth
    int cluster = kPickCluster;
    while (cluster > 1 && (static_cast<int64_t>(a.batch) * cluster > 2 * kRowBlocks || a.vocab <= cluster / 2 * 2 * kPickThreads)) cluster /= 2;
    // a short line leaves SMs to the blocks of the second kernel, which have something to do before they need its results
    const int64_t items = static_cast<int64_t>(a.batch) * rows * chunks;
    int64_t row_blocks = std::min<int64_t>(kRowBlocks, (items + 5) / 6);
    if (items <= 2 * kRowBlocks * (kRowThreads / 32)) row_blocks = std::min<int64_t>(row_blocks, std::max(kRowBlocks / 2, kRowBlocks - (a.batch * cluster + 1) / 2));
    verify_rows_kernel<T><<<static_cast<unsigned>(row_blocks), kRowThreads, 0, s>>>(a, stats, rows, chunks);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a.batch * cluster));
    cfg.blockDim = dim3(kPickThreads);
    cfg.dynamicSmemBytes = rows * sizeof(RowShare);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {static_cast<unsigned>(cluster), 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, verify_pick_kernel<T>, a, static_cast<const ChunkStat*>(stats), rows, chunks, cluster);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace
}  // namespace mtj

extern "C" {

int32_t mtj_set_error(int32_t code, const char* msg);   // defined next to mtj_last_error

int64_t mtj_verify_scratch_bytes(const mtj_verify_args* a) {
  std::string err;
  const int32_t rc = mtj::check_args(a, &err);
  if (rc) {
    mtj_set_error(rc, err.c_str());
    return -1;
  }
  return mtj::stats_bytes(*a);
}

int32_t mtj_verify_drafts(const mtj_verify_args* a, void* scratch, int64_t scratch_bytes, mtj_stream stream) {
  std::string err;
  const int32_t rc = mtj::check_args(a, &err);
  if (rc) return mtj_set_error(rc, err.c_str());
  if (!scratch || scratch_bytes < mtj::stats_bytes(*a) || (reinterpret_cast<uintptr_t>(scratch) & 15))
    return mtj_set_error(MTJ_ERR_INVALID, "scratch too small or not 16-byte aligned");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto* stats = static_cast<mtj::ChunkStat*>(scratch);
  const cudaError_t e = a->dtype == MTJ_F32 ? mtj::run<float>(*a, stats, s) : mtj::run<__nv_bfloat16>(*a, stats, s);
  if (e != cudaSuccess) return mtj_set_error(MTJ_ERR_CUDA, cudaGetErrorString(e));
  return MTJ_OK;
}

}  // extern "C"

// Verification of drafted tokens against the target model's logits (mtj_verify_drafts).
//
// verify_rows_kernel: every row of logits that takes part is read once, in chunks of kChunk entries, one block each: the
//   chunk's maximum (and where it first stands) and the sum of exp((l - maximum) / temp).  A thread holds its entries in
//   registers, so the maximum is known before the first exponential.
// verify_pick_kernel: a cluster of blocks a sequence.  Every block joins the chunks of all rows to shares, in 64 bits, and
//   decides alike how many drafts are taken; then the cluster shares out the one row that the next token comes from.
//   The race r_i / -log(noise_i) is run in 32 bits with a bound on the error of every entry; those that can win it are run
//   again in 64 bits, so that the token does not hang on the rounding of a near-tie or of a difference of near-equal shares.
//
// Bound by the bytes of the logits: 32-bit sums of exponentials of a chunk, 64-bit sums over chunks.
#include <math.h>

#include <string>

#include "mtj_cache.cuh"
#include "mtj_kernels.h"

namespace mtj {
namespace {

constexpr int kRowThreads = 256;
constexpr int kPerThread = 16;
constexpr int kChunk = kRowThreads * kPerThread;
constexpr int kPickThreads = 512;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kPickCluster = 8;

struct ChunkStat {
  float top, sum;      // largest entry; sum of exp((l - top) / temp) over the chunk
  int32_t at, pad;     // where it first stands
};

__device__ __forceinline__ float value_at(const float* p, int i) { return p[i]; }
__device__ __forceinline__ float value_at(const __nv_bfloat16* p, int i) { return __bfloat162float(p[i]); }

__device__ __forceinline__ int drafts_of(const mtj_verify_args& a, int b) {
  return a.counts_dev ? min(max(a.counts_dev[b], 0), a.drafts) : a.drafts;
}
__device__ __forceinline__ float temp_of(const mtj_verify_args& a, int b) { return a.temp_dev ? a.temp_dev[b] : a.temp; }

// exp((l - top) / temp) = 2^((l - top) * scale), the scale as the sum of two numbers so that its rounding does not lean on every entry
struct ExpScale {
  float hi, lo;
  __device__ __forceinline__ explicit ExpScale(float temp) {
    const double c = 1.4426950408889634074 / static_cast<double>(temp);
    hi = static_cast<float>(c);
    lo = isfinite(hi) ? static_cast<float>(c - static_cast<double>(hi)) : 0.f;
  }
  __device__ __forceinline__ float operator()(float l, float top) const {
    const float d = fmaxf(l - top, -1e30f);      // -inf (and NaN): a finite number whose products cannot cancel
    return d == 0.f ? 1.f : exp2f(fmaf(d, hi, d * lo));
  }
};

// rows of one sequence: 0 .. drafts the target's, then the draft's
template <typename T>
__device__ __forceinline__ const T* row_of(const mtj_verify_args& a, int b, int r) {
  return r <= a.drafts ? static_cast<const T*>(a.target_dev) + b * a.batch_target + r * a.ld_target
                       : static_cast<const T*>(a.draft_dev) + b * a.batch_draft + (r - a.drafts - 1) * a.ld_draft;
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) verify_rows_kernel(const mtj_verify_args a, ChunkStat* stats, int rows, int chunks) {
  const int c = blockIdx.x % chunks, r = blockIdx.x / chunks % rows, b = blockIdx.x / chunks / rows;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ float sm_top[kRowThreads / 32], sm_sum[kRowThreads / 32];
  __shared__ int sm_at[kRowThreads / 32];
  pdl_launch_dependents();
  const int n = drafts_of(a, b);
  const float temp = temp_of(a, b);
  const bool greedy = !(temp > 0.f);
  if (r <= a.drafts ? r > n : (r - a.drafts - 1 >= n || greedy)) return;      // this row takes no part
  const T* row = row_of<T>(a, b, r);
  constexpr int kVec = 16 / sizeof(T);
  // chunks begin at 16-byte boundaries: `skew` entries before the row's first one
  const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  float v[kPerThread];
  float top = -INFINITY;
  int at = 0x7fffffff;
#pragma unroll
  for (int u = 0; u < kPerThread / kVec; ++u) {
    const int i0 = c * kChunk + (u * kRowThreads + tid) * kVec - skew;
    float* w = v + u * kVec;
    if (i0 >= 0 && i0 + kVec <= a.vocab) {
      const uint4 x = ld_cached16(row + i0);
      if constexpr (sizeof(T) == 2) {
        unpack8(x, w);
      } else {
        w[0] = __uint_as_float(x.x);
        w[1] = __uint_as_float(x.y);
        w[2] = __uint_as_float(x.z);
        w[3] = __uint_as_float(x.w);
      }
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) w[e] = i0 + e >= 0 && i0 + e < a.vocab ? value_at(row, i0 + e) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      if (w[e] > top) {
        top = w[e];
        at = i0 + e;
      }
  }
  // the block's maximum, at its lowest place
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t2 = __shfl_xor_sync(0xffffffffu, top, o);
    const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
    if (t2 > top || (t2 == top && a2 < at)) {
      top = t2;
      at = a2;
    }
  }
  if (lane == 0) {
    sm_top[warp] = top;
    sm_at[warp] = at;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w)
    if (sm_top[w] > top || (sm_top[w] == top && sm_at[w] < at)) {
      top = sm_top[w];
      at = sm_at[w];
    }
  float sum = 0.f;
  if (!greedy && top > -INFINITY) {
    const ExpScale e(temp);
#pragma unroll
    for (int u = 0; u < kPerThread; ++u) sum += e(v[u], top);
  }
  sum = warp_sum(sum);
  if (lane == 0) sm_sum[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < kRowThreads / 32; ++w) sum += sm_sum[w];
    stats[blockIdx.x] = {top, sum, at, 0};
  }
}

struct RowShare {
  float top;           // largest logit of the row
  int at;              // its first place
  double sum;          // sum of exp((l - top) / temp)
};

// log of the share of logit l in a row
__device__ __forceinline__ double log_share(const RowShare& s, float l, double temp) {
  return (static_cast<double>(l) - static_cast<double>(s.top)) / temp - log(s.sum);
}
__device__ __forceinline__ double share(const RowShare& s, float l, double temp) {
  return l == s.top ? 1.0 / s.sum : exp((static_cast<double>(l) - static_cast<double>(s.top)) / temp) / s.sum;
}

struct Racer {
  double score;
  int at;
};
__device__ __forceinline__ void take_better(Racer& x, double score, int at) {
  if (score > x.score || (score == x.score && at < x.at)) {
    x.score = score;
    x.at = at;
  }
}

__device__ __forceinline__ uint32_t pick_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void pick_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <typename V>
__device__ __forceinline__ V peer_value(const V* p, uint32_t rank) {
  static_assert(sizeof(V) == 4 || sizeof(V) == 8, "one register or a pair");
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  V v;
  if constexpr (sizeof(V) == 4) {
    uint32_t x;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
    memcpy(&v, &x, 4);
  } else {
    unsigned long long x;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(x) : "r"(at) : "memory");
    memcpy(&v, &x, 8);
  }
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kPickThreads) verify_pick_kernel(const mtj_verify_args a, const ChunkStat* stats, int rows, int chunks,
                                                                   int cluster) {
  extern __shared__ RowShare row_share[];          // [rows]
  __shared__ float sm_best[kPickWarps], s_best;
  __shared__ double sm_score[kPickWarps], s_score;
  __shared__ int sm_at[kPickWarps], s_at, s_taken;
  const int b = blockIdx.x / cluster, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = pick_rank();
  const int n = drafts_of(a, b), n_out = a.drafts + 1;
  const float temp = temp_of(a, b);
  const bool greedy = !(temp > 0.f);
  const int32_t* tokens = a.draft_tokens_dev + static_cast<size_t>(b) * a.drafts;
  pdl_wait();
  for (int r = warp; r < rows; r += kPickWarps) {
    if (r <= a.drafts ? r > n : (r - a.drafts - 1 >= n || greedy)) continue;
    const ChunkStat* st = stats + (static_cast<size_t>(b) * rows + r) * chunks;
    float top = -INFINITY;
    int at = 0x7fffffff;
    for (int c = lane; c < chunks; c += 32)
      if (st[c].top > top) {
        top = st[c].top;
        at = st[c].at;
      }
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
    if (!greedy)
      for (int c = lane; c < chunks; c += 32)
        if (st[c].top > -INFINITY)
          sum += static_cast<double>(st[c].sum) *
                 (st[c].top == top ? 1.0 : exp((static_cast<double>(st[c].top) - static_cast<double>(top)) / static_cast<double>(temp)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) row_share[r] = {top, top > -INFINITY ? at : 0, sum};
  }
  __syncthreads();
  const double t64 = greedy ? 1.0 : static_cast<double>(temp);
  if (warp == 0) {
    int taken = 0;
    for (int k0 = 0; k0 < n && taken == k0; k0 += 32) {
      const int k = k0 + lane;
      bool good = false;
      if (k < n) {
        const int x = tokens[k];
        if (x >= 0 && x < a.vocab) {
          if (greedy) {
            good = x == row_share[k].at;
          } else {
            const double p = share(row_share[k], value_at(row_of<T>(a, b, k), x), t64);
            const double q = a.draft_dev ? share(row_share[a.drafts + 1 + k], value_at(row_of<T>(a, b, a.drafts + 1 + k), x), t64) : 1.0;
            good = static_cast<double>(a.accept_dev[static_cast<size_t>(b) * a.drafts + k]) * q < p;
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
  int next;
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
    const float* noise = a.noise_dev + static_cast<size_t>(b) * a.vocab;
    const ExpScale e(temp);
    const float p_inv = static_cast<float>(1.0 / ps.sum), q_inv = known ? static_cast<float>(1.0 / qs.sum) : 0.f;
    const int per = (a.vocab + cluster - 1) / cluster;
    const int i0 = static_cast<int>(rank) * per, i1 = min(a.vocab, i0 + per);
    // 32 bits: lower bounds first, their best over the cluster, then whoever's upper bound reaches it
    constexpr float kSlack = 4e-6f;       // on a share: argument, exponential, sum and product, each below 2^-20 of it in all
    auto bounds = [&](int i, float* lower, float* upper) {
      const float p = e(value_at(prow, i), ps.top) * p_inv;
      const float q = known ? e(value_at(qrow, i), qs.top) * q_inv : 0.f;
      const float x = -logf(noise[i]);
      const float r = i == without ? 0.f : p - q, slack = i == without ? 0.f : kSlack * (p + q);
      *lower = (r - slack) / x * (1.f - 1e-6f);
      *upper = (r + slack) / x * (1.f + 1e-6f);
    };
    float best = 0.f;
    for (int i = i0 + tid; i < i1; i += kPickThreads) {
      float lower, upper;
      bounds(i, &lower, &upper);
      best = fmaxf(best, lower);
    }
    best = warp_max(best);
    if (lane == 0) sm_best[warp] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < kPickWarps; ++w) best = fmaxf(best, sm_best[w]);
      s_best = best;
    }
    pick_sync();
    best = 0.f;
    for (int r = 0; r < cluster; ++r) best = fmaxf(best, peer_value(&s_best, r));
    Racer win = {0.0, 0x7fffffff};
    bool difference = true;
    for (int pass = 0; pass < 2; ++pass) {
      for (int i = i0 + tid; i < i1; i += kPickThreads) {
        float lower, upper;
        if (difference) bounds(i, &lower, &upper);
        if (difference && !(upper > 0.f && upper >= best)) continue;
        const double p = share(ps, value_at(prow, i), t64);
        const double q = !difference ? 0.0 : known ? share(qs, value_at(qrow, i), t64) : i == without ? p : 0.0;
        const double r = p - q;
        if (r > 0.0) take_better(win, r / -log(static_cast<double>(noise[i])), i);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double s2 = __shfl_xor_sync(0xffffffffu, win.score, o);
        const int a2 = __shfl_xor_sync(0xffffffffu, win.at, o);
        take_better(win, s2, a2);
      }
      if (lane == 0) {
        sm_score[warp] = win.score;
        sm_at[warp] = win.at;
      }
      __syncthreads();
      if (tid == 0) {
        for (int w = 0; w < kPickWarps; ++w) take_better(win, sm_score[w], sm_at[w]);
        s_score = win.score;
        s_at = win.at;
      }
      pick_sync();
      for (int r = 0; r < cluster; ++r) take_better(win, peer_value(&s_score, r), peer_value(&s_at, r));
      pick_sync();                                    // all have read: the next pass may overwrite, and a block may leave
      if (win.at < a.vocab) break;                    // alike in every thread of the cluster
      difference = false;                             // the difference is zero everywhere: the target's own shares
    }
    next = win.at < a.vocab ? win.at : ps.at;
  }
  if (rank == 0)
    for (int k = tid; k < n_out; k += kPickThreads) {
      const int x = k < taken ? tokens[k] : k == taken ? next : -1;
      a.tokens_out_dev[static_cast<size_t>(b) * n_out + k] = x;
      if (a.logprobs_out_dev)
        a.logprobs_out_dev[static_cast<size_t>(b) * n_out + k] =
            x < 0 || greedy ? 0.f : static_cast<float>(log_share(row_share[k], value_at(row_of<T>(a, b, k), x), t64));
      if (k == 0) a.accepted_out_dev[b] = taken;
    }
}

int rows_of(const mtj_verify_args& a) { return a.drafts + 1 + (a.draft_dev ? a.drafts : 0); }
int chunks_of(const mtj_verify_args& a) { return (a.vocab + kChunk + 15) / kChunk; }      // room for the skew of a row's start
int64_t stats_bytes(const mtj_verify_args& a) {
  return static_cast<int64_t>(a.batch) * rows_of(a) * chunks_of(a) * static_cast<int64_t>(sizeof(ChunkStat));
}

int32_t check_args(const mtj_verify_args* a, std::string* err) {
  auto bad = [&](const char* what) {
    *err = what;
    return static_cast<int32_t>(MTJ_ERR_INVALID);
  };
  if (!a || !a->target_dev || !a->noise_dev || !a->tokens_out_dev || !a->accepted_out_dev) return bad("null argument");
  if (a->batch <= 0 || a->vocab <= 0 || a->drafts < 0) return bad("batch and vocab must be positive, drafts not negative");
  if (a->drafts > 0 && (!a->draft_tokens_dev || !a->accept_dev)) return bad("null argument");
  if (a->drafts > 1024) return bad("at most 1024 drafted tokens a sequence");
  if (a->dtype != MTJ_F32 && a->dtype != MTJ_BF16) {
    *err = "dtype must be MTJ_F32 or MTJ_BF16";
    return MTJ_ERR_UNSUPPORTED;
  }
  const uintptr_t size = a->dtype == MTJ_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(a->target_dev) | reinterpret_cast<uintptr_t>(a->draft_dev)) & (size - 1))
    return bad("logits must be aligned to their type");
  if (a->ld_target < a->vocab || (a->draft_dev && a->ld_draft < a->vocab)) return bad("a row's stride is shorter than the vocabulary");
  if (a->batch_target < 0 || a->batch_draft < 0) return bad("strides must not be negative");
  if (a->vocab > 0x7fffffff - 2 * kChunk) return bad("the vocabulary is too large");
  if (static_cast<int64_t>(a->batch) * rows_of(*a) > 0x7fffffff / chunks_of(*a)) return bad("batch * drafts * vocab is too large");
  return MTJ_OK;
}

template <typename T>
cudaError_t run(const mtj_verify_args& a, ChunkStat* stats, cudaStream_t s) {
  const int rows = rows_of(a), chunks = chunks_of(a);
  verify_rows_kernel<T><<<static_cast<unsigned>(a.batch * rows * chunks), kRowThreads, 0, s>>>(a, stats, rows, chunks);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int cluster = a.vocab > 2 * kPickThreads ? kPickCluster : 1;
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
  return cudaLaunchKernelEx(&cfg, verify_pick_kernel<T>, a, static_cast<const ChunkStat*>(stats), rows, chunks, cluster);
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

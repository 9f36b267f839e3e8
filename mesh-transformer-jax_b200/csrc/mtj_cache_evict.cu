// Eviction from a paged cache by accumulated attention weight (mtj_k_cache_evict).
//
// cache_select_kernel: one block a (sequence, key head).  The weights become integers that order as the numbers do; a
//   radix selection over four digits of eight bits finds the key of the last one that is kept and how many of its equals are,
//   and a pass in slot order writes the kept slots and their weights.
// cache_move_kernel: one block a (spare page, key head, sequence) copies the kept rows of keys and values.
#include <string>

#include "mtj_cache.cuh"
#include "mtj_kernels.h"

namespace mtj {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kMoveThreads = 256;

// ascending integer order is ascending order of the numbers; -0 and +0 are equal
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v == 0.0f) v = 0.0f;
  const uint32_t u = __float_as_uint(v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// the sum over the threads before this one and, in *all, over the block; every thread takes part
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int w = warp_sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  *all = __shfl_sync(0xffffffffu, w, 31);
  const int before = warp ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
  return before + x - v;
}

__global__ void __launch_bounds__(kSelThreads) cache_select_kernel(const mtj_cache_evict_args a) {
  __shared__ int hist[256], warp_sums[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int b = blockIdx.x / a.kv_heads, tid = threadIdx.x;
  const int slots = a.pages * kPageTokens;
  const CacheSeq s = cache_seq(a.lengths_dev, nullptr, b, 0, a.pages);
  const bool moves = s.length > a.keep;
  const float* w = a.weights_dev + static_cast<size_t>(blockIdx.x) * slots;
  float* w_out = a.weights_out_dev + static_cast<size_t>(blockIdx.x) * slots;
  int32_t* kept = a.kept_out_dev + static_cast<size_t>(blockIdx.x) * a.keep;
  const int held = min(s.length, a.keep);
  if (blockIdx.x % a.kv_heads == 0) {
    if (tid == 0) {
      a.lengths_out_dev[b] = held;
      if (s.bad && a.status_dev) atomicOr(a.status_dev, kDevErrBadIndex);
    }
    const int spare = (a.keep + kPageTokens - 1) / kPageTokens;
    for (int i = tid; i < a.pages; i += kSelThreads) {
      const size_t at = static_cast<size_t>(b) * a.pages + i;
      a.page_table_out_dev[at] = !moves ? a.page_table_dev[at] : i < spare ? a.spare_pages_dev[static_cast<size_t>(b) * spare + i] : -1;
    }
  }
  if (!moves) {
    for (int i = tid; i < slots; i += kSelThreads) w_out[i] = i < s.length ? w[i] : 0.f;
    for (int i = tid; i < a.keep; i += kSelThreads) kept[i] = i < s.length ? i : -1;
    return;
  }
  const int lo = a.first, hi = s.length - a.last, need = a.keep - a.first - a.last;
  // the `need` largest of [lo, hi): all keys above `prefix`, and the first `ties` equal to it
  uint32_t prefix = 0, mask = 0;
  int ties = need;
  if (need > 0) {
    if (tid == 0) s_need = need;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += kSelThreads) {
        const uint32_t k = order_key(w[i]);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      // digits from the largest down: thread t holds digit 255 - t
      int all;
      const int here = tid < 256 ? hist[255 - tid] : 0;
      const int above = block_scan(here, warp_sums, &all);
      const int want = s_need;
      __syncthreads();
      if (tid < 256 && above < want && above + here >= want) {
        s_prefix = prefix | (static_cast<uint32_t>(255 - tid) << shift);
        s_need = want - above;
      }
      __syncthreads();
      prefix = s_prefix;
      mask |= 255u << shift;
    }
    ties = s_need;
  }
  int out = 0, equal_before = 0;
  for (int i0 = 0; i0 < s.length; i0 += kSelThreads) {
    const int i = i0 + tid;
    const bool in = i < s.length;
    const float v = in ? w[i] : 0.f;
    const bool middle = in && i >= lo && i < hi && need > 0;
    const uint32_t k = order_key(v);
    const bool equal = middle && k == prefix;
    int all_equal, all_keep;
    const int rank = block_scan(equal ? 1 : 0, warp_sums, &all_equal);
    const bool keep = in && (i < lo || i >= hi || (middle && (k > prefix || (equal && equal_before + rank < ties))));
    const int at = block_scan(keep ? 1 : 0, warp_sums, &all_keep);
    if (keep) {
      kept[out + at] = i;
      w_out[out + at] = v;      // at or before slot i, which this block has read
    }
    out += all_keep;
    equal_before += all_equal;
  }
  __syncthreads();
  for (int i = held + tid; i < slots; i += kSelThreads) w_out[i] = 0.f;
}

__global__ void __launch_bounds__(kMoveThreads) cache_move_kernel(const mtj_cache_evict_args a) {
  const int spare = (a.keep + kPageTokens - 1) / kPageTokens;
  const int i = blockIdx.x % spare, kvh = blockIdx.x / spare % a.kv_heads, b = blockIdx.x / spare / a.kv_heads;
  const CacheSeq s = cache_seq(a.lengths_dev, nullptr, b, 0, a.pages);
  if (s.length <= a.keep) return;
  const int to = a.spare_pages_dev[static_cast<size_t>(b) * spare + i];
  if (!cache_page_ok(to, a.n_pages)) {
    if (threadIdx.x == 0 && a.status_dev) atomicOr(a.status_dev, kDevErrBadIndex);
    return;
  }
  const int rows = min(kPageTokens, a.keep - i * kPageTokens), vecs = a.d_head / 8;
  const int32_t* kept = a.kept_out_dev + (static_cast<size_t>(b) * a.kv_heads + kvh) * a.keep + i * kPageTokens;
  for (int v = threadIdx.x; v < rows * vecs; v += kMoveThreads) {
    const int r = v / vecs, slot = kept[r];
    const int from = a.page_table_dev[static_cast<size_t>(b) * a.pages + slot / kPageTokens];
    if (!cache_page_ok(from, a.n_pages)) {
      if (a.status_dev) atomicOr(a.status_dev, kDevErrBadIndex);
      continue;
    }
    const size_t src = ((static_cast<size_t>(from) * a.kv_heads + kvh) * kPageTokens + slot % kPageTokens) * vecs + v % vecs;
    const size_t dst = ((static_cast<size_t>(to) * a.kv_heads + kvh) * kPageTokens) * vecs + v;
    static_cast<uint4*>(a.kpool_dev)[dst] = static_cast<const uint4*>(a.kpool_dev)[src];
    static_cast<uint4*>(a.vpool_dev)[dst] = static_cast<const uint4*>(a.vpool_dev)[src];
  }
}

int32_t check_args(const mtj_cache_evict_args* a, std::string* err) {
  auto bad = [&](const char* what) {
    *err = what;
    return static_cast<int32_t>(MTJ_ERR_INVALID);
  };
  if (!a || !a->kpool_dev || !a->vpool_dev || !a->page_table_dev || !a->lengths_dev || !a->weights_dev || !a->spare_pages_dev ||
      !a->kept_out_dev || !a->lengths_out_dev || !a->weights_out_dev || !a->page_table_out_dev)
    return bad("null argument");
  if (a->d_head != 64 && a->d_head != 128 && a->d_head != 256) {
    *err = "d_head must be 64, 128 or 256";
    return MTJ_ERR_UNSUPPORTED;
  }
  if (a->n_pages <= 0 || a->batch <= 0 || a->pages <= 0 || a->kv_heads <= 0) return bad("n_pages, batch, pages and kv_heads must be positive");
  if (a->keep < 1 || a->first < 0 || a->last < 0 || a->first > a->keep || a->last > a->keep - a->first)
    return bad("keep must be positive and hold the first and the last slots");
  if (a->lengths_out_dev == a->lengths_dev || a->page_table_out_dev == a->page_table_dev)
    return bad("the new lengths and the new page table are arrays of their own");
  if ((reinterpret_cast<uintptr_t>(a->kpool_dev) | reinterpret_cast<uintptr_t>(a->vpool_dev)) & 15)
    return bad("pools must be 16-byte aligned");
  const int64_t most = 0x7fffffff;
  if (a->pages > most / kPageTokens || static_cast<int64_t>(a->batch) * a->kv_heads > most / kPageTokens / a->pages ||
      a->keep > most - kPageTokens || static_cast<int64_t>(a->batch) * a->kv_heads > most / ((a->keep + kPageTokens - 1) / kPageTokens))
    return bad("batch * kv_heads * slots is too large");
  return MTJ_OK;
}

}  // namespace
}  // namespace mtj

extern "C" {

int32_t mtj_set_error(int32_t code, const char* msg);   // defined next to mtj_last_error

int32_t mtj_k_cache_evict(const mtj_cache_evict_args* a, mtj_stream stream) {
  std::string err;
  const int32_t rc = mtj::check_args(a, &err);
  if (rc) return mtj_set_error(rc, err.c_str());
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  mtj::cache_select_kernel<<<a->batch * a->kv_heads, mtj::kSelThreads, 0, s>>>(*a);
  const int spare = (a->keep + mtj::kPageTokens - 1) / mtj::kPageTokens;
  mtj::cache_move_kernel<<<static_cast<unsigned>(spare * a->kv_heads * a->batch), mtj::kMoveThreads, 0, s>>>(*a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return mtj_set_error(MTJ_ERR_CUDA, cudaGetErrorString(e));
  return MTJ_OK;
}

}  // extern "C"

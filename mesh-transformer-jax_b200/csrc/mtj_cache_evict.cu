// Eviction from a paged cache by accumulated attention weight (mtj_k_cache_evict).
//
// cache_select_kernel: one block a (sequence, key head).  The weights become integers that order as the numbers do; a
//   radix selection over digits of 11, 11 and 10 bits finds the key of the last one that is kept and how many of its equals are
//   (it ends early when a digit's whole bin is kept); a thread has kEach neighbouring slots, so that two sums over the block
//   give every kept slot its place.  Up to kEach * kSelThreads slots are read once and stay in registers.  A block has a whole head,
//   and not a cluster of them: the sums over the block are the chain, and would cross the cluster.
// cache_move_kernel: one block a (spare page, key head, sequence) copies the kept rows of keys and values; bound by their bytes.
//
// 8 sequences of 3000 to 16383 slots, 8 key heads of 128, 4096 kept: 19 us (64 blocks, three rounds of counting in shared memory) and
// 44 us, 118 MB read and as many written at 5.4 TB/s.
#include <string>

#include "mtj_cache.cuh"
#include "mtj_kernels.h"

namespace mtj {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kMoveThreads = 256;
constexpr int kEach = 16;                  // neighbouring slots of a thread
constexpr int kStage = 4096;               // kept slots on their way out
constexpr int kBins = 2048;                // the first digit is sign, exponent and two bits: weights of one size are in several bins

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
  __shared__ int hist[kBins], warp_sums[32];
  __shared__ int stage_slot[kStage];
  __shared__ float stage_weight[kStage];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need, s_all;
  const int b = blockIdx.x / a.kv_heads, tid = threadIdx.x;
  const int slots = a.pages * kPageTokens;
  pdl_launch_dependents();
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
  // neighbouring slots of a thread, fewer where the sequence is short; a block goes over the sequence in steps of `span`
  const int each = min(kEach, (s.length + 4 * kSelThreads - 1) / (4 * kSelThreads) * 4), span = each * kSelThreads;
  const bool once = s.length <= span;
  float v[kEach];
  auto load = [&](int base) {
    const int i0 = base + tid * each;
#pragma unroll
    for (int e0 = 0; e0 < kEach; e0 += 4) {
      if (e0 >= each) break;
      if (i0 + e0 + 4 <= s.length && !(reinterpret_cast<uintptr_t>(w) & 15)) {
        const float4 x = *reinterpret_cast<const float4*>(w + i0 + e0);
        v[e0] = x.x;
        v[e0 + 1] = x.y;
        v[e0 + 2] = x.z;
        v[e0 + 3] = x.w;
      } else {
#pragma unroll
        for (int e = e0; e < e0 + 4; ++e) v[e] = i0 + e < s.length ? w[i0 + e] : 0.f;
      }
    }
  };
  if (once) load(0);
  // the `need` largest of [lo, hi): all keys above `prefix` in the digits of `mask`, and the first `ties` equal to it there
  uint32_t prefix = 0, mask = 0;
  int ties = need;
  if (need > 0) {
    if (tid == 0) s_need = need;
    for (int digit = 0; digit < 3; ++digit) {
      const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
      const uint32_t digits = digit == 2 ? 1023u : 2047u;
      for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int base = 0; base < s.length; base += span) {
        if (!once) load(base);
        const int i0 = base + tid * each;
        if (i0 >= s.length) continue;
#pragma unroll
        for (int e0 = 0; e0 < kEach; e0 += 4) {
          if (e0 >= each) break;
#pragma unroll
          for (int e = e0; e < e0 + 4; ++e) {
            const uint32_t k = order_key(v[e]);
            if (i0 + e >= lo && i0 + e < hi && (k & mask) == prefix) atomicAdd(&hist[(k >> shift) & digits], 1);
          }
        }
      }
      __syncthreads();
      // digits from the largest down: a thread holds two
      const int top = kBins - 1 - 2 * tid;
      int all;
      const int first = hist[top], second = hist[top - 1];
      const int above = block_scan(first + second, warp_sums, &all);
      const int want = s_need;
      __syncthreads();
      if (above < want && above + first + second >= want) {
        const bool upper = above + first >= want;
        s_prefix = prefix | (static_cast<uint32_t>(upper ? top : top - 1) << shift);
        s_need = want - above - (upper ? 0 : first);
        s_all = above + first + (upper ? 0 : second) == want;
      }
      __syncthreads();
      prefix = s_prefix;
      mask |= digits << shift;
      if (s_all) break;
    }
    ties = s_need;
  }
  int out = 0, equal_before = 0;
  for (int base = 0; base < s.length; base += span) {
    if (!once) load(base);
    const int i0 = base + tid * each;
    uint32_t equal = 0, sure = 0;          // bits of this thread's slots
    if (i0 < s.length) {
#pragma unroll
      for (int e0 = 0; e0 < kEach; e0 += 4) {
        if (e0 >= each) break;
#pragma unroll
        for (int e = e0; e < e0 + 4; ++e) {
          const int i = i0 + e;
          const uint32_t k = order_key(v[e]) & mask;
          const bool middle = i >= lo && i < hi;
          if (i < s.length && (!middle || (need > 0 && k > prefix))) sure |= 1u << e;
          if (middle && need > 0 && k == prefix) equal |= 1u << e;
        }
      }
    }
    int all_equal, all_keep;
    int rank = equal_before + block_scan(__popc(equal), warp_sums, &all_equal);
    for (uint32_t rest = equal; rest && rank < ties; rest &= rest - 1, ++rank) sure |= rest & (0u - rest);
    const int first_place = block_scan(__popc(sure), warp_sums, &all_keep);
    // through shared memory: neighbouring threads' places are neighbours, a thread's own are too, a warp's at one time are not
    for (int r0 = 0; r0 < all_keep; r0 += kStage) {
      int place = first_place - r0;
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (sure >> e & 1u) {
          if (place >= 0 && place < kStage) {
            stage_slot[place] = i0 + e;
            stage_weight[place] = v[e];
          }
          ++place;
        }
      __syncthreads();
      for (int i = tid; i < min(kStage, all_keep - r0); i += kSelThreads) {
        kept[out + r0 + i] = stage_slot[i];
        w_out[out + r0 + i] = stage_weight[i];      // at or before its slot, which this block has read
      }
      __syncthreads();
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
  if (s.length <= a.keep) {
    pdl_wait();                            // a launch that ends before the one it is chained to would let the next one overtake both
    return;
  }
  const int to = a.spare_pages_dev[static_cast<size_t>(b) * spare + i];
  pdl_wait();
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
  if (a->pages > kMostPages || static_cast<int64_t>(a->batch) * a->kv_heads > most / kPageTokens / a->pages ||
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
  cudaError_t e = cudaGetLastError();
  const int spare = (a->keep + mtj::kPageTokens - 1) / mtj::kPageTokens;
  if (e == cudaSuccess)
    e = mtj::launch_pdl(mtj::cache_move_kernel, dim3(static_cast<unsigned>(spare * a->kv_heads * a->batch)), dim3(mtj::kMoveThreads), 0, s, true, *a);
  if (e != cudaSuccess) return mtj_set_error(MTJ_ERR_CUDA, cudaGetErrorString(e));
  return MTJ_OK;
}

}  // extern "C"

// Geometry of the paged caches of mtj_k_cache_attn and mtj_k_cache_evict, shared by their kernels.
#pragma once
#include "../../include/mtj_b200.h"
#include "mtj_common.cuh"

namespace mtj {

constexpr int kMostPages = 1 << 24;         // of a sequence: places of slots, and a few steps behind the last, are 32-bit numbers

// Slots in use and new tokens of one sequence; numbers that do not fit the cache make it an empty one.
struct CacheSeq {
  int length, fresh;
  bool bad;
};
__device__ __forceinline__ CacheSeq cache_seq(const int32_t* lengths, const int32_t* new_tokens, int b, int tokens, int pages) {
  CacheSeq s;
  s.length = lengths[b];
  s.fresh = new_tokens ? new_tokens[b] : tokens;
  s.bad = s.fresh < 0 || s.fresh > tokens || s.length < s.fresh || s.length > pages * kPageTokens;
  if (s.bad) s.length = s.fresh = 0;
  return s;
}
__device__ __forceinline__ bool cache_page_ok(int page, int n_pages) { return page >= 0 && page < n_pages; }

// Slots visible to the token in slot p: [0, min(sinks, low)) and [low, p]
__device__ __forceinline__ int cache_window_low(int p, int window) { return p >= window ? p - window + 1 : 0; }

}  // namespace mtj

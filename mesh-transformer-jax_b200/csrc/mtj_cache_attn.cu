// Attention of new tokens over a paged cache with a sliding window and first tokens that stay visible (mtj_k_cache_attn).
#include <math.h>

#include <string>

#include "mtj_cache_kernels.h"

namespace mtj {
namespace {

int32_t check_args(const mtj_cache_attn_args* a, std::string* err) {
  auto bad = [&](const char* what) {
    *err = what;
    return static_cast<int32_t>(MTJ_ERR_INVALID);
  };
  if (!a) return bad("null argument");
  if (!a->kpool_dev || !a->vpool_dev || !a->page_table_dev || !a->lengths_dev || !a->q_dev || !a->out_dev) return bad("null argument");
  if (!a->k_new_dev != !a->v_new_dev) return bad("new keys and new values come together");
  if (a->d_head != 64 && a->d_head != 128 && a->d_head != 256) {
    *err = "d_head must be 64, 128 or 256";
    return MTJ_ERR_UNSUPPORTED;
  }
  if (a->dtype != MTJ_F32 && a->dtype != MTJ_BF16) {
    *err = "dtype must be MTJ_F32 or MTJ_BF16";
    return MTJ_ERR_UNSUPPORTED;
  }
  if (a->n_pages <= 0 || a->batch <= 0 || a->pages <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->tokens <= 0)
    return bad("n_pages, batch, pages, heads, kv_heads and tokens must be positive");
  if (a->pages > kMostPages) return bad("more than 2^30 slots a sequence");
  if (a->tokens > a->pages * kPageTokens) return bad("more tokens than the pages of a sequence hold");
  if (a->heads % a->kv_heads || a->heads / a->kv_heads > MTJ_CACHE_MAX_GROUP)
    return bad("heads must be a multiple of kv_heads, at most MTJ_CACHE_MAX_GROUP times as many");
  if (a->window < 1 || a->sinks < 0) return bad("window must be positive and sinks not negative");
  if (!(a->scale > 0.f) || !(a->scale < INFINITY)) return bad("scale must be positive and finite");
  if (a->weights_in_dev && !a->weights_out_dev) return bad("weights_in without weights_out");
  const int64_t cols = static_cast<int64_t>(a->heads) * a->d_head, kv_cols = static_cast<int64_t>(a->kv_heads) * a->d_head;
  if (a->ld_q < cols || a->ld_out < cols || (a->k_new_dev && (a->ld_k < kv_cols || a->ld_v < kv_cols)))
    return bad("a row's stride is shorter than its heads");
  if ((a->ld_q | a->ld_out | (a->k_new_dev ? a->ld_k | a->ld_v : 0)) & 7) return bad("row strides must be multiples of 8 elements");
  const uintptr_t all = reinterpret_cast<uintptr_t>(a->kpool_dev) | reinterpret_cast<uintptr_t>(a->vpool_dev) |
                        reinterpret_cast<uintptr_t>(a->q_dev) | reinterpret_cast<uintptr_t>(a->out_dev) |
                        reinterpret_cast<uintptr_t>(a->k_new_dev) | reinterpret_cast<uintptr_t>(a->v_new_dev);
  if (all & 15) return bad("pools and rows must be 16-byte aligned");
  const int64_t most = 0x7fffffff, rows = static_cast<int64_t>(a->batch) * a->tokens;
  if (rows > most || rows * a->heads > most) return bad("batch * tokens * heads is too large");
  if (static_cast<int64_t>(a->batch) * a->kv_heads > most / kPageTokens / a->pages) return bad("batch * kv_heads * slots is too large");
  if (!cache_prompt_fits(*a)) return bad("too many new tokens for one call");
  if (a->kv_heads > 65535) return bad("too many key heads");
  if (static_cast<int64_t>(a->n_pages) * a->kv_heads > most / kPageTokens) return bad("n_pages * kv_heads is too large");
  return MTJ_OK;
}

// Few rows per key head, one or two tokens, queries in 32 bits and calls that add up weights go tile by tile over the cache; other
// prompts have the tensor cores' tiles of 128 rows.  At 64 rows the two are equal or the first ahead (8 x 128, one sequence of 2000 slots:
// 23 against 31 us; 8 sequences of 8000, 4 heads a key head: 152 against 162), at 128 the second is (35 / 31 and 275 / 165).
constexpr int kFewRows = 64;
bool takes_few(const mtj_cache_attn_args& a) {
  return a.dtype == MTJ_F32 || a.weights_out_dev || a.tokens <= 2 || a.tokens * static_cast<int64_t>(a.heads / a.kv_heads) <= kFewRows;
}

}  // namespace
}  // namespace mtj

extern "C" {

int32_t mtj_set_error(int32_t code, const char* msg);   // defined next to mtj_last_error

int64_t mtj_k_cache_attn_scratch_bytes(const mtj_cache_attn_args* a) {
  std::string err;
  const int32_t rc = mtj::check_args(a, &err);
  if (rc) {
    mtj_set_error(rc, err.c_str());
    return -1;
  }
  return mtj::takes_few(*a) ? mtj::plan_cache_few(*a).total : mtj::cache_prompt_scratch(*a);
}

int32_t mtj_k_cache_attn(const mtj_cache_attn_args* a, void* scratch, int64_t scratch_bytes, mtj_stream s) {
  std::string err;
  const int32_t rc = mtj::check_args(a, &err);
  if (rc) return mtj_set_error(rc, err.c_str());
  const bool few = mtj::takes_few(*a);
  mtj::CacheFewPlan p = {};
  if (few) p = mtj::plan_cache_few(*a);
  else p.total = mtj::cache_prompt_scratch(*a);
  if (!scratch || scratch_bytes < p.total || (reinterpret_cast<uintptr_t>(scratch) & 255))
    return mtj_set_error(MTJ_ERR_INVALID, "scratch too small or not 256-byte aligned");
  const cudaStream_t st = static_cast<cudaStream_t>(s);
  const cudaError_t e = few ? mtj::run_cache_few(*a, p, static_cast<char*>(scratch), st)
                            : mtj::run_cache_prompt(*a, static_cast<char*>(scratch), st);
  if (e != cudaSuccess) return mtj_set_error(MTJ_ERR_CUDA, cudaGetErrorString(e));
  return MTJ_OK;
}

}  // extern "C"

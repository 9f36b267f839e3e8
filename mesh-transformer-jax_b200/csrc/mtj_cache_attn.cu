// Attention of new tokens over a paged cache with a sliding window and first tokens that stay visible (mtj_k_cache_attn).
#include <math.h>

#include <string>

#include "mtj_cache_kernels.h"

namespace mtj {
namespace {

constexpr int kRowThreads = 128;
constexpr int kRowWarps = kRowThreads / 32;

__device__ __forceinline__ float load_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_value(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// The new tokens' keys and values into their slots: one block a token and sequence.
template <typename T>
__global__ void __launch_bounds__(256) cache_append_kernel(const mtj_cache_attn_args a) {
  const int t = blockIdx.x % a.tokens, b = blockIdx.x / a.tokens;
  const CacheSeq s = cache_seq(a.lengths_dev, a.new_tokens_dev, b, a.tokens, a.pages);
  if (t >= s.fresh) return;
  const int slot = s.length - s.fresh + t;
  const int page = a.page_table_dev[static_cast<size_t>(b) * a.pages + slot / kPageTokens];
  if (!cache_page_ok(page, a.n_pages)) {
    if (threadIdx.x == 0 && a.status_dev) atomicOr(a.status_dev, kDevErrBadIndex);
    return;
  }
  const int cols = a.kv_heads * a.d_head;
  const T* k = static_cast<const T*>(a.k_new_dev) + (static_cast<size_t>(b) * a.tokens + t) * a.ld_k;
  const T* v = static_cast<const T*>(a.v_new_dev) + (static_cast<size_t>(b) * a.tokens + t) * a.ld_v;
  for (int c = threadIdx.x; c < cols; c += 256) {
    const int h = c / a.d_head, e = c % a.d_head;
    const size_t at = ((static_cast<size_t>(page) * a.kv_heads + h) * kPageTokens + slot % kPageTokens) * a.d_head + e;
    static_cast<__nv_bfloat16*>(a.kpool_dev)[at] = __float2bfloat16_rn(load_value(k + c));
    static_cast<__nv_bfloat16*>(a.vpool_dev)[at] = __float2bfloat16_rn(load_value(v + c));
  }
}

// One block a query row: its warps walk the visible slots in turn, each with a running maximum, sum and weighted value.
template <typename T, int DH>
__global__ void __launch_bounds__(kRowThreads) cache_row_kernel(const mtj_cache_attn_args a, float2* lse) {
  constexpr int EPL = DH / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.x % a.heads, t = blockIdx.x / a.heads % a.tokens, b = blockIdx.x / a.heads / a.tokens;
  const CacheSeq s = cache_seq(a.lengths_dev, a.new_tokens_dev, b, a.tokens, a.pages);
  if (s.bad && h == 0 && t == 0 && threadIdx.x == 0 && a.status_dev) atomicOr(a.status_dev, kDevErrBadIndex);
  __shared__ float sm_m[kRowWarps], sm_l[kRowWarps], sm_o[kRowWarps][DH];
  const size_t row = static_cast<size_t>(b) * a.tokens + t;
  float q[EPL], o[EPL], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    q[e] = t < s.fresh ? load_value(static_cast<const T*>(a.q_dev) + row * a.ld_q + h * DH + e * 32 + lane) * a.scale : 0.f;
    o[e] = 0.f;
  }
  const int p = t < s.fresh ? s.length - s.fresh + t : -1;
  const int low = cache_window_low(p, a.window), sinks = min(a.sinks, low);
  const int seen = p < 0 ? 0 : sinks + p + 1 - low;
  const int kvh = h / (a.heads / a.kv_heads);
  for (int i = warp; i < seen; i += kRowWarps) {
    const int j = i < sinks ? i : low + i - sinks;
    const int page = a.page_table_dev[static_cast<size_t>(b) * a.pages + j / kPageTokens];
    if (!cache_page_ok(page, a.n_pages)) {
      if (lane == 0 && a.status_dev) atomicOr(a.status_dev, kDevErrBadIndex);
      continue;
    }
    const size_t at = ((static_cast<size_t>(page) * a.kv_heads + kvh) * kPageTokens + j % kPageTokens) * DH + lane;
    const __nv_bfloat16 *k = static_cast<const __nv_bfloat16*>(a.kpool_dev) + at, *v = static_cast<const __nv_bfloat16*>(a.vpool_dev) + at;
    float d = 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) d = fmaf(q[e], load_value(k + e * 32), d);
    d = warp_sum(d);
    const float m_new = fmaxf(m, d);
    const float corr = __expf(m - m_new), w = __expf(d - m_new);
    l = fmaf(l, corr, w);
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] = fmaf(o[e], corr, w * load_value(v + e * 32));
    m = m_new;
  }
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < EPL; ++e) sm_o[warp][e * 32 + lane] = o[e];
  __syncthreads();
  float M = -INFINITY, L = 0.f;
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) M = fmaxf(M, sm_m[w]);
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) L += sm_m[w] == -INFINITY ? 0.f : sm_l[w] * __expf(sm_m[w] - M);
  for (int c = threadIdx.x; c < DH; c += kRowThreads) {
    float O = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) O += sm_m[w] == -INFINITY ? 0.f : sm_o[w][c] * __expf(sm_m[w] - M);
    store_value(static_cast<T*>(a.out_dev) + row * a.ld_out + h * DH + c, L > 0.f ? O / L : 0.f);
  }
  if (lse && threadIdx.x == 0) lse[row * a.heads + h] = make_float2(M, L);
}

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
  if (a->pages > 0x7fffffff / kPageTokens || a->tokens > a->pages * kPageTokens) return bad("more tokens than the pages of a sequence hold");
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
  if (static_cast<int64_t>(a->n_pages) * a->kv_heads > most / kPageTokens) return bad("n_pages * kv_heads is too large");
  return MTJ_OK;
}

// Few rows per key head, queries in 32 bits and calls that add up weights go tile by tile over the cache; other prompts row by row.
bool takes_few(const mtj_cache_attn_args& a) {
  return a.dtype == MTJ_F32 || a.weights_out_dev || a.tokens * static_cast<int64_t>(a.heads / a.kv_heads) <= 64;
}

template <int DH>
cudaError_t run_prompt(const mtj_cache_attn_args& a, cudaStream_t s) {
  if (a.k_new_dev) cache_append_kernel<__nv_bfloat16><<<a.batch * a.tokens, 256, 0, s>>>(a);
  cache_row_kernel<__nv_bfloat16, DH><<<a.batch * a.tokens * a.heads, kRowThreads, 0, s>>>(a, nullptr);
  return cudaGetLastError();
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
  return mtj::takes_few(*a) ? mtj::plan_cache_few(*a).total : 256;
}

int32_t mtj_k_cache_attn(const mtj_cache_attn_args* a, void* scratch, int64_t scratch_bytes, mtj_stream s) {
  std::string err;
  const int32_t rc = mtj::check_args(a, &err);
  if (rc) return mtj_set_error(rc, err.c_str());
  const bool few = mtj::takes_few(*a);
  mtj::CacheFewPlan p = {};
  if (few) p = mtj::plan_cache_few(*a);
  else p.total = 256;
  if (!scratch || scratch_bytes < p.total || (reinterpret_cast<uintptr_t>(scratch) & 255))
    return mtj_set_error(MTJ_ERR_INVALID, "scratch too small or not 256-byte aligned");
  const cudaStream_t st = static_cast<cudaStream_t>(s);
  const cudaError_t e = few ? mtj::run_cache_few(*a, p, static_cast<char*>(scratch), st)
                        : a->d_head == 64 ? mtj::run_prompt<64>(*a, st)
                        : a->d_head == 128 ? mtj::run_prompt<128>(*a, st) : mtj::run_prompt<256>(*a, st);
  if (e != cudaSuccess) return mtj_set_error(MTJ_ERR_CUDA, cudaGetErrorString(e));
  return MTJ_OK;
}

}  // extern "C"

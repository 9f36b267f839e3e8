// Shared device helpers for the sm_100a kernels of libmtj_b200.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace mtj {

constexpr int kPageTokens = 64;          // tokens per KV page
constexpr int kWarp = 32;

// Device-side error word bits (one word per handle, read by mtj_check_device_status).
constexpr uint32_t kDevErrTimeout = 1u;
constexpr uint32_t kDevErrBadIndex = 2u;

// A kernel's dynamic shared memory limit is an attribute of the (kernel, device) pair: set it once per
// device, with that device current.  One DeviceOnce object per kernel instantiation.
struct DeviceOnce {
  bool done[64] = {};
  template <typename F>
  cudaError_t run(F&& set_attribute) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const bool tracked = dev >= 0 && dev < 64;
    if (tracked && done[dev]) return cudaSuccess;
    e = set_attribute();
    if (e == cudaSuccess && tracked) done[dev] = true;
    return e;
  }
};

// 16-byte streaming load of data that nobody writes while the kernel is there (weights) and that is touched once per pass: bypass
// L1 so the activations stay resident there.
__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
// The same for cached keys and values, whose newest rows other blocks or the predecessor of a chained launch write while the kernel
// is there: a coherent load.
__device__ __forceinline__ uint4 ld_cached16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ld_cached4(const void* p) {
  uint32_t v;
  asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// bf16 pair packed in a 32-bit word -> two floats (bf16 is the top half of fp32).
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ __forceinline__ void unpack8(const uint4& v, float* f) {
  f[0] = bf16_lo(v.x); f[1] = bf16_hi(v.x);
  f[2] = bf16_lo(v.y); f[3] = bf16_hi(v.y);
  f[4] = bf16_lo(v.z); f[5] = bf16_hi(v.z);
  f[6] = bf16_lo(v.w); f[7] = bf16_hi(v.w);
}

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&t);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// jax.nn.gelu's default tanh approximation.
__device__ __forceinline__ float gelu_tanh(float x) {
  const float c = 0.7978845608028654f;   // sqrt(2/pi)
  return 0.5f * x * (1.0f + tanhf(c * (x + 0.044715f * x * x * x)));
}

// Programmatic dependent launch: a kernel launched with the programmatic
// stream-serialisation attribute may start while its predecessor drains; it
// must not touch the predecessor's outputs before pdl_wait().
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ---- mbarrier + 1-D bulk copy (TMA) helpers ---------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_fence_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Bounded wait: returns false (instead of spinning forever) if the phase does
// not complete; the caller records kDevErrTimeout and carries on.
#ifndef MTJ_WAIT_POLLS
#define MTJ_WAIT_POLLS (1 << 18)           // behind the first look; 0 in a build that tests what a wait that runs out leaves behind
#endif
template <int POLLS = MTJ_WAIT_POLLS>
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
  {
    // a phase that is already complete is seen without the (possibly suspending) try_wait
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
  }
  for (int i = 0; i < POLLS; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return false;
}
// The chance that a copy in flight is given to land before its block leaves, whatever the limit of the waits that ran out.
__device__ __forceinline__ void mbar_settle(uint32_t bar, uint32_t parity) { mbar_wait<(1 << 18)>(bar, parity); }
__device__ __forceinline__ uint64_t l2_evict_first_policy() {
  uint64_t pol;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(pol));
  return pol;
}
// global -> this block's shared memory, `bytes` a multiple of 16, both 16-byte aligned
__device__ __forceinline__ void bulk_load(uint32_t dst_smem, const void* src, uint32_t bytes, uint32_t bar,
                                          uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
      ::"r"(dst_smem), "l"(src), "r"(bytes), "r"(bar), "l"(policy)
      : "memory");
}

// Physical location of (page-table row, absolute position) in a KV pool laid
// out [page][head][kPageTokens][d_head].
__device__ __forceinline__ size_t kv_offset(const int32_t* __restrict__ table_row, int ring_pages,
                                            int heads, int d_head, int head, int pos) {
  const int slot = (pos / kPageTokens) % ring_pages;
  const int page = table_row[slot];
  return ((static_cast<size_t>(page) * heads + head) * kPageTokens + (pos % kPageTokens)) *
         static_cast<size_t>(d_head);
}

}  // namespace mtj

// What the kernels of serving from a paged cache share: the three element types of activations, caches and logits, and the
// checks of a cache's view.
#pragma once
#include "common.cuh"
#include "tc_ptx.cuh"

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// Waits for a phase of an mbarrier, for two seconds at most: false when it gave up. A parity only tells a phase from its
// neighbours, so whoever waits has to meet every phase of the barrier in order.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity) {
  if (tc::mbar_try_wait(bar, parity)) return true;
  unsigned long long t0, t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
  do {
    if (tc::mbar_try_wait_for(bar, parity, 1000)) return true;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  } while (t - t0 < 2000000000ull);
  return tc::mbar_try_wait(bar, parity);
}

// Counts an arrival, after whatever this thread, and through a barrier its warp or CTA, has written; what those counted before
// had written is visible behind it, through a barrier to the others too. (One instruction: a relaxed one between two fences
// took 0.4 us longer.)
__device__ __forceinline__ uint32_t arrive_at(uint32_t* counter) {
  uint32_t before;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
  return before;
}

static inline bool paged_kind(int kind) { return kind == FC_F32 || kind == FC_F16 || kind == FC_BF16; }
static inline size_t paged_bytes(int kind) { return kind == FC_F32 ? 4 : 2; }
static inline bool aligned_to(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
constexpr uint32_t PAGED_MAX_PAGE = 256, PAGED_MAX_HEAD_DIM = 256;

// paged_plan.cu: the fields of a view that every entry point reads, and those of its k and v
int paged_check_pages(FcDevice* dev, const FcPagedCache* c);
int paged_check_pool(FcDevice* dev, const FcPagedCache* c);
// An operator's scratch, `bytes` for the handle's life, of which the first `zero` start at zero. Allocated by the operator's
// first call, under a stream capture too (no stream operation).
int serving_scratch(FcDevice* dev, ServingScratch* s, size_t zero, size_t bytes, void** out);

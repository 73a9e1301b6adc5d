// Log-probabilities of given tokens, the distribution's entropy, the target's rank and the largest alternatives of rows of
// logits.
//
// With m the row's maximum, S = sum e^(x - m) and T = sum e^(x - m) (x - m): lse = m + ln S, the log-probability of token t is
// x_t - lse and the entropy ln S - T / S. S and T are f32 sums of one thread's share, then of the row in a fixed order.
#include "paged.cuh"

namespace {

constexpr uint32_t TOP_MAX = 32;
constexpr int LP_THREADS = 512;

struct LogprobArgs {
  const void* logits;
  uint64_t stride;
  uint32_t vocab, top;
  const int32_t* targets;
  float *logprob, *entropy;
  int32_t* rank;
  int32_t* top_index;
  float* top_logprob;
};

// larger values first, equal ones by lower index: the larger key wins; 0 is no candidate (NaN)
__device__ __forceinline__ unsigned long long key_of(float x, uint32_t i) {
  if (x != x) return 0ull;
  const uint32_t b = __float_as_uint(x + 0.0f); // (-0 + 0 = +0)
  return ((unsigned long long)(b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u)) << 32) | (0xffffffffu - i);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float(b ^ ((b >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ unsigned long long block_max(unsigned long long v, unsigned long long* sm) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int i = 0; i < LP_THREADS / 32; i++) v = max(v, sm[i]);
  __syncthreads();
  return v;
}
template <typename V>
__device__ __forceinline__ V block_sum(V v, V* sm) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < LP_THREADS / 32; i++) v += sm[i];
  __syncthreads();
  return v;
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(LogprobArgs a) {
  __shared__ unsigned long long sm_k[LP_THREADS / 32];
  __shared__ float sm_f[LP_THREADS / 32];
  __shared__ uint32_t sm_u[LP_THREADS / 32];
  grid_wait();
  const uint32_t r = blockIdx.x;
  const T* x = (const T*)a.logits + (size_t)r * a.stride;
  const int32_t t = a.targets ? a.targets[r] : -1;
  const bool has = (uint32_t)t < a.vocab;
  const unsigned long long mine = has ? key_of(to_f32(x[t]), (uint32_t)t) : 0ull;
  unsigned long long best = 0;
  for (uint32_t i = threadIdx.x; i < a.vocab; i += LP_THREADS) best = max(best, key_of(to_f32(x[i]), i));
  best = block_max(best, sm_k);
  const float m = best ? key_value(best) : 0.0f, base = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f, of = 0.0f;
  uint32_t above = 0;
  for (uint32_t i = threadIdx.x; i < a.vocab; i += LP_THREADS) {
    const float v = to_f32(x[i]), d = v - base, e = expf(d);
    sum += e;
    of += e == 0.0f ? 0.0f : e * d;
    above += key_of(v, i) > mine;
  }
  sum = block_sum(sum, sm_f), of = block_sum(of, sm_f), above = block_sum(above, sm_u);
  const float log_sum = sum == 0.0f ? 0.0f : logf(sum);
  if (threadIdx.x == 0) {
    if (a.logprob) a.logprob[r] = has ? to_f32(x[t]) - base - log_sum : __int_as_float(0x7fffffff);
    if (a.entropy) a.entropy[r] = sum == 0.0f ? 0.0f : log_sum - of / sum;
    if (a.rank) a.rank[r] = has ? (int32_t)above : -1;
  }
  for (uint32_t k = 0; k < a.top; k++) {
    if (k) {
      const unsigned long long below = best;
      best = 0;
      if (below)
        for (uint32_t i = threadIdx.x; i < a.vocab; i += LP_THREADS) {
          const unsigned long long key = key_of(to_f32(x[i]), i);
          if (key < below) best = max(best, key);
        }
      best = block_max(best, sm_k);
    }
    if (threadIdx.x == 0) {
      if (a.top_index) a.top_index[(size_t)r * a.top + k] = best ? (int32_t)(0xffffffffu - (uint32_t)best) : -1;
      if (a.top_logprob) a.top_logprob[(size_t)r * a.top + k] = best ? key_value(best) - base - log_sum : -INFINITY;
    }
  }
}

} // namespace

FC_API int fc_logprobs_dev(FcDevice* dev, const void* logits, int kind, uint32_t rows, uint64_t stride, uint32_t vocab, const int32_t* targets,
                           uint32_t top, float* logprob, float* entropy, int32_t* rank, int32_t* top_index, float* top_logprob) {
  if (!dev) return FC_ERR_ARG;
  cudaSetDevice(dev->ordinal);
  if (!paged_kind(kind)) return fc_fail(dev, FC_ERR_UNSUPPORTED, "logits are f32, f16 or bf16, not kind %d", kind);
  if (rows && !logits) return fc_fail(dev, FC_ERR_ARG, "fc_logprobs_dev: logits are NULL");
  if (vocab == 0 || vocab > (1u << 30)) return fc_fail(dev, FC_ERR_SHAPE, "rows of %u logits", vocab);
  if (rows > 1 && stride < vocab) return fc_fail(dev, FC_ERR_SHAPE, "rows of %u logits %llu apart", vocab, (unsigned long long)stride);
  if (top > TOP_MAX) return fc_fail(dev, FC_ERR_UNSUPPORTED, "at most %u alternatives, not %u", TOP_MAX, top);
  if (rows && !aligned_to(logits, paged_bytes(kind))) return fc_fail(dev, FC_ERR_ARG, "logits must be aligned to their elements");
  if (rows > (1u << 30)) return fc_fail(dev, FC_ERR_SHAPE, "%u rows", rows);
  if (!rows) return FC_OK;
  const LogprobArgs a{logits, stride, vocab, top_index || top_logprob ? top : 0u, targets, logprob, entropy, rank, top_index, top_logprob};
  auto kern = kind == FC_F32 ? logprobs_kernel<float> : kind == FC_F16 ? logprobs_kernel<__half> : logprobs_kernel<__nv_bfloat16>;
  FC_LAUNCH(dev, "logprobs", launch_on(dev, true, kern, dim3(rows), dim3(LP_THREADS), 0, a));
  return FC_OK;
}

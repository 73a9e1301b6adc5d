// Attention of new tokens over a paged key-value cache: out = sum_j p_j v_j with p the softmax of scale * q . k_j over the
// positions j a row may see, found through its request's page table.
//
// One pass with the softmax's running maximum and sum: where a later score raises the maximum from m to m', the sum and
// the weighted values so far are multiplied by 2^(m - m') (scores are held times log2 e).
#include <cmath>

#include "paged.cuh"

namespace {

struct AttendArgs {
  const void *q, *k, *v;
  void* out;
  const int32_t *request, *position, *table;
  uint64_t q_stride, out_stride;
  uint32_t heads, kv_heads, hd, requests, max_pages, n_pages, page_shift;
  float scale; // times log2 e
};

// One CTA per (row, query head); a warp takes every fourth position, a lane channels lane, lane + 32, ..
template <typename T, typename C>
__global__ void __launch_bounds__(128) attend_kernel(AttendArgs a) {
  constexpr int E = PAGED_MAX_HEAD_DIM / 32;
  __shared__ float sm_m[4], sm_l[4], sm_o[4][PAGED_MAX_HEAD_DIM];
  grid_wait();
  const uint32_t h = blockIdx.x, r = blockIdx.y, kvh = h / (a.heads / a.kv_heads);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int32_t req = a.request ? a.request[r] : (int32_t)r;
  const uint64_t cap = (uint64_t)a.max_pages << a.page_shift;
  const uint32_t len = (uint32_t)req < a.requests && a.position[r] >= 0 ? (uint32_t)min((uint64_t)a.position[r] + 1, cap) : 0u;
  const int32_t* table = a.table + (size_t)(len ? req : 0) * a.max_pages;
  const uint32_t mask = (1u << a.page_shift) - 1;
  float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < E; i++) {
    const uint32_t e = lane + 32 * i;
    q[i] = e < a.hd ? to_f32(((const T*)a.q)[(size_t)r * a.q_stride + (size_t)h * a.hd + e]) * a.scale : 0.0f;
    o[i] = 0.0f;
  }
  for (uint32_t j = warp; j < len; j += 4) {
    const uint32_t page = (uint32_t)table[j >> a.page_shift];
    if (page >= a.n_pages) continue;
    const size_t at = ((((size_t)page * a.kv_heads + kvh) << a.page_shift) + (j & mask)) * a.hd;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; i++)
      if (lane + 32 * i < a.hd) s = fmaf(q[i], to_f32(((const C*)a.k)[at + lane + 32 * i]), s);
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.0f : mn;
    const float keep = exp2f(m - base), p = exp2f(s - base);
    m = mn, l = fmaf(l, keep, p);
#pragma unroll
    for (int i = 0; i < E; i++)
      if (lane + 32 * i < a.hd) o[i] = fmaf(o[i], keep, p * to_f32(((const C*)a.v)[at + lane + 32 * i]));
  }
  if (lane == 0) sm_m[warp] = m, sm_l[warp] = l;
#pragma unroll
  for (int i = 0; i < E; i++) sm_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float mx = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
  if (mx == -INFINITY) mx = 0.0f;
  float sum = 0.0f, w[4];
  for (int i = 0; i < 4; i++) w[i] = exp2f(sm_m[i] - mx), sum = fmaf(sm_l[i], w[i], sum);
  for (uint32_t e = threadIdx.x; e < a.hd; e += 128) {
    float v = 0.0f;
    for (int i = 0; i < 4; i++) v = fmaf(sm_o[i][e], w[i], v);
    ((T*)a.out)[(size_t)r * a.out_stride + (size_t)h * a.hd + e] = from_f32<T>(sum == 0.0f ? 0.0f : v / sum);
  }
}

template <typename T>
int launch_attend(FcDevice* dev, int cache_kind, uint32_t rows, const AttendArgs& a) {
  auto kern = cache_kind == FC_F32 ? attend_kernel<T, float> : cache_kind == FC_F16 ? attend_kernel<T, __half> : attend_kernel<T, __nv_bfloat16>;
  FC_LAUNCH(dev, "paged_attend", launch_on(dev, true, kern, dim3(a.heads, rows), dim3(128), 0, a));
  return FC_OK;
}

} // namespace

FC_API int fc_paged_attend_dev(FcDevice* dev, const FcPagedCache* c, const void* q, int kind, uint64_t q_stride, uint32_t rows, uint32_t heads,
                               const int32_t* request, const int32_t* position, float scale, void* out, uint64_t out_stride) {
  if (!dev) return FC_ERR_ARG;
  cudaSetDevice(dev->ordinal);
  FC_TRY(paged_check_pool(dev, c));
  if (!c->table || !c->requests || !c->max_pages) return fc_fail(dev, FC_ERR_ARG, "attention needs the cache's page table");
  if (!paged_kind(kind)) return fc_fail(dev, FC_ERR_UNSUPPORTED, "rows are f32, f16 or bf16, not kind %d", kind);
  if (rows && (!q || !position || !out)) return fc_fail(dev, FC_ERR_ARG, "fc_paged_attend_dev: a pointer is NULL");
  if (heads == 0 || heads % c->kv_heads) return fc_fail(dev, FC_ERR_SHAPE, "heads %u is not a multiple of kv_heads %u", heads, c->kv_heads);
  const uint64_t width = (uint64_t)heads * c->head_dim;
  if (width > (1u << 30) || rows > 65535) return fc_fail(dev, FC_ERR_UNSUPPORTED, "%u rows of %llu elements", rows, (unsigned long long)width);
  if (rows > 1 && (q_stride < width || out_stride < width))
    return fc_fail(dev, FC_ERR_SHAPE, "rows of %llu elements %llu and %llu apart", (unsigned long long)width, (unsigned long long)q_stride,
                   (unsigned long long)out_stride);
  if (rows && (!aligned_to(q, paged_bytes(kind)) || !aligned_to(out, paged_bytes(kind))))
    return fc_fail(dev, FC_ERR_ARG, "q and the result must be aligned to their elements");
  if (!std::isfinite(scale)) return fc_fail(dev, FC_ERR_ARG, "the scale is not finite");
  if (!request && rows > c->requests) return fc_fail(dev, FC_ERR_RANGE, "%u rows in a table of %u requests", rows, c->requests);
  if (!rows) return FC_OK;
  AttendArgs a = {};
  a.q = q, a.k = c->k, a.v = c->v, a.out = out, a.request = request, a.position = position, a.table = c->table;
  a.q_stride = q_stride, a.out_stride = out_stride, a.heads = heads, a.kv_heads = c->kv_heads, a.hd = c->head_dim;
  a.requests = c->requests, a.max_pages = c->max_pages, a.n_pages = c->n_pages, a.page_shift = (uint32_t)__builtin_ctz(c->page);
  a.scale = (scale == 0.0f ? 1.0f / sqrtf((float)c->head_dim) : scale) * 1.44269504088896340736f;
  return kind == FC_F32   ? launch_attend<float>(dev, c->kind, rows, a)
         : kind == FC_F16 ? launch_attend<__half>(dev, c->kind, rows, a)
                          : launch_attend<__nv_bfloat16>(dev, c->kind, rows, a);
}

// Rotary positions on the q and k heads of fused qkv rows, and k and v written to their slots of a paged cache: one launch
// that reads every row once.
//
// A pair (a, b) of channels becomes (a c - b s, a s + b c) with c, s of the row's position and the pair's index, in f32
// whatever the rows' and the cache's type, rounded once when it is stored. The tables come with the call
// (fc_rope_tables): angles of long contexts need 64 bits, the rotation does not.
#include <cmath>
#include <vector>

#include "paged.cuh"

namespace {

struct AppendArgs {
  const void* qkv;
  void *q_out, *k, *v;
  const float *cos, *sin;
  const int64_t* slot;
  const int32_t* position;
  uint64_t stride, q_stride, slots;
  uint32_t heads, kv_heads, hd, half, positions, page_shift;
  bool neox;
};

// element e of a head at x, rotated where it belongs to a pair
template <typename T>
__device__ __forceinline__ float turned(const AppendArgs& a, const T* x, uint32_t e, const float* c, const float* s) {
  if (e >= 2 * a.half) return to_f32(x[e]);
  const uint32_t p = a.neox ? (e < a.half ? e : e - a.half) : e / 2;
  const bool second = a.neox ? e >= a.half : e & 1;
  const float u = to_f32(x[a.neox ? p : 2 * p]), w = to_f32(x[a.neox ? p + a.half : 2 * p + 1]);
  return second ? fmaf(u, s[p], w * c[p]) : fmaf(u, c[p], -(w * s[p]));
}

template <typename T, typename C>
__global__ void __launch_bounds__(256) append_kernel(AppendArgs a) {
  grid_wait();
  const uint32_t r = blockIdx.x;
  const T* row = (const T*)a.qkv + (size_t)r * a.stride;
  const int64_t slot = a.slot[r];
  const int32_t pos = a.position[r];
  const bool dead = pos < 0 || (a.half && (uint32_t)pos >= a.positions);
  const bool stored = !dead && (uint64_t)slot < a.slots;
  const float* c = a.cos + (dead ? 0 : (size_t)pos * a.half);
  const float* s = a.sin + (dead ? 0 : (size_t)pos * a.half);
  const uint64_t page = (uint64_t)slot >> a.page_shift, in_page = (uint64_t)slot & ((1u << a.page_shift) - 1);
  const uint32_t n = (a.heads + 2 * a.kv_heads) * a.hd;
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
    const uint32_t h = i / a.hd, e = i % a.hd;
    if (h < a.heads) {
      ((T*)a.q_out)[(size_t)r * a.q_stride + i] = from_f32<T>(dead ? 0.0f : turned(a, row + (size_t)h * a.hd, e, c, s));
    } else if (stored) {
      const bool is_k = h < a.heads + a.kv_heads;
      const uint32_t kh = h - a.heads - (is_k ? 0 : a.kv_heads);
      const float v = is_k ? turned(a, row + (size_t)h * a.hd, e, c, s) : to_f32(row[i]);
      ((C*)(is_k ? a.k : a.v))[(((page * a.kv_heads + kh) << a.page_shift) + in_page) * a.hd + e] = from_f32<C>(v);
    }
  }
}

template <typename T>
int launch_append(FcDevice* dev, int cache_kind, uint32_t rows, const AppendArgs& a) {
  auto kern = cache_kind == FC_F32 ? append_kernel<T, float> : cache_kind == FC_F16 ? append_kernel<T, __half> : append_kernel<T, __nv_bfloat16>;
  FC_LAUNCH(dev, "paged_append", launch_on(dev, true, kern, dim3(rows), dim3(256), 0, a));
  return FC_OK;
}

} // namespace

FC_API int fc_paged_append_dev(FcDevice* dev, const FcPagedCache* c, const FcRotary* rotary, const void* qkv, int kind, uint64_t stride,
                               uint32_t rows, uint32_t heads, const int64_t* slot, const int32_t* position, void* q_out, uint64_t q_stride) {
  if (!dev) return FC_ERR_ARG;
  cudaSetDevice(dev->ordinal);
  FC_TRY(paged_check_pool(dev, c));
  if (!paged_kind(kind)) return fc_fail(dev, FC_ERR_UNSUPPORTED, "rows are f32, f16 or bf16, not kind %d", kind);
  if (rows && (!qkv || !slot || !position || !q_out)) return fc_fail(dev, FC_ERR_ARG, "fc_paged_append_dev: a pointer is NULL");
  if (heads == 0 || heads % c->kv_heads) return fc_fail(dev, FC_ERR_SHAPE, "heads %u is not a multiple of kv_heads %u", heads, c->kv_heads);
  const uint64_t width = ((uint64_t)heads + 2ull * c->kv_heads) * c->head_dim;
  if (width > (1u << 30)) return fc_fail(dev, FC_ERR_UNSUPPORTED, "rows of %llu elements", (unsigned long long)width);
  if (rows > 1 && (stride < width || q_stride < (uint64_t)heads * c->head_dim))
    return fc_fail(dev, FC_ERR_SHAPE, "rows of %llu elements %llu apart (q: %llu)", (unsigned long long)width, (unsigned long long)stride,
                   (unsigned long long)q_stride);
  if (rows && (!aligned_to(qkv, paged_bytes(kind)) || !aligned_to(q_out, paged_bytes(kind))))
    return fc_fail(dev, FC_ERR_ARG, "qkv and q must be aligned to their elements");
  AppendArgs a = {};
  if (rotary) {
    if (!rotary->cos || !rotary->sin || !rotary->positions) return fc_fail(dev, FC_ERR_ARG, "rotary tables are NULL or empty");
    if (rotary->rope_dim == 0 || rotary->rope_dim % 2 || rotary->rope_dim > c->head_dim)
      return fc_fail(dev, FC_ERR_SHAPE, "rope_dim %u must be even and at most head_dim %u", rotary->rope_dim, c->head_dim);
    if (rotary->rope_type != FC_ROPE_NORM && rotary->rope_type != FC_ROPE_NEOX) return fc_fail(dev, FC_ERR_ARG, "unknown rope type %u", rotary->rope_type);
    a.cos = rotary->cos, a.sin = rotary->sin, a.half = rotary->rope_dim / 2, a.positions = rotary->positions, a.neox = rotary->rope_type == FC_ROPE_NEOX;
  }
  if (!rows) return FC_OK;
  if (rows > (1u << 30)) return fc_fail(dev, FC_ERR_SHAPE, "%u rows", rows);
  a.qkv = qkv, a.q_out = q_out, a.k = c->k, a.v = c->v, a.slot = slot, a.position = position, a.stride = stride, a.q_stride = q_stride;
  a.slots = (uint64_t)c->n_pages * c->page, a.heads = heads, a.kv_heads = c->kv_heads, a.hd = c->head_dim;
  a.page_shift = (uint32_t)__builtin_ctz(c->page);
  return kind == FC_F32   ? launch_append<float>(dev, c->kind, rows, a)
         : kind == FC_F16 ? launch_append<__half>(dev, c->kind, rows, a)
                          : launch_append<__nv_bfloat16>(dev, c->kind, rows, a);
}

FC_API int fc_rope_tables(const FcRopeScaling* s, uint32_t positions, float* cos_out, float* sin_out) {
  if (!s || !cos_out || !sin_out) return fc_fail(nullptr, FC_ERR_ARG, "fc_rope_tables: a pointer is NULL");
  const uint32_t half = s->rope_dim / 2;
  auto bad = [](float v) { return !std::isfinite(v) || v <= 0.0f; };
  if (s->rope_dim == 0 || s->rope_dim % 2 || s->rope_dim > (1u << 16)) return fc_fail(nullptr, FC_ERR_SHAPE, "rope_dim %u must be even and positive", s->rope_dim);
  if (bad(s->base) || bad(s->linear_factor)) return fc_fail(nullptr, FC_ERR_ARG, "base and linear_factor must be finite and positive");
  if (s->n_freq_factors && (s->n_freq_factors != half || !s->freq_factors)) return fc_fail(nullptr, FC_ERR_SHAPE, "%u frequency factors for %u pairs", s->n_freq_factors, half);
  if (s->original_ctx && (bad(s->factor) || bad(s->beta_fast) || bad(s->beta_slow) || s->base == 1.0f || !std::isfinite(s->attn_factor) || s->attn_factor < 0.0f))
    return fc_fail(nullptr, FC_ERR_ARG, "factor, beta_fast and beta_slow must be finite and positive");
  for (uint32_t i = 0; i < s->n_freq_factors; i++)
    if (bad(s->freq_factors[i])) return fc_fail(nullptr, FC_ERR_ARG, "frequency factor %u must be finite and positive", i);
  std::vector<double> freq;
  try {
    freq.resize(half);
  } catch (...) {
    return fc_fail(nullptr, FC_ERR_OOM, "no host memory");
  }
  double low = 0.0, high = 0.0, mag = 1.0;
  if (s->original_ctx) {
    // the pair that turns `beta` times in original_ctx positions: base^(-2i / d) * ctx = 2 pi beta
    auto pair_of = [&](double beta) { return s->rope_dim * std::log(s->original_ctx / (beta * 2.0 * M_PI)) / (2.0 * std::log((double)s->base)); };
    low = std::fmax(std::floor(pair_of(s->beta_fast)), 0.0);
    high = std::fmin(std::ceil(pair_of(s->beta_slow)), (double)s->rope_dim - 1.0);
    mag = s->attn_factor != 0.0f ? (double)s->attn_factor : s->factor > 1.0f ? 0.1 * std::log((double)s->factor) + 1.0 : 1.0;
  }
  for (uint32_t i = 0; i < half; i++) {
    double f = std::pow((double)s->base, -2.0 * i / s->rope_dim) / s->linear_factor;
    if (s->n_freq_factors) f /= s->freq_factors[i];
    if (s->original_ctx) {
      const double slow = std::fmin(std::fmax((i - low) / std::fmax(high - low, 1e-3), 0.0), 1.0);
      f = f * (1.0 - slow) + f / s->factor * slow;
    }
    freq[i] = f;
  }
  for (uint32_t p = 0; p < positions; p++)
    for (uint32_t i = 0; i < half; i++) {
      const double angle = p * freq[i];
      cos_out[(size_t)p * half + i] = (float)(std::cos(angle) * mag);
      sin_out[(size_t)p * half + i] = (float)(std::sin(angle) * mag);
    }
  return FC_OK;
}

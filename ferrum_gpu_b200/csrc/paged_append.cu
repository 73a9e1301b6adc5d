// Rotary positions on the q and k heads of fused qkv rows, and k and v written to their slots of a paged cache: one launch
// that reads every row once.
//
// A pair (a, b) of channels becomes (a c - b s, a s + b c) with c, s of the row's position and the pair's index, in f32
// whatever the rows' and the cache's type, rounded once when it is stored. The tables come with the call
// (fc_rope_tables): angles of long contexts need 64 bits, the rotation does not.
//
// What bounds it is bytes: every row read and written once. A row is cut into items of up to N elements a load (16 bytes of a
// 16-bit row): a run of N pairs of a head - one piece for neighbouring pairs, two for the half layout -, or N channels that are
// only copied. Items of all rows are one line, so that small heads and few rows fill warps too; a thread has the loads of
// two items in flight. The tables' rows are shared by all heads and come from L1 / L2.
#include <algorithm>
#include <cmath>
#include <vector>

#include "paged.cuh"

namespace {

struct Div { // by a constant: (n * mul) >> 32 >> shift, for n below 2^31
  uint32_t d, mul, shift;
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return d == 1 ? n : __umulhi(n, mul) >> shift; }
};
Div div_by(uint32_t d) {
  Div r{d, 0, 0};
  while ((2ull << r.shift) < d) r.shift++; // 2^shift < d <= 2^(shift + 1)
  r.mul = (uint32_t)(((1ull << (32 + r.shift)) + d - 1) / d);
  return r;
}

struct AppendArgs {
  const void* qkv;
  void *q_out, *k, *v;
  const float *cos, *sin;
  const int64_t* slot;
  const int32_t* position;
  uint64_t stride, q_stride, slots;
  uint32_t rows, heads, kv_heads, hd, half, positions, page_shift;
  bool neox;
  uint32_t turned;               // items of a head that are rotated
  Div items, per_head, per_v;    // items of a row, of a q or k head, of a v head
};

constexpr int APPEND_THREADS = 256, IN_FLIGHT = 2;

// N elements side by side, one or two accesses of up to 16 bytes
template <typename T, int N>
__device__ __forceinline__ void load_run(const T* p, float (&x)[N]) {
  constexpr int BYTES = N * (int)sizeof(T);
  if constexpr (N == 1) {
    x[0] = to_f32(*p);
  } else {
    union {
      T e[N];
      uint4 v16[(BYTES + 15) / 16];
      uint2 v8;
      uint32_t v4;
    } u;
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; i++) u.v16[i] = *(reinterpret_cast<const uint4*>(p) + i);
    } else if constexpr (BYTES == 8) {
      u.v8 = *reinterpret_cast<const uint2*>(p);
    } else {
      u.v4 = *reinterpret_cast<const uint32_t*>(p);
    }
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = to_f32(u.e[i]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_run(T* p, const float (&x)[N]) {
  constexpr int BYTES = N * (int)sizeof(T);
  if constexpr (N == 1) {
    *p = from_f32<T>(x[0]);
  } else {
    union {
      T e[N];
      uint4 v16[(BYTES + 15) / 16];
      uint2 v8;
      uint32_t v4;
    } u;
#pragma unroll
    for (int i = 0; i < N; i++) u.e[i] = from_f32<T>(x[i]);
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; i++) *(reinterpret_cast<uint4*>(p) + i) = u.v16[i];
    } else if constexpr (BYTES == 8) {
      *reinterpret_cast<uint2*>(p) = u.v8;
    } else {
      *reinterpret_cast<uint32_t*>(p) = u.v4;
    }
  }
}

// N: elements of an item's piece; 1 also takes pairs that no wider piece meets, and rows aligned to nothing but elements
template <typename T, typename C, int N>
__global__ void __launch_bounds__(APPEND_THREADS) append_kernel(AppendArgs a) {
  grid_wait();
  const uint32_t all = a.rows * a.items.d, threads = gridDim.x * APPEND_THREADS;
  for (uint32_t first = blockIdx.x * APPEND_THREADS + threadIdx.x; first < all; first += threads * IN_FLIGHT) {
    float x[IN_FLIGHT][N], y[IN_FLIGHT][N];
    uint32_t row[IN_FLIGHT], head[IN_FLIGHT], ch[IN_FLIGHT]; // ch: the first piece's first channel; the second's lies `apart` behind
    bool turn[IN_FLIGHT];
    int32_t pos[IN_FLIGHT];
    int64_t slot[IN_FLIGHT];
    const uint32_t apart = a.neox ? a.half : 1u;
#pragma unroll
    for (int i = 0; i < IN_FLIGHT; i++) {
      const uint32_t id = first + i * threads;
      if (id >= all) break;
      row[i] = a.items.of(id);
      uint32_t it = id - row[i] * a.items.d;
      const uint32_t rotating = (a.heads + a.kv_heads) * a.per_head.d;
      if (it < rotating) {
        head[i] = a.per_head.of(it), it -= head[i] * a.per_head.d;
        turn[i] = it < a.turned;
        ch[i] = turn[i] ? (N == 1 && !a.neox ? 2 * it : it * N) : 2 * a.half + (it - a.turned) * N;
      } else {
        it -= rotating;
        const uint32_t h = a.per_v.of(it);
        head[i] = a.heads + a.kv_heads + h, ch[i] = (it - h * a.per_v.d) * N, turn[i] = false;
      }
      const T* src = static_cast<const T*>(a.qkv) + (size_t)row[i] * a.stride + (size_t)head[i] * a.hd + ch[i];
      load_run<T, N>(src, x[i]);
      if (turn[i] && (a.neox || N == 1)) load_run<T, N>(src + apart, y[i]);
      pos[i] = a.position[row[i]], slot[i] = a.slot[row[i]];
    }
#pragma unroll
    for (int i = 0; i < IN_FLIGHT; i++) {
      if (first + i * threads >= all) break;
      const bool dead = pos[i] < 0 || (a.half && (uint32_t)pos[i] >= a.positions);
      const bool second = turn[i] && (a.neox || N == 1);
      if (turn[i] && !dead) {
        const float* c = a.cos + (size_t)pos[i] * a.half;
        const float* s = a.sin + (size_t)pos[i] * a.half;
        if (second) {
          float cs[N], sn[N];
          load_run<float, N>(c + (N == 1 && !a.neox ? ch[i] / 2 : ch[i]), cs), load_run<float, N>(s + (N == 1 && !a.neox ? ch[i] / 2 : ch[i]), sn);
#pragma unroll
          for (int e = 0; e < N; e++) {
            const float u = x[i][e], w = y[i][e];
            x[i][e] = fmaf(u, cs[e], -(w * sn[e])), y[i][e] = fmaf(u, sn[e], w * cs[e]);
          }
        } else if constexpr (N > 1) {
          float cs[N / 2], sn[N / 2];
          load_run<float, N / 2>(c + ch[i] / 2, cs), load_run<float, N / 2>(s + ch[i] / 2, sn);
#pragma unroll
          for (int e = 0; e < N / 2; e++) {
            const float u = x[i][2 * e], w = x[i][2 * e + 1];
            x[i][2 * e] = fmaf(u, cs[e], -(w * sn[e])), x[i][2 * e + 1] = fmaf(u, sn[e], w * cs[e]);
          }
        }
      }
      if (head[i] < a.heads) {
        if (dead) {
#pragma unroll
          for (int e = 0; e < N; e++) x[i][e] = y[i][e] = 0.0f;
        }
        T* to = static_cast<T*>(a.q_out) + (size_t)row[i] * a.q_stride + (size_t)head[i] * a.hd + ch[i];
        store_run<T, N>(to, x[i]);
        if (second) store_run<T, N>(to + apart, y[i]);
      } else if (!dead && (uint64_t)slot[i] < a.slots) {
        const bool is_k = head[i] < a.heads + a.kv_heads;
        const uint32_t kh = head[i] - a.heads - (is_k ? 0 : a.kv_heads);
        const uint64_t page = (uint64_t)slot[i] >> a.page_shift, in_page = (uint64_t)slot[i] & ((1u << a.page_shift) - 1);
        C* to = static_cast<C*>(is_k ? a.k : a.v) + (((page * a.kv_heads + kh) << a.page_shift) + in_page) * a.hd + ch[i];
        store_run<C, N>(to, x[i]);
        if (second) store_run<C, N>(to + apart, y[i]);
      }
    }
  }
}

template <typename T, typename C>
int launch_append(FcDevice* dev, AppendArgs a, uint32_t rope_dim, bool aligned8, bool aligned4, bool aligned2) {
  // the widest piece that pairs, tables and addresses allow (8192 rows of 48 x 128 in bf16, L2 flushed: 70 us with 8, 86 with 4, 121 with 2, 174 with 1)
  const uint32_t whole = rope_dim == 0 ? 8 : a.neox ? a.half : rope_dim, table = a.neox ? a.half : a.half;
  auto fits = [&](uint32_t n, bool aligned) { return aligned && whole % n == 0 && table % (a.neox ? n : n / 2) == 0; };
  const uint32_t n = fits(8, aligned8) ? 8 : fits(4, aligned4) ? 4 : fits(2, aligned2) ? 2 : 1;
  a.turned = n == 1 ? a.half : (a.neox ? a.half : rope_dim) / n;
  a.per_head = div_by(a.turned + (a.hd - rope_dim) / n), a.per_v = div_by(a.hd / n);
  const uint64_t items = (uint64_t)(a.heads + a.kv_heads) * a.per_head.d + (uint64_t)a.kv_heads * a.per_v.d;
  // (items are counted in 31 bits: more rows go in several launches)
  const uint32_t at_once = (uint32_t)std::min<uint64_t>(a.rows, 0x7fffffffull / items);
  a.items = div_by((uint32_t)items);
  auto kern = n == 8 ? append_kernel<T, C, 8> : n == 4 ? append_kernel<T, C, 4> : n == 2 ? append_kernel<T, C, 2> : append_kernel<T, C, 1>;
  const uint32_t rows = a.rows;
  for (uint32_t r = 0; r < rows; r += at_once) {
    AppendArgs b = a;
    b.rows = std::min(at_once, rows - r);
    b.qkv = static_cast<const T*>(a.qkv) + (size_t)r * a.stride, b.q_out = static_cast<T*>(a.q_out) + (size_t)r * a.q_stride;
    b.slot += r, b.position += r;
    const uint64_t all = (uint64_t)b.rows * items, ctas = (all + APPEND_THREADS - 1) / APPEND_THREADS, most = (uint64_t)dev->prop.multiProcessorCount * 64;
    FC_LAUNCH(dev, "paged_append", launch_on(dev, true, kern, dim3((unsigned)std::min(ctas, most)), dim3(APPEND_THREADS), 0, b));
  }
  return FC_OK;
}
template <typename T>
int launch_append(FcDevice* dev, int cache_kind, const AppendArgs& a, uint32_t rope_dim) {
  auto aligned = [&](uint32_t n) {
    const size_t bytes = std::min<size_t>(16, n * sizeof(T));
    return aligned_to(a.qkv, bytes) && aligned_to(a.q_out, bytes) && a.stride * sizeof(T) % bytes == 0 && a.q_stride * sizeof(T) % bytes == 0 &&
           (!rope_dim || (aligned_to(a.cos, 16) && aligned_to(a.sin, 16)));
  };
  const bool b8 = aligned(8), b4 = aligned(4), b2 = aligned(2);
  return cache_kind == FC_F32   ? launch_append<T, float>(dev, a, rope_dim, b8, b4, b2)
         : cache_kind == FC_F16 ? launch_append<T, __half>(dev, a, rope_dim, b8, b4, b2)
                                : launch_append<T, __nv_bfloat16>(dev, a, rope_dim, b8, b4, b2);
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
  if (width > (1u << 28)) return fc_fail(dev, FC_ERR_UNSUPPORTED, "rows of %llu elements", (unsigned long long)width);
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
  a.rows = rows, a.slots = (uint64_t)c->n_pages * c->page, a.heads = heads, a.kv_heads = c->kv_heads, a.hd = c->head_dim;
  a.page_shift = (uint32_t)__builtin_ctz(c->page);
  const uint32_t rope_dim = 2 * a.half;
  return kind == FC_F32   ? launch_append<float>(dev, c->kind, a, rope_dim)
         : kind == FC_F16 ? launch_append<__half>(dev, c->kind, a, rope_dim)
                          : launch_append<__nv_bfloat16>(dev, c->kind, a, rope_dim);
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

// Log-probabilities of given tokens, the distribution's entropy, the target's rank and the largest alternatives of rows of
// logits.
//
// With m a maximum, S = sum 2^d and T = sum 2^d d over d = (x - m) log2 e: the log-probability of token t is
// x_t - m - ln 2 log2 S, the entropy ln 2 (log2 S - T / S). Two shares (m, S, T) of a row are joined at the larger maximum:
// S f and f (T + S delta) with delta <= 0 the difference of the maxima and f = 2^delta.
//
// What bounds it is the logits' bytes (16-bit rows: also instructions, about nine per logit). A row is read once, eight
// 16-byte loads of a thread in flight; each thread keeps a running (m, S, T) and the number of logits that rank before the
// target, all of it in f32 registers. For the alternatives it only writes down the maximum of every group of logits it has
// passed. The k-th largest of the threads' largest group maxima bounds the k-th largest logit from below: only the groups
// that reach it (k and a few) are read again, and the logits that reach it are put in order by counting, for each, those
// before it. Many equal logits at that bound (forbidden tokens, a row of one value) are taken in index order instead.
//
// Few rows are cut into shares for several CTAs, so that all SMs load; the CTA of a row that arrives last joins them, in
// the shares' order: the same bits every time.
#include <type_traits>

#include "paged.cuh"

namespace {

constexpr uint32_t TOP_MAX = 32;
constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32;
constexpr int LP_VECS = 8;          // 16-byte loads of a thread in flight
constexpr uint32_t LP_GROUPS = 8;   // groups of a thread: their maxima are written down
constexpr uint32_t LP_CTAS = 4;     // CTAs resident on an SM
constexpr uint32_t LP_CAND = 1024;  // logits put in order by counting
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

struct Share { // of a row
  float m, s, t;
  uint32_t above;
};

struct LogprobArgs {
  const void* logits;
  uint64_t stride;
  uint32_t vocab, top, splits;
  const int32_t* targets;
  float *logprob, *entropy;
  int32_t* rank;
  int32_t* top_index;
  float* top_logprob;
  Share* shares;      // [rows][splits]
  float* maxima;      // [rows][splits][LP_GROUPS][LP_THREADS]
  uint32_t* arrived;  // [rows]
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) { // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// larger values first: an order-preserving integer, 0 for NaN (never listed); -0 is +0
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x != x ? 0u : b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu)); }

// Distances from a maximum, in log2 units. m log2 e is rounded once for all of a share's logits, and the share's sums are
// relative to that; where the rounding would be more than 2^-9 (logits past 2^16) the difference is formed first.
struct Base {
  float m, l2, left; // left: m log2 e - l2, what the rounding left out
  bool big;
  __device__ __forceinline__ explicit Base(float top) {
    m = top == -INFINITY ? 0.0f : top; // (nothing but forbidden tokens so far: they stay at -inf)
    big = fabsf(m) > 65536.0f;
    l2 = __fmul_rn(m, LOG2E); // (wherever it is used: never part of a fused multiply-add)
    left = big ? 0.0f : fmaf(m, LOG2E, -l2);
  }
  __device__ __forceinline__ float of(float x) const { return big ? (x - m) * LOG2E : fmaf(x, LOG2E, -l2); }
};
// from sums relative to one maximum to sums relative to a larger one
__device__ __forceinline__ float below(float from, float to) {
  const Base a(from), b(to);
  return fmaxf(a.big || b.big ? (a.m - b.m) * LOG2E - a.left + b.left : a.l2 - b.l2, -300.0f);
}
__device__ __forceinline__ void move_to(float m, Share& a) {
  if (a.m == m) return;
  const float delta = a.m == -INFINITY ? 0.0f : below(a.m, m), f = a.m == -INFINITY ? 0.0f : ex2(delta);
  a.t = f * fmaf(a.s, delta, a.t), a.s *= f, a.m = m;
}

template <typename T>
struct Vec { // 16 bytes of logits
  static constexpr int E = 16 / sizeof(T);
  static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[E]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (sizeof(T) == 4) {
        x[i] = __uint_as_float(w[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
      } else {
        x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
};

// (exponentials below 2^-150 are 0, and so is their part of T: no 0 * inf)
__device__ __forceinline__ void add(float d, float& s, float& t) {
  d = max_nan(d, -160.0f);
  const float e = ex2(d);
  s += e, t = fmaf(e, d, t);
}

template <typename V, typename F>
__device__ __forceinline__ V warp_reduce(V v, F f) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// of the whole CTA; `sm`: a word per warp, free again after the call's second barrier
template <typename V, typename F>
__device__ __forceinline__ V reduce(V v, V* sm, F f) {
  v = warp_reduce(v, f);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sm[0];
#pragma unroll
  for (int w = 1; w < LP_WARPS; w++) v = f(v, sm[w]);
  __syncthreads();
  return v;
}
// The warp's 32 keys in descending order over the lanes (bitonic); `from`: of a sequence that rises and falls only the last
// rounds are needed.
__device__ __forceinline__ uint32_t sort_lanes(uint32_t v, int from) {
  const uint32_t lane = threadIdx.x & 31;
  for (int size = from; size <= 32; size <<= 1)
    for (int stride = size >> 1; stride; stride >>= 1) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, v, stride);
      const bool low = (lane & stride) == 0, down = (lane & size) == 0 || size == 32;
      v = low == down ? max(v, other) : min(v, other);
    }
  return v;
}

// Where a row's logits lie: vectors from the first 16-byte boundary on, and the few before and behind them.
template <typename T>
struct Row {
  const T* x;
  uint32_t head, vecs, rest, vocab; // rest: logits outside the vectors
  __device__ __forceinline__ Row(const LogprobArgs& a, uint32_t r) {
    x = static_cast<const T*>(a.logits) + (size_t)r * a.stride;
    vocab = a.vocab;
    head = min(a.vocab, (uint32_t)((16 - ((uintptr_t)x & 15)) & 15) / (uint32_t)sizeof(T));
    vecs = (a.vocab - head) / Vec<T>::E;
    rest = a.vocab - vecs * Vec<T>::E;
  }
  __device__ __forceinline__ const uint4* vec(uint32_t i) const { return reinterpret_cast<const uint4*>(x + head) + i; }
  __device__ __forceinline__ uint32_t rest_at(uint32_t i) const { return i < head ? i : vocab - rest + i; }
};

template <typename T>
__global__ void __launch_bounds__(LP_THREADS, LP_CTAS) logprobs_kernel(LogprobArgs a) {
  constexpr int E = Vec<T>::E;
  __shared__ float sm_f[LP_WARPS];
  __shared__ uint32_t sm_u[LP_WARPS];
  __shared__ float own_maxima[LP_GROUPS * LP_THREADS];
  __shared__ uint32_t sm_sorted[LP_WARPS][32], sm_n, sm_ties, sm_last;
  __shared__ unsigned long long cand[LP_CAND];
  grid_wait();
  const uint32_t r = blockIdx.x / a.splits, split = blockIdx.x - r * a.splits, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Row<T> row(a, r);
  const int32_t target = a.targets ? a.targets[r] : -1;
  const bool has = (uint32_t)target < a.vocab;
  const float xt = has ? to_f32(row.x[target]) : 0.0f;
  // Logits before the target count where they are equal to it, those behind it where they are larger: larger than the next
  // smaller value, and than it. A NaN target counts all that are no NaN; nothing else does.
  const float behind = !has ? INFINITY : xt != xt ? -INFINITY : xt, before = !has ? INFINITY : xt != xt ? -INFINITY : xt == -INFINITY ? -INFINITY : nextafterf(xt, -INFINITY);
  const bool floor_too = has && (xt != xt || xt == -INFINITY); // (nothing is smaller than -inf: compared with >= there)
  auto ranks_before = [&](float x, uint32_t i) { return has && (xt != xt ? x == x : x > xt || (x == xt && i < (uint32_t)target)); };

  // this CTA's share of the vectors, a thread's in steps of LP_VECS, `per` steps to a group
  const uint32_t v0 = (uint32_t)((uint64_t)row.vecs * split / a.splits), v1 = (uint32_t)((uint64_t)row.vecs * (split + 1) / a.splits);
  constexpr uint32_t STEP = LP_THREADS * LP_VECS;
  const uint32_t steps = (v1 - v0 + STEP - 1) / STEP, per = (steps + LP_GROUPS - 1) / LP_GROUPS;
  float* maxima = a.splits == 1 ? own_maxima : a.maxima + (size_t)blockIdx.x * (LP_GROUPS * LP_THREADS);
  Share own{-INFINITY, 0.0f, 0.0f, 0u};
  float group_max = -INFINITY;
  uint32_t group = 0;
  for (uint32_t st = 0; st < steps; st++) {
    uint4 v[LP_VECS];
    const uint32_t at = v0 + st * STEP + tid;
#pragma unroll
    for (int i = 0; i < LP_VECS; i++)
      if (at + i * LP_THREADS < v1) v[i] = __ldg(row.vec(at + i * LP_THREADS));
    const int n = at < v1 ? min(LP_VECS, (int)((v1 - at + LP_THREADS - 1) / LP_THREADS)) : 0;
    float high = -INFINITY;
#pragma unroll
    for (int i = 0; i < LP_VECS; i++)
      if (i < n) {
        float x[E];
        Vec<T>::unpack(v[i], x);
#pragma unroll
        for (int e = 0; e < E; e++) high = fmaxf(high, x[e]); // (a group of NaN: -inf, which reaches nothing that it should not)
      }
    group_max = fmaxf(group_max, high);
    if (high > own.m) move_to(high, own);
    const Base base(own.m);
    auto sums = [&](auto big) {
#pragma unroll
      for (int i = 0; i < LP_VECS; i++)
        if (i < n) {
          float x[E];
          Vec<T>::unpack(v[i], x);
          const uint32_t first = row.head + (at + i * LP_THREADS) * E;
          const float thr = first + E <= (uint32_t)target ? before : behind; // (the target's own vector: looked at below)
#pragma unroll
          for (int e = 0; e < E; e++) {
            add(decltype(big)::value ? (x[e] - base.m) * LOG2E : fmaf(x[e], LOG2E, -base.l2), own.s, own.t);
            own.above += x[e] > thr;
          }
          if (floor_too || (has && first <= (uint32_t)target && (uint32_t)target < first + E)) {
#pragma unroll
            for (int e = 0; e < E; e++) own.above += (uint32_t)ranks_before(x[e], first + e) - (uint32_t)(x[e] > thr);
          }
        }
    };
    if (base.big) sums(std::true_type());
    else sums(std::false_type());
    if (a.top && ((st + 1) % per == 0 || st + 1 == steps)) {
      maxima[group++ * LP_THREADS + tid] = group_max;
      group_max = -INFINITY;
    }
  }
  if (split == 0 && tid < row.rest) {
    const uint32_t i = row.rest_at(tid);
    const float x = to_f32(row.x[i]);
    if (x > own.m) move_to(x, own);
    add(Base(own.m).of(x), own.s, own.t);
    own.above += ranks_before(x, i);
  }
  // the share
  auto larger = [](float x, float y) { return fmaxf(x, y); };
  auto plus = [](auto x, auto y) { return x + y; };
  const float m = reduce(own.m, sm_f, larger);
  move_to(m, own);
  Share all{m, reduce(own.s, sm_f, plus), reduce(own.t, sm_f, plus), reduce(own.above, sm_u, plus)};
  uint32_t groups = (steps + max(per, 1u) - 1) / max(per, 1u);
  if (a.splits > 1) {
    if (tid == 0) a.shares[blockIdx.x] = all;
    __threadfence();
    __syncthreads();
    if (tid == 0) sm_last = atomicAdd(&a.arrived[r], 1u) == a.splits - 1;
    __syncthreads();
    if (!sm_last) return;
    __threadfence();
    if (tid == 0) a.arrived[r] = 0; // for the next call
    const Share* shares = a.shares + (size_t)r * a.splits;
    Share mine{-INFINITY, 0.0f, 0.0f, 0u};
    for (uint32_t i = tid; i < a.splits; i += LP_THREADS) {
      const float4 raw = __ldcg(reinterpret_cast<const float4*>(shares + i));
      Share one{raw.x, raw.y, raw.z, __float_as_uint(raw.w)};
      const float high = fmaxf(mine.m, one.m);
      move_to(high, mine), move_to(high, one);
      mine.s += one.s, mine.t += one.t, mine.above += one.above;
    }
    const float top = reduce(mine.m, sm_f, larger);
    move_to(top, mine);
    all = Share{top, reduce(mine.s, sm_f, plus), reduce(mine.t, sm_f, plus), reduce(mine.above, sm_u, plus)};
  }
  const Base base(all.m);
  const float log_s = all.s == 0.0f ? 0.0f : log2f(all.s);
  // ln of the sum relative to the maximum itself: less what rounding m log2 e left out
  const float ln_s = LN2 * (log_s - base.left);
  auto logprob_of = [&](float x) { return x - base.m - ln_s; };
  if (tid == 0) {
    if (a.logprob) a.logprob[r] = has ? logprob_of(xt) : __int_as_float(0x7fffffff);
    if (a.entropy) a.entropy[r] = all.s == 0.0f ? 0.0f : LN2 * (log_s - all.t / all.s);
    if (a.rank) a.rank[r] = has ? (int32_t)all.above : -1;
  }
  if (!a.top) return;

  // ---- the alternatives ----
  auto put = [&](uint32_t k, unsigned long long key) { // key 0: there is none
    const float x = value_of((uint32_t)(key >> 32));
    if (a.top_index) a.top_index[(size_t)r * a.top + k] = key ? (int32_t)(0xffffffffu - (uint32_t)key) : -1;
    if (a.top_logprob) a.top_logprob[(size_t)r * a.top + k] = key ? logprob_of(x) : -INFINITY;
  };
  auto key_of = [](uint32_t order, uint32_t i) { return (unsigned long long)order << 32 | (0xffffffffu - i); };
  // the shares' maxima: group g of thread t of share s covers steps g per .. of that share
  const float* row_maxima = a.splits == 1 ? own_maxima : a.maxima + (size_t)r * a.splits * (LP_GROUPS * LP_THREADS);
  auto share_groups = [&](uint32_t s, uint32_t& first, uint32_t& last, uint32_t& per) {
    first = (uint32_t)((uint64_t)row.vecs * s / a.splits), last = (uint32_t)((uint64_t)row.vecs * (s + 1) / a.splits);
    const uint32_t steps = (last - first + STEP - 1) / STEP;
    per = (steps + LP_GROUPS - 1) / LP_GROUPS;
    return per ? (steps + per - 1) / per : 0u;
  };
  __syncthreads(); // (own_maxima)
  uint32_t best = 0;
  for (uint32_t s = 0; s < a.splits; s++) {
    uint32_t first, last, per_s;
    const uint32_t n = share_groups(s, first, last, per_s);
    for (uint32_t g = 0; g < n; g++) {
      const float* p = row_maxima + (size_t)(s * LP_GROUPS + g) * LP_THREADS + tid;
      best = max(best, order_of(a.splits == 1 ? *p : __ldcg(p)));
    }
  }
  // the k-th largest of the threads' maxima: sorted per warp, then the larger halves of pairs of warps
  uint32_t sorted = sort_lanes(best, 2);
  sm_sorted[warp][lane] = sorted;
  if (tid == 0) sm_n = 0, sm_ties = 0;
  __syncthreads();
#pragma unroll
  for (int half = LP_WARPS / 2; half; half >>= 1) {
    if (warp < half) {
      sorted = sort_lanes(max(sorted, sm_sorted[warp + half][31 - lane]), 32);
      sm_sorted[warp][lane] = sorted;
    }
    __syncthreads();
  }
  const uint32_t bound = sm_sorted[0][a.top - 1];
  // The logits above the bound, from the front of the list, and those equal to it, from its end.
  auto offer = [&](float x, uint32_t i, bool equal_too) {
    const uint32_t o = order_of(x);
    if (!o || o < bound || (o == bound && !equal_too)) return;
    const uint32_t p = atomicAdd(o > bound ? &sm_n : &sm_ties, 1u);
    if (p < LP_CAND) cand[o > bound ? p : LP_CAND - 1 - p] = key_of(o, i);
  };
  auto gather = [&](bool equal_too) {
    for (uint32_t s = 0; s < a.splits; s++) {
      uint32_t first, last, per_s;
      const uint32_t n = share_groups(s, first, last, per_s);
      for (uint32_t g = 0; g < n; g++) {
        const float* p = row_maxima + (size_t)(s * LP_GROUPS + g) * LP_THREADS + tid;
        const uint32_t o = order_of(a.splits == 1 ? *p : __ldcg(p));
        // a warp reads its groups that reach the bound one after another, a vector per lane
        for (uint32_t reach = __ballot_sync(0xffffffffu, o > bound || (o == bound && equal_too)); reach; reach &= reach - 1) {
          if (*(volatile uint32_t*)&sm_n + *(volatile uint32_t*)&sm_ties > LP_CAND) break; // (the list runs over: no use)
          const uint32_t begin = first + g * per_s * STEP + warp * 32 + __ffs(reach) - 1;
          for (uint32_t i = lane; i < per_s * LP_VECS; i += 32) {
            const uint32_t at = begin + i * LP_THREADS;
            if (at >= last) break;
            float x[E];
            Vec<T>::unpack(__ldg(row.vec(at)), x);
#pragma unroll
            for (int e = 0; e < E; e++) offer(x[e], row.head + at * E + e, equal_too);
          }
          __syncwarp();
        }
      }
    }
    if (tid < row.rest) offer(to_f32(row.x[row.rest_at(tid)]), row.rest_at(tid), equal_too);
    __syncthreads();
  };
  gather(true);
  const bool over = sm_n + sm_ties > LP_CAND;
  __syncthreads();
  if (over) { // many equal ones, as a rule: those above the bound alone
    if (tid == 0) sm_n = 0, sm_ties = 0;
    __syncthreads();
    gather(false);
  }
  const uint32_t above = sm_n, n = above + sm_ties;
  if (n <= LP_CAND) {
    // a candidate's place is the number of larger ones
    for (uint32_t i = tid; i < n; i += LP_THREADS) {
      const unsigned long long key = cand[i < above ? i : LP_CAND - 1 - (i - above)];
      uint32_t place = 0;
      for (uint32_t j = 0; j < above; j++) place += cand[j] > key;
      if (i >= above)
        for (uint32_t j = above; j < n; j++) place += cand[LP_CAND - 1 - (j - above)] > key;
      if (place < a.top) put(place, key);
    }
    uint32_t filled = n;
    if (over) // then the first ones equal to it, in index order
      for (uint32_t i0 = 0; i0 < a.vocab && filled < a.top; i0 += LP_THREADS) {
        const uint32_t i = i0 + tid;
        const bool equal = i < a.vocab && order_of(to_f32(row.x[i])) == bound;
        const uint32_t votes = __ballot_sync(0xffffffffu, equal);
        if (lane == 0) sm_u[warp] = __popc(votes);
        __syncthreads();
        uint32_t place = filled + __popc(votes & ((1u << lane) - 1));
#pragma unroll
        for (int w = 0; w < LP_WARPS; w++) {
          if (w < (int)warp) place += sm_u[w];
          filled += sm_u[w];
        }
        if (equal && place < a.top) put(place, key_of(bound, i));
        __syncthreads();
      }
    for (uint32_t k = filled + tid; k < a.top; k += LP_THREADS) put(k, 0ull);
    return;
  }
  // More logits above the bound than the list holds (a thread's groups hold nearly all that is large): one sweep for each
  // alternative, for the largest key below the last.
  unsigned long long last_key = ~0ull;
  for (uint32_t k = 0; k < a.top; k++) {
    unsigned long long mine = 0;
    for (uint32_t i = tid; i < a.vocab; i += LP_THREADS) {
      const uint32_t o = order_of(to_f32(row.x[i]));
      const unsigned long long key = o ? key_of(o, i) : 0ull;
      if (key < last_key) mine = max(mine, key);
    }
    last_key = reduce(mine, cand, [](unsigned long long x, unsigned long long y) { return max(x, y); });
    if (tid == 0) put(k, last_key);
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
  LogprobArgs a{logits, stride, vocab, top_index || top_logprob ? top : 0u, 1u, targets, logprob, entropy, rank, top_index, top_logprob, nullptr, nullptr, nullptr};
  // shares of a row: as many as there are SMs' CTAs left for it, each of whole steps
  const uint32_t ctas = (uint32_t)dev->prop.multiProcessorCount * LP_CTAS;
  const uint64_t vecs = (uint64_t)vocab * paged_bytes(kind) / 16, steps = (vecs + LP_THREADS * LP_VECS - 1) / (LP_THREADS * LP_VECS);
  if (rows < ctas && steps > 1) a.splits = (uint32_t)(steps < ctas / rows ? steps : ctas / rows);
  if (a.splits > 1) {
    const size_t words = ((size_t)ctas * 4 + 255) / 256 * 256, shares = ((size_t)ctas * sizeof(Share) + 255) / 256 * 256;
    void* p;
    FC_TRY(serving_scratch(dev, &dev->logprobs, words, words + shares + (size_t)ctas * LP_GROUPS * LP_THREADS * 4, &p));
    a.arrived = static_cast<uint32_t*>(p);
    a.shares = reinterpret_cast<Share*>(static_cast<char*>(p) + words);
    a.maxima = reinterpret_cast<float*>(static_cast<char*>(p) + words + shares);
  }
  auto kern = kind == FC_F32 ? logprobs_kernel<float> : kind == FC_F16 ? logprobs_kernel<__half> : logprobs_kernel<__nv_bfloat16>;
  FC_LAUNCH(dev, "logprobs", launch_on(dev, true, kern, dim3(rows * a.splits), dim3(LP_THREADS), 0, a));
  return FC_OK;
}

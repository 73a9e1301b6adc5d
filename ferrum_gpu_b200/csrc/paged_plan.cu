// Pages and slots of one serving step, from the requests' lengths: prefix sums over the requests, then every row of the
// step finds its request, position and slot for itself.
//
// With o_i positions held, g_i to come and P(x) = ceil(x / page): request i takes need_i = P(o_i + g_i) - P(o_i) pages, the
// j-th of them being free[n_free - 1 - (need_0 + .. + need_{i-1} + j)]; row t of request i has position o_i + t - start_i.
// Nothing depends on the order in which threads run.
//
// One cluster: each CTA forms the prefix sums of all requests for itself (a few KB from L2), then writes its share of the
// rows. Only in-place updates (lengths, stack height) have to wait until every CTA has read, which is the cluster's barrier.
#include <climits>
#include <cmath>

#include "paged.cuh"

namespace {

constexpr uint32_t PLAN_THREADS = 1024;
constexpr uint32_t PLAN_MAX = 8192; // requests of a call: their prefix sums lie in shared memory (16 bytes each)
constexpr uint32_t PLAN_CTAS = 8;   // CTAs of the cluster, where there are rows for them

struct PlanArgs {
  uint32_t page_shift, n_pages, requests, max_pages, n, rows;
  int32_t *table, *lens, *free, *n_free;
  const int32_t *req, *grow;
  int32_t* starts;
  int64_t* slot;
  int32_t *position, *request, *lens_out, *n_free_out, *status;
};

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// exclusive prefix sums of two 64-bit values per thread over the CTA, and their totals
struct Pair {
  long long a, b;
};
__device__ __forceinline__ Pair scan_pair(Pair v, Pair& total) {
  __shared__ Pair warps[32];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Pair s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, s.a, o), b = __shfl_up_sync(0xffffffffu, s.b, o);
    if (lane >= o) s.a += a, s.b += b;
  }
  if (lane == 31) warps[warp] = s;
  __syncthreads();
  if (warp == 0) {
    Pair w = lane < blockDim.x / 32 ? warps[lane] : Pair{0, 0};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long a = __shfl_up_sync(0xffffffffu, w.a, o), b = __shfl_up_sync(0xffffffffu, w.b, o);
      if (lane >= o) w.a += a, w.b += b;
    }
    warps[lane] = w;
  }
  __syncthreads();
  total = warps[blockDim.x / 32 - 1];
  const Pair before = warp ? warps[warp - 1] : Pair{0, 0};
  return {before.a + s.a - v.a, before.b + s.b - v.b};
}

__device__ __forceinline__ long long pages_of(long long len, uint32_t shift) { return (len + (1ll << shift) - 1) >> shift; }

// the faults of a step, in the order in which they are reported
enum { BAD_ROW = 1, BAD_LONG = 2, BAD_PAGE = 4 };

__global__ void __launch_bounds__(PLAN_THREADS) extend_kernel(PlanArgs a) {
  extern __shared__ int4 entry[]; // per request: rows up to and with it, positions held, pages taken before it, table row
  grid_wait();
  const uint32_t per = (a.n + blockDim.x - 1) / blockDim.x, i0 = threadIdx.x * per, i1 = min(a.n, i0 + per);
  const int32_t n_free = *a.n_free;
  int bad = 0;
  Pair mine{0, 0};
  for (uint32_t i = i0; i < i1; i++) {
    const int32_t r = a.req ? a.req[i] : (int32_t)i, g = a.grow[i];
    int32_t o = 0;
    if ((uint32_t)r >= a.requests || g < 0) bad |= BAD_ROW;
    else {
      o = a.lens[r];
      if (o < 0) bad |= BAD_ROW;
      else if ((long long)o + g > ((long long)a.max_pages << a.page_shift) || (long long)o + g > INT_MAX) bad |= BAD_LONG;
    }
    entry[i] = make_int4(g, o, 0, r);
    if (!bad) mine.a += g, mine.b += pages_of((long long)o + g, a.page_shift) - pages_of(o, a.page_shift);
  }
  bad = __syncthreads_or(bad & BAD_ROW) ? BAD_ROW : __syncthreads_or(bad) ? BAD_LONG : 0;
  Pair total;
  Pair at = scan_pair(mine, total);
  const bool held = (uint32_t)n_free <= a.n_pages; // (a stack height that is none: nothing can be taken from it)
  int32_t status = bad & BAD_ROW       ? FC_ERR_RANGE
                   : bad               ? FC_ERR_CONTEXT_FULL
                   : total.a > a.rows  ? FC_ERR_SHAPE
                   : !held             ? FC_ERR_RANGE
                   : total.b > n_free  ? (int32_t)(total.b - n_free)
                                       : 0;
  for (uint32_t i = i0; i < i1; i++) {
    const int4 e = entry[i];
    const long long o = e.y, g = e.x;
    entry[i] = make_int4((int32_t)(at.a + g), e.y, (int32_t)at.b, e.w);
    if (!status) at.a += g, at.b += pages_of(o + g, a.page_shift) - pages_of(o, a.page_shift);
  }
  __syncthreads();
  const uint32_t tokens = status ? 0u : (uint32_t)total.a;
  const uint32_t step = gridDim.x * blockDim.x, first = blockIdx.x * blockDim.x + threadIdx.x;
  const uint32_t mask = (1u << a.page_shift) - 1;
  for (uint32_t t = first; t < a.rows; t += step) {
    int64_t slot = -1;
    int32_t pos = -1, r = -1;
    if (t < tokens) {
      uint32_t lo = 0, hi = a.n - 1; // the first request whose rows end behind t
      while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if ((uint32_t)entry[mid].x > t) hi = mid;
        else lo = mid + 1;
      }
      const int4 e = entry[lo];
      const uint32_t start = lo ? (uint32_t)entry[lo - 1].x : 0u;
      pos = e.y + (int32_t)(t - start), r = e.w;
      const uint32_t p = (uint32_t)pos >> a.page_shift, had = (uint32_t)pages_of(e.y, a.page_shift);
      const int32_t page = p < had ? a.table[(size_t)r * a.max_pages + p] : a.free[n_free - 1 - (e.z + (int32_t)(p - had))];
      slot = ((int64_t)page << a.page_shift) + (pos & mask);
    }
    if (a.slot) a.slot[t] = slot;
    if (a.position) a.position[t] = pos;
    if (a.request) a.request[t] = r;
  }
  cluster_barrier(); // every CTA has read lengths, table and stack height
  for (uint32_t i = first; i < a.n; i += step) {
    const int4 e = entry[i];
    const uint32_t start = i ? (uint32_t)entry[i - 1].x : 0u;
    const int32_t g = status ? 0 : e.x - (int32_t)start;
    if (status) {
      a.starts[i] = 0;
      if (a.lens_out != a.lens && (uint32_t)e.w < a.requests) a.lens_out[e.w] = a.lens[e.w];
      continue;
    }
    a.starts[i] = (int32_t)start;
    const uint32_t had = (uint32_t)pages_of(e.y, a.page_shift), has = (uint32_t)pages_of((long long)e.y + g, a.page_shift);
    int32_t* row = a.table + (size_t)e.w * a.max_pages;
    for (uint32_t p = had; p < has; p++) row[p] = a.free[n_free - 1 - (e.z + (int32_t)(p - had))];
    a.lens_out[e.w] = e.y + g;
  }
  if (first == 0) {
    a.starts[a.n] = (int32_t)tokens;
    *a.n_free_out = status ? n_free : n_free - (int32_t)total.b;
    *a.status = status;
  }
}

__global__ void __launch_bounds__(PLAN_THREADS) release_kernel(PlanArgs a) {
  extern __shared__ int4 entry[]; // per request: pages held, -, pages of the requests before it, table row
  grid_wait();
  const uint32_t per = (a.n + blockDim.x - 1) / blockDim.x, i0 = threadIdx.x * per, i1 = min(a.n, i0 + per);
  const int32_t n_free = *a.n_free;
  int bad = (uint32_t)n_free > a.n_pages ? BAD_ROW : 0;
  Pair mine{0, 0};
  for (uint32_t i = i0; i < i1; i++) {
    const int32_t r = a.req ? a.req[i] : (int32_t)i;
    long long held = 0;
    if ((uint32_t)r >= a.requests) bad = BAD_ROW;
    else {
      const int32_t o = a.lens[r];
      if (o < 0 || (long long)o > ((long long)a.max_pages << a.page_shift)) bad = BAD_ROW;
      else held = pages_of(o, a.page_shift);
    }
    entry[i] = make_int4((int32_t)held, 0, 0, r);
    mine.b += held;
  }
  bad = __syncthreads_or(bad);
  Pair total;
  Pair at = scan_pair(mine, total);
  for (uint32_t i = i0; i < i1; i++) {
    entry[i].z = (int32_t)at.b;
    at.b += entry[i].x;
  }
  int32_t status = bad ? FC_ERR_RANGE : total.b > (long long)a.n_pages - n_free ? FC_ERR_SHAPE : 0;
  __syncthreads();
  const uint32_t lane = threadIdx.x & 31, warp = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, warps = gridDim.x * blockDim.x / 32;
  // (a table entry that is no page would come back as one: looked for before anything is pushed)
  int wrong = 0;
  if (!status)
    for (uint32_t i = warp; i < a.n; i += warps) {
      const int4 e = entry[i];
      const int32_t* row = a.table + (size_t)e.w * a.max_pages;
      for (uint32_t p = lane; p < (uint32_t)e.x; p += 32) wrong |= (uint32_t)row[p] >= a.n_pages;
    }
  wrong = __syncthreads_or(wrong);
  __shared__ int any_wrong;
  if (threadIdx.x == 0) any_wrong = 0;
  cluster_barrier();
  if (wrong && threadIdx.x < gridDim.x) { // one word in each CTA of the cluster
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(&any_wrong)), "r"(threadIdx.x));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(1) : "memory");
  }
  cluster_barrier(); // and every CTA has read lengths, table and stack height
  if (!status && any_wrong) status = FC_ERR_RANGE;
  for (uint32_t i = warp; i < a.n; i += warps) {
    const int4 e = entry[i];
    if (status) {
      if (lane == 0 && a.lens_out != a.lens && (uint32_t)e.w < a.requests) a.lens_out[e.w] = a.lens[e.w];
      continue;
    }
    const int32_t* row = a.table + (size_t)e.w * a.max_pages;
    for (uint32_t p = lane; p < (uint32_t)e.x; p += 32) a.free[n_free + e.z + (int32_t)p] = row[p];
    if (lane == 0) a.lens_out[e.w] = 0;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *a.n_free_out = status ? n_free : n_free + (int32_t)total.b;
    *a.status = status;
  }
}

int launch_plan(FcDevice* dev, const char* what, void (*kern)(PlanArgs), const PlanArgs& a, uint32_t work) {
  const size_t smem = (size_t)a.n * sizeof(int4);
  static OncePerDevice once[2];
  if (once[kern == release_kernel].first(dev->ordinal))
    FC_CUDA(dev, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(PLAN_MAX * sizeof(int4))));
  // one CTA up to a row per thread, else the whole cluster
  const uint32_t ctas = work <= PLAN_THREADS ? 1 : PLAN_CTAS;
  const uint32_t threads = work <= 256 && a.n <= 256 ? 256 : PLAN_THREADS;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = ctas, at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.gridDim = ctas, cfg.blockDim = threads, cfg.dynamicSmemBytes = smem, cfg.stream = dev->stream, cfg.attrs = at, cfg.numAttrs = 2;
  FC_LAUNCH(dev, what, cudaLaunchKernelEx(&cfg, kern, a));
  return FC_OK;
}

int plan_args(FcDevice* dev, const FcPagedCache* c, const int32_t* req, uint32_t n, int32_t* lens_out, int32_t* n_free_out, int32_t* status,
              PlanArgs* a) {
  FC_TRY(paged_check_pages(dev, c));
  if (!c->table || !c->lens || !c->free || !c->n_free || !status) return fc_fail(dev, FC_ERR_ARG, "a page plan needs the table, lengths, free pages and a status word");
  if (!c->requests || !c->max_pages) return fc_fail(dev, FC_ERR_SHAPE, "empty page table");
  if (n > PLAN_MAX) return fc_fail(dev, FC_ERR_UNSUPPORTED, "a page plan takes at most %u requests, not %u", PLAN_MAX, n);
  if (!req && n > c->requests) return fc_fail(dev, FC_ERR_RANGE, "%u requests in a table of %u", n, c->requests);
  a->page_shift = (uint32_t)__builtin_ctz(c->page), a->n_pages = c->n_pages, a->requests = c->requests, a->max_pages = c->max_pages;
  a->n = n, a->table = c->table, a->lens = c->lens, a->free = c->free, a->n_free = c->n_free, a->req = req;
  a->lens_out = lens_out ? lens_out : c->lens, a->n_free_out = n_free_out ? n_free_out : c->n_free, a->status = status;
  return FC_OK;
}

} // namespace

int serving_scratch(FcDevice* dev, ServingScratch* s, size_t zero, size_t bytes, void** out) {
  const bool fresh = !s->ws.p;
  if (fresh || !s->clear) {
    const bool capturing = stream_capturing(dev);
    if (fresh) {
      cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
      cudaThreadExchangeStreamCaptureMode(&mode);
      void* p = nullptr;
      const cudaError_t e = capturing ? cudaMalloc(&p, bytes) : device_malloc(dev, &p, bytes);
      cudaThreadExchangeStreamCaptureMode(&mode);
      FC_CUDA(dev, e);
      s->ws = Workspace{p, bytes};
    }
    FC_CUDA(dev, cudaMemsetAsync(s->ws.p, 0, zero, dev->stream)); // (captured: a node of the graph; the handle's own calls still do it once)
    s->clear = !capturing;
  }
  *out = s->ws.p;
  return FC_OK;
}

int paged_check_pages(FcDevice* dev, const FcPagedCache* c) {
  if (!c) return fc_fail(dev, FC_ERR_ARG, "the cache's view is NULL");
  if (c->page == 0 || c->page > PAGED_MAX_PAGE || (c->page & (c->page - 1)))
    return fc_fail(dev, FC_ERR_UNSUPPORTED, "a page holds a power of two of positions up to %u, not %u", PAGED_MAX_PAGE, c->page);
  if (c->n_pages == 0 || c->n_pages > (uint32_t)INT_MAX) return fc_fail(dev, FC_ERR_SHAPE, "a pool of %u pages", c->n_pages);
  return FC_OK;
}

int paged_check_pool(FcDevice* dev, const FcPagedCache* c) {
  FC_TRY(paged_check_pages(dev, c));
  if (!paged_kind(c->kind)) return fc_fail(dev, FC_ERR_UNSUPPORTED, "a paged cache holds f32, f16 or bf16, not kind %d", c->kind);
  if (c->head_dim == 0 || c->head_dim % 8 || c->head_dim > PAGED_MAX_HEAD_DIM)
    return fc_fail(dev, FC_ERR_UNSUPPORTED, "head_dim %u is not a multiple of 8 up to %u", c->head_dim, PAGED_MAX_HEAD_DIM);
  if (c->kv_heads == 0 || c->kv_heads > 65535) return fc_fail(dev, FC_ERR_SHAPE, "%u kv heads", c->kv_heads);
  if (!c->k || !c->v) return fc_fail(dev, FC_ERR_ARG, "the cache's k or v is NULL");
  if (!aligned_to(c->k, 16) || !aligned_to(c->v, 16)) return fc_fail(dev, FC_ERR_ARG, "the cache's k and v must be 16-byte aligned");
  return FC_OK;
}

FC_API int fc_paged_extend_dev(FcDevice* dev, const FcPagedCache* c, const int32_t* requests, const int32_t* grow, uint32_t n, uint32_t rows,
                               int32_t* starts, int64_t* slot, int32_t* position, int32_t* request, int32_t* lens_out, int32_t* n_free_out,
                               int32_t* status) {
  if (!dev) return FC_ERR_ARG;
  cudaSetDevice(dev->ordinal);
  PlanArgs a = {};
  FC_TRY(plan_args(dev, c, requests, n, lens_out, n_free_out, status, &a));
  if ((n && !grow) || !starts) return fc_fail(dev, FC_ERR_ARG, "fc_paged_extend_dev: grow or starts is NULL");
  if (rows > (uint32_t)INT_MAX) return fc_fail(dev, FC_ERR_SHAPE, "%u rows in a step", rows);
  a.grow = grow, a.rows = rows, a.starts = starts, a.slot = slot, a.position = position, a.request = request;
  return launch_plan(dev, "paged_extend", extend_kernel, a, rows > n ? rows : n);
}

FC_API int fc_paged_release_dev(FcDevice* dev, const FcPagedCache* c, const int32_t* requests, uint32_t n, int32_t* lens_out,
                                int32_t* n_free_out, int32_t* status) {
  if (!dev) return FC_ERR_ARG;
  cudaSetDevice(dev->ordinal);
  PlanArgs a = {};
  FC_TRY(plan_args(dev, c, requests, n, lens_out, n_free_out, status, &a));
  return launch_plan(dev, "paged_release", release_kernel, a, n * 32);
}

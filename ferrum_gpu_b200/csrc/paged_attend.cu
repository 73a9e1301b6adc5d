// Attention of new tokens over a paged key-value cache: out = sum_j p_j v_j with p the softmax of scale * q . k_j over the
// positions j a row may see, found through its request's page table.
//
// One pass with the softmax's running maximum and sum: where a later score raises the maximum from m to m', the sum and
// the weighted values so far are multiplied by 2^(m - m') (scores are held times log2 e).
//
// What bounds it is the cache's bytes, so everything is laid out for reading them once, in 16-byte pieces, straight into the
// registers that the matrix instructions take - no tile in shared memory, no copy between lanes:
//  * mma.sync with the heads of a kv head as the 16 rows: 8 heads, each as two terms (row g the high one, row g + 8 the
//    low one; q = high + low to 22 bits for f16 and tf32, 16 for bf16, where f32 rows bring a third term in a second
//    instruction). The two partial results of a head end up in one thread and are added there.
//  * scores: positions are the 8 columns, channels the depth. The order of channels along the depth is free as long as q has
//    the same, so a lane takes the 16 consecutive bytes of its row that it can load at once.
//  * p v: positions are the depth - the scores' own layout is the layout of the first operand, no shuffle between the two
//    products - and channels the columns, again in the order that 16-byte pieces of a position's row give.
//  * an f32 cache goes as two tf32 terms (11 + 11 bits) made in registers.
// p is at most 2^P_LIFT instead of 1 so that its low f16 term keeps its bits far below the maximum.
//
// Work: tiles of 64 positions of (row, kv head, 8 heads), all of a step in one line, cut evenly over the CTAs that are
// resident at once: a row alone is spread over the GPU, rows of unequal length cost what they hold. A CTA's four warps take
// 16 positions in turn and join through shared memory; a (row, kv head) that several CTAs share is joined by the one
// that arrives last, from f32 partial results in the order of the positions - the same bits every time.
#include <cmath>
#include <type_traits>

#include "paged.cuh"

namespace {

constexpr int WARPS = 4, TILE = 64, ROWS8 = 8; // warps of a CTA, positions of a tile, heads of one matrix operand
constexpr float P_LIFT = 10.0f;

struct AttendArgs {
  const void *q, *k, *v;
  void* out;
  const int32_t *request, *position, *table;
  uint64_t q_stride, out_stride;
  uint32_t rows, heads, kv_heads, group, blocks, hd, requests, max_pages, n_pages, page_shift; // blocks: of 8 heads, per kv head
  int act;
  float scale; // times log2 e
  float* parts;
  uint32_t* arrived;
};
// a part: 8 maxima, 8 sums, 8 rows of weighted values
constexpr uint32_t part_floats(uint32_t hdp) { return 2 * ROWS8 + ROWS8 * hdp; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename C>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<float>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x as tf32 terms: the upper 11 bits (to nearest), then the upper 11 of what is left
__device__ __forceinline__ uint32_t tf32_high(uint32_t x) { return (x + 0x1000u) & 0xffffe000u; }
__device__ __forceinline__ uint32_t tf32_low(uint32_t x, uint32_t high) {
  return __float_as_uint(__uint_as_float(x) - __uint_as_float(high)) & 0xffffe000u;
}
// two values as one register of 16-bit terms, and what the terms leave of them
template <typename C>
__device__ __forceinline__ uint32_t take_term(float& x, float& y);
template <>
__device__ __forceinline__ uint32_t take_term<__half>(float& x, float& y) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  x -= f.x, y -= f.y;
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t take_term<__nv_bfloat16>(float& x, float& y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const float2 f = __bfloat1622float2(h);
  x -= f.x, y -= f.y;
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 load16(const char* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
__device__ __forceinline__ float load_act(const void* p, int act, size_t i) {
  return act == FC_F32 ? static_cast<const float*>(p)[i] : act == FC_F16 ? to_f32(static_cast<const __half*>(p)[i]) : to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_act(void* p, int act, size_t i, float v) {
  if (act == FC_F32) static_cast<float*>(p)[i] = v;
  else if (act == FC_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// positions a row sees, and the row of the table they are found in
__device__ __forceinline__ uint32_t row_len(const AttendArgs& a, uint32_t r, uint32_t& req) {
  const int32_t q = a.request ? a.request[r] : (int32_t)r, p = a.position[r];
  const bool ok = (uint32_t)q < a.requests && p >= 0;
  req = ok ? (uint32_t)q : 0u;
  const uint64_t cap = (uint64_t)a.max_pages << a.page_shift;
  return ok ? (uint32_t)min((uint64_t)p + 1, cap) : 0u;
}
__device__ __forceinline__ uint32_t row_tiles(uint32_t len) { return max(1u, (len + TILE - 1) / TILE); }

// HDP: channels rounded up to what the registers are laid out for; FULL: head_dim is HDP; TERMS: of q and p (bf16: 2 or 3)
template <typename C, int HDP, bool FULL, int TERMS>
__global__ void __launch_bounds__(WARPS * 32, HDP == 64 ? 3 : 2) attend_kernel(AttendArgs a) {
  constexpr bool F32 = sizeof(C) == 4;
  constexpr int E = 16 / sizeof(C);             // elements of a 16-byte piece
  constexpr int NJ = HDP / (4 * E);             // pieces of a k row per lane (4 lanes share a row)
  constexpr int NI = HDP / (8 * E);             // pieces of a v row per lane (8 lanes share a row)
  constexpr int PS = F32 && HDP > 64 ? 8 : 16;  // positions of a warp's step
  constexpr int NT = PS / 8;
  constexpr bool SIZED = std::is_same<C, __half>::value; // its terms have a range to keep to
  constexpr bool AHEAD = HDP <= 128;            // the next step's k is requested before this one's softmax
  __shared__ union { // q while positions are multiplied, then the warps' results
    uint4 q[NJ][TERMS][32];
    float o[WARPS][ROWS8][HDP];
  } sm;
  auto& sm_q = sm.q;
  auto& sm_o = sm.o;
  __shared__ float sm_m[WARPS][ROWS8], sm_l[WARPS][ROWS8];
  __shared__ uint32_t sm_big[ROWS8];
  __shared__ uint32_t sm_scan[WARPS], sm_row, sm_at, sm_last;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t per_row = a.kv_heads * a.blocks;
  grid_wait();

  // Where this CTA's share of the tiles begins: prefix sums over the rows' tiles, a run of rows per thread.
  const uint32_t run = (a.rows + WARPS * 32 - 1) / (WARPS * 32), r0 = min(a.rows, tid * run), r1 = min(a.rows, r0 + run);
  uint32_t mine = 0, req;
  for (uint32_t r = r0; r < r1; r++) mine += row_tiles(row_len(a, r, req));
  uint32_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) sm_scan[warp] = upto;
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (int w = 0; w < WARPS; w++) {
    if (w < (int)warp) upto += sm_scan[w];
    all += sm_scan[w];
  }
  all *= per_row, upto *= per_row, mine *= per_row;
  const uint32_t n_cta = min(gridDim.x, all), share = all / n_cta, extra = all % n_cta; // (the first `extra` CTAs take one more)
  if (blockIdx.x >= n_cta) return;
  auto begin_of = [&](uint32_t c) { return c * share + min(c, extra); };
  auto owner_of = [&](uint32_t tile) {
    const uint32_t longer = extra * (share + 1);
    return tile < longer ? tile / (share + 1) : extra + (tile - longer) / share;
  };
  const uint32_t begin = begin_of(blockIdx.x), end = begin_of(blockIdx.x + 1);
  if (upto - mine <= begin && begin < upto) {
    uint32_t at = upto - mine, r = r0;
    for (;; r++) {
      const uint32_t n = row_tiles(row_len(a, r, req)) * per_row;
      if (begin < at + n) break;
      at += n;
    }
    sm_row = r, sm_at = at;
  }
  __syncthreads();
  uint32_t r = sm_row, len = row_len(a, r, req), tiles = row_tiles(len);
  uint32_t row_at = sm_at; // the row's first tile
  uint32_t which = (begin - row_at) / tiles, tile = (begin - row_at) % tiles;

  const size_t row_bytes = (size_t)a.hd * sizeof(C);
  for (uint32_t at = begin; at < end;) {
    const uint32_t tile_end = min(tiles, tile + (end - at));
    const uint32_t kvh = which / a.blocks, h0 = kvh * a.group + (which % a.blocks) * ROWS8;
    const uint32_t heads = min((uint32_t)ROWS8, (kvh + 1) * a.group - h0);
    // q's terms as the matrix operand wants them: lane (g, t) of piece j has channels (4 j + t) E .. of head h0 + g
    if (SIZED) { // (the f16 terms of a head: of q divided by a power of two near its largest)
      if (tid < ROWS8) sm_big[tid] = 0;
      __syncthreads();
    }
    float mul = a.scale;
    constexpr int ITEMS = (NJ * 32 + WARPS * 32 - 1) / (WARPS * 32);
    float qv[ITEMS][E];
#pragma unroll
    for (int it = 0; it < ITEMS; it++) {
      const uint32_t id = tid + it * WARPS * 32, j = id / 32;
      if (NJ * 32 % (WARPS * 32) && id >= NJ * 32) continue;
      float big = 0.0f;
#pragma unroll
      for (int e = 0; e < E; e++) {
        const uint32_t ch = (4 * j + t) * E + e;
        qv[it][e] = g < heads && (FULL || ch < a.hd) ? load_act(a.q, a.act, (size_t)r * a.q_stride + (size_t)(h0 + g) * a.hd + ch) : 0.0f;
        big = fmaxf(big, fabsf(qv[it][e]));
      }
      if (SIZED) atomicMax(&sm_big[g], __float_as_uint(big));
    }
    float down = 1.0f;
    if (SIZED) {
      __syncthreads();
      const int ex = min(max((int)(sm_big[g] >> 23), 27), 253) - 127; // (a power of two that has an inverse, whatever the largest is)
      down = __uint_as_float((uint32_t)(127 - ex) << 23), mul *= __uint_as_float((uint32_t)(127 + ex) << 23);
    }
#pragma unroll
    for (int it = 0; it < ITEMS; it++) {
      const uint32_t id = tid + it * WARPS * 32, j = id / 32;
      if (NJ * 32 % (WARPS * 32) && id >= NJ * 32) continue;
      uint32_t w[TERMS][4];
      if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < E; e++) {
          const uint32_t x = __float_as_uint(qv[it][e]);
          w[0][e] = tf32_high(x), w[1][e] = tf32_low(x, w[0][e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          float x = qv[it][e] * down, y = qv[it][e + 1] * down;
#pragma unroll
          for (int m = 0; m < TERMS; m++) w[m][e / 2] = take_term<C>(x, y);
        }
      }
#pragma unroll
      for (int m = 0; m < TERMS; m++) sm_q[j][m][lane] = make_uint4(w[m][0], w[m][1], w[m][2], w[m][3]);
    }
    __syncthreads();

    float o[NI][E][4], top = -INFINITY, sum = 0.0f; // of head g: the maximum is the lane's four's, the sum its own positions'
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
      for (int e = 0; e < E; e++)
#pragma unroll
        for (int c = 0; c < 4; c++) o[i][e][c] = 0.0f;

    const uint32_t p_end = min(len, tile_end * TILE), mask = (1u << a.page_shift) - 1;
    const int32_t* table = a.table + (size_t)req * a.max_pages;
    const uint64_t page_rows = (uint64_t)a.kv_heads << a.page_shift, head_row = (uint64_t)kvh << a.page_shift;
    // the page of position p + lane (mod the step's), none past the end
    auto look = [&](uint32_t p) {
      const uint32_t pos = p + (lane & (PS - 1));
      const uint32_t page = pos < p_end ? (uint32_t)table[pos >> a.page_shift] : 0xffffffffu;
      return page < a.n_pages ? page : 0xffffffffu;
    };
    auto row_of = [&](uint32_t page, uint32_t pos) { // (a page that is none: the pool's first, to be masked)
      return ((page == 0xffffffffu ? 0 : page) * page_rows + head_row + (pos & mask)) * row_bytes;
    };
    uint4 kk[NT][NJ];
    auto load_k = [&](uint32_t p, uint32_t pages) {
#pragma unroll
      for (int n = 0; n < NT; n++) {
        const uint32_t i = n * 8 + g;
        const char* src = static_cast<const char*>(a.k) + row_of(__shfl_sync(0xffffffffu, pages, i), p + i) + t * 16;
#pragma unroll
        for (int j = 0; j < NJ; j++) kk[n][j] = FULL || (4 * j + t) * E < a.hd ? load16(src + j * 64) : make_uint4(0, 0, 0, 0);
      }
    };
    uint32_t p = tile * TILE + warp * PS;
    uint32_t pages = look(p), pages_next = look(p + WARPS * PS);
    if (AHEAD && p < p_end) load_k(p, pages);
    for (; p < p_end; p += WARPS * PS) {
      if (!AHEAD) load_k(p, pages);
      uint4 vv[NT][2][NI];
      bool ok[NT][2];
      bool clean = true;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const uint32_t i = n * 8 + 2 * t + x, page = __shfl_sync(0xffffffffu, pages, i);
          ok[n][x] = page != 0xffffffffu;
          clean = clean && ok[n][x];
          const char* src = static_cast<const char*>(a.v) + row_of(page, p + i) + g * 16;
#pragma unroll
          for (int c = 0; c < NI; c++) vv[n][x][c] = FULL || (8 * c + g) * E < a.hd ? load16(src + c * 128) : make_uint4(0, 0, 0, 0);
        }
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int c = 0; c < 4; c++) s[n][c] = 0.0f;
#pragma unroll
      for (int j = 0; j < NJ; j++) {
        const uint4 hi = sm_q[j][0][lane], lo = sm_q[j][1][lane];
        const uint32_t a0[4] = {hi.x, lo.x, hi.y, lo.y}, a1[4] = {hi.z, lo.z, hi.w, lo.w};
        if constexpr (F32) {
#pragma unroll
          for (int n = 0; n < NT; n++) {
            const uint32_t k0 = tf32_high(kk[n][j].x), k1 = tf32_high(kk[n][j].y), k2 = tf32_high(kk[n][j].z), k3 = tf32_high(kk[n][j].w);
            mma<C>(s[n], a0, k0, k1);
            mma<C>(s[n], a1, k2, k3);
            mma<C>(s[n], a0, tf32_low(kk[n][j].x, k0), tf32_low(kk[n][j].y, k1));
            mma<C>(s[n], a1, tf32_low(kk[n][j].z, k2), tf32_low(kk[n][j].w, k3));
          }
        } else {
#pragma unroll
          for (int n = 0; n < NT; n++) {
            mma<C>(s[n], a0, kk[n][j].x, kk[n][j].y);
            mma<C>(s[n], a1, kk[n][j].z, kk[n][j].w);
          }
          if constexpr (TERMS == 3) {
            const uint4 ll = sm_q[j][TERMS - 1][lane];
            const uint32_t b0[4] = {ll.x, 0, ll.y, 0}, b1[4] = {ll.z, 0, ll.w, 0};
#pragma unroll
            for (int n = 0; n < NT; n++) {
              mma<C>(s[n], b0, kk[n][j].x, kk[n][j].y);
              mma<C>(s[n], b1, kk[n][j].z, kk[n][j].w);
            }
          }
        }
      }
      pages = pages_next, pages_next = look(p + 2 * WARPS * PS);
      if (AHEAD && p + WARPS * PS < p_end) load_k(p + WARPS * PS, pages);
      clean = __all_sync(0xffffffffu, clean);
      float best = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const float v = (s[n][x] + s[n][x + 2]) * mul;
          s[n][x] = clean || ok[n][x] ? v : -INFINITY;
          best = fmaxf(best, s[n][x]);
        }
      best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
      best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
      if (__any_sync(0xffffffffu, best > top)) {
        const float higher = fmaxf(top, best), keep = higher == -INFINITY ? 1.0f : ex2(top - higher);
        top = higher, sum *= keep;
#pragma unroll
        for (int i = 0; i < NI; i++)
#pragma unroll
          for (int e = 0; e < E; e++)
#pragma unroll
            for (int c = 0; c < 4; c++) o[i][e][c] *= keep; // (rows g and g + 8 are one head)
      }
      const float base = top == -INFINITY ? 0.0f : top - P_LIFT;
      float pr[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int x = 0; x < 2; x++) pr[n][x] = ex2(s[n][x] - base), sum += pr[n][x];
      if (!clean) { // what no position holds may be NaN, and 0 * NaN is not 0
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int x = 0; x < 2; x++)
            if (!ok[n][x])
#pragma unroll
              for (int c = 0; c < NI; c++) vv[n][x][c] = make_uint4(0, 0, 0, 0);
      }
      if constexpr (F32) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const uint32_t x = __float_as_uint(pr[n][0]), y = __float_as_uint(pr[n][1]), xh = tf32_high(x), yh = tf32_high(y);
          const uint32_t pa[4] = {xh, tf32_low(x, xh), yh, tf32_low(y, yh)};
#pragma unroll
          for (int c = 0; c < NI; c++) {
            const uint32_t u[4] = {vv[n][0][c].x, vv[n][0][c].y, vv[n][0][c].z, vv[n][0][c].w};
            const uint32_t w[4] = {vv[n][1][c].x, vv[n][1][c].y, vv[n][1][c].z, vv[n][1][c].w};
#pragma unroll
            for (int e = 0; e < E; e++) {
              const uint32_t uh = tf32_high(u[e]), wh = tf32_high(w[e]);
              mma<C>(o[c][e], pa, uh, wh);
              mma<C>(o[c][e], pa, tf32_low(u[e], uh), tf32_low(w[e], wh));
            }
          }
        }
      } else {
        uint32_t pa[4], pb[4];
        pa[0] = take_term<C>(pr[0][0], pr[0][1]), pa[1] = take_term<C>(pr[0][0], pr[0][1]);
        pa[2] = take_term<C>(pr[1][0], pr[1][1]), pa[3] = take_term<C>(pr[1][0], pr[1][1]);
        if (TERMS == 3) pb[0] = take_term<C>(pr[0][0], pr[0][1]), pb[2] = take_term<C>(pr[1][0], pr[1][1]), pb[1] = pb[3] = 0;
#pragma unroll
        for (int c = 0; c < NI; c++) {
          const uint32_t u[4][4] = {{vv[0][0][c].x, vv[0][0][c].y, vv[0][0][c].z, vv[0][0][c].w}, {vv[0][1][c].x, vv[0][1][c].y, vv[0][1][c].z, vv[0][1][c].w},
                                    {vv[1][0][c].x, vv[1][0][c].y, vv[1][0][c].z, vv[1][0][c].w}, {vv[1][1][c].x, vv[1][1][c].y, vv[1][1][c].z, vv[1][1][c].w}};
#pragma unroll
          for (int e = 0; e < E; e++) {
            const uint32_t pick = e & 1 ? 0x7632u : 0x5410u;
            const uint32_t b0 = __byte_perm(u[0][e / 2], u[1][e / 2], pick), b1 = __byte_perm(u[2][e / 2], u[3][e / 2], pick);
            mma<C>(o[c][e], pa, b0, b1);
            if constexpr (TERMS == 3) mma<C>(o[c][e], pb, b0, b1);
          }
        }
      }
    }

    // join the four warps
    __syncthreads(); // (all have read q)
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (t == 0) sm_m[warp][g] = top, sm_l[warp][g] = sum;
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
      for (int e = 0; e < E; e++)
#pragma unroll
        for (int x = 0; x < 2; x++) sm_o[warp][g][(8 * i + 2 * t + x) * E + e] = o[i][e][x] + o[i][e][x + 2];
    __syncthreads();
    const bool whole = tile == 0 && tile_end == tiles;
    const uint32_t first_tile = row_at + which * tiles;
    const uint32_t c0 = whole ? 0 : owner_of(first_tile), c1 = whole ? 0 : owner_of(first_tile + tiles - 1);
    auto part_of = [&](uint32_t c) { // a CTA has two: one for where it begins, one for where it ends
      return a.parts + (size_t)(2 * c + (begin_of(c) >= first_tile ? 0 : 1)) * part_floats(HDP);
    };
    float* part = whole ? nullptr : part_of(blockIdx.x);
    for (uint32_t i = tid; i < heads * a.hd; i += WARPS * 32) {
      const uint32_t h = i / a.hd, ch = i - h * a.hd;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; w++) m = fmaxf(m, sm_m[w][h]);
      const float base = m == -INFINITY ? 0.0f : m;
      float l = 0.0f, v = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; w++) {
        const float f = ex2(sm_m[w][h] - base);
        l = fmaf(sm_l[w][h], f, l), v = fmaf(sm_o[w][h][ch], f, v);
      }
      if (whole) {
        store_act(a.out, a.act, (size_t)r * a.out_stride + (size_t)(h0 + h) * a.hd + ch, l == 0.0f ? 0.0f : v / l);
      } else {
        if (ch == 0) part[h] = m, part[ROWS8 + h] = l;
        part[2 * ROWS8 + h * HDP + ch] = v;
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) sm_last = atomicAdd(&a.arrived[c0], 1u) == c1 - c0;
      __syncthreads();
      if (sm_last) {
        __threadfence();
        // Each warp finds two heads' maxima over the parts; then, JOIN parts at a time, their weights go to shared memory and
        // every thread adds its channels' values, all loads of a turn in flight together.
        float (*sm_w)[ROWS8] = reinterpret_cast<float (*)[ROWS8]>(&sm);
        constexpr int JOIN = 32, OWN = (ROWS8 * HDP / 4 + WARPS * 32 - 1) / (WARPS * 32);
        {
          const uint32_t h = warp * 2 + (lane >> 4);
          float m = -INFINITY;
          for (uint32_t c = c0 + (lane & 15); c <= c1; c += 16) m = fmaxf(m, __ldcg(part_of(c) + h));
#pragma unroll
          for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          sm_m[0][h] = m == -INFINITY ? 0.0f : m; // (all lanes of a head write the same)
        }
        __syncthreads();
        float4 v[OWN];
        float l[OWN];
#pragma unroll
        for (int n = 0; n < OWN; n++) v[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f), l[n] = 0.0f;
        for (uint32_t c = c0; c <= c1; c += JOIN) {
          const uint32_t here = min((uint32_t)JOIN, c1 - c + 1);
          for (uint32_t i = tid; i < here * ROWS8; i += WARPS * 32) {
            const uint32_t h = i % ROWS8;
            const float* q = part_of(c + i / ROWS8);
            const float f = ex2(__ldcg(q + h) - sm_m[0][h]);
            sm_w[i / ROWS8][h] = f, sm_w[JOIN + i / ROWS8][h] = f * __ldcg(q + ROWS8 + h);
          }
          __syncthreads();
#pragma unroll
          for (int n = 0; n < OWN; n++) {
            const uint32_t i = tid + n * WARPS * 32, h = i / (HDP / 4), ch = i % (HDP / 4) * 4;
            if (h >= heads || (!FULL && ch >= a.hd)) continue;
            const float* q = a.parts + 2 * ROWS8 + h * HDP + ch;
#pragma unroll 8
            for (uint32_t k = 0; k < here; k++) {
              const float4 x = __ldcg(reinterpret_cast<const float4*>(q + (part_of(c + k) - a.parts)));
              const float f = sm_w[k][h];
              v[n].x = fmaf(x.x, f, v[n].x), v[n].y = fmaf(x.y, f, v[n].y), v[n].z = fmaf(x.z, f, v[n].z), v[n].w = fmaf(x.w, f, v[n].w);
              l[n] += sm_w[JOIN + k][h];
            }
          }
          __syncthreads();
        }
#pragma unroll
        for (int n = 0; n < OWN; n++) {
          const uint32_t i = tid + n * WARPS * 32, h = i / (HDP / 4), ch = i % (HDP / 4) * 4;
          if (h >= heads || (!FULL && ch >= a.hd)) continue;
          const float f = l[n] == 0.0f ? 0.0f : 1.0f / l[n];
          const float x[4] = {v[n].x * f, v[n].y * f, v[n].z * f, v[n].w * f};
#pragma unroll
          for (int e = 0; e < 4; e++) store_act(a.out, a.act, (size_t)r * a.out_stride + (size_t)(h0 + h) * a.hd + ch + e, x[e]);
        }
        if (tid == 0) a.arrived[c0] = 0; // for the next call
      }
    }
    __syncthreads(); // shared memory is free again
    at += tile_end - tile;
    tile = 0;
    if (tile_end == tiles && ++which == per_row) {
      row_at += tiles * per_row;
      which = 0;
      if (++r < a.rows) len = row_len(a, r, req), tiles = row_tiles(len);
    }
  }
}

constexpr uint32_t MAX_CTAS_PER_SM = 4;

template <typename C, int HDP, bool FULL, int TERMS>
int launch_attend(FcDevice* dev, AttendArgs a) {
  auto kern = attend_kernel<C, HDP, FULL, TERMS>;
  static int resident[64]; // CTAs of an SM, by device
  int& fit = resident[dev->ordinal & 63];
  if (!fit) {
    FC_CUDA(dev, cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kern, WARPS * 32, 0));
    if (fit < 1 || fit > (int)MAX_CTAS_PER_SM) fit = fit < 1 ? 1 : MAX_CTAS_PER_SM;
  }
  const uint64_t most = (uint64_t)a.rows * a.kv_heads * a.blocks * (((((uint64_t)a.max_pages << a.page_shift) + TILE - 1) / TILE));
  const uint64_t ctas = (uint64_t)dev->prop.multiProcessorCount * fit;
  FC_LAUNCH(dev, "paged_attend", launch_on(dev, true, kern, dim3((unsigned)(most < ctas ? most : ctas)), dim3(WARPS * 32), 0, a));
  return FC_OK;
}
template <typename C, int TERMS>
int launch_attend(FcDevice* dev, const AttendArgs& a) {
  return a.hd == 64    ? launch_attend<C, 64, true, TERMS>(dev, a)
         : a.hd < 64   ? launch_attend<C, 64, false, TERMS>(dev, a)
         : a.hd == 128 ? launch_attend<C, 128, true, TERMS>(dev, a)
         : a.hd < 128  ? launch_attend<C, 128, false, TERMS>(dev, a)
         : a.hd == 256 ? launch_attend<C, 256, true, TERMS>(dev, a)
                       : launch_attend<C, 256, false, TERMS>(dev, a);
}

// Partial results and arrival counters, for the handle's life: two parts per CTA that can be resident. The counters start at
// zero and every call leaves them there.
int attend_scratch(FcDevice* dev, AttendArgs* a) {
  const size_t ctas = (size_t)dev->prop.multiProcessorCount * MAX_CTAS_PER_SM, words = (ctas * 4 + 255) / 256 * 256;
  if (!dev->attend.p) {
    const size_t bytes = words + ctas * 2 * part_floats(PAGED_MAX_HEAD_DIM) * 4;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed; // (an allocation of its own, no stream operation: fine under a capture)
    cudaThreadExchangeStreamCaptureMode(&mode);
    void* p = nullptr;
    const cudaError_t e = stream_capturing(dev) ? cudaMalloc(&p, bytes) : device_malloc(dev, &p, bytes);
    cudaThreadExchangeStreamCaptureMode(&mode);
    FC_CUDA(dev, e);
    dev->attend = Workspace{p, bytes};
    dev->attend_clear = false;
  }
  if (!dev->attend_clear) { // (captured: a node of the graph, and the handle's own calls still have to do it once)
    FC_CUDA(dev, cudaMemsetAsync(dev->attend.p, 0, words, dev->stream));
    dev->attend_clear = !stream_capturing(dev);
  }
  a->arrived = static_cast<uint32_t*>(dev->attend.p);
  a->parts = reinterpret_cast<float*>(static_cast<char*>(dev->attend.p) + words);
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
  const uint64_t row_most = ((uint64_t)c->max_pages * c->page + TILE - 1) / TILE;
  if ((uint64_t)rows * heads * row_most > 0xffffffffull) // (tiles are counted in 32 bits)
    return fc_fail(dev, FC_ERR_UNSUPPORTED, "%u rows of %u heads over page tables of %u x %u positions: more than one call holds", rows, heads,
                   c->max_pages, c->page);
  AttendArgs a = {};
  a.q = q, a.k = c->k, a.v = c->v, a.out = out, a.request = request, a.position = position, a.table = c->table;
  a.q_stride = q_stride, a.out_stride = out_stride, a.heads = heads, a.kv_heads = c->kv_heads, a.hd = c->head_dim;
  a.requests = c->requests, a.max_pages = c->max_pages, a.n_pages = c->n_pages, a.page_shift = (uint32_t)__builtin_ctz(c->page);
  a.rows = rows, a.group = heads / c->kv_heads, a.blocks = (a.group + ROWS8 - 1) / ROWS8, a.act = kind;
  a.scale = (scale == 0.0f ? 1.0f / sqrtf((float)c->head_dim) : scale) * 1.44269504088896340736f;
  FC_TRY(attend_scratch(dev, &a));
  if (c->kind == FC_F32) return launch_attend<float, 2>(dev, a);
  if (c->kind == FC_F16) return launch_attend<__half, 2>(dev, a);
  // bf16 terms have 8 bits: two hold a 16-bit row, f32 rows take three
  return kind == FC_F32 ? launch_attend<__nv_bfloat16, 3>(dev, a) : launch_attend<__nv_bfloat16, 2>(dev, a);
}

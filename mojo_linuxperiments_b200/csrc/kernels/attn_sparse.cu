// Attention of single rows of queries over the pages of their sequences that look most promising: scores of all pages, selection and attention in one launch.
//
// A page's score for a KV head bounds what any of its query heads can get from any key of the page: with lo <= k <= hi per dimension,
//   q . k <= sum_d max(q_d lo_d, q_d hi_d) = q+ . hi + q- . lo,      q+ = max(q, 0), q- = min(q, 0),
// and the score is the largest of the group's heads.  The first pages, and the last up to the row's own position, are read always; the others compete.
//
// Grid (split, KV head x group of up to 16 query heads, row); the splits of a row are a thread-block cluster.  Each scores its share of the pages into
// shared memory, the cluster selects (page_select.cuh), each reads its share of the selected pages, and the parts are joined through distributed
// shared memory.  Bound by the bytes of the bounds, 2 dk per page, and of the pages taken.
//
#include "ptx.cuh"
#include "api.h"
#include "launch.cuh"
#include "decode_warp.cuh"
#include "page_select.cuh"
#include "attn_sparse.cuh"

namespace b200 {

__device__ __forceinline__ float as_f(float v) { return v; }
__device__ __forceinline__ float as_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_max(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// ---- any head size up to 512, bf16 or fp32: a warp per page, lanes along the dimensions ------------------------------------------------
constexpr int AS_MAX_D = 512, AS_PER_LANE = AS_MAX_D / 32;

template <typename T>
__global__ void __launch_bounds__(PS_THREADS) attn_sparse_any_kernel(const __grid_constant__ SparseParams p) {
  extern __shared__ __align__(16) uint8_t as_smem[];
  __shared__ PageSelectShared sel;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x, S = p.splits, tok = blockIdx.z;
  const int kvh = blockIdx.y / p.hgroups, hg = blockIdx.y - kvh * p.hgroups;
  const int group = p.hq / p.c.kv_heads, g0 = hg * 16, G = min(16, group - g0), h0 = kvh * group + g0;
  const int dk = p.c.dk, dv = p.c.dv, ps = p.c.page_size;
  SparseRow row;
  if (!row.find(p, tok)) {                       // the same for all CTAs of the cluster
    if (rank == 0) {
      T* o = static_cast<T*>(p.out) + static_cast<size_t>(tok) * p.ldo + static_cast<size_t>(h0) * dv;
      for (int i = tid; i < G * dv; i += PS_THREADS) o[i] = T(0.f);
      if (p.chosen && hg == 0)
        for (int i = tid; i < p.top; i += PS_THREADS) p.chosen[(static_cast<size_t>(tok) * p.c.kv_heads + kvh) * p.top + i] = -1;
    }
    return;
  }
  const T* q = static_cast<const T*>(p.q) + static_cast<size_t>(tok) * p.ldq;
  const int* pt = p.c.page_table + static_cast<size_t>(row.seq) * p.c.max_pages;
  // shared memory: scores, list, [8 warps][dv + 2], [16 heads][dv + 2]
  unsigned* keys = reinterpret_cast<unsigned*>(as_smem);
  int* list = reinterpret_cast<int*>(keys + p.score_cap);
  float* part = reinterpret_cast<float*>(list + p.list_cap);
  const int pitch = dv + 2;
  float* joined = part + PS_WARPS * pitch;

  const int share = row.lists(p, rank, list, S);          // without a selection the list is known
  if (row.selects) {
    const int i0 = ps_share(row.candidates, rank, S), i1 = ps_share(row.candidates, rank + 1, S);
    for (int i = i0 + warp; i < i1; i += PS_WARPS) {
      const int page = pt[row.place0 + i];
      float s = -INFINITY;
      if (page >= 0 && page < p.c.num_pages) {
        const T* lo = static_cast<const T*>(p.bounds) + (static_cast<size_t>(page) * p.c.kv_heads + kvh) * 2 * dk;
        float a[AS_PER_LANE], b[AS_PER_LANE];
#pragma unroll
        for (int j = 0; j < AS_PER_LANE; ++j) {
          const int d = lane + 32 * j;
          a[j] = d < dk ? as_f(lo[d]) : 0.f;
          b[j] = d < dk ? as_f(lo[dk + d]) : 0.f;
        }
        for (int h = 0; h < group; ++h) {
          float t = 0.f;
#pragma unroll
          for (int j = 0; j < AS_PER_LANE; ++j) {
            const int d = lane + 32 * j;
            if (d < dk) {
              const float x = as_f(q[static_cast<size_t>(kvh * group + h) * dk + d]);
              t = fmaf(fmaxf(x, 0.f), b[j], fmaf(fminf(x, 0.f), a[j], t));
            }
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
          s = as_max(s, t);
        }
      }
      if (lane == 0) keys[i - i0] = ps_order(s);
    }
    __syncthreads();
    select_pages(sel, keys, i1 - i0, i0, row.take, row.first, row.entries, row.place0, list, rank, S);
  }
  if (S > 1) cluster_sync_all(); else __syncthreads();
  if (p.chosen && hg == 0) row.tell(p, tok, kvh, rank, share, list, S);

  // a head at a time, a page per warp: 32 keys or the page's, then the values with the lanes along their dimensions
  const size_t rec = static_cast<size_t>(p.c.kv_heads) * ps * (dk + dv);
  for (int g = 0; g < G; ++g) {
    const T* qh = q + static_cast<size_t>(h0 + g) * dk;
    float m = -INFINITY, l = 0.f, acc[AS_PER_LANE];
#pragma unroll
    for (int j = 0; j < AS_PER_LANE; ++j) acc[j] = 0.f;
    for (int i = warp; i < share; i += PS_WARPS) {
      const int place = list[i], page = pt[place];
      if (page < 0 || page >= p.c.num_pages) continue;
      const T* kp = static_cast<const T*>(p.c.data) + static_cast<size_t>(page) * rec + static_cast<size_t>(kvh) * ps * dk;
      const T* vp = static_cast<const T*>(p.c.data) + static_cast<size_t>(page) * rec + static_cast<size_t>(p.c.kv_heads) * ps * dk + static_cast<size_t>(kvh) * ps * dv;
      const int r0 = max(0, row.low - place * ps), r1 = min(ps, row.pos + 1 - place * ps);
      for (int k0 = r0; k0 < r1; k0 += 32) {
        const int n = min(32, r1 - k0);
        float s = -INFINITY;
        for (int r = 0; r < n; ++r) {
          float t = 0.f;
          for (int d = lane; d < dk; d += 32) t = fmaf(as_f(qh[d]), as_f(kp[static_cast<size_t>(k0 + r) * dk + d]), t);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
          if (lane == r) s = t * p.s.scale;
        }
        float mx = s;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mn = fmaxf(m, mx);
        if (mn == -INFINITY) continue;
        const float a = m == -INFINITY ? 0.f : expf(m - mn), e = s == -INFINITY ? 0.f : expf(s - mn);
        float sum = e;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l = l * a + sum;
        m = mn;
#pragma unroll
        for (int j = 0; j < AS_PER_LANE; ++j) acc[j] *= a;
        for (int r = 0; r < n; ++r) {
          const float w = __shfl_sync(0xffffffffu, e, r);
#pragma unroll
          for (int j = 0; j < AS_PER_LANE; ++j)
            if (lane + 32 * j < dv) acc[j] = fmaf(w, as_f(vp[static_cast<size_t>(k0 + r) * dv + lane + 32 * j]), acc[j]);
        }
      }
    }
    float* mine = part + warp * pitch;
    if (lane == 0) { mine[dv] = m; mine[dv + 1] = l; }
#pragma unroll
    for (int j = 0; j < AS_PER_LANE; ++j)
      if (lane + 32 * j < dv) mine[lane + 32 * j] = acc[j];
    __syncthreads();
    float* to = joined + g * pitch;
    float top = -INFINITY, total = 0.f;
    for (int w = 0; w < PS_WARPS; ++w) top = fmaxf(top, part[w * pitch + dv]);
    for (int d = tid; d < dv; d += PS_THREADS) {
      float v = 0.f;
      for (int w = 0; w < PS_WARPS; ++w) {
        const float mw = part[w * pitch + dv];
        if (mw != -INFINITY) v = fmaf(expf(mw - top), part[w * pitch + d], v);
      }
      to[d] = v;
    }
    if (tid == 0) {
      for (int w = 0; w < PS_WARPS; ++w) {
        const float mw = part[w * pitch + dv];
        if (mw != -INFINITY) total = fmaf(expf(mw - top), part[w * pitch + dv + 1], total);
      }
      to[dv] = top;
      to[dv + 1] = total;
    }
    __syncthreads();
  }
  if (S > 1) cluster_sync_all();
  const uint32_t j_addr = smem_u32(joined);
  T* o = static_cast<T*>(p.out) + static_cast<size_t>(tok) * p.ldo + static_cast<size_t>(h0) * dv;
  for (int i = rank * PS_THREADS + tid; i < G * dv; i += S * PS_THREADS) {
    const int g = i / dv, d = i - g * dv;
    float m = p.s.sink ? p.s.sink[h0 + g] : -INFINITY, l = p.s.sink ? 1.f : 0.f, v = 0.f;
    for (int r = 0; r < S; ++r) {
      const uint32_t base = (S > 1 ? mapa_shared(j_addr, r) : j_addr) + 4u * (g * pitch);
      const float mr = __uint_as_float(ps_ld_cluster(base + 4u * dv));
      if (mr == -INFINITY) continue;
      const float mn = fmaxf(m, mr), fo = m == -INFINITY ? 0.f : expf(m - mn), fn = expf(mr - mn);
      l = l * fo + fn * __uint_as_float(ps_ld_cluster(base + 4u * (dv + 1)));
      v = v * fo + fn * __uint_as_float(ps_ld_cluster(base + 4u * d));
      m = mn;
    }
    float f = l > 0.f ? 1.f / l : 0.f;
    if (p.s.gate) f *= 1.f / (1.f + expf(-as_f(static_cast<const T*>(p.s.gate)[static_cast<size_t>(tok) * p.s.ldg + h0 + g])));
    o[i] = T(v * f);
  }
  if (S > 1) cluster_sync_all();                 // no CTA leaves while a peer may still read its part
}

// ---- bf16, head sizes up to 128, pages of 16: tensor cores --------------------------------------------------------------------------
// Eight warps, one CTA per SM.  Scores are products with [lo, hi] of 2 dk numbers, q- against lo and q+ against hi: the same MMAs as for keys, eight
// pages in the place of eight keys (decode_warp.cuh has the order of the dimensions).  Sums are fp32 and their terms exact.
constexpr int AST_PITCH_PAD = 4;
template <int DV> struct SparseShape {
  static constexpr int PITCH = DV + AST_PITCH_PAD, SIZE = 16 * PITCH + 32;
  static constexpr int FLOATS = (PS_WARPS + 1) * SIZE + 16 * 8;
};

__device__ __forceinline__ uint32_t as_above(uint32_t x) {      // the larger of each half and zero; NaN stays
  const __nv_bfloat162 v = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&x), __floats2bfloat162_rn(0.f, 0.f));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t as_below(uint32_t x) {
  const __nv_bfloat162 v = __hmin2_nan(*reinterpret_cast<const __nv_bfloat162*>(&x), __floats2bfloat162_rn(0.f, 0.f));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// s += q' . bound of eight pages, over one half of the bounds
template <int DK, bool UP>
__device__ __forceinline__ void score_half(float (&s)[4], const DwQuery<DK>& q, const uint4 (&b)[DK / 32]) {
#pragma unroll
  for (int c = 0; c < DK / 32; ++c) {
    auto f = [](uint32_t x) { return UP ? as_above(x) : as_below(x); };
    dw_mma(s, f(q.lo[c].x), f(q.hi[c].x), f(q.lo[c].y), f(q.hi[c].y), b[c].x, b[c].y);
    dw_mma(s, f(q.lo[c].z), f(q.hi[c].z), f(q.lo[c].w), f(q.hi[c].w), b[c].z, b[c].w);
  }
}

template <int DK, int DV, bool FULL>
__global__ void __launch_bounds__(PS_THREADS, 1) attn_sparse_kernel(const __grid_constant__ SparseParams p) {
  using Sh = SparseShape<DV>;
  using bf16 = __nv_bfloat16;
  extern __shared__ __align__(16) uint8_t as_smem[];
  __shared__ PageSelectShared sel;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x, S = p.splits, tok = blockIdx.z;
  const int kvh = blockIdx.y / p.hgroups, hg = blockIdx.y - kvh * p.hgroups;
  const int group = p.hq / p.c.kv_heads, g0 = hg * 16, G = min(16, group - g0), h0 = kvh * group + g0;
  const int dk = FULL ? DK : p.c.dk, dv = FULL ? DV : p.c.dv;
  SparseRow row;
  if (!row.find(p, tok)) {                       // the same for all CTAs of the cluster
    if (rank == 0) {
      bf16* o = static_cast<bf16*>(p.out) + static_cast<size_t>(tok) * p.ldo + static_cast<size_t>(h0) * dv;
      for (int i = tid; i < G * dv; i += PS_THREADS) o[i] = __float2bfloat16(0.f);
      if (p.chosen && hg == 0)
        for (int i = tid; i < p.top; i += PS_THREADS) p.chosen[(static_cast<size_t>(tok) * p.c.kv_heads + kvh) * p.top + i] = -1;
    }
    return;
  }
  const bf16* q = static_cast<const bf16*>(p.q) + static_cast<size_t>(tok) * p.ldq;
  const int* pt = p.c.page_table + static_cast<size_t>(row.seq) * p.c.max_pages;
  float* parts = reinterpret_cast<float*>(as_smem);          // [8 warps], then the CTA's own, then shares [16][8]
  unsigned* keys = reinterpret_cast<unsigned*>(parts + Sh::FLOATS);
  int* list = reinterpret_cast<int*>(keys + p.score_cap);

  const int share = row.lists(p, rank, list, S);             // without a selection the list is known
  DecodeWarp<DK, DV, FULL> w;
  if (row.selects) {
    const int i0 = ps_share(row.candidates, rank, S), i1 = ps_share(row.candidates, rank + 1, S);
    const int a = i0 + static_cast<int>(static_cast<long long>(i1 - i0) * warp / PS_WARPS), b = i0 + static_cast<int>(static_cast<long long>(i1 - i0) * (warp + 1) / PS_WARPS);
    const int r = lane >> 2, d = (lane & 3) * 8, blocks = (group + 15) / 16;
    if (blocks == 1) w.q.load(q + static_cast<size_t>(kvh) * group * dk, group, dk);
    uint4 lo[DK / 32], hi[DK / 32];
    int ids = 0, ids_from = a - 32;
    auto request = [&](int i) {                  // bounds of pages i .. i + 7: a lane has part of page i + r
      if (i >= ids_from + 32) {
        ids_from = i;
        ids = i + lane < b ? pt[row.place0 + i + lane] : -1;
      }
      const int page = __shfl_sync(0xffffffffu, ids, i - ids_from + r);
      const bool on = page >= 0 && page < p.c.num_pages;
      const bf16* x = static_cast<const bf16*>(p.bounds) + (static_cast<size_t>(on ? page : 0) * p.c.kv_heads + kvh) * 2 * dk;
#pragma unroll
      for (int c = 0; c < DK / 32; ++c) {
        const bool in = on && (FULL || c * 32 + d < dk);
        lo[c] = dw_load(x + c * 32 + d, in);
        hi[c] = dw_load(x + dk + c * 32 + d, in);
      }
      return on;
    };
    if (a < b) {
      bool on = request(a);
      for (int i = a; i < b; i += 8) {
        float best[2] = {-INFINITY, -INFINITY};
        uint4 l8[DK / 32], h8[DK / 32];
#pragma unroll
        for (int c = 0; c < DK / 32; ++c) { l8[c] = lo[c]; h8[c] = hi[c]; }
        const unsigned there = __ballot_sync(0xffffffffu, on);
        if (i + 8 < b) on = request(i + 8);
        for (int k = 0; k < blocks; ++k) {
          const int n = min(16, group - 16 * k);
          if (blocks > 1) w.q.load(q + (static_cast<size_t>(kvh) * group + 16 * k) * dk, n, dk);
          float s[4] = {0.f, 0.f, 0.f, 0.f};
          score_half<DK, false>(s, w.q, l8);
          score_half<DK, true>(s, w.q, h8);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (r < n) best[e] = as_max(best[e], s[e]);
            if (r + 8 < n) best[e] = as_max(best[e], s[2 + e]);
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          best[e] = as_max(best[e], __shfl_xor_sync(0xffffffffu, best[e], 4));
          best[e] = as_max(best[e], __shfl_xor_sync(0xffffffffu, best[e], 8));
          best[e] = as_max(best[e], __shfl_xor_sync(0xffffffffu, best[e], 16));
          const int page = 2 * (lane & 3) + e;   // of the eight
          if (r == 0 && i + page < b) keys[i + page - i0] = ps_order((there >> (4 * page)) & 1u ? best[e] : -INFINITY);
        }
      }
    }
    __syncthreads();
    select_pages(sel, keys, i1 - i0, i0, row.take, row.first, row.entries, row.place0, list, rank, S);
  }
  w.begin(dk, dv, p.s.scale);
  w.q.load(q + static_cast<size_t>(h0) * dk, G, dk);
  if (S > 1) cluster_sync_all(); else __syncthreads();
  if (p.chosen && hg == 0) row.tell(p, tok, kvh, rank, share, list, S);

  const size_t rec = static_cast<size_t>(p.c.kv_heads) * 16 * (dk + dv);
  const bf16* kbase = static_cast<const bf16*>(p.c.data) + static_cast<size_t>(kvh) * 16 * dk;
  const bf16* vbase = static_cast<const bf16*>(p.c.data) + static_cast<size_t>(p.c.kv_heads) * 16 * dk + static_cast<size_t>(kvh) * 16 * dv;
  // the places and pages of this warp's next 32 entries are in its lanes
  int ids = 0, places = 0, ids_from = -32, place = 0, page = -1;
  const int mine = share > warp ? (share - warp + PS_WARPS - 1) / PS_WARPS : 0;
  auto next = [&](int i) {
    if (i >= ids_from + 32) {
      ids_from = i;
      places = i + lane < mine ? list[warp + (i + lane) * PS_WARPS] : 0;
      ids = i + lane < mine ? pt[places] : -1;
    }
    place = __shfl_sync(0xffffffffu, places, i - ids_from);
    page = __shfl_sync(0xffffffffu, ids, i - ids_from);
    if (page >= p.c.num_pages) page = -1;
  };
  if (mine > 0) {
    next(0);
    int lo = max(0, row.low - place * 16), hi = min(16, row.pos + 1 - place * 16);
    w.load_k(kbase + (page >= 0 ? page * rec : 0), page >= 0);
    w.load_v(vbase + (page >= 0 ? page * rec : 0), lo, page >= 0 ? hi : 0);
    for (int i = 0; i < mine; ++i) {
      float s[2][4];
      w.scores(s);
      const int here = page, lo_here = lo, hi_here = hi;
      if (i + 1 < mine) {
        next(i + 1);
        lo = max(0, row.low - place * 16);
        hi = min(16, row.pos + 1 - place * 16);
        w.load_k(kbase + (page >= 0 ? page * rec : 0), page >= 0);
      }
      if (here >= 0) {
        uint32_t pr[4];
        w.weigh(s, lo_here, hi_here, pr);
        w.add(pr);
      } else if (lane == 0 && p.status) {
        atomicCAS(p.status, 0, static_cast<int>(ST_BAD_ARGUMENT) | (25 << 8));
      }
      if (i + 1 < mine) w.load_v(vbase + (page >= 0 ? page * rec : 0), lo, page >= 0 ? hi : 0);
    }
  }
  w.end();
  w.put(parts + warp * Sh::SIZE, Sh::PITCH, G);
  __syncthreads();
  float* own = parts + PS_WARPS * Sh::SIZE;
  float* shares = own + Sh::SIZE;
  dw_join<PS_WARPS, PS_THREADS>(parts, Sh::SIZE, Sh::PITCH, G, dv, own);
  if (S > 1) cluster_sync_all(); else __syncthreads();
  const uint32_t own_addr = smem_u32(own);
  if (tid < 16 * 8) {                            // eight lanes per row, a CTA of the cluster each
    const int g = tid >> 3, i = tid & 7;
    float m = -INFINITY, l = 0.f;
    if (g < G && i < S) {
      const uint32_t base = S > 1 ? mapa_shared(own_addr, i) : own_addr;
      m = dw_ld_cluster(base + 4u * (16 * Sh::PITCH + g));
      l = dw_ld_cluster(base + 4u * (16 * Sh::PITCH + 16 + g));
    }
    const float sink2 = p.s.sink && g < G ? p.s.sink[h0 + g] * DW_LOG2E : -INFINITY;
    float top = fmaxf(m, sink2);
#pragma unroll
    for (int o = 1; o < 8; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float use = top == -INFINITY ? 0.f : top, f0 = m == -INFINITY ? 0.f : dw_exp2(m - use);
    float total = f0 * l;
#pragma unroll
    for (int o = 1; o < 8; o *= 2) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (p.s.sink) total += dw_exp2(sink2 - use);
    float f = total > 0.f ? 1.f / total : 0.f;
    if (p.s.gate && g < G) f *= 1.f / (1.f + __expf(-__bfloat162float(static_cast<const bf16*>(p.s.gate)[static_cast<size_t>(tok) * p.s.ldg + h0 + g])));
    shares[tid] = f0 * f;
  }
  __syncthreads();
  bf16* out = static_cast<bf16*>(p.out) + static_cast<size_t>(tok) * p.ldo + static_cast<size_t>(h0) * dv;
  for (int i = rank * PS_THREADS + tid; i < G * dv; i += S * PS_THREADS) {
    const int g = i / dv, x = i - g * dv;
    float v = 0.f;
    for (int r = 0; r < S; ++r) {
      const float f = shares[g * 8 + r];
      if (f != 0.f) v += f * dw_ld_cluster((S > 1 ? mapa_shared(own_addr, r) : own_addr) + 4u * (g * Sh::PITCH + x));
    }
    out[i] = __float2bfloat16(v);
  }
  if (S > 1) cluster_sync_all();                 // no CTA leaves while a peer may still read its part
}

template <int DK, int DV, bool FULL>
static int launch_sparse(const SparseParams& p, cudaStream_t stream) {
  const size_t smem = 4 * (static_cast<size_t>(SparseShape<DV>::FLOATS) + p.score_cap + p.list_cap);
  if (smem > SPARSE_MAX_SMEM) return -5;
  cudaError_t e = cudaFuncSetAttribute(attn_sparse_kernel<DK, DV, FULL>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SPARSE_MAX_SMEM));
  if (e != cudaSuccess) return -1000 - static_cast<int>(e);
  launch_ex(attn_sparse_kernel<DK, DV, FULL>, dim3(p.splits, p.c.kv_heads * p.hgroups, p.M), dim3(PS_THREADS), smem, stream, p.splits, p);
  e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -2000 - static_cast<int>(e);
}

template <typename T>
static int launch_sparse_any(const SparseParams& p, cudaStream_t stream) {
  const size_t smem = 4 * (static_cast<size_t>(p.score_cap) + p.list_cap + static_cast<size_t>(PS_WARPS + 16) * (p.c.dv + 2));
  if (smem > SPARSE_MAX_SMEM) return -5;
  cudaError_t e = cudaFuncSetAttribute(attn_sparse_any_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SPARSE_MAX_SMEM));
  if (e != cudaSuccess) return -1000 - static_cast<int>(e);
  launch_ex(attn_sparse_any_kernel<T>, dim3(p.splits, p.c.kv_heads * p.hgroups, p.M), dim3(PS_THREADS), smem, stream, p.splits, p);
  e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -2000 - static_cast<int>(e);
}

}  // namespace b200

using namespace b200;

extern "C" int b200_attn_paged_sparse(const void* q, long long ldq, void* out, long long ldo, int hq, int M, const int* positions, const int* seq_ids,
                                      const int* seq_lens, const b200_paged_cache* c, const void* bounds, const b200_attn_spec* s, int top, int first,
                                      int last, int splits, int* chosen, int* status, cudaStream_t stream) {
  if (M <= 0) return 0;
  if (!q || !out || !positions || !c || !c->data || !c->page_table || !bounds || !s) return -1;
  if (hq <= 0 || c->kv_heads <= 0 || hq % c->kv_heads || c->page_size <= 0 || c->dk <= 0 || c->dv <= 0 || c->dk > AS_MAX_D || c->dv > AS_MAX_D ||
      c->num_pages <= 0) return -2;
  if (first < 0 || last < 1 || top < first + last || splits < 1 || splits > 8 || M > 65535 || !(s->scale > 0.f)) return -3;
  SparseParams p = {};
  p.q = q; p.ldq = ldq; p.out = out; p.ldo = ldo; p.hq = hq; p.M = M; p.hgroups = (hq / c->kv_heads + 15) / 16;
  p.positions = positions; p.seq_ids = seq_ids; p.seq_lens = seq_lens; p.c = *c; p.s = *s; p.bounds = bounds;
  p.top = top; p.first = first; p.last = last; p.splits = splits; p.chosen = chosen; p.status = status;
  p.score_cap = (((c->max_pages + splits - 1) / splits + 1) + 3) & ~3;
  p.list_cap = (((top < c->max_pages ? top : c->max_pages) + splits - 1) / splits + 1 + 3) & ~3;
  if (static_cast<long long>(c->kv_heads) * p.hgroups > 65535) return -3;
  if (c->f32) return launch_sparse_any<float>(p, stream);
  if (c->page_size != 16 || c->dk > 128 || c->dv > 128 || c->dk % 8 || c->dv % 8 || ldq % 8 || (reinterpret_cast<uintptr_t>(q) & 15) ||
      (reinterpret_cast<uintptr_t>(c->data) & 15) || (reinterpret_cast<uintptr_t>(bounds) & 15)) return launch_sparse_any<__nv_bfloat16>(p, stream);
  const int d = c->dk > c->dv ? c->dk : c->dv;
  if (c->dk == 64 && c->dv == 64) return launch_sparse<64, 64, true>(p, stream);
  if (c->dk == 128 && c->dv == 128) return launch_sparse<128, 128, true>(p, stream);
  if (d <= 64) return launch_sparse<64, 64, false>(p, stream);
  return launch_sparse<128, 128, false>(p, stream);
}

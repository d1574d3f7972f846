// Attention of single rows of queries over the pages of their sequences that look most promising.
//
// A page's score for a KV head bounds what any of its query heads can get from any key of the page: with lo <= k <= hi per dimension,
//   q . k <= sum_d max(q_d lo_d, q_d hi_d) = q+ . hi + q- . lo,      q+ = max(q, 0), q- = min(q, 0),
// and the score is the largest of the group's heads.  The first pages, and the last up to the row's own position, are read always; the others compete.
//
// Two launches.  The first scores all pages of all rows, spread over the whole chip; bound by the bytes of the bounds, 2 dk per page.  The second has a
// cluster of CTAs per row and group of heads: each selects (page_select.cuh), reads its share of the pages taken, and the sums are joined
// through distributed shared memory, every CTA joining a slice of the dimensions.  (One launch of clusters that scored, selected and read took 32 us where these
// two take 20, 131,071 keys and 8 KV heads: eight clusters keep 64 of 148 SMs busy with the scores, and clusters of 16 do not all run at once.)
//
// One row behind 131,071 keys, 128 of 8,192 pages taken, 8 KV heads of 128: 7.5 us for the scores (33.5 MB of bounds, 4.5 TB/s), 1.7 between the launches, 5 for the
// selection, 4 for 8.4 MB of pages, 2 for the join.  16 rows behind 8,000 to 16,001 keys, 64 pages each, 4 KV heads: 22 us for 59 MB.
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

// =====================================================================================================================================
// scores.  Grid (pages, KV head, row)
// =====================================================================================================================================
constexpr int SC_WARPS = 8, SC_THREADS = 32 * SC_WARPS;

// ---- any head size, bf16 or fp32: four pages per warp, lanes along the dimensions, the queries in shared memory -------------------------
constexpr int SCA_EACH = 4, SCA_PAGES = SCA_EACH * SC_WARPS;
constexpr int AS_MAX_D = 512, AS_RUNS = AS_MAX_D / 128;      // dimensions 128 at a time: four for a lane

// elements d .. d + 3 of a row of n, zeros behind it; VEC: rows are whole fours of elements that lie on as many bytes
template <bool VEC, typename T>
__device__ __forceinline__ float4 as_f4(const T* row, int d, int n) {
  if constexpr (VEC) {
    if (d >= n) return make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (sizeof(T) == 4) return __ldcg(reinterpret_cast<const float4*>(row + d));
    else {
      const uint2 r = __ldcg(reinterpret_cast<const uint2*>(row + d));
      return make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16), __uint_as_float(r.y & 0xffff0000u));
    }
  }
  return make_float4(d < n ? as_f(row[d]) : 0.f, d + 1 < n ? as_f(row[d + 1]) : 0.f, d + 2 < n ? as_f(row[d + 2]) : 0.f, d + 3 < n ? as_f(row[d + 3]) : 0.f);
}
__device__ __forceinline__ int as_padded(int d) { return (d + 127) & ~127; }

template <typename T, bool VEC>
__global__ void __launch_bounds__(SC_THREADS) page_scores_any_kernel(const __grid_constant__ SparseParams p) {
  extern __shared__ __align__(16) float sc_q[];      // [heads of the group][dk, zeros up to whole 128]
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tok = blockIdx.z, kvh = blockIdx.y;
  const int group = p.hq / p.c.kv_heads, dk = p.c.dk, wide = as_padded(dk);
  SparseRow row;
  if (!row.find(p, tok) || !row.selects || static_cast<int>(blockIdx.x) * SCA_PAGES >= row.candidates) return;
  const T* q = static_cast<const T*>(p.q) + static_cast<size_t>(tok) * p.ldq + static_cast<size_t>(kvh) * group * dk;
  for (int i = threadIdx.x; i < group * wide; i += SC_THREADS) {
    const int h = i / wide, d = i - h * wide;
    sc_q[i] = d < dk ? as_f(q[static_cast<size_t>(h) * dk + d]) : 0.f;
  }
  __syncthreads();
  const int i0 = blockIdx.x * SCA_PAGES + warp * SCA_EACH, n = min(row.candidates - i0, SCA_EACH);
  if (n <= 0) return;
  const int* pt = p.c.page_table + static_cast<size_t>(row.seq) * p.c.max_pages + row.place0 + i0;
  const T* lo[SCA_EACH];
  bool there[SCA_EACH];
  float s[SCA_EACH];
#pragma unroll
  for (int j = 0; j < SCA_EACH; ++j) {
    const int page = j < n ? pt[j] : -1;
    there[j] = page >= 0 && page < p.c.num_pages;
    lo[j] = static_cast<const T*>(p.bounds) + (static_cast<size_t>(there[j] ? page : 0) * p.c.kv_heads + kvh) * 2 * dk;
    s[j] = -INFINITY;
  }
  // four heads at a time, so that the bounds are read once for them
  for (int h0 = 0; h0 < group; h0 += 4) {
    float t[SCA_EACH][4] = {};
    for (int d0 = 0; d0 < dk; d0 += 128) {
      float4 a[SCA_EACH], b[SCA_EACH];
#pragma unroll
      for (int j = 0; j < SCA_EACH; ++j) { a[j] = as_f4<VEC>(lo[j], d0 + 4 * lane, dk); b[j] = as_f4<VEC>(lo[j] + dk, d0 + 4 * lane, dk); }
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if (h0 + h >= group) break;
        const float4 x = *reinterpret_cast<const float4*>(sc_q + (h0 + h) * wide + d0 + 4 * lane);
#pragma unroll
        for (int j = 0; j < SCA_EACH; ++j) {
          float u = fmaf(fmaxf(x.x, 0.f), b[j].x, fmaf(fminf(x.x, 0.f), a[j].x, t[j][h]));
          u = fmaf(fmaxf(x.y, 0.f), b[j].y, fmaf(fminf(x.y, 0.f), a[j].y, u));
          u = fmaf(fmaxf(x.z, 0.f), b[j].z, fmaf(fminf(x.z, 0.f), a[j].z, u));
          t[j][h] = fmaf(fmaxf(x.w, 0.f), b[j].w, fmaf(fminf(x.w, 0.f), a[j].w, u));
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      if (h0 + h >= group) break;
#pragma unroll
      for (int j = 0; j < SCA_EACH; ++j) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t[j][h] += __shfl_xor_sync(0xffffffffu, t[j][h], o);
        s[j] = as_max(s[j], t[j][h]);
      }
    }
  }
  unsigned* to = p.scores + (static_cast<size_t>(tok) * p.c.kv_heads + kvh) * p.c.max_pages + i0;
#pragma unroll
  for (int j = 0; j < SCA_EACH; ++j)
    if (lane == j && j < n) to[j] = ps_order(there[j] ? s[j] : -INFINITY);
}

// ---- bf16, head sizes up to 128: tensor cores ----------------------------------------------------------------------------------------------
// Products with [lo, hi] of 2 dk numbers, q- against lo and q+ against hi: the same MMAs as for keys, 16 pages in the place of 16 keys
// (decode_warp.cuh has the order of the dimensions).  A warp has one or two steps of 16 pages, 8 KiB of bounds each, the second's requested as the first's are used.  Sums are
// fp32 and their terms exact.
constexpr int SC_CTAS = 296;

__device__ __forceinline__ uint32_t as_above(uint32_t x) {      // the larger of each half and zero; NaN stays
  const __nv_bfloat162 v = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&x), __floats2bfloat162_rn(0.f, 0.f));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t as_below(uint32_t x) {
  const __nv_bfloat162 v = __hmin2_nan(*reinterpret_cast<const __nv_bfloat162*>(&x), __floats2bfloat162_rn(0.f, 0.f));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// s += q' . bounds, one half of the bounds of sixteen pages (rows lane / 4 and lane / 4 + 8): pages g, g, g + 8, g + 8 of heads 2 t, 2 t + 1.  Two
// sums each, so that an MMA need not wait for the one before.
template <int DK, int NH, bool UP>
__device__ __forceinline__ void score_half(float (&s)[NH][2][4], const DwQuery<DK, NH>& q, const uint4 (&b)[2][DK / 32]) {
  auto f = [](uint32_t x) { return UP ? as_above(x) : as_below(x); };
#pragma unroll
  for (int c = 0; c < DK / 32; ++c)
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      const uint4 x = q.h[n][c];
      dw_mma(s[n][0], b[0][c].x, b[1][c].x, b[0][c].y, b[1][c].y, f(x.x), f(x.y));
      dw_mma(s[n][1], b[0][c].z, b[1][c].z, b[0][c].w, b[1][c].w, f(x.z), f(x.w));
    }
}

template <int DK, int NH, bool FULL, int EACH>
__global__ void __launch_bounds__(SC_THREADS, NH == 1 ? 2 : 1) page_scores_kernel(const __grid_constant__ SparseParams p) {
  using bf16 = __nv_bfloat16;
  B200_TRACE_INIT();
  if (threadIdx.x == 0) B200_TRACE(TK_ATTN_OWN, TP_START);
  pdl_wait();
  pdl_launch_dependents();       // what starts now may read all that was written before this kernel
  if (threadIdx.x == 0) B200_TRACE(TK_ATTN_OWN, TP_DEPS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tok = blockIdx.z, kvh = blockIdx.y;
  const int group = p.hq / p.c.kv_heads, dk = FULL ? DK : p.c.dk, g = lane >> 2, t = lane & 3;
  SparseRow row;
  if (!row.find(p, tok) || !row.selects || static_cast<int>(blockIdx.x) * SC_WARPS * EACH >= row.candidates) return;
  const bf16* q = static_cast<const bf16*>(p.q) + static_cast<size_t>(tok) * p.ldq + static_cast<size_t>(kvh) * group * dk;
  unsigned* to = p.scores + (static_cast<size_t>(tok) * p.c.kv_heads + kvh) * p.c.max_pages;
  const int a = blockIdx.x * SC_WARPS * EACH + warp * EACH, b = min(row.candidates, a + EACH);
  if (a < b) {
    const int ids = a + lane < b ? p.c.page_table[static_cast<size_t>(row.seq) * p.c.max_pages + row.place0 + a + lane] : -1;
    DwQuery<DK, NH> w;
    uint4 lo[2][DK / 32], hi[2][DK / 32];
    const bf16* from[2];
    auto find = [&](int i) {                     // pages a + i .. a + i + 15: this lane's two; whether they are there
      unsigned there = 0u;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int page = __shfl_sync(0xffffffffu, ids, i + g + 8 * u);
        const bool on = page >= 0 && page < p.c.num_pages;
        from[u] = static_cast<const bf16*>(p.bounds) + (static_cast<size_t>(on ? page : 0) * p.c.kv_heads + kvh) * 2 * dk + t * 8;
        there |= static_cast<unsigned>(on) << u;
      }
      return there;
    };
    auto request = [&](uint4 (&x)[2][DK / 32], int at, unsigned there) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < DK / 32; ++c) x[u][c] = dw_load(from[u] + at + c * 32, ((there >> u) & 1u) && (FULL || c * 32 + t * 8 < dk));
    };
    for (int n0 = 0; n0 < group; n0 += 8 * NH) {             // more than 16 heads: the bounds once for every 16
      const int n = min(8 * NH, group - n0);
      unsigned there = find(0);
      request(lo, 0, there);
      request(hi, dk, there);
      w.load(q + static_cast<size_t>(n0) * dk, n, dk);
#pragma unroll 1
      for (int i = 0; i < b - a; i += 16) {
        float s[NH][2][4];
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[h][0][e] = s[h][1][e] = 0.f;
        const unsigned here = there;
        const bool more = i + 16 < b - a;
        score_half<DK, NH, false>(s, w, lo);
        if (more) { there = find(16); request(lo, 0, there); }
        score_half<DK, NH, true>(s, w, hi);
        if (more) request(hi, dk, there);
        float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (8 * h + 2 * t + (e & 1) < n) best[e >> 1] = as_max(best[e >> 1], s[h][0][e] + s[h][1][e]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          best[u] = as_max(best[u], __shfl_xor_sync(0xffffffffu, best[u], 1));
          best[u] = as_max(best[u], __shfl_xor_sync(0xffffffffu, best[u], 2));
          const int at = a + i + g + 8 * u;
          if (t == 0 && at < b) {
            const unsigned key = ps_order((here >> u) & 1u ? best[u] : -INFINITY);
            to[at] = n0 > 0 ? max(to[at], key) : key;
          }
        }
      }
    }
  }
  if (threadIdx.x == 0) B200_TRACE(TK_ATTN_OWN, TP_EXIT);
  B200_TRACE_FLUSH(TK_ATTN_OWN);
}

// =====================================================================================================================================
// selection and attention.  Grid (split, KV head x group of up to 16 query heads, row); the splits of a row are a cluster
// =====================================================================================================================================

// zeros for a row that sees nothing
template <typename T>
__device__ __forceinline__ void sparse_nothing(const SparseParams& p, int tok, int kvh, int hg, int h0, int G, int rank) {
  if (rank != 0) return;
  T* o = static_cast<T*>(p.out) + static_cast<size_t>(tok) * p.ldo + static_cast<size_t>(h0) * p.c.dv;
  for (int i = threadIdx.x; i < G * p.c.dv; i += PS_THREADS) o[i] = T(0.f);
  if (p.chosen && hg == 0)
    for (int i = threadIdx.x; i < p.top; i += PS_THREADS) p.chosen[(static_cast<size_t>(tok) * p.c.kv_heads + kvh) * p.top + i] = -1;
}

// ---- any head size, bf16 or fp32 ------------------------------------------------------------------------------------------------------------
// A warp takes 16 keys of a page for four heads at a time, lanes along the dimensions: all rows of the keys, then of the values, are on their way at once.
constexpr int ASA_HEADS = 4;

template <typename T, bool VEC>
__global__ void __launch_bounds__(PS_THREADS) attn_sparse_any_kernel(const __grid_constant__ SparseParams p) {
  extern __shared__ __align__(16) uint8_t as_smem[];
  __shared__ PageSelectShared sel;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x, S = p.splits, tok = blockIdx.z;
  const int kvh = blockIdx.y / p.hgroups, hg = blockIdx.y - kvh * p.hgroups;
  const int group = p.hq / p.c.kv_heads, g0 = hg * 16, G = min(16, group - g0), h0 = kvh * group + g0;
  const int dk = p.c.dk, dv = p.c.dv, ps = p.c.page_size, wide = as_padded(dk), pitch = as_padded(dv) + 4;
  SparseRow row;
  if (!row.find(p, tok)) { sparse_nothing<T>(p, tok, kvh, hg, h0, G, rank); return; }      // the same for all CTAs of the cluster
  const T* q = static_cast<const T*>(p.q) + static_cast<size_t>(tok) * p.ldq + static_cast<size_t>(h0) * dk;
  const int* pt = p.c.page_table + static_cast<size_t>(row.seq) * p.c.max_pages;
  // [8 warps][4 heads][pitch], [16 heads][pitch] (the last four of a row: m, l), queries [16][wide], scores, list
  float* part = reinterpret_cast<float*>(as_smem);
  float* joined = part + PS_WARPS * ASA_HEADS * pitch;
  float* qs = joined + 16 * pitch;
  unsigned* room = reinterpret_cast<unsigned*>(qs + 16 * wide);
  int* list = reinterpret_cast<int*>(room + p.score_cap);
  for (int i = tid; i < 16 * wide; i += PS_THREADS) {
    const int h = i / wide, d = i - h * wide;
    qs[i] = h < G && d < dk ? as_f(q[static_cast<size_t>(h) * dk + d]) : 0.f;
  }
  const int share = row.lists(p, sel, room, tok, kvh, rank, S, list);
  __syncthreads();
  if (p.chosen && hg == 0) row.tell(p, tok, kvh, rank, share, list, S);

  const size_t rec = static_cast<size_t>(p.c.kv_heads) * ps * (dk + dv);
  const int per = (ps + 15) / 16;                // runs of 16 keys of a page
  for (int g4 = 0; g4 < G; g4 += ASA_HEADS) {
    float m[ASA_HEADS], l[ASA_HEADS];
    float4 acc[ASA_HEADS][AS_RUNS];
#pragma unroll
    for (int h = 0; h < ASA_HEADS; ++h) {
      m[h] = -INFINITY; l[h] = 0.f;
#pragma unroll
      for (int j = 0; j < AS_RUNS; ++j) acc[h][j] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int i = warp; i < share * per; i += PS_WARPS) {
      const int place = list[i / per], page = pt[place];
      if (page < 0 || page >= p.c.num_pages) {
        if (lane == 0 && p.status) atomicCAS(p.status, 0, static_cast<int>(ST_BAD_ARGUMENT) | (25 << 8));
        continue;
      }
      const int k0 = i % per * 16, r0 = max(0, row.low - place * ps), r1 = min(ps, row.pos + 1 - place * ps);
      if (k0 >= r1 || k0 + 16 <= r0) continue;
      const T* kp = static_cast<const T*>(p.c.data) + static_cast<size_t>(page) * rec + static_cast<size_t>(kvh) * ps * dk;
      const T* vp = static_cast<const T*>(p.c.data) + static_cast<size_t>(page) * rec + static_cast<size_t>(p.c.kv_heads) * ps * dk + static_cast<size_t>(kvh) * ps * dv;
      auto seen = [&](int r) { return k0 + r >= r0 && k0 + r < r1; };
      float s[ASA_HEADS] = {};                   // of key lane / 2
      for (int d0 = 0; d0 < dk; d0 += 128) {
        float4 k[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) k[r] = as_f4<VEC>(kp + static_cast<size_t>(seen(r) ? k0 + r : max(k0, r0)) * dk, d0 + 4 * lane, dk);
#pragma unroll
        for (int h = 0; h < ASA_HEADS; ++h) {
          if (g4 + h >= G) break;
          const float4 x = *reinterpret_cast<const float4*>(qs + (g4 + h) * wide + d0 + 4 * lane);
          // sixteen sums over the lanes: half of what is left goes to the partner each time
          float t[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) t[r] = fmaf(x.x, k[r].x, fmaf(x.y, k[r].y, fmaf(x.z, k[r].z, x.w * k[r].w)));
#pragma unroll
          for (int o = 16, half = 8; o > 1; o >>= 1, half >>= 1)
#pragma unroll
            for (int r = 0; r < half; ++r) {
              const bool upper = lane & o;
              const float mine = upper ? t[r + half] : t[r], other = upper ? t[r] : t[r + half];
              t[r] = mine + __shfl_xor_sync(0xffffffffu, other, o);
            }
          s[h] += t[0] + __shfl_xor_sync(0xffffffffu, t[0], 1);
        }
      }
      float e[ASA_HEADS], a[ASA_HEADS];
#pragma unroll
      for (int h = 0; h < ASA_HEADS; ++h) {
        const float x = seen(lane >> 1) ? s[h] * p.s.scale : -INFINITY;
        float mx = x;
#pragma unroll
        for (int o = 16; o > 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mn = fmaxf(m[h], mx), use = mn == -INFINITY ? 0.f : mn;
        a[h] = m[h] == -INFINITY ? 0.f : expf(m[h] - use);
        e[h] = x == -INFINITY ? 0.f : expf(x - use);
        float sum = e[h];
#pragma unroll
        for (int o = 16; o > 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l[h] = l[h] * a[h] + sum;
        m[h] = mn;
      }
#pragma unroll
      for (int j = 0; j < AS_RUNS; ++j) {
        if (128 * j >= dv) break;
        float4 v[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = seen(r) ? as_f4<VEC>(vp + static_cast<size_t>(k0 + r) * dv, 128 * j + 4 * lane, dv) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int h = 0; h < ASA_HEADS; ++h) {
          if (g4 + h >= G) break;
          float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float w = __shfl_sync(0xffffffffu, e[h], 2 * r);
            t.x = fmaf(w, v[r].x, t.x); t.y = fmaf(w, v[r].y, t.y); t.z = fmaf(w, v[r].z, t.z); t.w = fmaf(w, v[r].w, t.w);
          }
          float4& c = acc[h][j];
          c.x = fmaf(c.x, a[h], t.x); c.y = fmaf(c.y, a[h], t.y); c.z = fmaf(c.z, a[h], t.z); c.w = fmaf(c.w, a[h], t.w);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < ASA_HEADS; ++h) {
      float* mine = part + (warp * ASA_HEADS + h) * pitch;
#pragma unroll
      for (int j = 0; j < AS_RUNS; ++j)
        if (128 * j < dv) *reinterpret_cast<float4*>(mine + 128 * j + 4 * lane) = acc[h][j];
      if (lane == 0) { mine[pitch - 4] = m[h]; mine[pitch - 3] = l[h]; }
    }
    __syncthreads();
    for (int i = tid; i < min(ASA_HEADS, G - g4) * (dv + 1); i += PS_THREADS) {      // the last of a head: the sums of its weights
      const int h = i / (dv + 1), d = i - h * (dv + 1);
      float top = -INFINITY, v = 0.f;
#pragma unroll
      for (int w = 0; w < PS_WARPS; ++w) top = fmaxf(top, part[(w * ASA_HEADS + h) * pitch + pitch - 4]);
      const float use = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < PS_WARPS; ++w) {
        const float* x = part + (w * ASA_HEADS + h) * pitch;
        v = fmaf(expf(x[pitch - 4] - use), d < dv ? x[d] : x[pitch - 3], v);
      }
      float* to = joined + (g4 + h) * pitch;
      if (d < dv) to[d] = v;
      else { to[pitch - 4] = top; to[pitch - 3] = v; }
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
      const float mr = dw_ld_cluster(base + 4u * (pitch - 4));
      const float mn = fmaxf(m, mr), use = mn == -INFINITY ? 0.f : mn, fo = expf(m - use), fn = expf(mr - use);
      l = l * fo + fn * dw_ld_cluster(base + 4u * (pitch - 3));
      v = v * fo + fn * dw_ld_cluster(base + 4u * d);
      m = mn;
    }
    float f = l > 0.f ? 1.f / l : l;             // nothing, or not a number
    if (p.s.gate) f *= 1.f / (1.f + expf(-as_f(static_cast<const T*>(p.s.gate)[static_cast<size_t>(tok) * p.s.ldg + h0 + g])));
    o[i] = T(v * f);
  }
  if (S > 1) cluster_sync_all();                 // no CTA leaves while a peer may still read its part
}

// ---- bf16, head sizes up to 128, pages of 16: tensor cores ------------------------------------------------------------------------------------
// Eight warps, one CTA per SM, a page per warp and step (decode_warp.cuh).
template <int DV> struct SparseShape {
  static constexpr int MAX_CLUSTER = 8, PITCH = DV + 4, SIZE = 16 * PITCH + 32;
  static constexpr int SLICES = 16 * DV + 4 * MAX_CLUSTER, FLOATS = PS_WARPS * SIZE + SLICES + 32 * MAX_CLUSTER;
};

template <int DK, int DV, int NH, bool FULL>
__global__ void __launch_bounds__(PS_THREADS, 1) attn_sparse_kernel(const __grid_constant__ SparseParams p) {
  using Sh = SparseShape<DV>;
  using bf16 = __nv_bfloat16;
  extern __shared__ __align__(16) uint8_t as_smem[];
  __shared__ PageSelectShared sel;
  B200_TRACE_INIT();
  if (threadIdx.x == 0) B200_TRACE(TK_ATTN_SPARSE, TP_START);
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x, S = p.splits, tok = blockIdx.z;
  const int kvh = blockIdx.y / p.hgroups, hg = blockIdx.y - kvh * p.hgroups;
  const int group = p.hq / p.c.kv_heads, g0 = hg * 16, G = min(16, group - g0), h0 = kvh * group + g0;
  const int dk = FULL ? DK : p.c.dk, dv = FULL ? DV : p.c.dv;
  // the kernel in front of this one starts it after its own wait: all but the scores is settled
  SparseRow row;
  const bool any = row.find(p, tok);
  const bf16* q = static_cast<const bf16*>(p.q) + static_cast<size_t>(tok) * p.ldq + static_cast<size_t>(h0) * dk;
  DecodeWarp<DK, DV, NH, FULL> w;
  w.begin(dk, dv, p.s.scale);
  w.q.load(q, any ? G : 0, dk);
  pdl_wait();
  if (tid == 0) B200_TRACE(TK_ATTN_SPARSE, TP_DEPS);
  if (!any) { sparse_nothing<bf16>(p, tok, kvh, hg, h0, G, rank); return; }      // the same for all CTAs of the cluster
  const int* pt = p.c.page_table + static_cast<size_t>(row.seq) * p.c.max_pages;
  // [8 warps], slices of every CTA's O for this one to join, (m, l) of every CTA [8][2][16], scores, list
  float* parts = reinterpret_cast<float*>(as_smem);
  float* slices = parts + PS_WARPS * Sh::SIZE;
  float* ml = slices + Sh::SLICES;
  unsigned* room = reinterpret_cast<unsigned*>(parts + Sh::FLOATS);
  int* list = reinterpret_cast<int*>(room + p.score_cap);
  const int share = row.lists(p, sel, room, tok, kvh, rank, S, list);
  __syncthreads();
  if (S > 1) cluster_arrive_relaxed();           // all CTAs have started when theirs is waited for, in front of the first access
  if (tid == 0) B200_TRACE(TK_ATTN_SPARSE, 3);               // lists
  if (p.chosen && hg == 0) row.tell(p, tok, kvh, rank, share, list, S);

  const size_t rec = static_cast<size_t>(p.c.kv_heads) * 16 * (dk + dv);
  const bf16* kbase = static_cast<const bf16*>(p.c.data) + static_cast<size_t>(kvh) * 16 * dk;
  const bf16* vbase = static_cast<const bf16*>(p.c.data) + static_cast<size_t>(p.c.kv_heads) * 16 * dk + static_cast<size_t>(kvh) * 16 * dv;
  // the places and pages of this warp's next 32 entries are in its lanes
  int ids = 0, places = 0, ids_from = -32;
  const int mine = share > warp ? (share - warp + PS_WARPS - 1) / PS_WARPS : 0;
  w.walk(mine, [&](int i) {
    if (i >= ids_from + 32) {
      ids_from = i;
      places = i + lane < mine ? list[warp + (i + lane) * PS_WARPS] : 0;
      ids = i + lane < mine ? pt[places] : -1;
    }
    const int place = __shfl_sync(0xffffffffu, places, i - ids_from), page = __shfl_sync(0xffffffffu, ids, i - ids_from);
    const bool there = page >= 0 && page < p.c.num_pages;
    if (!there && lane == 0 && p.status) atomicCAS(p.status, 0, static_cast<int>(ST_BAD_ARGUMENT) | (25 << 8));
    const size_t at = there ? page * rec : 0;
    return DwPage{kbase + at, vbase + at, max(0, row.low - place * 16), there ? min(16, row.pos + 1 - place * 16) : 0};
  }, [] {});
  w.put(parts + warp * Sh::SIZE, Sh::PITCH, G);
  __syncthreads();
  if (tid == 0) B200_TRACE(TK_ATTN_SPARSE, 4);               // attention
  if (S > 1) cluster_wait_acquire();
  // The CTA's sums go to the CTAs that join them: every one has a slice of the output's quads of dimensions.
  const int quads = dv >> 2, total = G * quads, slice = (total + S - 1) / S;
  for (int i = tid; i < total; i += PS_THREADS) {
    const int g = i / quads, d = (i - g * quads) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
#pragma unroll 4
    for (int k = 0; k < PS_WARPS; ++k) m = fmaxf(m, parts[k * Sh::SIZE + 16 * Sh::PITCH + g]);
    const float use = m == -INFINITY ? 0.f : m;
#pragma unroll 4
    for (int k = 0; k < PS_WARPS; ++k) {         // a warp without pages has left zeros
      const float* x = parts + k * Sh::SIZE;
      const float f = dw_exp2(x[16 * Sh::PITCH + g] - use);
      const float4 y = *reinterpret_cast<const float4*>(x + g * Sh::PITCH + d);
      v.x += f * y.x; v.y += f * y.y; v.z += f * y.z; v.w += f * y.w;
      l += f * x[16 * Sh::PITCH + 16 + g];
    }
    const int r = static_cast<int>(((static_cast<long long>(i) + 1) * S - 1) / total);       // whose slice has it
    const uint32_t to = smem_u32(slices + 4 * (rank * slice + i - ps_share(total, r, S)));
    st_shared_cluster_v4(S > 1 ? mapa_shared(to, r) : to, __float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w));
    // the threads of a head's quads tell the CTAs its (m, l)
#pragma unroll 1
    for (int k = i - g * quads; k < S; k += quads) {
      const uint32_t at = smem_u32(ml + 32 * rank + g);
      st_shared_cluster_u32(S > 1 ? mapa_shared(at, k) : at, __float_as_uint(m));
      st_shared_cluster_u32((S > 1 ? mapa_shared(at, k) : at) + 64, __float_as_uint(l));
    }
  }
  if (S > 1) cluster_sync_all(); else __syncthreads();       // nothing of another CTA is touched behind this
  const int x0 = ps_share(total, rank, S), x1 = ps_share(total, rank + 1, S);
  bf16* out = static_cast<bf16*>(p.out) + static_cast<size_t>(tok) * p.ldo + static_cast<size_t>(h0) * dv;
  for (int i = x0 + tid; i < x1; i += PS_THREADS) {
    const int g = i / quads, d = (i - g * quads) * 4;
    const float sink2 = p.s.sink ? p.s.sink[h0 + g] * DW_LOG2E : -INFINITY;
    float m = sink2;
#pragma unroll 4
    for (int r = 0; r < S; ++r) m = fmaxf(m, ml[32 * r + g]);
    const float use = m == -INFINITY ? 0.f : m;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = dw_exp2(sink2 - use);
#pragma unroll 4
    for (int r = 0; r < S; ++r) {
      const float f = dw_exp2(ml[32 * r + g] - use);
      const float4 y = *reinterpret_cast<const float4*>(slices + 4 * (r * slice + i - x0));
      v.x += f * y.x; v.y += f * y.y; v.z += f * y.z; v.w += f * y.w;
      l += f * ml[32 * r + 16 + g];
    }
    float f = l > 0.f ? 1.f / l : l;             // nothing, or not a number
    if (p.s.gate) f *= 1.f / (1.f + __expf(-__bfloat162float(static_cast<const bf16*>(p.s.gate)[static_cast<size_t>(tok) * p.s.ldg + h0 + g])));
    *reinterpret_cast<uint2*>(out + g * dv + d) = make_uint2(dw_pack(v.x * f, v.y * f), dw_pack(v.z * f, v.w * f));
  }
  if (tid == 0) B200_TRACE(TK_ATTN_SPARSE, TP_EXIT);
  B200_TRACE_FLUSH(TK_ATTN_SPARSE);
}

// ---- launches ---------------------------------------------------------------------------------------------------------------------------------
template <auto Scores, auto Attend>
static int launch_sparse_pair(dim3 grid1, size_t smem1, size_t smem2, const SparseParams& p, cudaStream_t stream) {
  if (smem1 > SPARSE_MAX_SMEM || smem2 > SPARSE_MAX_SMEM) return -5;
  cudaError_t e = smem1 > (48u << 10) ? allow_smem<Scores>(static_cast<int>(SPARSE_MAX_SMEM)) : cudaSuccess;
  if (e == cudaSuccess) e = allow_smem<Attend>(static_cast<int>(SPARSE_MAX_SMEM));
  if (e != cudaSuccess) return -1000 - static_cast<int>(e);
  launch_ex(Scores, grid1, dim3(SC_THREADS), smem1, stream, 0, p);
  launch_ex(Attend, dim3(p.splits, p.c.kv_heads * p.hgroups, p.M), dim3(PS_THREADS), smem2, stream, p.splits, p);
  e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -2000 - static_cast<int>(e);
}

// scores stay in shared memory up to what a CTA has left; more are looked at where the first kernel left them
static void fit_scores(SparseParams& p, size_t floats) {
  const size_t used = 4 * (floats + p.list_cap + p.score_cap);
  const size_t room = used < SPARSE_MAX_SMEM ? (SPARSE_MAX_SMEM - used) / 4 : 0, most = (static_cast<size_t>(p.c.max_pages) + 3) & ~size_t(3);
  p.score_cap = static_cast<int>(most < room ? most : room & ~size_t(3));
}

template <typename T, bool VEC>
static int launch_sparse_any_as(SparseParams p, cudaStream_t stream) {
  const size_t wide = (static_cast<size_t>(p.c.dk) + 127) & ~size_t(127), pitch = ((static_cast<size_t>(p.c.dv) + 127) & ~size_t(127)) + 4;
  const size_t floats = (PS_WARPS * ASA_HEADS + 16) * pitch + 16 * wide;
  fit_scores(p, floats);
  const dim3 grid((p.c.max_pages + SCA_PAGES - 1) / SCA_PAGES, p.c.kv_heads, p.M);
  return launch_sparse_pair<page_scores_any_kernel<T, VEC>, attn_sparse_any_kernel<T, VEC>>(grid, 4 * static_cast<size_t>(p.hq / p.c.kv_heads) * wide,
                                                                                           4 * (floats + p.list_cap + p.score_cap), p, stream);
}

template <typename T>
static int launch_sparse_any(const SparseParams& p, cudaStream_t stream) {
  const bool vec = p.c.dk % 4 == 0 && p.c.dv % 4 == 0 && (reinterpret_cast<uintptr_t>(p.c.data) | reinterpret_cast<uintptr_t>(p.bounds)) % (4 * sizeof(T)) == 0;
  return vec ? launch_sparse_any_as<T, true>(p, stream) : launch_sparse_any_as<T, false>(p, stream);
}

template <int DK, int DV, int NH, bool FULL, int EACH>
static int launch_sparse_as(SparseParams p, cudaStream_t stream) {
  fit_scores(p, SparseShape<DV>::FLOATS);
  const dim3 grid((p.c.max_pages + EACH * SC_WARPS - 1) / (EACH * SC_WARPS), p.c.kv_heads, p.M);
  return launch_sparse_pair<page_scores_kernel<DK, NH, FULL, EACH>, attn_sparse_kernel<DK, DV, NH, FULL>>(
      grid, 0, 4 * (static_cast<size_t>(SparseShape<DV>::FLOATS) + p.score_cap + p.list_cap), p, stream);
}

// A warp scores 16 pages, in one step, or 32 where not all CTAs would run at once (one row behind 8,000 keys, 8 heads of 128: 13.1 us with 16, 14.0 with 32)
template <int DK, int DV, int NH, bool FULL>
static int launch_sparse(const SparseParams& p, cudaStream_t stream) {
  const long long ctas = static_cast<long long>((p.c.max_pages + 16 * SC_WARPS - 1) / (16 * SC_WARPS)) * p.c.kv_heads * p.M;
  return ctas <= SC_CTAS ? launch_sparse_as<DK, DV, NH, FULL, 16>(p, stream) : launch_sparse_as<DK, DV, NH, FULL, 32>(p, stream);
}

template <int DK, int DV, bool FULL>
static int launch_sparse_heads(const SparseParams& p, cudaStream_t stream) {
  return p.hq / p.c.kv_heads <= 8 ? launch_sparse<DK, DV, 1, FULL>(p, stream) : launch_sparse<DK, DV, 2, FULL>(p, stream);
}

}  // namespace b200

using namespace b200;

// Clusters of so many CTAs, one per SM, that run at once on the current device (which of a GPU's SMs make up a cluster depends on how many of them each part of it has);
// 0 where that cannot be told
extern "C" int b200_sparse_clusters(int size) {
  if (size < 1 || size > 8) return 0;
  if (allow_smem<attn_sparse_kernel<128, 128, 1, true>>(static_cast<int>(SPARSE_MAX_SMEM)) != cudaSuccess) return 0;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = size; attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size); cfg.blockDim = dim3(PS_THREADS); cfg.dynamicSmemBytes = SPARSE_MAX_SMEM; cfg.attrs = &attr; cfg.numAttrs = 1;
  int n = 0;
  return cudaOccupancyMaxActiveClusters(&n, attn_sparse_kernel<128, 128, 1, true>, &cfg) == cudaSuccess ? n : (static_cast<void>(cudaGetLastError()), 0);
}

extern "C" int b200_attn_paged_sparse(const void* q, long long ldq, void* out, long long ldo, int hq, int M, const int* positions, const int* seq_ids,
                                      const int* seq_lens, const b200_paged_cache* c, const void* bounds, const b200_attn_spec* s, int top, int first,
                                      int last, int splits, unsigned* scores, int* chosen, int* status, cudaStream_t stream) {
  if (M <= 0) return 0;
  if (!q || !out || !positions || !c || !c->data || !c->page_table || !bounds || !s || !scores) return -1;
  if (hq <= 0 || c->kv_heads <= 0 || hq % c->kv_heads || c->page_size <= 0 || c->dk <= 0 || c->dv <= 0 || c->dk > AS_MAX_D || c->dv > AS_MAX_D ||
      c->num_pages <= 0) return -2;
  if (first < 0 || last < 1 || top < first + last || splits < 1 || splits > 8 || M > 65535 || !(s->scale > 0.f)) return -3;
  SparseParams p = {};
  p.q = q; p.ldq = ldq; p.out = out; p.ldo = ldo; p.hq = hq; p.M = M; p.hgroups = (hq / c->kv_heads + 15) / 16;
  p.positions = positions; p.seq_ids = seq_ids; p.seq_lens = seq_lens; p.c = *c; p.s = *s; p.bounds = bounds; p.scores = scores;
  p.top = top; p.first = first; p.last = last; p.splits = splits; p.chosen = chosen; p.status = status;
  // pages of a row at most: those asked for, of those that it sees
  int read = top < c->max_pages ? top : c->max_pages;
  if (s->chunk > 0 && s->chunk / c->page_size + 2 < read) read = s->chunk / c->page_size + 2;
  p.list_cap = ((read + splits - 1) / splits + 1 + 3) & ~3;
  if (static_cast<long long>(c->kv_heads) * p.hgroups > 65535) return -3;
  if (c->f32) return launch_sparse_any<float>(p, stream);
  if (c->page_size != 16 || c->dk > 128 || c->dv > 128 || c->dk % 8 || c->dv % 8 || ldq % 8 || ldo % 4 || (reinterpret_cast<uintptr_t>(q) & 15) ||
      (reinterpret_cast<uintptr_t>(out) & 7) || (reinterpret_cast<uintptr_t>(c->data) & 15) || (reinterpret_cast<uintptr_t>(bounds) & 15))
    return launch_sparse_any<__nv_bfloat16>(p, stream);
  const int d = c->dk > c->dv ? c->dk : c->dv;
  if (c->dk == 64 && c->dv == 64) return launch_sparse_heads<64, 64, true>(p, stream);
  if (c->dk == 128 && c->dv == 128) return launch_sparse_heads<128, 128, true>(p, stream);
  if (d <= 64) return launch_sparse_heads<64, 64, false>(p, stream);
  return launch_sparse_heads<128, 128, false>(p, stream);
}

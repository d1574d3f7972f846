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
// This form takes any head size up to 512, bf16 or fp32: a warp per page, lanes along the dimensions.
#include "ptx.cuh"
#include "api.h"
#include "launch.cuh"
#include "page_select.cuh"
#include "attn_sparse.cuh"

namespace b200 {

__device__ __forceinline__ float as_f(float v) { return v; }
__device__ __forceinline__ float as_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_max(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

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
  return c->f32 ? launch_sparse_any<float>(p, stream) : launch_sparse_any<__nv_bfloat16>(p, stream);
}

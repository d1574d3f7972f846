// Records of a paged cache as such: copies from page to page in all layers at once, and the bounds of the keys of a page.
//
// copy_pages: y[dst_i] = y[src_i] for every array y of records.  The page numbers come from the host, which has handed the pages out,
// and travel in the kernel's parameters: no copy to the device in front of the launch, no look-up behind a load.  Bound by the bytes, read once and
// written once; a CTA takes 16 KiB of one record, four loads of 16 bytes per thread in flight.
//
// page_bounds: lo[d] = min_t k[t][d], hi[d] = max_t k[t][d] over the tokens of a page that a sequence has, per KV head.  Both are values of the
// keys' own type, so nothing is rounded.  A warp takes one head of one page; lanes lie along the row of 16-byte pieces and, where a row has fewer
// than 32 of them, along the tokens.
#include "ptx.cuh"
#include "api.h"
#include "launch.cuh"

namespace b200 {

constexpr int CP_THREADS = 256, CP_PER_THREAD = 4, CP_CHUNK = CP_THREADS * CP_PER_THREAD;      // in units of 16 bytes
constexpr int CP_ARRAYS = 64;

// a kernel's parameters may be 32,764 bytes; few pages, the common case, travel in few
template <int PAIRS>
struct CopyPagesParams {
  uint4* base[CP_ARRAYS];
  unsigned record[CP_ARRAYS];            // in units of 16 bytes
  int src[PAIRS], dst[PAIRS];
};

template <int PAIRS>
__global__ void __launch_bounds__(CP_THREADS) copy_pages_kernel(const __grid_constant__ CopyPagesParams<PAIRS> p) {
  pdl_launch_dependents();
  const unsigned record = p.record[blockIdx.y], at = blockIdx.x * CP_CHUNK + threadIdx.x;
  if (blockIdx.x * CP_CHUNK >= record) return;
  uint4* base = p.base[blockIdx.y];
  const uint4* from = base + static_cast<size_t>(p.src[blockIdx.z]) * record;
  uint4* to = base + static_cast<size_t>(p.dst[blockIdx.z]) * record;
  pdl_wait();
  uint4 v[CP_PER_THREAD];
#pragma unroll
  for (int i = 0; i < CP_PER_THREAD; ++i)
    if (at + i * CP_THREADS < record) v[i] = from[at + i * CP_THREADS];
#pragma unroll
  for (int i = 0; i < CP_PER_THREAD; ++i)
    if (at + i * CP_THREADS < record) to[at + i * CP_THREADS] = v[i];
}

template <int PAIRS>
static int copy_pages_some(void* const* arrays, const long long* records, int n_arrays, const int* src, const int* dst, int n, cudaStream_t stream) {
  CopyPagesParams<PAIRS> p;
  unsigned longest = 0;
  for (int i = 0; i < n_arrays; ++i) {
    p.base[i] = static_cast<uint4*>(arrays[i]);
    p.record[i] = static_cast<unsigned>(records[i] >> 4);
    if (p.record[i] > longest) longest = p.record[i];
  }
  for (int i = 0; i < n; ++i) { p.src[i] = src[i]; p.dst[i] = dst[i]; }
  launch_ex(copy_pages_kernel<PAIRS>, dim3((longest + CP_CHUNK - 1) / CP_CHUNK, n_arrays, n), dim3(CP_THREADS), 0, stream, 0, p);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -2000 - static_cast<int>(e);
}

// ---- bounds ------------------------------------------------------------------------------------------------------------------
constexpr int PB_WARPS = 8;

struct PageBoundsParams {
  b200_paged_cache c;
  const int* starts; const int* ends; const int* seq_ids;
  void* out;                             // [pages][kv_heads][2][dk]
  int* status;
};

// the smaller and the larger of two, NaN where one of them is: a page with a key that is not a number is not left out
__device__ __forceinline__ float pb_min(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float pb_max(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
template <typename T> struct PbVec;
template <> struct PbVec<float> {
  static __device__ void first(float (&x)[4], uint4 r) { x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w); }
};
template <> struct PbVec<__nv_bfloat16> {
  static __device__ void first(float (&x)[8], uint4 r) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
};
__device__ __forceinline__ float pb_f(float v) { return v; }
__device__ __forceinline__ float pb_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void pb_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void pb_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }      // exact: the value is one of the keys'

// VEC: rows are whole pieces of 16 bytes
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * PB_WARPS) page_bounds_kernel(const __grid_constant__ PageBoundsParams p) {
  constexpr int N = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, b = blockIdx.y, ps = p.c.page_size, dk = p.c.dk;
  const int unit = blockIdx.x * PB_WARPS + (threadIdx.x >> 5), at = unit / p.c.kv_heads, h = unit - at * p.c.kv_heads;
  const int start = p.starts[b], end = p.ends[b], seq = p.seq_ids ? p.seq_ids[b] : b;
  if (end <= start) return;
  if (start < 0 || seq < 0 || seq >= p.c.num_seqs || (end - 1) / ps >= p.c.max_pages) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && p.status) atomicCAS(p.status, 0, static_cast<int>(ST_BAD_ARGUMENT) | (24 << 8));
    return;
  }
  const int place = start / ps + at;
  if (place > (end - 1) / ps) return;
  const int page = p.c.page_table[static_cast<size_t>(seq) * p.c.max_pages + place];
  if (page < 0 || page >= p.c.num_pages) {
    if (lane == 0 && p.status) atomicCAS(p.status, 0, static_cast<int>(ST_BAD_ARGUMENT) | (24 << 8));
    return;
  }
  const int rows = min(ps, end - place * ps), pieces = dk / N;
  const T* k = static_cast<const T*>(p.c.data) + static_cast<size_t>(page) * p.c.kv_heads * ps * (dk + p.c.dv) + static_cast<size_t>(h) * ps * dk;
  T* lo = static_cast<T*>(p.out) + (static_cast<size_t>(page) * p.c.kv_heads + h) * 2 * dk;
  // lanes along a row: the least power of two that holds it, at most the warp; the others take other rows
  int wide = 1;
  while (wide < pieces && wide < 32) wide *= 2;
  const int col = lane & (wide - 1), r0 = lane / wide, step = 32 / wide;
  for (int c0 = 0; c0 < pieces; c0 += wide) {
    const int c = c0 + col;
    float mn[N], mx[N];
#pragma unroll
    for (int i = 0; i < N; ++i) { mn[i] = INFINITY; mx[i] = -INFINITY; }
    if (c < pieces) {
#pragma unroll 8
      for (int r = r0; r < rows; r += step) {
        float x[N];
        if constexpr (VEC) PbVec<T>::first(x, *reinterpret_cast<const uint4*>(k + static_cast<size_t>(r) * dk + c * N));
        else x[0] = pb_f(k[static_cast<size_t>(r) * dk + c]);
#pragma unroll
        for (int i = 0; i < N; ++i) { mn[i] = pb_min(mn[i], x[i]); mx[i] = pb_max(mx[i], x[i]); }
      }
    }
    for (int o = wide; o < 32; o *= 2) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        mn[i] = pb_min(mn[i], __shfl_xor_sync(0xffffffffu, mn[i], o));
        mx[i] = pb_max(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
      }
    }
    if (c < pieces && r0 == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) { pb_put(lo + c * N + i, mn[i]); pb_put(lo + dk + c * N + i, mx[i]); }
    }
  }
}

template <typename T, bool VEC>
static int launch_page_bounds(const PageBoundsParams& p, dim3 grid, cudaStream_t stream) {
  launch_ex(page_bounds_kernel<T, VEC>, grid, dim3(32 * PB_WARPS), 0, stream, 0, p);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -2000 - static_cast<int>(e);
}

}  // namespace b200

using namespace b200;

extern "C" int b200_copy_pages(void* const* arrays, const long long* records, int n_arrays, const int* src, const int* dst, int n, cudaStream_t stream) {
  if (n_arrays <= 0 || n <= 0) return 0;
  if (!arrays || !records || !src || !dst) return -1;
  for (int i = 0; i < n_arrays; ++i) {
    if (!arrays[i] || (reinterpret_cast<uintptr_t>(arrays[i]) & 15)) return -4;
    if (records[i] <= 0 || (records[i] & 15) || records[i] > (1ll << 31)) return -2;
  }
  for (int i = 0; i < n; ++i) if (src[i] < 0 || dst[i] < 0) return -3;
  constexpr int FEW = 64, MANY = 3900;
  for (int a = 0; a < n_arrays; a += CP_ARRAYS)
    for (int i = 0; i < n; i += MANY) {
      const int na = n_arrays - a < CP_ARRAYS ? n_arrays - a : CP_ARRAYS, ni = n - i < MANY ? n - i : MANY;
      const int rc = ni <= FEW ? copy_pages_some<FEW>(arrays + a, records + a, na, src + i, dst + i, ni, stream)
                               : copy_pages_some<MANY>(arrays + a, records + a, na, src + i, dst + i, ni, stream);
      if (rc) return rc;
    }
  return 0;
}

extern "C" int b200_page_bounds(const b200_paged_cache* c, const int* starts, const int* ends, const int* seq_ids, int portions, int max_tokens, void* out,
                                int* status, cudaStream_t stream) {
  if (portions <= 0 || max_tokens <= 0) return 0;
  if (!c || !c->data || !c->page_table || !starts || !ends || !out) return -1;
  if (c->kv_heads <= 0 || c->dk <= 0 || c->dv < 0 || c->page_size <= 0 || c->num_pages <= 0 || portions > 65535) return -2;
  PageBoundsParams p{*c, starts, ends, seq_ids, out, status};
  const long long pages = (static_cast<long long>(max_tokens) + 2 * c->page_size - 2) / c->page_size;
  const long long most = pages < c->max_pages ? pages : c->max_pages;
  const dim3 grid(static_cast<unsigned>((most * c->kv_heads + PB_WARPS - 1) / PB_WARPS), portions);
  const size_t size = c->f32 ? 4 : 2;
  const bool vec = c->dk * size % 16 == 0 && static_cast<size_t>(c->kv_heads) * c->page_size * (c->dk + c->dv) * size % 16 == 0 &&
                   (reinterpret_cast<uintptr_t>(c->data) & 15) == 0;
  if (c->f32) return vec ? launch_page_bounds<float, true>(p, grid, stream) : launch_page_bounds<float, false>(p, grid, stream);
  return vec ? launch_page_bounds<__nv_bfloat16, true>(p, grid, stream) : launch_page_bounds<__nv_bfloat16, false>(p, grid, stream);
}

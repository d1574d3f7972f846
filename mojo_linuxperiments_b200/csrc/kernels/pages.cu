// Records of a paged cache as such: copies from page to page in all layers at once, and the bounds of the keys of a page.
//
// copy_pages: y[dst_i] = y[src_i] for every array y of records.  The page numbers come from the host, which has handed the pages out,
// and travel in the kernel's parameters: no copy to the device in front of the launch, no look-up behind a load.  Bound by the bytes, read once and
// written once; a CTA takes 16 KiB of one record, four loads of 16 bytes per thread in flight.  1,500 pages in each of 16 layers, 3.1 GB, take 482 us, 6.5 TB/s,
// the rate of a plain copy; one page in each of 32 layers 1.6 us.
//
// page_bounds: lo[d] = min_t k[t][d], hi[d] = max_t k[t][d] over the tokens of a page that a sequence has, per KV head.  Both are values of the
// keys' own type, so nothing is rounded.  Bound by the bytes of the keys.  A CTA takes some pages, whose numbers it looks up at once, and a warp one head of one of
// them after the other; lanes lie along the row of 16-byte pieces and, where a row has fewer than 32 of them, along the tokens.
// 382 MB of prompts take 62 us (6.1 TB/s), the pages of a step's tokens 2.6 us.
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
constexpr int PB_WARPS = 8, PB_MOST = 32, PB_UNITS = 6, PB_CTAS = 592;

struct PageBoundsParams {
  b200_paged_cache c;
  const int* starts; const int* ends; const int* seq_ids;
  void* out;                             // [pages][kv_heads][2][dk]
  int each;                              // pages of a CTA
  int* status;
};

// The smaller and the larger of two (of two pairs, in bf16), NaN where one of them is: a page with a key that is not a number is not left out.  All on the words that
// a row is read in: nothing is converted.
template <typename T> struct PbWord;
template <> struct PbWord<float> {
  using W = uint32_t;
  static constexpr uint32_t MOST = 0x7f800000u, LEAST = 0xff800000u;
  static __device__ __forceinline__ uint32_t lesser(uint32_t a, uint32_t b) { uint32_t r; asm("min.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { uint32_t r; asm("max.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
};
template <> struct PbWord<__nv_bfloat16> {
  using W = uint16_t;
  static constexpr uint32_t MOST = 0x7f807f80u, LEAST = 0xff80ff80u;
  static __device__ __forceinline__ uint32_t lesser(uint32_t a, uint32_t b) { uint32_t r; asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { uint32_t r; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
};

// VEC: rows are whole pieces of 16 bytes; otherwise a piece is one element
template <typename T, bool VEC>
__global__ void __launch_bounds__(32 * PB_WARPS) page_bounds_kernel(const __grid_constant__ PageBoundsParams p) {
  using P = PbWord<T>;
  constexpr int N = VEC ? 16 / static_cast<int>(sizeof(T)) : 1, WORDS = VEC ? 4 : 1, BATCH = 8;
  pdl_launch_dependents();
  pdl_wait();
  __shared__ int ids[PB_MOST];
  const int lane = threadIdx.x & 31, b = blockIdx.y, ps = p.c.page_size, dk = p.c.dk;
  const int start = p.starts[b], end = p.ends[b], seq = p.seq_ids ? p.seq_ids[b] : b;
  if (end <= start) return;
  const int last = (end - 1) / ps;
  if (start < 0 || seq < 0 || seq >= p.c.num_seqs || last >= p.c.max_pages || last - start / ps >= static_cast<int>(gridDim.x) * p.each) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && p.status) atomicCAS(p.status, 0, static_cast<int>(ST_BAD_ARGUMENT) | (24 << 8));
    return;
  }
  const int place0 = start / ps + blockIdx.x * p.each, pages = min(p.each, last + 1 - place0);
  if (pages <= 0) return;
  if (static_cast<int>(threadIdx.x) < pages) {
    const int page = p.c.page_table[static_cast<size_t>(seq) * p.c.max_pages + place0 + threadIdx.x];
    const bool there = page >= 0 && page < p.c.num_pages;
    if (!there && p.status) atomicCAS(p.status, 0, static_cast<int>(ST_BAD_ARGUMENT) | (24 << 8));
    ids[threadIdx.x] = there ? page : -1;
  }
  __syncthreads();
  const int pieces = dk / N;
  // lanes along a row: the least power of two that holds it, at most the warp; the others take other rows
  int wide = 1;
  while (wide < pieces && wide < 32) wide *= 2;
  const int col = lane & (wide - 1), r0 = lane / wide, step = 32 / wide;
  for (int unit = threadIdx.x >> 5; unit < pages * p.c.kv_heads; unit += PB_WARPS) {
    const int at = unit / p.c.kv_heads, h = unit - at * p.c.kv_heads, page = ids[at], rows = min(ps, end - (place0 + at) * ps);
    if (page < 0) continue;
    const T* k = static_cast<const T*>(p.c.data) + static_cast<size_t>(page) * p.c.kv_heads * ps * (dk + p.c.dv) + static_cast<size_t>(h) * ps * dk;
    T* lo = static_cast<T*>(p.out) + (static_cast<size_t>(page) * p.c.kv_heads + h) * 2 * dk;
    for (int c0 = 0; c0 < pieces; c0 += wide) {
      const int c = c0 + col;
      uint32_t mn[WORDS], mx[WORDS];
#pragma unroll
      for (int i = 0; i < WORDS; ++i) { mn[i] = P::MOST; mx[i] = P::LEAST; }
      if (c < pieces)
        for (int r1 = r0; r1 < rows; r1 += BATCH * step) {
          uint32_t x[BATCH][WORDS];
#pragma unroll
          for (int j = 0; j < BATCH; ++j) {
            // rows behind the end: the first of the batch once more, which changes nothing
            const T* at_row = k + static_cast<size_t>(r1 + j * step < rows ? r1 + j * step : r1) * dk + c * N;
            if constexpr (VEC) {
              const uint4 v = __ldcg(reinterpret_cast<const uint4*>(at_row));
              x[j][0] = v.x; x[j][1] = v.y; x[j][2] = v.z; x[j][3] = v.w;
            } else {
              const typename P::W w = *reinterpret_cast<const typename P::W*>(at_row);
              x[j][0] = sizeof(T) == 2 ? w * 0x10001u : w;
            }
          }
#pragma unroll
          for (int j = 0; j < BATCH; ++j)
#pragma unroll
            for (int i = 0; i < WORDS; ++i) { mn[i] = P::lesser(mn[i], x[j][i]); mx[i] = P::larger(mx[i], x[j][i]); }
        }
      for (int o = wide; o < 32; o *= 2) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
          mn[i] = P::lesser(mn[i], __shfl_xor_sync(0xffffffffu, mn[i], o));
          mx[i] = P::larger(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
        }
      }
      if (c < pieces && r0 == 0) {
        if constexpr (VEC) {
          *reinterpret_cast<uint4*>(lo + c * N) = make_uint4(mn[0], mn[1], mn[2], mn[3]);
          *reinterpret_cast<uint4*>(lo + dk + c * N) = make_uint4(mx[0], mx[1], mx[2], mx[3]);
        } else {
          *reinterpret_cast<typename P::W*>(lo + c) = static_cast<typename P::W>(mn[0]);
          *reinterpret_cast<typename P::W*>(lo + dk + c) = static_cast<typename P::W>(mx[0]);
        }
      }
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
  const long long pages = (static_cast<long long>(max_tokens) + 2 * c->page_size - 2) / c->page_size;
  const long long most = pages < c->max_pages ? pages : c->max_pages;
  // Pages of a CTA: so many that a warp has six heads, one after the other, and no more than leave four CTAs per SM (8 heads of 128, 240,000 tokens: 62 us with 6
  // pages, 68 with 8; 8 heads of 64, 32,000 tokens: 8.5 us with 3 pages, 16 with 8; one head, 144,000 tokens: 10.6 with 3, 7.1 with 8)
  const long long heads = PB_UNITS * PB_WARPS / c->kv_heads, share = most * portions / PB_CTAS, each = heads < share ? heads : share;
  PageBoundsParams p{*c, starts, ends, seq_ids, out, static_cast<int>(each < 1 ? 1 : each > PB_MOST ? PB_MOST : each), status};
  const dim3 grid(static_cast<unsigned>((most + p.each - 1) / p.each), portions);
  const size_t size = c->f32 ? 4 : 2;
  const bool vec = c->dk * size % 16 == 0 && static_cast<size_t>(c->kv_heads) * c->page_size * (c->dk + c->dv) * size % 16 == 0 &&
                   ((reinterpret_cast<uintptr_t>(c->data) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  if (c->f32) return vec ? launch_page_bounds<float, true>(p, grid, stream) : launch_page_bounds<float, false>(p, grid, stream);
  return vec ? launch_page_bounds<__nv_bfloat16, true>(p, grid, stream) : launch_page_bounds<__nv_bfloat16, false>(p, grid, stream);
}

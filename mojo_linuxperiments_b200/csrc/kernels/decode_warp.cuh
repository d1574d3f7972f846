// Attention of up to 8 or 16 query rows (the heads of a KV head) of one token over pages of 16 keys, by one warp: m16n8k16 MMAs in bf16 with fp32 sums.
//
// Decoding reads every key and value once, so the pages go straight from memory into the registers that the MMAs read, with no stop in shared memory.  The
// keys of a page are the 16 rows of the first product, S^T = K Q^T, and the dimensions of the values those of the second, O^T = V^T P^T, so that
// eight heads fill the eight columns.  The order of the dimensions inside a dot product is free: a lane takes eight neighbouring ones of a key, 16 bytes, as
// its share of two MMA steps (the queries are read in the same order).  Of the values a lane takes eight neighbouring dimensions of four keys and pairs
// them up key by key; P^T is P through two 8 x 8 transpositions in registers.
//
// The next page's keys are requested into the same registers as soon as the scores are issued, its values after the last MMA: 8 KiB on the way per warp of heads
// of 128, 96 KiB per SM with twelve warps, where 45 KiB are the full rate of the memory.  (Two pages in registers, one on its way while the other is used, or two in a
// ring in shared memory, brought by bulk copies: no faster.)  128 sequences with 500 own keys each, 8 heads of 128, take 54 us for 267 MB behind their prefix: 4.9 TB/s, with the waits for
// places and the joins in it.
#pragma once
#include "ptx.cuh"

namespace b200 {

constexpr float DW_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ void dw_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t dw_transpose(uint32_t x) {      // 8 x 8 of 16 bits, row lane / 4, columns 2 (lane & 3) and the next
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint4 dw_load(const __nv_bfloat16* p, bool on) {
  return on ? __ldcg(reinterpret_cast<const uint4*>(p)) : make_uint4(0u, 0u, 0u, 0u);
}
__device__ __forceinline__ float dw_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float dw_ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t dw_pack(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// heads lane / 4 and lane / 4 + 8 in the order that the keys are read in
template <int DK, int NH>
struct DwQuery {
  uint4 h[NH][DK / 32];
  // q: first of G rows, dk apart; rows beyond are zero
  __device__ __forceinline__ void load(const __nv_bfloat16* q, int G, int dk) {
    const int lane = threadIdx.x & 31, d = (lane & 3) * 8;
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int c = 0; c < DK / 32; ++c) {
        const int r = (lane >> 2) + 8 * n;
        h[n][c] = dw_load(q + static_cast<size_t>(r) * dk + c * 32 + d, c * 32 + d < dk && r < G);
      }
  }
};

// where a page is and which of its keys count
struct DwPage { const __nv_bfloat16* k; const __nv_bfloat16* v; int lo, hi; };      // lo >= hi: none

template <int DK, int DV, int NH, bool FULL>
struct DecodeWarp {
  DwQuery<DK, NH> q;
  float o[NH][DV / 64][4][4];            // dimensions 64 c + 8 (lane / 4) + 2 j and the next of heads 2 (lane & 3) and the next
  float m[NH][2], l[NH][2];              // of the same heads, in powers of two; l: this lane's share
  float scale_log2;
  int dk, dv;
  struct Held { uint4 k[2][DK / 32], v[DV / 64][4]; int lo, hi; };

  __device__ __forceinline__ void begin(int dk_, int dv_, float scale) {
    dk = FULL ? DK : dk_; dv = FULL ? DV : dv_; scale_log2 = scale * DW_LOG2E;
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      m[n][0] = m[n][1] = -INFINITY; l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int c = 0; c < DV / 64; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[n][c][j][i] = 0.f;
    }
  }
  // A page that is not there (lo >= hi) has addresses of one that is: what is read is not used.
  __device__ __forceinline__ void load_k(Held& p, const DwPage& at) const {
    const int lane = threadIdx.x & 31, d = (lane & 3) * 8;
    const __nv_bfloat16* k = at.k + (lane >> 2) * dk + d;
#pragma unroll
    for (int c = 0; c < DK / 32; ++c) {
      p.k[0][c] = dw_load(k + c * 32, FULL || c * 32 + d < dk);
      p.k[1][c] = dw_load(k + 8 * dk + c * 32, FULL || c * 32 + d < dk);
    }
  }
  __device__ __forceinline__ void load_v(Held& p, const DwPage& at) const {
    const int lane = threadIdx.x & 31, d = (lane >> 2) * 8;
    const __nv_bfloat16* v = at.v + 2 * (lane & 3) * dv + d;
#pragma unroll
    for (int c = 0; c < DV / 64; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) p.v[c][i] = dw_load(v + ((i & 1) + (i >> 1) * 8) * dv + c * 64, FULL || c * 64 + d < dv);
    p.lo = at.lo;
    p.hi = at.hi;
  }
  // one page; then, if there is one, the page `next` is requested into the same registers
  template <typename Next>
  __device__ __forceinline__ void step(Held& p, bool more, Next&& next) {
    const int lane = threadIdx.x & 31, g = lane >> 2;
    float s[NH][4];                      // keys g, g, g + 8, g + 8 of heads 2 t, 2 t + 1
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
#pragma unroll
    for (int c = 0; c < DK / 32; ++c)
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        dw_mma(s[n], p.k[0][c].x, p.k[1][c].x, p.k[0][c].y, p.k[1][c].y, q.h[n][c].x, q.h[n][c].y);
        dw_mma(s[n], p.k[0][c].z, p.k[1][c].z, p.k[0][c].w, p.k[1][c].w, q.h[n][c].z, q.h[n][c].w);
      }
    const int lo = p.lo, hi = p.hi;
    DwPage at;
    if (more) { at = next(); load_k(p, at); }
    if (lo < hi) {
      const bool on0 = g >= lo && g < hi, on1 = g + 8 >= lo && g + 8 < hi;
      uint32_t b[NH][2];
      bool grows = false;
      float a[NH][2];
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float x = on0 ? s[n][i] * scale_log2 : -INFINITY, y = on1 ? s[n][2 + i] * scale_log2 : -INFINITY;
          float top = fmaxf(x, y);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const float mn = fmaxf(m[n][i], top), use = mn == -INFINITY ? 0.f : mn;
          a[n][i] = dw_exp2(m[n][i] - use);
          grows = grows || a[n][i] != 1.f;
          m[n][i] = mn;
          e[i] = dw_exp2(x - use);
          e[2 + i] = dw_exp2(y - use);
        }
        // rounded to bf16 for the MMA; the denominator adds what the MMA sees
        const uint32_t p0 = dw_pack(e[0], e[1]), p1 = dw_pack(e[2], e[3]);
        l[n][0] = l[n][0] * a[n][0] + (__uint_as_float(p0 << 16) + __uint_as_float(p1 << 16));
        l[n][1] = l[n][1] * a[n][1] + (__uint_as_float(p0 & 0xffff0000u) + __uint_as_float(p1 & 0xffff0000u));
        b[n][0] = dw_transpose(p0);
        b[n][1] = dw_transpose(p1);
      }
      if (lo > 0 || hi < 16) {                   // rows outside may hold anything: a weight of zero must not meet a NaN
        const int t = 2 * (lane & 3);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = t + (i & 1) + (i >> 1) * 8;
          if (r < lo || r >= hi) {
#pragma unroll
            for (int c = 0; c < DV / 64; ++c) p.v[c][i] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
      }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int c = 0; c < DV / 64; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) { o[n][c][j][0] *= a[n][0]; o[n][c][j][1] *= a[n][1]; o[n][c][j][2] *= a[n][0]; o[n][c][j][3] *= a[n][1]; }
      }
#pragma unroll
      for (int c = 0; c < DV / 64; ++c) {
        const uint32_t w[4][4] = {{p.v[c][0].x, p.v[c][0].y, p.v[c][0].z, p.v[c][0].w}, {p.v[c][1].x, p.v[c][1].y, p.v[c][1].z, p.v[c][1].w},
                                  {p.v[c][2].x, p.v[c][2].y, p.v[c][2].z, p.v[c][2].w}, {p.v[c][3].x, p.v[c][3].y, p.v[c][3].z, p.v[c][3].w}};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a0 = __byte_perm(w[0][j], w[1][j], 0x5410), a1 = __byte_perm(w[0][j], w[1][j], 0x7632);
          const uint32_t a2 = __byte_perm(w[2][j], w[3][j], 0x5410), a3 = __byte_perm(w[2][j], w[3][j], 0x7632);
#pragma unroll
          for (int n = 0; n < NH; ++n) dw_mma(o[n][c][j], a0, a1, a2, a3, b[n][0], b[n][1]);
        }
      }
    }
    if (more) load_v(p, at);
  }
  // pages 0 .. n - 1; page(i) is asked for in this order.  start() runs once the first requests are out.
  template <typename Page, typename Start>
  __device__ __forceinline__ void walk(int n, Page&& page, Start&& start) {
    if (n <= 0) return;
    Held x;
    DwPage at = page(0);
    load_k(x, at);
    load_v(x, at);
    start();
    for (int i = 0; i < n; ++i) step(x, i + 1 < n, [&] { return page(i + 1); });
  }
  // O and (m, l) of the first G heads to shared memory, rows `pitch` floats apart: [16][pitch], then m [16], l [16]
  __device__ __forceinline__ void put(float* to, int pitch, int G) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[n][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int h = 8 * n + 2 * t + e;
        if (h < G) {
          if (g == 0) { to[16 * pitch + h] = m[n][e]; to[16 * pitch + 16 + h] = sum; }
#pragma unroll
          for (int c = 0; c < DV / 64; ++c) {
            const int d = c * 64 + 8 * g;
            if (FULL || d < dv) {
              float4* row = reinterpret_cast<float4*>(to + h * pitch + d);
              row[0] = make_float4(o[n][c][0][e], o[n][c][0][2 + e], o[n][c][1][e], o[n][c][1][2 + e]);
              row[1] = make_float4(o[n][c][2][e], o[n][c][2][2 + e], o[n][c][3][e], o[n][c][3][2 + e]);
            }
          }
        }
      }
  }
};

// The lane's page (if it is one) is asked for into L2: pages lie anywhere, and the first access to one takes more than a microsecond
__device__ __forceinline__ void dw_prefetch(const __nv_bfloat16* kbase, const __nv_bfloat16* vbase, int page, size_t rec, int dk, int dv, int num_pages) {
  if (page < 0 || page >= num_pages) return;
  bulk_prefetch_l2(kbase + page * rec, 32 * dk);
  bulk_prefetch_l2(vbase + page * rec, 32 * dv);
}

// Parts of several warps, as put() leaves them `size` floats apart, joined into `to` by all threads (THREADS of them), four dimensions each
template <int WARPS, int THREADS>
__device__ __forceinline__ void dw_join(const float* parts, int size, int pitch, int G, int dv, float* to) {
  const int quads = dv >> 2;
  for (int i = threadIdx.x; i < G * quads; i += THREADS) {
    const int g = i / quads, d = (i - g * quads) * 4;
    float mw[WARPS], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) { mw[w] = parts[w * size + 16 * pitch + g]; m = fmaxf(m, mw[w]); }
    const float use = m == -INFINITY ? 0.f : m;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {            // a warp without pages has left zeros
      const float f = dw_exp2(mw[w] - use);
      const float4 x = *reinterpret_cast<const float4*>(parts + w * size + g * pitch + d);
      v.x += f * x.x; v.y += f * x.y; v.z += f * x.z; v.w += f * x.w;
      l += f * parts[w * size + 16 * pitch + 16 + g];
    }
    *reinterpret_cast<float4*>(to + g * pitch + d) = v;
    if (d == 0) { to[16 * pitch + g] = m; to[16 * pitch + 16 + g] = l; }
  }
}

// four numbers of shared memory of CTA r of the cluster, if there is one (addr: this CTA's address of the same place)
__device__ __forceinline__ float4 dw_ld_cluster4(uint32_t addr, int r, bool cluster) {
  const uint32_t a = cluster ? mapa_shared(addr, r) : addr;
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

}  // namespace b200

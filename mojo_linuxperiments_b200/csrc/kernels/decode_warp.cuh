// Attention of up to 16 query rows (the heads of a KV head) of one token over pages of 16 keys, by one warp: m16n8k16 MMAs in bf16 with fp32 sums.
//
// Decoding reads every key and value once, so the pages go straight from memory into the registers that the MMAs read, with no stop in shared memory: the
// order of the dimensions inside a dot product is free, and a lane takes eight neighbouring ones of a key, 16 bytes, as its share of two MMA steps
// (the queries are read in the same order); of the values a lane takes eight neighbouring dimensions of four keys and pairs them up key by key.  The keys of
// the next page are requested as soon as the scores of this one are issued, its values after the last MMA of this one: up to 8 KiB per warp are on
// their way at any time, 64 KiB per SM with eight warps, where 45 are in flight at the full rate of the memory.
#pragma once
#include "ptx.cuh"

namespace b200 {

constexpr float DW_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ void dw_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// the queries' rows lane / 4 and lane / 4 + 8 in the order that the keys are read in
template <int DK>
struct DwQuery {
  uint4 lo[DK / 32], hi[DK / 32];
  // q: first of G rows, dk apart; rows beyond are zero
  __device__ __forceinline__ void load(const __nv_bfloat16* q, int G, int dk) {
    const int lane = threadIdx.x & 31, r = lane >> 2, d = (lane & 3) * 8;
#pragma unroll
    for (int c = 0; c < DK / 32; ++c) {
      const bool in = c * 32 + d < dk;
      lo[c] = dw_load(q + static_cast<size_t>(r) * dk + c * 32 + d, in && r < G);
      hi[c] = dw_load(q + static_cast<size_t>(r + 8) * dk + c * 32 + d, in && r + 8 < G);
    }
  }
};

template <int DK, int DV, bool FULL>
struct DecodeWarp {
  DwQuery<DK> q;
  uint4 k[2][DK / 32], v[DV / 64][4];
  float o[DV / 64][8][4];
  float m0, m1, l0, l1;                  // of rows lane / 4 and lane / 4 + 8, in powers of two
  float scale_log2;
  int dk, dv;

  __device__ __forceinline__ void begin(int dk_, int dv_, float scale) {
    dk = FULL ? DK : dk_; dv = FULL ? DV : dv_; scale_log2 = scale * DW_LOG2E;
    m0 = m1 = -INFINITY; l0 = l1 = 0.f;
#pragma unroll
    for (int c = 0; c < DV / 64; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[c][j][i] = 0.f;
  }
  __device__ __forceinline__ void load_k(const __nv_bfloat16* kp, bool on) {
    const int lane = threadIdx.x & 31, r = lane >> 2, d = (lane & 3) * 8;
#pragma unroll
    for (int c = 0; c < DK / 32; ++c) {
      const bool in = on && (FULL || c * 32 + d < dk);
      k[0][c] = dw_load(kp + r * dk + c * 32 + d, in);
      k[1][c] = dw_load(kp + (r + 8) * dk + c * 32 + d, in);
    }
  }
  // rows outside [lo, hi) may hold anything: a weight of zero must not meet a NaN
  __device__ __forceinline__ void load_v(const __nv_bfloat16* vp, int lo, int hi) {
    const int lane = threadIdx.x & 31, d = (lane >> 2) * 8, t = 2 * (lane & 3);
#pragma unroll
    for (int c = 0; c < DV / 64; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = t + (i & 1) + (i >> 1) * 8;
        v[c][i] = dw_load(vp + r * dv + c * 64 + d, (FULL || c * 64 + d < dv) && r >= lo && r < hi);
      }
  }
  __device__ __forceinline__ void scores(float (&s)[2][4]) const {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
#pragma unroll
      for (int c = 0; c < DK / 32; ++c) {
        dw_mma(s[n], q.lo[c].x, q.hi[c].x, q.lo[c].y, q.hi[c].y, k[n][c].x, k[n][c].y);
        dw_mma(s[n], q.lo[c].z, q.hi[c].z, q.lo[c].w, q.hi[c].w, k[n][c].z, k[n][c].w);
      }
    }
  }
  // keys [lo, hi) of the page count, at least one
  __device__ __forceinline__ void weigh(float (&s)[2][4], int lo, int hi, uint32_t (&p)[4]) {
    const int t = 2 * (threadIdx.x & 3);
    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int key = n * 8 + t + e;
        const bool on = key >= lo && key < hi;
        s[n][e] = on ? s[n][e] * scale_log2 : -INFINITY;
        s[n][2 + e] = on ? s[n][2 + e] * scale_log2 : -INFINITY;
        x0 = fmaxf(x0, s[n][e]);
        x1 = fmaxf(x1, s[n][2 + e]);
      }
    x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1)); x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
    x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1)); x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
    const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
    const float u0 = n0 == -INFINITY ? 0.f : n0, u1 = n1 == -INFINITY ? 0.f : n1;
    const float a0 = dw_exp2(m0 - u0), a1 = dw_exp2(m1 - u1);
    m0 = n0; m1 = n1;
    float t0 = 0.f, t1 = 0.f;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      // rounded to bf16 for the MMA; the denominator adds what the MMA sees
      const __nv_bfloat162 b0 = __floats2bfloat162_rn(dw_exp2(s[n][0] - u0), dw_exp2(s[n][1] - u0));
      const __nv_bfloat162 b1 = __floats2bfloat162_rn(dw_exp2(s[n][2] - u1), dw_exp2(s[n][3] - u1));
      t0 += __low2float(b0) + __high2float(b0);
      t1 += __low2float(b1) + __high2float(b1);
      p[2 * n] = *reinterpret_cast<const uint32_t*>(&b0);
      p[2 * n + 1] = *reinterpret_cast<const uint32_t*>(&b1);
    }
    l0 = l0 * a0 + t0;
    l1 = l1 * a1 + t1;
    if (__any_sync(0xffffffffu, a0 != 1.f || a1 != 1.f)) {
#pragma unroll
      for (int c = 0; c < DV / 64; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) { o[c][j][0] *= a0; o[c][j][1] *= a0; o[c][j][2] *= a1; o[c][j][3] *= a1; }
    }
  }
  __device__ __forceinline__ void add(const uint32_t (&p)[4]) {
#pragma unroll
    for (int c = 0; c < DV / 64; ++c) {
      const uint32_t w[4][4] = {{v[c][0].x, v[c][0].y, v[c][0].z, v[c][0].w}, {v[c][1].x, v[c][1].y, v[c][1].z, v[c][1].w},
                                {v[c][2].x, v[c][2].y, v[c][2].z, v[c][2].w}, {v[c][3].x, v[c][3].y, v[c][3].z, v[c][3].w}};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dw_mma(o[c][2 * i], p[0], p[1], p[2], p[3], __byte_perm(w[0][i], w[1][i], 0x5410), __byte_perm(w[2][i], w[3][i], 0x5410));
        dw_mma(o[c][2 * i + 1], p[0], p[1], p[2], p[3], __byte_perm(w[0][i], w[1][i], 0x7632), __byte_perm(w[2][i], w[3][i], 0x7632));
      }
    }
  }
  // sums of a row live in four lanes until here
  __device__ __forceinline__ void end() {
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
  }
  // O and (m, l) of the first G rows to shared memory, rows `pitch` floats apart: [16][pitch], then m [16], l [16]
  __device__ __forceinline__ void put(float* to, int pitch, int G) const {
    const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
#pragma unroll
    for (int c = 0; c < DV / 64; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          // column n of the tiles is dimension 64 c + 8 n + tile
          const int d = c * 64 + 16 * t + 8 * e + j;
          if (FULL || d < dv) {
            if (r < G) *reinterpret_cast<float4*>(to + r * pitch + d) = make_float4(o[c][j][e], o[c][j + 1][e], o[c][j + 2][e], o[c][j + 3][e]);
            if (r + 8 < G) *reinterpret_cast<float4*>(to + (r + 8) * pitch + d) = make_float4(o[c][j][2 + e], o[c][j + 1][2 + e], o[c][j + 2][2 + e], o[c][j + 3][2 + e]);
          }
        }
    if (t == 0) { to[16 * pitch + r] = m0; to[16 * pitch + 8 + r] = m1; to[16 * pitch + 16 + r] = l0; to[16 * pitch + 24 + r] = l1; }
  }
};

// Parts of several warps, as put() leaves them `size` floats apart, joined into `to` by all threads (THREADS of them)
template <int WARPS, int THREADS>
__device__ __forceinline__ void dw_join(const float* parts, int size, int pitch, int G, int dv, float* to) {
  for (int i = threadIdx.x; i < G * dv; i += THREADS) {
    const int g = i / dv, d = i - g * dv;
    float m = -INFINITY, v = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, parts[w * size + 16 * pitch + g]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float* p = parts + w * size;
      const float mw = p[16 * pitch + g];
      if (mw == -INFINITY) continue;             // its numbers are nobody's
      const float f = dw_exp2(mw - m);
      v += f * p[g * pitch + d];
      l += f * p[16 * pitch + 16 + g];
    }
    to[g * pitch + d] = v;
    if (d == 0) { to[16 * pitch + g] = m; to[16 * pitch + 16 + g] = l; }
  }
}

}  // namespace b200

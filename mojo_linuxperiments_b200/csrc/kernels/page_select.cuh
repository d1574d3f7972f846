// Which pages a row of queries reads: the pages of its sequence that always count, and those of the others whose scores are highest.
//
// The CTAs of a cluster hold the scores of a share of the pages each, as integers of the same order.  Four rounds of eight bits find the score of the
// last page taken: every CTA counts its digits, and all read all counts through distributed shared memory.  Then the pages go, in their own order, to the
// list of the CTA that will read them: an equal share for each, wherever the pages lie.  Equal scores: the lower page first.
#pragma once
#include "ptx.cuh"

namespace b200 {

constexpr int PS_THREADS = 256, PS_WARPS = 8;

struct PageSelectShared {
  unsigned hist[4][256];                 // digits of this CTA's scores, a round each
  unsigned warp_counts[PS_WARPS][2];     // above the last score taken, equal to it
  unsigned counts[2];
  unsigned scan[PS_WARPS];
  unsigned found[2];                     // digit of the round, pages still to be taken within it
};

__device__ __forceinline__ unsigned ps_order(float s) {
  const unsigned b = __float_as_uint(s);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;       // not a number: taken rather than lost
  return b ^ (static_cast<unsigned>(static_cast<int>(b) >> 31) | 0x80000000u);
}

__device__ __forceinline__ unsigned ps_ld_cluster(uint32_t addr) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// the CTA that reads entry x of a list of n that S CTAs share, and the first entry of CTA r
__device__ __forceinline__ int ps_owner(int x, int n, int S) { return static_cast<int>(((static_cast<long long>(x) + 1) * S - 1) / n); }
__device__ __forceinline__ int ps_share(int n, int r, int S) { return static_cast<int>(static_cast<long long>(n) * r / S); }

// keys[0 .. n): the scores of this CTA's candidates, number from .. of all; `take` (> 0) of the cluster's candidates are wanted, fewer than there are.
// They become entries first .. of lists of `entries`, as numbers place0 + candidate.  All threads of all CTAs of the cluster call it with the same
// arguments but for keys, n and from; afterwards the lists are complete once the cluster has met (cluster_sync_all).
__device__ __forceinline__ void select_pages(PageSelectShared& sh, const unsigned* keys, int n, int from, int take, int first, int entries, int place0,
                                             int* list, int rank, int S) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < 4 * 256; i += PS_THREADS) sh.hist[0][i] = 0u;
  __syncthreads();
  unsigned prefix = 0u, left = static_cast<unsigned>(take);
#pragma unroll 1
  for (int round = 0; round < 4; ++round) {
    const int shift = 24 - 8 * round;
    for (int i = tid; i < n; i += PS_THREADS) {
      const unsigned k = keys[i];
      if (round == 0 || (k >> (shift + 8)) == prefix) atomicAdd(&sh.hist[round][(k >> shift) & 255u], 1u);
    }
    if (S > 1) cluster_sync_all(); else __syncthreads();
    // thread t has digit 255 - t: how many candidates have that digit, and how many a higher one
    const uint32_t at = smem_u32(&sh.hist[round][255 - tid]);
    unsigned mine = 0u;
    if (S > 1) { for (int r = 0; r < S; ++r) mine += ps_ld_cluster(mapa_shared(at, r)); }
    else mine = sh.hist[round][255 - tid];
    unsigned upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) { const unsigned x = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += x; }
    if (lane == 31) sh.scan[warp] = upto;
    __syncthreads();
    for (int w = 0; w < warp; ++w) upto += sh.scan[w];
    if (upto >= left && upto - mine < left) { sh.found[0] = 255u - tid; sh.found[1] = left - (upto - mine); }
    __syncthreads();
    prefix = prefix << 8 | sh.found[0];
    left = sh.found[1];
    __syncthreads();
  }
  // every warp takes a run of the CTA's candidates, in order
  const int a = static_cast<int>(static_cast<long long>(n) * warp / PS_WARPS), b = static_cast<int>(static_cast<long long>(n) * (warp + 1) / PS_WARPS);
  unsigned above = 0u, equal = 0u;
  for (int i = a; i < b; i += 32) {
    const unsigned k = i + lane < b ? keys[i + lane] : 0u;
    const bool on = i + lane < b;
    above += __popc(__ballot_sync(0xffffffffu, on && k > prefix));
    equal += __popc(__ballot_sync(0xffffffffu, on && k == prefix));
  }
  if (lane == 0) { sh.warp_counts[warp][0] = above; sh.warp_counts[warp][1] = equal; }
  __syncthreads();
  if (tid < 2) {
    unsigned t = 0u;
    for (int w = 0; w < PS_WARPS; ++w) t += sh.warp_counts[w][tid];
    sh.counts[tid] = t;
  }
  if (S > 1) cluster_sync_all(); else __syncthreads();
  unsigned at = static_cast<unsigned>(first), equals_before = 0u;
  const uint32_t c_addr = smem_u32(sh.counts);
  for (int r = 0; r < rank; ++r) { at += ps_ld_cluster(mapa_shared(c_addr, r)); equals_before += ps_ld_cluster(mapa_shared(c_addr + 4, r)); }
  for (int w = 0; w < warp; ++w) { at += sh.warp_counts[w][0]; equals_before += sh.warp_counts[w][1]; }
  at += min(equals_before, left);
  for (int i = a; i < b; i += 32) {
    const bool on = i + lane < b;
    const unsigned k = on ? keys[i + lane] : 0u;
    const unsigned below = (1u << lane) - 1u;
    const unsigned eq = __ballot_sync(0xffffffffu, on && k == prefix);
    const bool taken = on && (k > prefix || (k == prefix && equals_before + __popc(eq & below) < left));
    const unsigned all = __ballot_sync(0xffffffffu, taken);
    if (taken) {
      const int x = static_cast<int>(at + __popc(all & below)), r = ps_owner(x, entries, S);
      const uint32_t to = smem_u32(list + (x - ps_share(entries, r, S)));
      st_shared_cluster_u32(S > 1 ? mapa_shared(to, r) : to, static_cast<uint32_t>(place0 + from + i + lane));
    }
    at += __popc(all);
    equals_before += __popc(eq);
  }
}

}  // namespace b200

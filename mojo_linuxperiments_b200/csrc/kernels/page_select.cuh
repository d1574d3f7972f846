// Which pages a row of queries reads: the pages of its sequence that always count, and those of the others whose scores are highest.
//
// Scores are integers of the same order.  A thread's largest score stands for all of its own: a digit below the take-th largest of those of 256 threads is no
// larger than the score of the last page taken, so only candidates from there on count, twice as many as are taken or so; they are put together in their own
// order.  Rounds of eight bits, from the highest in which scores differ, then find the score of the last page taken, and end as soon as a whole
// digit is taken; rounds over all candidates where that leaves too many (many pages taken, many equal scores).  Equal scores: the lower page
// first.  Every CTA that reads a part of the pages selects by itself: an exchange between CTAs costs more than looking at thousands of scores again.
// Loops are short rather than unrolled: a selection is run once per launch, and its instructions have to be fetched for that.  125 of 8,189 take 5 us.
#pragma once
#include "ptx.cuh"

namespace b200 {

constexpr int PS_THREADS = 256, PS_WARPS = 8, PS_BATCH = 16, PS_FEW = 768;

struct PageSelectShared {
  uint2 few[PS_FEW];                     // score and number of the candidates that may be taken
  unsigned hist[5][256];                 // digits, a round each; digit d at 255 - d
  unsigned scan[PS_WARPS][2], tally[PS_WARPS][2];
  unsigned found[3];                     // digit of the round, scores still to be taken within it, scores within it
};

__device__ __forceinline__ unsigned ps_order(float s) {
  const unsigned b = __float_as_uint(s);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;       // not a number: taken rather than lost
  return b ^ (static_cast<unsigned>(static_cast<int>(b) >> 31) | 0x80000000u);
}

// part r of n things that S share begins here
__device__ __forceinline__ int ps_share(int n, int r, int S) { return static_cast<int>(static_cast<long long>(n) * r / S); }

// f(number, score) for the scores of this thread: numbers tid, tid + 256, .. below n, sixteen loads at a time
template <typename F>
__device__ __forceinline__ void ps_each(const unsigned* keys, int n, F&& f) {
#pragma unroll 1
  for (int i0 = threadIdx.x; i0 < n; i0 += PS_BATCH * PS_THREADS) {
    unsigned k[PS_BATCH];
#pragma unroll
    for (int j = 0; j < PS_BATCH; ++j) k[j] = i0 + j * PS_THREADS < n ? keys[i0 + j * PS_THREADS] : 0u;
#pragma unroll
    for (int j = 0; j < PS_BATCH; ++j)
      if (i0 + j * PS_THREADS < n) f(i0 + j * PS_THREADS, k[j]);
  }
}

// In which digit the left-th largest is, of what has been counted in `hist` (all counts are in place): found[0], and found[1] of found[2] there
__device__ __forceinline__ void ps_digit(PageSelectShared& sh, const unsigned* hist, unsigned left) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned mine = hist[tid];
  unsigned upto = mine;                          // with digit 255 - tid or a higher one
#pragma unroll
  for (int o = 1; o < 32; o *= 2) { const unsigned x = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += x; }
  if (lane == 31) sh.tally[warp][0] = upto;
  __syncthreads();
  upto += __reduce_add_sync(0xffffffffu, lane < warp ? sh.tally[lane][0] : 0u);
  if (upto - mine < left && left <= upto) { sh.found[0] = 255u - tid; sh.found[1] = left - (upto - mine); sh.found[2] = mine; }
  __syncthreads();
}

// Sums of two counts over the warps before this thread's, and over all
__device__ __forceinline__ void ps_before(PageSelectShared& sh, unsigned x, unsigned y, unsigned& x0, unsigned& y0, unsigned& all_x) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  x = __reduce_add_sync(0xffffffffu, x);
  y = __reduce_add_sync(0xffffffffu, y);
  __syncthreads();                               // nobody reads what is written here any more
  if (lane == 0) { sh.scan[warp][0] = x; sh.scan[warp][1] = y; }
  __syncthreads();
  const unsigned u = lane < PS_WARPS ? sh.scan[lane][0] : 0u, v = lane < PS_WARPS ? sh.scan[lane][1] : 0u;
  x0 = __reduce_add_sync(0xffffffffu, lane < warp ? u : 0u);
  y0 = __reduce_add_sync(0xffffffffu, lane < warp ? v : 0u);
  all_x = __reduce_add_sync(0xffffffffu, u);
}

// Of the n candidates with scores `keys` (shared or global memory) `take` are wanted (0 < take < n).  They are entries first .. of the row's list, as
// numbers place0 + candidate; entries list0 .. list0 + share are written to list[0 .. share).  low, high: the least and the largest score that this thread saw.
__device__ __forceinline__ void select_pages(PageSelectShared& sh, const unsigned* keys, int n, unsigned low, unsigned high, int take, int first, int place0,
                                             int* list, int list0, int share) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned best = high;
  const bool some = tid < n;                     // a thread without scores stands for none
#pragma unroll
  for (int i = 0; i < 5; ++i) sh.hist[i][tid] = 0u;
  low = __reduce_min_sync(0xffffffffu, low);
  high = __reduce_max_sync(0xffffffffu, high);
  if (lane == 0) { sh.scan[warp][0] = low; sh.scan[warp][1] = high; }
  __syncthreads();
  low = __reduce_min_sync(0xffffffffu, sh.scan[lane & (PS_WARPS - 1)][0]);
  high = __reduce_max_sync(0xffffffffu, sh.scan[lane & (PS_WARPS - 1)][1]);
  const int width = high > low ? 32 - __clz(high - low) : 0;     // differences of scores have that many bits; none: all are equal
  unsigned bound = low;
  if (take <= min(n, PS_THREADS) && width > 0) {
    const int cut = max(0, width - 8);
    if (some) atomicAdd(&sh.hist[4][255u - ((best - low) >> cut)], 1u);
    __syncthreads();
    ps_digit(sh, sh.hist[4], static_cast<unsigned>(take));
    bound = low + (sh.found[0] << cut);
  }
  // Every warp has a run of the candidates, 1,024 at a time: lane j keeps which of numbers 32 j .. 32 j + 31 may be taken
  const int steps = (n + PS_THREADS - 1) / PS_THREADS, a = warp * 32 * steps, b = min(n, a + 32 * steps);
  auto look = [&](int from, auto&& test) {
    unsigned mask = 0u;
#pragma unroll 8
    for (int j = 0; j < 32; ++j) {
      const int i = from + 32 * j + lane;
      const unsigned x = __ballot_sync(0xffffffffu, i < b && test(keys[i < b ? i : a]));
      if (lane == j) mask = x;
    }
    return mask;
  };
  auto may = [&](unsigned k) { return k >= bound; };
  unsigned mask = 0u, count = 0u, before, unused, m;
#pragma unroll 1
  for (int from = a; from < b; from += 1024) { mask = look(from, may); count += __popc(mask); }
  ps_before(sh, count, 0u, before, unused, m);
  const bool few = m <= PS_FEW;
  if (few) {
#pragma unroll 1
    for (int from = a; from < b; from += 1024) {
      if (steps > 32) mask = look(from, may);
      unsigned at = __popc(mask);
#pragma unroll
      for (int o = 1; o < 32; o *= 2) { const unsigned x = __shfl_up_sync(0xffffffffu, at, o); if (lane >= o) at += x; }
      const unsigned all = __shfl_sync(0xffffffffu, at, 31);
      at += before - __popc(mask);
      for (unsigned any = mask; any; any &= any - 1u) {
        const int i = from + 32 * lane + __ffs(any) - 1;
        sh.few[at++] = make_uint2(keys[i], static_cast<unsigned>(i));
      }
      before += all;
    }
    __syncthreads();
  }
  const unsigned base = few ? bound : low;
  int shift = high > base ? 32 - __clz(high - base) : 0;
  unsigned prefix = 0u, left = static_cast<unsigned>(take);
#pragma unroll 1
  for (int round = 0; shift > 0; ++round) {
    const int bits = min(8, shift), above = round > 0 ? bits : 31;               // a first round has no digits in front
    shift -= bits;
    auto tally = [&](unsigned k) {
      k = (k - base) >> shift;
      if (round == 0 || (k >> above) == prefix) atomicAdd(&sh.hist[round][255u - (k & ((1u << bits) - 1u))], 1u);
    };
    if (few) { for (int c = tid; c < static_cast<int>(m); c += PS_THREADS) tally(sh.few[c].x); }
    else ps_each(keys, n, [&](int, unsigned k) { tally(k); });
    __syncthreads();
    ps_digit(sh, sh.hist[round], left);
    prefix = prefix << bits | sh.found[0];
    left = sh.found[1];
    if (left == sh.found[2]) break;              // the whole digit is taken
  }
  // in order: those above the last one taken, and the first `left` of those equal to it
  if (few) {
    const int c0 = static_cast<int>(m) * tid / PS_THREADS, c1 = static_cast<int>(m) * (tid + 1) / PS_THREADS;
    unsigned na = 0u, ne = 0u, ua, ue;
    for (int c = c0; c < c1; ++c) {
      const unsigned k = (sh.few[c].x - base) >> shift;
      na += k > prefix;
      ne += k == prefix;
    }
    ps_before(sh, na, ne, ua, ue, count);
    unsigned ia = na, ie = ne;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const unsigned x = __shfl_up_sync(0xffffffffu, ia, o), y = __shfl_up_sync(0xffffffffu, ie, o);
      if (lane >= o) { ia += x; ie += y; }
    }
    unsigned e = ue + ie - ne;
    int x = first + static_cast<int>(ua + ia - na + min(e, left)) - list0;
    for (int c = c0; c < c1; ++c) {
      const uint2 f = sh.few[c];
      const unsigned k = (f.x - base) >> shift;
      if (k < prefix || (k == prefix && e++ >= left)) continue;
      if (x >= 0 && x < share) list[x] = place0 + static_cast<int>(f.y);
      ++x;
    }
    return;
  }
  unsigned na = 0u, ne = 0u, a0, e0;
  auto over = [&](unsigned k) { return ((k - base) >> shift) > prefix; };
  auto same = [&](unsigned k) { return ((k - base) >> shift) == prefix; };
#pragma unroll 1
  for (int from = a; from < b; from += 1024) { na += __popc(look(from, over)); ne += __popc(look(from, same)); }
  ps_before(sh, na, ne, a0, e0, count);
#pragma unroll 1
  for (int from = a; from < b; from += 1024) {
    const unsigned above = look(from, over), equal = look(from, same);
    unsigned ua = __popc(above), ue = __popc(equal);
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const unsigned x = __shfl_up_sync(0xffffffffu, ua, o), y = __shfl_up_sync(0xffffffffu, ue, o);
      if (lane >= o) { ua += x; ue += y; }
    }
    unsigned e = e0 + ue - __popc(equal);        // before this lane's
    int x = first + static_cast<int>(a0 + ua - __popc(above) + min(e, left)) - list0;
    for (unsigned any = above | equal; any; any &= any - 1u) {
      const int bit = __ffs(any) - 1;
      if (!((above >> bit) & 1u) && e++ >= left) continue;
      if (x >= 0 && x < share) list[x] = place0 + from + 32 * lane + bit;
      ++x;
    }
    a0 += __shfl_sync(0xffffffffu, ua, 31);
    e0 += __shfl_sync(0xffffffffu, ue, 31);
  }
}

}  // namespace b200

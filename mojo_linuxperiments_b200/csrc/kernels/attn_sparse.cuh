// What the forms of attention over selected pages share: their parameters, and what a row of queries sees.
#pragma once
#include "ptx.cuh"
#include "api.h"
#include "page_select.cuh"

namespace b200 {

constexpr size_t SPARSE_MAX_SMEM = 200u << 10;

struct SparseParams {
  const void* q; long long ldq;
  void* out; long long ldo;
  int hq, M, hgroups;
  const int* positions; const int* seq_ids; const int* seq_lens;
  b200_paged_cache c;
  b200_attn_spec s;
  const void* bounds;                    // [pages][kv_heads][2][dk]
  unsigned* scores;                      // [M][kv_heads][max_pages], candidates' in their order
  int top, first, last;
  int splits, list_cap, score_cap;       // entries and scores that a CTA has room for
  int* chosen;                           // [M][kv_heads][top] or NULL
  int* status;
};

struct SparseRow {
  int seq, pos, low;                     // keys low .. pos are seen
  int page0, pages;                      // first page of them, number of pages
  int entries;                           // pages read
  bool selects;                          // more pages than are read
  int first, take, candidates, place0;   // pages read in any case at the front; of `candidates` from page place0 on `take` are taken

  // false: nothing to see (an empty slot, or a row that names no place of the cache, which the status word then says)
  __device__ __forceinline__ bool find(const SparseParams& p, int tok) {
    seq = p.seq_ids ? p.seq_ids[tok] : tok;
    pos = p.positions[tok];
    if (p.seq_lens && p.seq_lens[tok] <= 0) return false;
    if (pos < 0 || seq < 0 || seq >= p.c.num_seqs || pos / p.c.page_size >= p.c.max_pages) {
      if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, static_cast<int>(ST_BAD_ARGUMENT) | (25 << 8));
      return false;
    }
    low = p.s.chunk > 0 ? pos - pos % p.s.chunk : 0;
    page0 = low / p.c.page_size;
    pages = pos / p.c.page_size - page0 + 1;
    entries = min(pages, p.top);
    first = p.first;
    take = p.top - p.first - p.last;
    selects = pages > p.top && take > 0;
    candidates = pages - p.first - p.last;
    place0 = page0 + p.first;
    return true;
  }
  // The entries of this CTA's list: those that need no score (all of them, or the first and the last), and those that do.  All threads; the list is
  // complete behind the next barrier.
  __device__ __forceinline__ int lists(const SparseParams& p, PageSelectShared& sel, unsigned* room, int tok, int kvh, int rank, int S, int* list) const {
    const int a = ps_share(entries, rank, S), b = ps_share(entries, rank + 1, S);
    for (int x = a + threadIdx.x; x < b; x += PS_THREADS) {
      if (pages == entries || x < first) list[x - a] = page0 + x;
      else if (x >= entries - p.last) list[x - a] = page0 + pages - (entries - x);
    }
    if (selects && a < entries - p.last && b > first) {
      const unsigned* keys = p.scores + (static_cast<size_t>(tok) * p.c.kv_heads + kvh) * p.c.max_pages;
      unsigned lo = 0xffffffffu, hi = 0u;
      const bool near = candidates <= p.score_cap;
      ps_each(keys, candidates, [&](int i, unsigned k) {
        lo = min(lo, k);
        hi = max(hi, k);
        if (near) room[i] = k;
      });
      select_pages(sel, near ? room : keys, candidates, lo, hi, take, first, place0, list, a, b - a);
    }
    return b - a;
  }
  __device__ __forceinline__ void tell(const SparseParams& p, int tok, int kvh, int rank, int share, const int* list, int S) const {
    int* to = p.chosen + (static_cast<size_t>(tok) * p.c.kv_heads + kvh) * p.top;
    const int a = ps_share(entries, rank, S);
    for (int i = threadIdx.x; i < share; i += PS_THREADS) to[a + i] = list[i];
    if (rank == 0)
      for (int i = entries + threadIdx.x; i < p.top; i += PS_THREADS) to[i] = -1;
  }
};

}  // namespace b200

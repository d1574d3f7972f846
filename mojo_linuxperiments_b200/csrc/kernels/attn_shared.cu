// Decode attention of sequences that share the pages of a prefix, on sm_100a tensor cores: the prefix is read once per group, not once per sequence.
//
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m):  keys of the prefix and a sequence's own keys give (m, l, O) each, which are joined by
//   m = max(m_1, m_2), l = sum l_i exp(m_i - m), O = sum O_i exp(m_i - m).
//
// Two launches.  The first takes the prefixes: the rows (member x query head) of a group are the M of tcgen05 MMAs over tiles of 128 keys, in pieces of
// up to 256 rows and of some tiles, which leave (m, l, O) in fp32.  Which pieces there are is a list on the device, made when groups change, so that a captured call
// follows them.  The second takes each sequence's own keys (decode_warp.cuh) while the first still runs, joins the pieces of the prefix, adds sink
// and gate and writes the output; it waits for the first only there.
//
// 4 sequences behind 512 tokens (32 heads over 8, rows of 128): 11.8 us, a chain of latencies: start 0.5, plan and queries 2, tiles 2.5, results 2.5, join 2, and a cluster
// of four CTAs per slot and KV head for what may be own keys.  32 behind 2,048 tokens with up to 300 of their own: 17.6 us.  128 behind 32,768 with up to 1,000 of their
// own: 132 us, 78 for the prefix, then 54 for the own keys, whose CTAs find no place beside the pieces.  (Where that was 125: in one kernel's registers beside the pieces
// 166 us and more; own keys by as many CTAs as there are places, one slot after the other and the joins shared out at the end, 135 us.)
#include "ptx.cuh"
#include "api.h"
#include "launch.cuh"
#include "gemm_common.cuh"
#include "decode_warp.cuh"

namespace b200 {

// ---- the plan: int32 on the device -------------------------------------------------------------------------------------------------
// [0] pieces; [4] pieces of this call that are done, [5] CTAs of the second kernel that have left (both zero between calls); at SP_INFO four numbers
// per slot: first row of its partial results, rows between the parts of the prefix, parts, tokens; then the pieces, eight numbers each; then the slots of the groups'
// members.
//
// A slot takes either all keys of the pieces of its group or none, so that no row meets a value that it does not see: none if it is shorter than the prefix,
// or if its chunk begins behind it.  A chunk that begins inside the prefix begins at the same key for every other slot, the last multiple of the chunk in front of
// the prefix's end; the pieces begin at the first page from there on, and what lies in front of that page is each slot's own.
constexpr int SP_DONE = 4, SP_LEFT = 5, SP_INFO = 16, SP_PIECE = 8;
// member0: of the group, in the list of slots; rows row0 .. row0 + rows of the group (member x query head); keys key0 .. key1; part: first row of the partial
// results of the group's rows for this run of keys; lead: slot whose pages are read; mode: what the two units of a CTA do, and above it the group's rows
struct SharedPiece { int member0, row0, rows, key0, key1, part, lead, mode, group_rows; };
// two tiles of 128 rows; the same 128 rows and every other tile of keys, whose results are the next part; one unit
enum SharedMode : int { SM_ROWS = 0, SM_KEYS = 1, SM_ONE = 2 };

struct SharedParams {
  const __nv_bfloat16* q; long long ldq;
  __nv_bfloat16* out; long long ldo;
  int hq, B;
  const int* seq_lens;
  int* plan; int pieces_at, slots_at, max_pieces;
  float* part; int part_rows;            // [kv_heads][dv / 4][part_rows][4], then (m, l) [kv_heads][part_rows][2]
  b200_paged_cache c;
  int chunk;
  float scale;
  const float* sink;
  const __nv_bfloat16* gate; long long ldg;
  int splits, hgroups;
  int* status;
  unsigned long long limit_ns;
};

// pairs of floats in a 64-bit register: one instruction for both
__device__ __forceinline__ uint64_t sx_pair(float a, float b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void sx_split(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t sx_fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ uint64_t sx_add2(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ float sx_max3(float a, float b, float c) { float r; asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }

__device__ __forceinline__ void sx_copy16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void sx_copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ---- prefixes -----------------------------------------------------------------------------------------------------------------------
// One CTA per SM with two units, which take turns on the tensor cores: warp 0 fetches pages by TMA (lane <-> page; one box for a page of rows of 128, whose
// requests take half the time of two) into two-stage rings, warp 1 issues the MMAs, warps 4..7 and 8..11 gather the queries of a unit, take its softmax
// (thread <-> row) and keep O in tensor memory.  Where a group has more than 128 rows the units share the keys, otherwise each has every other tile.  Results are
// stored with the rows of a tile next to each other, so that a warp's stores and the loads of a slot's heads are whole sectors.
//
// A step of both units, 2 x 128 x 128 scores and their products, takes 2.15 us at the 1.5 GHz that this load leaves, 2.4 to 2.7 where softmaxes are sharp and maxima
// move on; the tensor cores, the exponentials and the reads of shared memory would take 1.4 each.  The rest is the way of one unit from its scores to its weights and
// back, which the other unit covers in part.  Measured on 128 sequences behind 32,768 tokens, when the step kept took 124 to 136, and not kept: scores of 64 keys at a
// time, two ahead (144 us for 127: MMAs 64 wide read their rows as often as wide ones), two warpgroups per unit (156 for 136), a quarter or half of the exponentials as
// polynomials (125, 128 for 125), columns reread in short loops (130 for 125), pages asked for into L2 two or three tiles ahead (135 for 126).
constexpr int SX_THREADS = 384, SX_BN = 128, SX_PS = 16;
// registers: 384 x 168 at launch, 128 x (72 + 216 + 216) afterwards, which is as many
constexpr int SX_REGS_FEW = 72, SX_REGS_MANY = 216;
constexpr int SX_CHUNK = 128 * 128, SX_TILE = 2 * SX_CHUNK;
// A tile's weights are taken against an older maximum while a row's new largest weight, relative to that, is no more than 2^8 and a sixteenth of the row's sum.  Beyond
// that the reference moves on and O is scaled: the weight of the largest key is one then, and its rounding does not count.  Errors against 64 bits, 128 sequences
// behind 8,192 tokens, scores of a standard deviation of 1 and of 3: 2.28e-3 and 1.70e-3, as a maximum that always moves on gives 2.23e-3 and 1.70e-3 and one
// that moves beyond 2^8 alone 2.33e-3 and 1.96e-3; 128 behind 32,768: 131 us, 141 and 128.5.
constexpr float SX_LAZY = 8.f, SX_SHARE = 16.f;
constexpr int SX_SMEM = 6 * SX_TILE + 1024 + 256;

__global__ void __launch_bounds__(SX_THREADS, 1)
attn_shared_prefix_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ SharedParams p) {
  extern __shared__ uint8_t smem_raw[];
  B200_TRACE_INIT();
  if (threadIdx.x == 0) B200_TRACE(TK_ATTN_SHARED, TP_START);
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sQ = smem_u32(smem), sK = sQ + 2 * SX_TILE, sV = sK + 2 * SX_TILE;        // two units, two stages, two stages
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + 6 * SX_TILE);
  const uint32_t bar0 = smem_u32(bars);
  enum { B_KFULL = 0, B_KEMPTY = 2, B_VFULL = 4, B_VEMPTY = 6, B_SFULL = 8, B_PFULL = 10, B_OFULL = 14, B_COUNT = 16 };      // two of each: stages or units; P in two halves
  auto bar = [&](int i) { return bar0 + 8u * i; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + B_COUNT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* seen = reinterpret_cast<volatile int*>(tmem_slot + 2);       // with chunks: some row of the piece takes it; two pieces in turn
  volatile int* gaps = reinterpret_cast<volatile int*>(tmem_slot + 4);       // some page of the piece does not exist; two pieces in turn

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int dk = p.c.dk, dv = p.c.dv, hkv = p.c.kv_heads, group = p.hq / hkv;
  const int kchunks = (dk + 63) >> 6, vchunks = (dv + 63) >> 6, ksteps = (dk + 15) >> 4, dv16 = (dv + 15) & ~15;
  const bool kwhole = dk == 128, vwhole = dv == 128;
  if (threadIdx.x == 0) {
    for (int i = 0; i < B_COUNT; ++i) mbar_init(bar(i), i >= B_PFULL && i < B_OFULL ? 4 : 1);
    *abort_flag = 0;
    seen[0] = seen[1] = gaps[0] = gaps[1] = 0;
    mbar_fence_init();
  }
  if (warp == 1) { tmem_alloc(smem_u32(tmem_slot), 512); tmem_relinquish(); }
  if (threadIdx.x == 32 * 2) { prefetch_tmap(&tmap_k); prefetch_tmap(&tmap_v); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;              // S (then P) of unit u at 128 u, O at 256 + 128 u
  pdl_wait();
  if (threadIdx.x == 0) B200_TRACE(TK_ATTN_SHARED, TP_DEPS);
  pdl_launch_dependents();       // what starts now may read all that was written before this kernel

  auto wait = [&](int i, uint32_t par, int code) { return mbar_wait(bar(i), par, abort_flag, p.status, code | (26 << 8), p.limit_ns); };
  // all warps meet, from the two branches that they are in, where the queries are in place and at the end of a piece
  enum { M_QUERIES = 1, M_END = 2 };
  auto meet = [&](int id) { named_bar_sync(id, SX_THREADS); };
  auto piece_of = [&](int item) {
    const int4* at = reinterpret_cast<const int4*>(p.plan + p.pieces_at + (item / hkv) * SP_PIECE);
    const int4 a = at[0], b = at[1];
    return SharedPiece{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w & 3, b.w >> 2};
  };
  const int room = p.c.max_pages * SX_PS;
  // tiles of 128 keys; with chunks known when the queries are in place
  auto tiles_of = [&](const SharedPiece& e, int turn) {
    const int end = min(e.key1, room);
    return end > e.key0 && (p.chunk <= 0 || seen[turn]) ? (end - e.key0 + SX_BN - 1) / SX_BN : 0;
  };
  auto units_of = [&](const SharedPiece& e) { return e.mode == SM_KEYS || (e.mode == SM_ROWS && e.rows > 128) ? 2 : 1; };
  SharedPiece e = piece_of(blockIdx.x);          // there is room for as many pieces as there are CTAs
  const int pieces = min(p.plan[0], p.max_pieces) * hkv;
  int turn = 0;
  if (warp < 4) {
    warpgroup_regs_dec<SX_REGS_FEW>();
    uint32_t kv = 0, p_par = 0;                  // tiles so far; bit u: parity of unit u's P
    for (int item = blockIdx.x; item < pieces; item += gridDim.x, turn ^= 1) {
      const int kvh = item % hkv;
      int n = 0;
      if (warp == 0) {
        const int kv_end = min(e.key1, room);
        const int* pt = p.c.page_table + static_cast<size_t>(e.lead) * p.c.max_pages;
        bool ok = true;
        // the pages of four tiles are in the lanes, those of the next four on their way
        auto ids_of = [&](int j) {
          const int tok = e.key0 + j * SX_BN + lane * SX_PS;
          if (tok >= kv_end) return p.c.num_pages;       // pages behind the end are filled with zeros, and so are those that do not exist
          const int pg = pt[tok / SX_PS];
          if (pg >= 0 && pg < p.c.num_pages) return pg;
          if (p.status) atomicCAS(p.status, 0, static_cast<int>(ST_BAD_ARGUMENT) | (26 << 8));
          return p.c.num_pages;
        };
        int ids = 0, ids_next = 0;
        auto load = [&](uint32_t dst, const CUtensorMap* m, int b, int chunks, bool whole, int pg) {
          if (lane == 0) mbar_expect_tx(bar(b), chunks * SX_CHUNK);
          __syncwarp();
          if (lane < 8 && whole) tma_load_5d(dst + lane * 4096, m, bar(b), 0, 0, 0, 2 * kvh, pg);
          else if (lane < 8)
            for (int c = 0; c < chunks; ++c) tma_load_3d(dst + c * SX_CHUNK + lane * 2048, m, bar(b), c * 64, kvh * SX_PS, pg);
        };
        auto fetch = [&](int j) {
          if ((j & 3) == 0 && j > 0) { ids = ids_next; ids_next = ids_of(j + 4); }
          const int page = __shfl_sync(0xffffffffu, ids, (j & 3) * 8 + (lane & 7));
          const int st = (kv + j) & 1;
          const uint32_t ph = (((kv + j) >> 1) & 1u) ^ 1u;
          ok = __all_sync(0xffffffffu, wait(B_KEMPTY + st, ph, ST_TIMEOUT_SMEM_EMPTY)) != 0;
          if (!ok) return;
          load(sK + st * SX_TILE, &tmap_k, B_KFULL + st, kchunks, kwhole, page);
          ok = __all_sync(0xffffffffu, wait(B_VEMPTY + st, ph, ST_TIMEOUT_SMEM_EMPTY)) != 0;
          if (!ok) return;
          load(sV + st * SX_TILE, &tmap_v, B_VFULL + st, vchunks, vwhole, page);
        };
        // without chunks the keys are known before the queries are in place, and nobody waits for this warp
        if (p.chunk > 0) meet(M_QUERIES); else named_bar_arrive(M_QUERIES, SX_THREADS);
        n = tiles_of(e, turn);
        if (n > 0) { ids = ids_of(0); ids_next = ids_of(4); }
        for (int j = 0; j < n && ok; ++j) fetch(j);
        if (!ok) { const uint64_t t0 = globaltimer_ns(); while (globaltimer_ns() - t0 < 2000000ull) { } }   // copies in flight land
      } else {
        meet(M_QUERIES);
        n = tiles_of(e, turn);
        if (warp == 1) {
          const bool one = elect_one();
          constexpr uint32_t IDESC_S = umma_idesc_bf16(128, 128, 0, 0);
          const uint32_t idesc_pv = umma_idesc_bf16(128, dv16, 0, 1);
          const uint64_t q_desc = umma_desc_k_sw128(sQ), k_desc = umma_desc_mn_sw128(sK, 16, kwhole ? 2048 : 1024);
          const uint64_t v_desc = umma_desc_mn_sw128(sV, vwhole ? 1024 : SX_CHUNK, vwhole ? 2048 : 1024);
          const uint32_t k_chunk = (kwhole ? 1024 : SX_CHUNK) >> 4, v_step = (vwhole ? 4096 : 2048) >> 4;
          const int units = units_of(e), lag = e.mode == SM_KEYS ? 2 : 1;      // tiles between two of a unit
          bool ok = true;
          // the product of tile j - lag and the scores of tile j, which go to where its weights were
          for (int j = 0; j < n + lag && ok && n > 0; ++j) {
            const int past = j - lag;
            const uint32_t ks = (kv + j) & 1, vs = (kv + past) & 1;
            if (j < n) ok = wait(B_KFULL + ks, ((kv + j) >> 1) & 1u, ST_TIMEOUT_SMEM_FULL);
            if (ok && past >= 0) ok = wait(B_VFULL + vs, ((kv + past) >> 1) & 1u, ST_TIMEOUT_SMEM_FULL);
#pragma unroll 1
            for (int u = e.mode == SM_KEYS ? j & 1 : 0; u < (e.mode == SM_KEYS ? (j & 1) + 1 : units) && ok; ++u) {
              if (past >= 0) {
                const uint64_t bd = v_desc + vs * (SX_TILE >> 4);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  ok = wait(B_PFULL + 2 * u + half, (p_par >> u) & 1u, ST_TIMEOUT_TMEM_EMPTY);
                  if (!ok) break;
                  tc_fence_after();
#pragma unroll
                  for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
                    if (one) umma_f16_ts(tmem + 256 + u * 128, tmem + u * 128 + kk * 8, bd + kk * v_step, idesc_pv, (past >= lag || kk > 0) ? 1u : 0u);
                }
                if (!ok) break;
                p_par ^= 1u << u;
                if (one && past + lag >= n) umma_commit(bar(B_OFULL + u));
              }
              if (j < n) {
                tc_fence_after();
                const uint64_t ad = q_desc + static_cast<uint32_t>(u * (SX_TILE >> 4)), bd = k_desc + ks * (SX_TILE >> 4);
#pragma unroll
                for (int kk = 0; kk < 8; ++kk) {
                  const uint32_t at_q = (kk >> 2) * (SX_CHUNK >> 4) + 2 * (kk & 3), at_k = (kk >> 2) * k_chunk + 2 * (kk & 3);
                  if (one && kk < ksteps) umma_f16_ss(tmem + u * 128, ad + at_q, bd + at_k, IDESC_S, kk > 0 ? 1u : 0u);
                }
                if (one) umma_commit(bar(B_SFULL + u));
              }
            }
            if (ok && one) {
              if (j < n) umma_commit(bar(B_KEMPTY + ks));
              if (past >= 0) umma_commit(bar(B_VEMPTY + vs));
            }
          }
          __syncwarp();
        } else if (threadIdx.x == 64) {
          seen[turn ^ 1] = gaps[turn ^ 1] = 0;   // the other piece's, at which nobody looks any more
        }
      }
      kv += n;
      meet(M_END);
      if (*abort_flag) break;                    // the same for all: nobody sets it between here and the next meeting
      if (item + static_cast<int>(gridDim.x) < pieces) e = piece_of(item + gridDim.x);
    }
  } else {
    warpgroup_regs_inc<SX_REGS_MANY>();
    const int u = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;   // unit; row of its tile, TMEM lane
    const uint32_t t_s = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + u * 128, t_o = t_s + 256;
    const float scale_log2 = p.scale * DW_LOG2E;
    uint32_t tiles = 0, items = 0;               // of this unit: their parities
    for (int item = blockIdx.x; item < pieces; item += gridDim.x, turn ^= 1) {
      const int kvh = item % hkv;
      const int row0 = e.row0 + (e.mode == SM_ROWS ? 128 * u : 0), rows = u < units_of(e) ? min(128, e.rows - (row0 - e.row0)) : 0;
      const bool idle = (warp & 3) * 32 >= rows;             // rows that nobody asked for: their weights are never looked at
      const int keys = min(e.key1, room) - e.key0;
      const int* pt = p.c.page_table + static_cast<size_t>(e.lead) * p.c.max_pages + e.key0 / SX_PS;
      auto exists = [&](int t) { const int pg = pt[t]; return pg >= 0 && pg < p.c.num_pages; };
      bool gap = false;
      for (int t = threadIdx.x - 128; t * SX_PS < keys; t += 256) gap = gap || !exists(t);
      if (!idle) {
        const int row = row0 + r, member = row / group;
        const bool on = r < rows;
        const int slot = on ? p.plan[p.slots_at + e.member0 + member] : 0;
        const long long from = on ? slot * p.ldq + static_cast<long long>(kvh * group + row - member * group) * dk : -1;
        bool any = true;
        if (p.chunk > 0) {
          const int len = on ? p.seq_lens[slot] : 0, tokens = on ? p.plan[SP_INFO + 4 * slot + 3] : 0;
          any = __any_sync(0xffffffffu, on && len >= tokens && (len - 1) - (len - 1) % p.chunk < tokens);
          if (any && lane == 0) seen[turn] = 1;
        }
        // half a warp per row: 256 neighbouring bytes at a time
        const int col = lane & 15;
        if (any)
#pragma unroll 2
        for (int i = 0; i < 16; ++i) {
          const long long at = __shfl_sync(0xffffffffu, from, 2 * i + (lane >> 4));
          const int x = (warp & 3) * 32 + 2 * i + (lane >> 4);
          const bool there = at >= 0 && col * 8 < dk;        // zeros otherwise
          sx_copy16(sQ + u * SX_TILE + (col >> 3) * SX_CHUNK + x * 128 + (((col & 7) ^ (x & 7)) << 4), p.q + (there ? at + col * 8 : 0), there);
        }
        sx_copies_done();
        fence_proxy_async_smem();
      }
      if (gap) gaps[turn] = 1;
      meet(M_QUERIES);
      if (threadIdx.x == 128) B200_TRACE(TK_ATTN_SHARED, 2); // queries in place
      const int n = rows > 0 ? tiles_of(e, turn) : 0;
      const bool gapped = gaps[turn] != 0;
      const int j0 = e.mode == SM_KEYS ? u : 0, step = e.mode == SM_KEYS ? 2 : 1;
      float m_ref = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = j0; j < n && ok; j += step) {
        ok = __all_sync(0xffffffffu, wait(B_SFULL + u, tiles++ & 1u, ST_TIMEOUT_TMEM_FULL)) != 0;
        if (!ok) break;
        if (threadIdx.x == 128 && j == 0) B200_TRACE(TK_ATTN_SHARED, 3);       // first scores
        tc_fence_after();
        if (!idle) {
          uint32_t v[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_x32(t_s + c * 32, v[c]);
          tmem_ld_wait();
          const int here = keys - j * SX_BN;     // behind them the tile is zeros
          if (here < SX_BN || gapped) {
            unsigned on = 0xffu;                 // pages of the tile that exist
            if (gapped) on = __ballot_sync(0xffffffffu, lane < 8 && lane * SX_PS < here && exists(j * (SX_BN / SX_PS) + lane));
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (c * 32 + i >= here || !(on >> ((c * 32 + i) / SX_PS) & 1u)) v[c][i] = 0xff800000u;      // -inf
          }
          float mx[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            mx[c] = __uint_as_float(v[c][0]);
#pragma unroll
            for (int i = 1; i < 31; i += 2) mx[c] = sx_max3(mx[c], __uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1]));
            mx[c] = fmaxf(mx[c], __uint_as_float(v[c][31]));
          }
          const float m_new = fmaxf(m_ref, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale_log2);
          if (__any_sync(0xffffffffu, m_new > m_ref && (m_new > m_ref + SX_LAZY || SX_SHARE * dw_exp2(m_new - m_ref) > l))) {
            const float alpha = m_ref == -INFINITY ? 0.f : dw_exp2(m_ref - m_new);
            l *= alpha;
            m_ref = m_new;
            if (j > j0) {      // the product before has completed: S of this tile was issued after it
#pragma unroll 1
              for (int c = 0; c < dv16; c += 32) {
                uint32_t o[32];
                tmem_ld_x32(t_o + c, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                tmem_st_x32(t_o + c, o);
              }
            }
          }
          const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
          // two at a time; rounded to bf16 for the MMA, the denominator adds what the MMA sees, so that the rounding of a weight that outweighs all others
          // has no part in the result
          const uint64_t scale2 = sx_pair(scale_log2, scale_log2), shift2 = sx_pair(-m_use, -m_use);
          uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float e0, e1;
              sx_split(sx_fma2(sx_pair(__uint_as_float(v[c][2 * i]), __uint_as_float(v[c][2 * i + 1])), scale2, shift2), e0, e1);
              e0 = dw_exp2(e0);
              e1 = dw_exp2(e1);
              pk[i] = dw_pack(e0, e1);
              sum[i & 1] = sx_add2(sum[i & 1], sx_pair(__uint_as_float(pk[i] << 16), __uint_as_float(pk[i] & 0xffff0000u)));
            }
            tmem_st_x16(t_s + c * 16, pk);
            if (c == 1) {                        // the product of the first half may begin
              tmem_st_wait();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(B_PFULL + 2 * u));
            }
          }
          float l0, l1, l2, l3;
          sx_split(sum[0], l0, l1);
          sx_split(sum[1], l2, l3);
          l += (l0 + l1) + (l2 + l3);
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (idle) mbar_arrive(bar(B_PFULL + 2 * u));
          mbar_arrive(bar(B_PFULL + 2 * u + 1));
        }
      }
      if (threadIdx.x == 128) B200_TRACE(TK_ATTN_SHARED, 4); // last weights
      const bool some = j0 < n;
      if (ok && some) ok = __all_sync(0xffffffffu, wait(B_OFULL + u, items++ & 1u, ST_TIMEOUT_TMEM_FULL)) != 0;
      tc_fence_after();
      if (threadIdx.x == 128) B200_TRACE(TK_ATTN_SHARED, 5); // last product
      if (ok && !idle) {
        // the second unit's results of the same rows are the next part
        const size_t to = static_cast<size_t>(e.part) + (e.mode == SM_KEYS && u > 0 ? e.group_rows : 0) + row0 + r;
        const bool mine = r < rows;
        if (mine) {
          float2* ml = reinterpret_cast<float2*>(p.part + static_cast<size_t>(hkv) * p.part_rows * dv) + static_cast<size_t>(kvh) * p.part_rows + to;
          *ml = make_float2(some ? m_ref : -INFINITY, l);
        }
        // nothing for a run of keys that nobody sees: its weights say so
        float4* dst = reinterpret_cast<float4*>(p.part) + static_cast<size_t>(kvh) * (dv >> 2) * p.part_rows + to;
        if (some)
#pragma unroll 1
          for (int c = 0; c < dv16; c += 32) {
            uint32_t o[32];
            tmem_ld_x32(t_o + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (mine && c + i * 4 < dv)
                dst[static_cast<size_t>((c >> 2) + i) * p.part_rows] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
          }
      }
      tc_fence_before();
      meet(M_END);
      if (threadIdx.x == 128) {
        if (!*abort_flag) red_release_gpu_add(reinterpret_cast<uint32_t*>(p.plan + SP_DONE), 1u);
        B200_TRACE(TK_ATTN_SHARED, 6);           // a piece
      }
      tc_fence_after();
      if (*abort_flag) break;
      if (item + static_cast<int>(gridDim.x) < pieces) e = piece_of(item + gridDim.x);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem, 512); }
  if (threadIdx.x == 0) B200_TRACE(TK_ATTN_SHARED, TP_EXIT);
  B200_TRACE_FLUSH(TK_ATTN_SHARED);
}

// ---- own keys, and the join ---------------------------------------------------------------------------------------------------------
// Grid (split, KV head x group of up to 16 query heads, slot); the splits of a slot are a cluster.  Four warps take pages in turn.
constexpr int SO_THREADS = 128, SO_WARPS = 4, SO_PARTS = 32;
constexpr int SO_AHEAD = 3;              // pages of a warp asked for into L2 ahead of their use
template <int DV> struct SoShape {
  static constexpr int PITCH = DV + 4, SIZE = 16 * PITCH + 32;
  static constexpr int SMEM = ((SO_WARPS + 1) * SIZE + 16 * (8 + SO_PARTS)) * 4;
};

// The last CTA that has looked at the counters clears them for the next call, which starts behind this kernel, and this kernel ends behind the first one.  Which
// that is, thread 0 asks early: the answer comes meanwhile.
__device__ __forceinline__ unsigned so_looked(const SharedParams& p) {
  return threadIdx.x == 0 ? atomicAdd(reinterpret_cast<unsigned*>(p.plan + SP_LEFT), 1u) : 0u;
}
__device__ __forceinline__ void so_leave(const SharedParams& p, unsigned before) {
  if (threadIdx.x != 0 || before != gridDim.x * gridDim.y * gridDim.z - 1u) return;
  pdl_wait();                                    // no piece is still to be counted, not even one that was given up
  p.plan[SP_DONE] = 0;
  p.plan[SP_LEFT] = 0;
}

template <int DK, int DV, int NH, bool FULL>
__global__ void __launch_bounds__(SO_THREADS, NH == 1 ? 3 : 2) attn_shared_own_kernel(const __grid_constant__ SharedParams p) {
  using Sh = SoShape<DV>;
  extern __shared__ __align__(16) float so_smem[];
  B200_TRACE_INIT();
  if (threadIdx.x == 0) B200_TRACE(TK_ATTN_OWN, TP_START);
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x, S = p.splits, b = blockIdx.z;
  const int kvh = blockIdx.y / p.hgroups, hg = blockIdx.y - kvh * p.hgroups;
  const int group = p.hq / p.c.kv_heads, g0 = hg * 16, G = min(16, group - g0), h0 = kvh * group + g0;
  const int dk = FULL ? DK : p.c.dk, dv = FULL ? DV : p.c.dv;
  // the kernel in front of this one starts it after its own wait: lengths, queries, keys and plan are settled
  const int len = p.seq_lens[b];
  const int4 info = *reinterpret_cast<const int4*>(p.plan + SP_INFO + 4 * b);       // first row of the parts, rows between them, parts, tokens
  const bool bad = len > p.c.max_pages * SX_PS;
  if (len <= 0 || bad) {                         // the same for all CTAs of the cluster
    if (bad && tid == 0 && p.status) atomicCAS(p.status, 0, static_cast<int>(ST_BAD_ARGUMENT) | (26 << 8));
    if (rank == 0)
      for (int i = tid; i < G * dv; i += SO_THREADS) p.out[static_cast<size_t>(b) * p.ldo + static_cast<size_t>(h0) * dv + i] = __float2bfloat16(0.f);
    so_leave(p, so_looked(p));
    return;
  }
  const int low = p.chunk > 0 ? (len - 1) - (len - 1) % p.chunk : 0;
  const bool shares = info.z > 0 && len >= info.w && low < info.w;
  // pages of the keys that are this kernel's: from the first seen, or those behind the prefix and, in front of them, the one that a chunk begins in
  const bool head = shares && low % SX_PS != 0;
  const int t0 = shares ? info.w / SX_PS - head : low / SX_PS, tiles = (len + SX_PS - 1) / SX_PS - t0;
  auto place = [&](int t) { return head && t == t0 ? low / SX_PS : t; };
  const int ta = t0 + static_cast<int>(static_cast<long long>(tiles) * rank / S), tb = t0 + static_cast<int>(static_cast<long long>(tiles) * (rank + 1) / S);
  const int mine = tb - ta > warp ? (tb - ta - warp + SO_WARPS - 1) / SO_WARPS : 0;
  const int* pt = p.c.page_table + static_cast<size_t>(b) * p.c.max_pages;
  const size_t rec = static_cast<size_t>(p.c.kv_heads) * SX_PS * (dk + dv);
  const __nv_bfloat16* kbase = static_cast<const __nv_bfloat16*>(p.c.data) + static_cast<size_t>(kvh) * SX_PS * dk;
  const __nv_bfloat16* vbase = static_cast<const __nv_bfloat16*>(p.c.data) + static_cast<size_t>(p.c.kv_heads) * SX_PS * dk + static_cast<size_t>(kvh) * SX_PS * dv;

  DecodeWarp<DK, DV, NH, FULL> w;
  w.begin(dk, dv, p.scale);
  // the ids of this warp's next 32 pages are in its lanes
  int ids = 0, ids_from = -32;
  w.walk(mine, [&](int i) {
    if (i >= ids_from + 32) {
      ids_from = i;
      ids = i + lane < mine ? pt[place(ta + warp + (i + lane) * SO_WARPS)] : -1;
      if (lane > 0 && lane < SO_AHEAD) dw_prefetch(kbase, vbase, ids, rec, dk, dv, p.c.num_pages);
    } else if (lane == i - ids_from + SO_AHEAD - 1) {
      dw_prefetch(kbase, vbase, ids, rec, dk, dv, p.c.num_pages);
    }
    const int page = __shfl_sync(0xffffffffu, ids, i - ids_from), first = place(ta + warp + i * SO_WARPS) * SX_PS;
    const bool there = page >= 0 && page < p.c.num_pages;
    if (!there && lane == 0 && p.status) atomicCAS(p.status, 0, static_cast<int>(ST_BAD_ARGUMENT) | (26 << 8));
    const size_t at = there ? page * rec : 0;
    return DwPage{kbase + at, vbase + at, max(0, low - first), there ? min(SX_PS, len - first) : 0};
  }, [&] { w.q.load(p.q + static_cast<size_t>(b) * p.ldq + static_cast<size_t>(h0) * dk, G, dk); });
  w.put(so_smem + warp * Sh::SIZE, Sh::PITCH, G);
  __syncthreads();
  if (tid == 0) B200_TRACE(TK_ATTN_OWN, 2);                  // own keys
  float* own = so_smem + SO_WARPS * Sh::SIZE;
  float* share = own + Sh::SIZE;                 // [16][8 + SO_PARTS]: what each part counts in the end
  dw_join<SO_WARPS, SO_THREADS>(so_smem, Sh::SIZE, Sh::PITCH, G, dv, own);
  // The parts of the prefix.  All CTAs of the first kernel run when this one starts, so their pieces may be waited for; the wait for its end takes 2 us longer.
  if (tid == 0 && shares) {
    const uint32_t pieces = static_cast<uint32_t>(min(p.plan[0], p.max_pieces)) * p.c.kv_heads;
    wait_count_gpu(reinterpret_cast<const uint32_t*>(p.plan + SP_DONE), pieces, p.status, static_cast<int>(ST_TIMEOUT_PEER_FLAG) | (26 << 8), p.limit_ns);
  }
  const unsigned before = so_looked(p);
  if (S > 1) cluster_sync_all(); else __syncthreads();
  if (tid == 0) B200_TRACE(TK_ATTN_OWN, TP_DEPS);
  const uint32_t own_addr = smem_u32(own);
  const float4* parts = reinterpret_cast<const float4*>(p.part) + static_cast<size_t>(kvh) * (dv >> 2) * p.part_rows + info.x + g0;
  const float* ml = p.part + static_cast<size_t>(p.c.kv_heads) * p.part_rows * dv + 2 * (static_cast<size_t>(kvh) * p.part_rows + info.x + g0);
  const int n_parts = shares ? min(info.z, SO_PARTS) : 0, all = S + n_parts;
  // a warp per row: lanes take the parts
  for (int g = warp; g < G; g += SO_WARPS) {
    float m[2], l[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = lane + 32 * u;
      m[u] = -INFINITY; l[u] = 0.f;
      if (i < S) {
        const uint32_t base = S > 1 ? mapa_shared(own_addr, i) : own_addr;
        m[u] = dw_ld_cluster(base + 4u * (16 * Sh::PITCH + g));
        l[u] = dw_ld_cluster(base + 4u * (16 * Sh::PITCH + 16 + g));
      } else if (i < all) {
        const float2 x = __ldcg(reinterpret_cast<const float2*>(ml + 2 * (static_cast<size_t>(i - S) * info.y + g)));
        m[u] = x.x; l[u] = x.y;
      }
    }
    const float sink2 = p.sink ? p.sink[h0 + g] * DW_LOG2E : -INFINITY;
    float top = fmaxf(fmaxf(m[0], m[1]), sink2);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float use = top == -INFINITY ? 0.f : top;
    const float f0 = m[0] == -INFINITY ? 0.f : dw_exp2(m[0] - use), f1 = m[1] == -INFINITY ? 0.f : dw_exp2(m[1] - use);
    float total = f0 * l[0] + f1 * l[1];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (p.sink) total += dw_exp2(sink2 - use);
    float f = total > 0.f ? 1.f / total : total;      // nothing, or not a number
    if (p.gate) f *= 1.f / (1.f + __expf(-__bfloat162float(p.gate[static_cast<size_t>(b) * p.ldg + h0 + g])));
    if (lane < all) share[g * (8 + SO_PARTS) + lane] = f0 * f;
    if (lane + 32 < all) share[g * (8 + SO_PARTS) + lane + 32] = f1 * f;
  }
  __syncthreads();
  // four dimensions per thread, the parts in turn: their loads do not wait for one another
  const int quads = dv >> 2;
  for (int i = rank * SO_THREADS + tid; i < G * quads; i += S * SO_THREADS) {
    const int d = i / G * 4, g = i - i / G * G;              // heads side by side, as the parts of the prefix have them
    const float* f = share + g * (8 + SO_PARTS);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    // (in batches of which none is cut short: what is left of a loop would wait for each of its loads)
    auto take = [&](float w, const float4& x) { v.x += w * x.x; v.y += w * x.y; v.z += w * x.z; v.w += w * x.w; };
    const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int s = 0; s < S; s += 4) {
      float4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = s + k < S ? dw_ld_cluster4(own_addr + 4u * (g * Sh::PITCH + d), s + k, S > 1) : none;
#pragma unroll
      for (int k = 0; k < 4; ++k) if (s + k < S) take(f[s + k], x[k]);
    }
#pragma unroll 1
    for (int s = 0; s < n_parts; s += 8) {
      float4 x[8];
      float fs[8];                               // zero: perhaps a part without keys, which has left no numbers
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        fs[k] = s + k < n_parts ? f[S + s + k] : 0.f;
        x[k] = fs[k] != 0.f ? __ldcg(parts + static_cast<size_t>(d >> 2) * p.part_rows + static_cast<size_t>(s + k) * info.y + g) : none;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) take(fs[k], x[k]);
    }
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), c = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p.out + static_cast<size_t>(b) * p.ldo + static_cast<size_t>(h0 + g) * dv + d) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&c));
  }
  if (S > 1) cluster_sync_all(); else __syncthreads();       // no CTA leaves while a peer may still read its part
  so_leave(p, before);
  if (tid == 0) B200_TRACE(TK_ATTN_OWN, TP_EXIT);
  B200_TRACE_FLUSH(TK_ATTN_OWN);
}

template <int DK, int DV, int NH, bool FULL>
static int launch_shared_own_as(const SharedParams& p, cudaStream_t stream) {
  constexpr int SMEM = SoShape<DV>::SMEM;
  cudaError_t e = allow_smem<attn_shared_own_kernel<DK, DV, NH, FULL>>(SMEM);
  if (e != cudaSuccess) return -1000 - static_cast<int>(e);
  launch_ex(attn_shared_own_kernel<DK, DV, NH, FULL>, dim3(p.splits, p.c.kv_heads * p.hgroups, p.B), dim3(SO_THREADS), SMEM, stream, p.splits, p);
  e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -2000 - static_cast<int>(e);
}

template <int DK, int DV, bool FULL>
static int launch_shared_own(const SharedParams& p, cudaStream_t stream) {
  return p.hq / p.c.kv_heads <= 8 ? launch_shared_own_as<DK, DV, 1, FULL>(p, stream) : launch_shared_own_as<DK, DV, 2, FULL>(p, stream);
}

}  // namespace b200

using namespace b200;

static bool shared_takes(const b200_paged_cache* c, int hq, long long ldq, long long ldo) {
  return !c->f32 && c->page_size == SX_PS && c->dk > 0 && c->dv > 0 && c->dk <= 128 && c->dv <= 128 && c->dk % 8 == 0 && c->dv % 8 == 0 && c->kv_heads > 0 &&
         hq % c->kv_heads == 0 && ldq % 8 == 0 && ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(c->data) & 15) == 0;
}

extern "C" int b200_attn_decode_shared(const void* q, long long ldq, void* out, long long ldo, int hq, int B, const int* seq_lens, const b200_paged_cache* c,
                                       const b200_attn_spec* s, int* plan, int pieces_at, int slots_at, int max_pieces, float* part, int part_rows,
                                       int splits, int num_sms, int* status, cudaStream_t stream) {
  if (B <= 0) return 0;
  if (!q || !out || !seq_lens || !c || !c->data || !c->page_table || !s || !plan || !part) return -1;
  if (!shared_takes(c, hq, ldq, ldo) || hq <= 0 || c->num_pages <= 0) return -2;
  if (B > c->num_seqs || B > 65535 || splits < 1 || splits > 8 || max_pieces < 0 || part_rows <= 0 || num_sms <= 0 || !(s->scale > 0.f)) return -3;
  if ((reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(out) & 7) || (reinterpret_cast<uintptr_t>(plan) & 15) ||
      (reinterpret_cast<uintptr_t>(part) & 15)) return -4;
  const uint64_t rec = static_cast<uint64_t>(c->kv_heads) * SX_PS * (c->dk + c->dv) * 2, kbytes = static_cast<uint64_t>(c->kv_heads) * SX_PS * c->dk * 2;
  CUtensorMap tk, tv;
  // rows of 128 numbers: a page at once, its two groups of eight keys, in each the two halves of their rows
  auto whole = [&](CUtensorMap* m, const void* base) {
    const uint64_t row = 256, n[5] = {64, 8, 2, static_cast<uint64_t>(c->kv_heads) * 2, static_cast<uint64_t>(c->num_pages)}, pitch[4] = {row, 128, 8 * row, rec};
    const uint32_t box[5] = {64, 8, 2, 2, 1};
    return make_tmap_5d_bf16(m, base, n, pitch, box);
  };
  const uint8_t* values = static_cast<const uint8_t*>(c->data) + kbytes;
  const uint64_t keys = static_cast<uint64_t>(c->kv_heads) * SX_PS;
  if (c->dk == 128 ? whole(&tk, c->data) : make_tmap_3d_bf16(&tk, c->data, c->dk, keys, c->num_pages, static_cast<uint64_t>(c->dk) * 2, rec, SX_PS, 1)) return -12;
  if (c->dv == 128 ? whole(&tv, values) : make_tmap_3d_bf16(&tv, values, c->dv, keys, c->num_pages, static_cast<uint64_t>(c->dv) * 2, rec, SX_PS, 1)) return -13;
  SharedParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(q); p.ldq = ldq; p.out = static_cast<__nv_bfloat16*>(out); p.ldo = ldo; p.hq = hq; p.B = B; p.seq_lens = seq_lens;
  p.plan = plan; p.pieces_at = pieces_at; p.slots_at = slots_at; p.max_pieces = max_pieces; p.part = part; p.part_rows = part_rows; p.c = *c; p.chunk = s->chunk;
  p.scale = s->scale; p.sink = s->sink; p.gate = static_cast<const __nv_bfloat16*>(s->gate); p.ldg = s->ldg; p.splits = splits;
  p.hgroups = (hq / c->kv_heads + 15) / 16; p.status = status; p.limit_ns = 2000000000ull;
  if (static_cast<long long>(c->kv_heads) * p.hgroups > 65535) return -3;
  cudaError_t e = allow_smem<attn_shared_prefix_kernel>(SX_SMEM);
  if (e != cudaSuccess) return -1000 - static_cast<int>(e);
  const long long most = static_cast<long long>(max_pieces) * c->kv_heads;
  const int grid = most < num_sms ? static_cast<int>(most > 0 ? most : 1) : num_sms;
  launch_ex(attn_shared_prefix_kernel, dim3(grid), dim3(SX_THREADS), SX_SMEM, stream, 0, tk, tv, p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return -2000 - static_cast<int>(e);
  const int d = c->dk > c->dv ? c->dk : c->dv;
  if (c->dk == 64 && c->dv == 64) return launch_shared_own<64, 64, true>(p, stream);
  if (c->dk == 128 && c->dv == 128) return launch_shared_own<128, 128, true>(p, stream);
  if (d <= 64) return launch_shared_own<64, 64, false>(p, stream);
  return launch_shared_own<128, 128, false>(p, stream);
}

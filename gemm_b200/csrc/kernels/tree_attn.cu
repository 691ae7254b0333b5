// Attention of drafted tree nodes over a paged KV cache on tcgen05 (bf16, heads of 64 or 128 columns).
//
// What a node sees, and the formula: tree_any.cu.  A row is a (node, query head of the group) pair, a tile is 128 rows of one KV head: floor(128 / G) nodes.
// The context is long and the rows are few, so the kernel is built to stream K and V: one block per SM, its shared memory a ring of 32 KB tiles (K and V of
// 128 places in turn) that TMA keeps full across work items, and two softmax groups of 128 threads, one thread per TMEM lane.
//   one tile in the item:   the groups take alternate KV blocks, each with its own maximum, sum and output accumulator, joined at the end;
//   two tiles in the item:  each group has its tile, and both use the same K and V (wide trees: half the loads, which would bound the products).
// A tile of 64 rows or fewer is folded: its rows lie two or four times in the 128 lanes, and each copy's thread takes that share of a block's places (zeros stand in P
// for the others), with a maximum and a sum of its own.  The products cost the same, and the chain S -> weights -> P is half or a quarter as long.
// TMEM: S / P (128 columns, P overwrites S in place) and O (128 columns) per group: all of it.
//
// Work: KV blocks of all (sequence, KV head, tile pair) items in one line, cut into equal pieces, one per SM: a long context is shared by many SMs, short ones
// fill one, whatever the mix.  The cut goes by lengths that only the device knows (a captured launch may be replayed with other ones), so every block works out
// its piece from the lengths, and one warp hands its segments to the others.  A piece that holds an item's part leaves the part's output (f32, normalised) and base-2
// logarithm of its sum in a workspace; a second launch joins the parts in the order of their blocks.
//
// P is rounded to bf16 for the second product (the tensor cores' operand type; sums stay f32): at most 2^-8 of each weight.
//
// What it measures (kernel, then join; measured copy bandwidth 6.53 TB/s): 32 sequences of 16 nodes on 8192 places at most, 32 query and 8 KV heads of 128: 126 + 5 us, 5.7 TB/s of K and V;
// 4 of 32 nodes on 65536: 138 + 8 us, 6.0 TB/s; there the stream of K and V bounds it.  64 trees of 63 nodes on 2048, 32 query and 4 KV heads: 133 + 11 us; there it is the chain
// S -> weights -> P -> product of the two groups (the tensor pipe is busy for a third of the time).  One sequence of 5 nodes on 1500: 10 + 3 us, all of it starts and ends.
// A segment costs about 5000 cycles beside its blocks (barrier of the groups 400, factors 750, last product 900, rows 2900), the segments' handing out 4000 at the kernel's begin.
#include "sm100.cuh"
#include "host_common.h"
#include <algorithm>

namespace gb {

constexpr int kTaThreads = 384;     // warps 0-3, 4-7: softmax groups; 8: K / V loads; 9: MMA; 10: Q loads; 11: segments
constexpr int kTaTiles = 7;         // 32 KB tiles of shared memory: one or two of Q, one in which rows are joined and put in order, the rest is the ring
// Items of as many blocks or fewer are not cut (no parts to write and join).  64 sequences of 8 nodes on 500 places each: 24 us, cut 29; on 10 to 500: 24.4, cut 26.4; on 10 to
// 1000 (8 blocks): 35.4, cut 33.6.  With a window most items have the same length, and whole ones are faster where the last round of the SMs leaves half of them idle at most.
// Whole / cut in us, windows of 1000, 12 nodes, heads of 128, on 148 SMs: 80 items 23 / 24, 144 24 / 31, 150 41 / 32, 200 42 / 38, 294 44 / 48, 304 59 / 51, 400 61 / 61, 592 79 / 83,
// 800 114 / 108, 1024 135 to 140 / 137; heads of 64: 144 20 / 24, 150 33 / 25, 294 38 / 41, 304 50 / 44; windows of 512, heads of 128: 144 20 / 24, 150 29 / 25, 294 36 / 40, 400 50 / 47, 800 94 / 80, 1024 109 / 103.
constexpr int kTaWhole = 4, kTaWholeWindow = 12;
constexpr int kTaSegs = 4;          // segments handed out ahead
constexpr int kTaSide = 3 * 1024;   // bytes beside the tiles
constexpr int kTaSmem = kTaTiles * 32768 + kTaSide;      // (all there is)

struct TreeAttnArgs {
  const int* cu_q; const int* kv_len; const int* block_table; const unsigned long long* mask; const int* positions;
  int n_seqs, max_pages, page_size, words, window, hq, hkv, total_tokens;
  int max_nodes;
  int cap;                           // places that a row of the block table has room for
  int G, tpt;                        // query heads per KV head; nodes per tile
  int pair;                          // tiles per item: 1 or 2
  int fold;                          // copies of the rows in a tile: 1, 2 or 4 (pair = 1, and at most 128 / fold rows in any sequence)
  int whole;                         // items are not cut (short contexts): no parts
  int head;                          // cost of an item's start and end, in blocks of one tile
  __nv_bfloat16* out;                // [T, hq, DV]
  float* part_o; float* part_lse;    // [2 * grid][pair * 128][DV], [2 * grid][pair * 128]
  int4* part_of;                     // [grid]: the item that begins in a piece and goes on behind it {parts, first part's slot | KV head << 16, its first token, nodes from there on};
                                     // parts = 0: none
  const __nv_bfloat16* v_cache; long num_slots;
  KernelStatus* status;
};

// Shape of a sequence's work.
struct TaSeq {
  int begin, nodes, len, ctx, first, blocks, units, tiles, pairs, items, head;
  __device__ __forceinline__ void load(const TreeAttnArgs& a, int s) {
    const int tpt = a.tpt;
    begin = min(max(a.cu_q[s], 0), a.total_tokens);
    const int all = max(min(a.cu_q[s + 1], a.total_tokens) - begin, 0);
    nodes = min(all, a.max_nodes);                     // (the bounds on the line and the workspace go by max_nodes)
    const int kv = a.kv_len[s];
    len = max(0, min(kv, a.cap));
    ctx = max(0, kv - all);
    first = a.window > 0 ? max(0, ctx - a.window + 1) / 128 : 0;
    blocks = max(0, (len + 127) / 128 - first);
    units = a.whole ? 1 : max(1, blocks);
    tiles = (nodes + tpt - 1) / tpt;
    pairs = (tiles + a.pair - 1) >> (a.pair - 1);
    items = pairs * a.hkv;
    head = a.whole ? 0 : a.head;
  }
  // The line that is cut: an item takes `head` (its start and its end, in blocks of one tile) and, per block, one for each of its tiles.
  __device__ __forceinline__ int cost(const TreeAttnArgs& a) const { return a.whole ? items : a.hkv * (pairs * head + tiles * units); }
};

// The line is cut into `active` pieces that differ by one at most.  (The whole line is shorter than 2^31: the host sees to that.  64-bit divisions would cost more than all else here.)
struct TaPiece {
  int total, active, each, more;          // each: length of a piece; the first `more` are longer by one
  int pos, left, seq, item, off;          // off: place in the item
  __device__ __forceinline__ int begin(int c) const { return c * each + min(c, more); }
  __device__ __forceinline__ int piece_of(int at) const { return at < more * (each + 1) ? at / (each + 1) : more + (at - more * (each + 1)) / each; }
};

// The part of an item that a block works on.
struct TaSeg {
  TaSeq q;
  int seq, item, kvh, tile, n_tiles;      // first tile, 1 or 2 of them
  int lo, n;                              // KV blocks [lo, lo + n) of the sequence
  bool full;                              // all of the item's blocks
  int slot;                               // of its part in the workspace
  int parts;                              // the item begins here and is cut: into so many parts
};

struct TaWalk {
  TaPiece p;
  TaSeq q;
  int nth;
  __device__ __forceinline__ bool next(const TreeAttnArgs& a, TaSeg& s) {
    while (p.left > 0) {
      const int kvh = p.item / q.pairs, tile = (p.item - kvh * q.pairs) * a.pair, n_tiles = min(a.pair, q.tiles - tile), w = a.whole ? 1 : n_tiles;
      const int cost = q.head + w * q.units;
      const int take = min(cost - p.off, p.left);
      // block b belongs to the piece that holds place head + b * w of the item
      auto block_at = [&](int o) { return o <= q.head ? 0 : (o - q.head + w - 1) >> (w - 1); };
      const int b0 = block_at(p.off), b1 = block_at(p.off + take);
      const int pos = p.pos - p.off;                               // the item's
      s.q = q; s.seq = p.seq; s.item = p.item; s.kvh = kvh; s.tile = tile; s.n_tiles = n_tiles;
      p.left -= take; p.pos += take; p.off += take;
      if (p.off == cost) {
        p.off = 0;
        if (++p.item == q.items) {
          p.item = 0;
          if (p.left > 0) do { ++p.seq; q.load(a, p.seq); } while (q.items == 0 && p.seq + 1 < a.n_seqs);
        }
      }
      if (b1 == b0) continue;                                      // (the piece ends or begins beside the item's first or last block)
      s.full = b0 == 0 && b1 == s.q.units;
      s.lo = s.q.first + (a.whole ? 0 : b0); s.n = a.whole ? s.q.blocks : min(b1 - b0, s.q.blocks - b0);
      s.slot = 2 * (int)blockIdx.x + (nth++ == 0 ? 0 : 1);
      s.parts = 0;
      if (!s.full && b0 == 0) {
        const int last = pos + s.q.head + (s.q.units - 1) * w;     // the place of the item's last block; the piece that holds it is the last one that begins there or before
        s.parts = p.piece_of(last) - (int)blockIdx.x + 1;
      }
      return true;
    }
    return false;
  }
};

__device__ __forceinline__ bool bar256_and(bool pred) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.and.pred p, 2, 256, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(r) : "r"((uint32_t)pred) : "memory");
  return r != 0;
}

// A bounded wait: polls, and then the one that looks at the clock, which is not worth its place in the instruction cache at each wait.
__device__ __noinline__ bool ta_wait_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag, KernelStatus* st, int where, int aux) {
  return mbar_wait(bar, parity, abort_flag, st, where, aux);
}
__device__ __forceinline__ bool ta_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, KernelStatus* st, int where, int aux) {
#pragma unroll 1
  for (int it = 0; it < 256; ++it) if (mbar_try_wait(bar, parity)) return true;
  return ta_wait_long(bar, parity, abort_flag, st, where, aux);
}

// Bits [at, at + 32) of a node's mask row (at may be negative: zeros in front).
__device__ __forceinline__ uint32_t mask_bits(const unsigned long long* row, int words, int at) {
  if (at <= -32 || at >= words * 64) return 0;
  if (at < 0) return (uint32_t)row[0] << -at;
  const int w = at >> 6, sh = at & 63;
  unsigned long long v = row[w] >> sh;
  if (sh > 32 && w + 1 < words) v |= row[w + 1] << (64 - sh);
  return (uint32_t)v;
}
// Of the bits of 32 tree nodes those with a position of `lo` or more (positions: of the first of them; `n` have one, of `last` at most).  Trees are seldom as deep as a window: not inlined.
__device__ __noinline__ uint32_t near_bits(uint32_t bits, const int* positions, int n, int lo, int last) {
#pragma unroll 1
  for (uint32_t m = bits; m; m &= m - 1) {
    const int i = __ffs(m) - 1;
    if (i >= n || min(positions[i], last) < lo) bits &= ~(1u << i);
  }
  return bits;
}
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; }

// 128 threads of softmax group g.
__device__ __forceinline__ void bar_group(int g) { asm volatile("bar.sync %0, 128;" :: "r"(3 + g) : "memory"); }

// Two floats in a 64-bit register: one issue slot adds both.
__device__ __forceinline__ uint64_t pair2(float lo, float hi) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi)); return r; }
__device__ __forceinline__ void unpair2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

// One block's step of a softmax thread: NC = 128 / FOLD of the block's scores, from column `at` on.  Returns the factor that the sum and O were scaled by in `l`, `m`.
template <int DV, int FOLD>
__device__ __forceinline__ void softmax_step(uint32_t s_t, int fold, bool first, bool edge, const uint32_t* see, float& m, float& l) {
  constexpr float kTau = 8.0f;         // O and the sum are rescaled only where a row's maximum has grown by more than 2^kTau
  constexpr int NC = 128 / FOLD;
  const uint32_t s_at = s_t + fold * NC;
  float sv[32];
  auto load = [&](int c) {                                         // scores of columns c to c + 31 of the lane's share
    tmem_ld_x32(s_at + c, reinterpret_cast<uint32_t*>(sv));
    tc_wait_ld();
    if (edge) {
#pragma unroll
      for (int i = 0; i < 32; ++i) if (!((see[c >> 5] >> i) & 1)) sv[i] = -INFINITY;
    }
  };
  // 32 columns at a time, in loops: unrolled they are 5% to 20% slower, as the SM's instruction cache does not hold the kernel then.  (The scores are read twice: all 128
  // do not fit the registers.)
  float top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < NC; c += 32) {
    load(c);
    float mx[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 32; ++i) mx[i & 3] = fmaxf(mx[i & 3], sv[i]);
    top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
  }
  float alpha = 1.0f;
  const bool grow = top > m + kTau || (m == -INFINITY && top > -INFINITY);
  if (grow) { alpha = fast_exp2(m - top); m = top; }
  if (!first && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
    for (int c = 0; c < DV / 32; ++c) {
      uint32_t o[32];
      tmem_ld_x32(s_t + 128 + c * 32, o);
      tc_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
      tmem_st_x32(s_t + 128 + c * 32, o);
    }
  }
  const float ref = m == -INFINITY ? 0.f : m;
  const uint64_t ref2 = pair2(-ref, -ref);
  uint64_t rs2[2] = {pair2(0.f, 0.f), pair2(0.f, 0.f)};
  float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int c = 0; c < NC; c += 32) {
    if (NC > 32) load(c);
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      // (in pairs where a thread has all 128 columns: 3% on wide trees; with folded rows it costs as much)
      float p0, p1;
      if constexpr (FOLD == 1) {
        unpair2(add2(pair2(sv[2 * i], sv[2 * i + 1]), ref2), p0, p1);
        p0 = fast_exp2(p0); p1 = fast_exp2(p1);
        rs2[i & 1] = add2(rs2[i & 1], pair2(p0, p1));
      } else {
        p0 = fast_exp2(sv[2 * i] - ref); p1 = fast_exp2(sv[2 * i + 1] - ref);
        rs[i & 1] += p0; rs[2 + (i & 1)] += p1;
      }
      pk[i] = pack_bf16x2(p0, p1);
    }
    tmem_st_x16(s_t + (fold * NC + c) / 2, pk);
  }
  if constexpr (FOLD > 1) {                                        // the other copies' places
    uint32_t z[NC / 2];
#pragma unroll
    for (int i = 0; i < NC / 2; ++i) z[i] = 0;
#pragma unroll
    for (int f = 1; f < FOLD; ++f) {
      const int x = (fold + f) & (FOLD - 1);
      if constexpr (FOLD == 4) tmem_st_x16(s_t + x * 16, z);
      else tmem_st_x32(s_t + x * 32, z);
    }
  }
  if constexpr (FOLD == 1) unpair2(add2(rs2[0], rs2[1]), rs[0], rs[2]);
  l = l * alpha + ((rs[0] + rs[1]) + (rs[2] + rs[3]));
  tc_wait_st();
}

template <int DK, int DV, int FOLD>
__global__ void __launch_bounds__(kTaThreads, 1)
tree_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const TreeAttnArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {                                   // (the swizzled tiles need it; the compiler is asked for it)
    pdl_wait();
    if (threadIdx.x == 0) {
      report_status(a.status, ST_BAD_ARG, 850);
      if (a.part_of != nullptr) a.part_of[blockIdx.x] = make_int4(0, 0, 0, 0);
    }
    return;
  }
  constexpr uint32_t kQ = 256 * DK, kSlot = 256 * (DK > DV ? DK : DV), kStage = 32768;
  uint8_t* sQ = smem;                                             // pair x [128 rows] (64-column halves of 128 B, swizzled)
  uint8_t* s_stage = smem + a.pair * kQ;                          // [2 groups][128 lanes] of 128 B
  uint8_t* ring = smem + a.pair * kQ + kStage;
  const int slots = min(10, (int)((kTaTiles * 32768 - a.pair * kQ - kStage) / kSlot));
  uint64_t* bars = (uint64_t*)(smem + kTaTiles * 32768);
  uint64_t* q_full = bars; uint64_t* q_empty = bars + 1;
  uint64_t* s_full = bars + 2; uint64_t* p_ready = bars + 4; uint64_t* o_full = bars + 6;      // [2] each, by group
  uint64_t* t_full = bars + 8; uint64_t* t_empty = bars + 18;                                  // [10] each
  uint64_t* g_full = bars + 28; uint64_t* g_empty = bars + 32;                                 // [kTaSegs] each
  uint32_t* tmem_slot = (uint32_t*)(bars + 36);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  int* s_odd = (int*)(tmem_slot + 2);                             // [16] places of the segment whose value rows are not finite, as bits: tree nodes; context from the window's begin on
  float* s_m = (float*)(bars + 46);                               // [2][128] maxima and sums of the groups' lanes
  float* s_l = s_m + 256;
  unsigned short* s_row = (unsigned short*)(s_l + 256);           // [128] row of a tile: node << 8 | head of the group
  TaSeg* s_seg = (TaSeg*)(s_row + 128);                         // [kTaSegs]; n_tiles = 0: no more
  static_assert(46 * 8 + 2048 + 256 + kTaSegs * sizeof(TaSeg) <= kTaSide, "shared memory");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1); mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_ready[i], 128); mbar_init(&o_full[i], 1); }
    for (int i = 0; i < 10; ++i) { mbar_init(&t_full[i], 1); mbar_init(&t_empty[i], 1); }
    for (int i = 0; i < kTaSegs; ++i) { mbar_init(&g_full[i], 1); mbar_init(&g_empty[i], 4); }      // (a softmax thread and the warps 8, 9, 10 give a segment back)
    *abort_flag = 0;
    for (int i = 0; i < 16; ++i) s_odd[i] = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
  }
  if (threadIdx.x < 128) s_row[threadIdx.x] = (unsigned short)((int)threadIdx.x / a.G << 8 | (int)threadIdx.x % a.G);
  if (warp == 9) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem_base = *tmem_slot;
  const int G = a.G, tpt = a.tpt;

  if (warp == 11) {
    // ---------------------------------------------------------------- segments: this block's piece of the line, handed to the other warps
    const int per = (a.n_seqs + 31) / 32, i0 = min(a.n_seqs, lane * per), i1 = min(a.n_seqs, i0 + per);
    TaWalk walk;
    walk.nth = 0;
    int mine = 0;
#pragma unroll 2
    for (int i = i0; i < i1; ++i) { TaSeq q; q.load(a, i); mine += q.cost(a); }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += x; }
    TaPiece& p = walk.p;
    p.total = __shfl_sync(0xffffffffu, incl, 31);
    // at least two blocks a piece: a part costs more to write and join than a block to work on (and every piece inside an item must get a block of it)
    p.active = min((int)gridDim.x, a.whole ? p.total : max(p.total / (2 * a.pair), min(p.total, 1)));
    p.left = 0;
    if ((int)blockIdx.x < p.active) {
      p.each = p.total / p.active; p.more = p.total - p.each * p.active;
      const int lo = p.begin(blockIdx.x);
      // the lane whose sequences hold the place, then the sequence
      const int src = __ffs(__ballot_sync(0xffffffffu, incl > lo)) - 1;
      int at = __shfl_sync(0xffffffffu, incl - mine, src);
      p.seq = min(a.n_seqs, src * per);
      while (true) {
        walk.q.load(a, p.seq);
        const int c = walk.q.cost(a);
        if (lo < at + c) break;
        at += c; ++p.seq;
      }
      const int in_seq = lo - at;
      const TaSeq& q = walk.q;
      const int head_cost = a.whole ? q.pairs : q.pairs * q.head + q.tiles * q.units;          // a KV head's; all of its pairs but the last cost the same
      const int kvh = in_seq / head_cost, in_head = in_seq - kvh * head_cost, pair_cost = a.whole ? 1 : q.head + a.pair * q.units;
      const int pair = min(in_head / pair_cost, q.pairs - 1);
      p.item = kvh * q.pairs + pair; p.off = in_head - pair * pair_cost;
      p.pos = lo; p.left = p.begin(blockIdx.x + 1) - lo;
    }
    if (lane == 0) {
      if (a.part_of != nullptr) a.part_of[blockIdx.x] = make_int4(0, 0, 0, 0);
      for (int k = 0;; ++k) {
        const int i = k % kTaSegs;
        TaSeg s;
        const bool more = walk.next(a, s);
        if (!more) s.n_tiles = 0;
        if (!ta_wait(&g_empty[i], ((k / kTaSegs) & 1) ^ 1, abort_flag, a.status, 840, k)) break;
        s_seg[i] = s;
        mbar_arrive(&g_full[i]);
        if (!more) break;
        if (s.parts > 0) a.part_of[blockIdx.x] = make_int4(s.parts, s.slot | s.kvh << 16, s.q.begin + s.tile * tpt, s.q.nodes - s.tile * tpt);
      }
    }
  } else if (warp == 8) {
    // ---------------------------------------------------------------- K and V: the lanes fetch and issue a page each
    const int ppb = 128 / a.page_size;
    const uint32_t page_bytes = (uint32_t)a.page_size * 128;
    int slot = 0; uint32_t ph = 0;
    bool ok = true;
    for (int k = 0; ok; ++k) {
      const int i = k % kTaSegs;
      ok = __all_sync(0xffffffffu, ta_wait(&g_full[i], (k / kTaSegs) & 1, abort_flag, a.status, 801, k));
      if (!ok || s_seg[i].n_tiles == 0) break;
      const int lo = s_seg[i].lo, n = s_seg[i].n, kvh = s_seg[i].kvh, len = s_seg[i].q.len;
      const int* bt = a.block_table + (size_t)s_seg[i].seq * a.max_pages;
      __syncwarp();
      if (lane == 0) mbar_arrive(&g_empty[i]);
      const int last_page = (len + a.page_size - 1) / a.page_size - 1;
      int page = n > 0 && lane < ppb ? bt[min(lo * ppb + lane, last_page)] : 0;
      for (int j = 0; j < n && ok; ++j) {
        const int now = page;
        if (j + 1 < n && lane < ppb) page = bt[min((lo + j + 1) * ppb + lane, last_page)];      // (pages behind the end: the last one again; nothing of them counts)
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          ok = ok && ta_wait(&t_empty[slot], ph ^ 1, abort_flag, a.status, 800, j);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const int D = kv ? DV : DK;
          const CUtensorMap* tm = kv ? &tmV : &tmK;
          if (lane == 0) mbar_expect_tx(&t_full[slot], 256u * D);
          __syncwarp();
          if (lane < ppb) {
            uint8_t* dst = ring + slot * kSlot + lane * page_bytes;
            tma_load_3d(dst, tm, &t_full[slot], 0, kvh, now * a.page_size);
            if (D > 64) tma_load_3d(dst + 16384, tm, &t_full[slot], 64, kvh, now * a.page_size);
          }
          if (++slot == slots) { slot = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 10) {
    if (lane == 0) {
      uint32_t ph = 0;
      for (int k = 0;; ++k) {
        const int i = k % kTaSegs;
        if (!ta_wait(&g_full[i], (k / kTaSegs) & 1, abort_flag, a.status, 811, k) || s_seg[i].n_tiles == 0) break;
        const int n = s_seg[i].n, n_tiles = s_seg[i].n_tiles, kvh = s_seg[i].kvh, begin = s_seg[i].q.begin + s_seg[i].tile * tpt;
        mbar_arrive(&g_empty[i]);
        if (n <= 0) continue;
        if (!ta_wait(q_empty, ph ^ 1, abort_flag, a.status, 810, k)) break;
        mbar_expect_tx(q_full, (uint32_t)(2 * DK * G * tpt) * FOLD * n_tiles);
        for (int t = 0; t < n_tiles * FOLD; ++t) {
          uint8_t* dst = FOLD > 1 ? sQ + t * (128 / FOLD) * 128 : sQ + t * kQ;      // a copy of the rows, or the second tile
          const int tok = begin + (FOLD > 1 ? 0 : t * tpt);
          tma_load_3d(dst, &tmQ, q_full, 0, kvh * G, tok);
          if constexpr (DK > 64) tma_load_3d(dst + 16384, &tmQ, q_full, 64, kvh * G, tok);
        }
        ph ^= 1;
      }
    }
  } else if (warp == 9) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = make_idesc(128, 128, 1, 1, 0, 0);
      constexpr uint32_t idesc_o = make_idesc(128, DV, 1, 1, 0, 1);            // B (= V) is MN-major
      const uint32_t q_addr = smem_u32(sQ), r_addr = smem_u32(ring);
      uint32_t q_ph = 0, p_ph = 0;                                             // p_ph: a bit per group
      int k_slot = 0, v_slot = 1;                                              // ring places of the next K and V tile: every other one
      uint32_t k_ph = 0, v_ph = 0;
      auto step_on = [&](int& slot, uint32_t& ph) { slot += 2; if (slot >= slots) { slot -= slots; ph ^= 1; } };
      bool ok = true;
      for (int k = 0; ok; ++k) {
        const int sg = k % kTaSegs;
        if (!ta_wait(&g_full[sg], (k / kTaSegs) & 1, abort_flag, a.status, 824, k) || s_seg[sg].n_tiles == 0) break;
        const bool two = s_seg[sg].n_tiles == 2;
        const int n = s_seg[sg].n, steps = two ? 2 * n : n;
        mbar_arrive(&g_empty[sg]);
        if (n <= 0) continue;
        if (!ta_wait(q_full, q_ph, abort_flag, a.status, 820, k)) break;
        q_ph ^= 1;
        // Step i: group i & 1; KV block i, or i / 2 where the groups share the blocks.  S runs two steps ahead: S of step i + 2 overwrites P of step i, which the pipe, running
        // this thread's MMAs in order, has read by then; and its arrival tells that O holds all of the group's earlier products.
        for (int j = 0; j < steps + 2 && ok; ++j) {
          const int p = j & 1;
          if (j >= 2) {
            const int i = j - 2;
            if (!ta_wait(&p_ready[p], (p_ph >> p) & 1, abort_flag, a.status, 822, i)) { ok = false; break; }
            p_ph ^= 1u << p;
            if (!ta_wait(&t_full[v_slot], v_ph, abort_flag, a.status, 823, i)) { ok = false; break; }
            tc_fence_after();
            const uint64_t vd = make_sdesc_sw128_mn(r_addr + v_slot * kSlot, 16384);
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)                                     // (the group's first block of the segment: O starts from zero)
              mma_f16_ts(tmem_base + p * 256 + 128, tmem_base + p * 256 + ks * 8, sdesc_at(vd, ks * 2048), idesc_o, (i >= 2 || ks > 0) ? 1u : 0u);
            if (!two || p) { tc_commit(&t_empty[v_slot]); step_on(v_slot, v_ph); }
            if (j >= steps) tc_commit(&o_full[p]);                             // the group's last block
          }
          if (j < steps) {
            if (!ta_wait(&t_full[k_slot], k_ph, abort_flag, a.status, 821, j)) { ok = false; break; }
            tc_fence_after();
            const uint64_t qd = make_sdesc_sw128(q_addr + (two && p ? kQ : 0)), kd = make_sdesc_sw128(r_addr + k_slot * kSlot);
#pragma unroll
            for (int ks = 0; ks < DK / 16; ++ks) {
              const uint32_t off = (ks >> 2) * 16384 + (ks & 3) * 32;
              mma_f16_ss(tmem_base + p * 256, sdesc_at(qd, off), sdesc_at(kd, off), idesc_s, ks > 0 ? 1u : 0u);
            }
            tc_commit(&s_full[p]);
            if (!two || p) { tc_commit(&t_empty[k_slot]); step_on(k_slot, k_ph); }
            if (j == steps - 1) tc_commit(q_empty);
          }
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax: one TMEM lane per thread
    const int g = warp >> 2;                                                   // group
    const int r = threadIdx.x & 127, fold = r / (128 / FOLD), rr = r % (128 / FOLD);      // lane; copy of the rows; row (fold is the same for a warp)
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_t = tmem_base + g * 256 + lane_off;
    const int t_local = s_row[rr] >> 8;
    uint32_t s_ph = 0, o_ph0 = 0, o_ph1 = 0;
    uint32_t t0 = 0;                                                           // ring tiles in front of the segment
    bool ok = bar256_and(ta_wait(&g_full[0], 0, abort_flag, a.status, 834, 0));
    for (int k = 0; ok && s_seg[k % kTaSegs].n_tiles > 0; ++k) {
      const TaSeg& s = s_seg[k % kTaSegs];
      const bool two = FOLD == 1 && s.n_tiles == 2;
      const int n = s.n, ctx = s.q.ctx, len = s.q.len, blk0 = s.lo;
      const int node = (s.tile + (two ? g : 0)) * tpt + t_local;               // of the sequence
      const bool live = t_local < tpt && node < s.q.nodes;
      const bool warp_live = __any_sync(0xffffffffu, live);
      const int tok = s.q.begin + min(node, s.q.nodes - 1);
      const unsigned long long* mrow = a.mask + (size_t)tok * a.words;
      const int last_pos = ctx + s.q.nodes - 1;                                // nodes have positions ctx to this
      const int lo = a.window > 0 ? min(max(a.positions[tok], ctx), last_pos) - a.window + 1 : 0;      // first position that the row sees
      const int win0 = ctx - a.window + 1, win1 = a.window > 0 ? win0 + s.q.nodes - 1 : 0;         // places in front of win0 are out of every row's window, those in front of win1 out of some row's
      float m = -INFINITY, l = 0.f;
      bool first = true;
      for (int b = two ? 0 : g; b < n && ok; b += two ? 1 : 2) {
        const int kv0 = (blk0 + b) * 128;
        const bool tail = kv0 + 128 > min(ctx, len);                           // tree nodes, or places behind the end
        const bool edge = tail || kv0 < lo;
        uint32_t see[4 / FOLD];
        if (edge) {
#pragma unroll
          for (int c = 0; c < 4 / FOLD; ++c) {
            const int k0 = kv0 + (fold * (4 / FOLD) + c) * 32;
            see[c] = low_bits(ctx - k0) & ~low_bits(lo - k0);
            if (tail) {
              uint32_t nodes = mask_bits(mrow, a.words, k0 - ctx);
              if (lo > ctx && nodes) nodes = near_bits(nodes, a.positions + s.q.begin + k0 - ctx, s.q.nodes - (k0 - ctx), lo, last_pos);
              see[c] = (see[c] | nodes) & low_bits(len - k0);
            }
          }
        }
        ok = __all_sync(0xffffffffu, ta_wait(&s_full[g], s_ph, abort_flag, a.status, 831, b));        // (a warp leaves as one)
        if (!ok) break;
        s_ph ^= 1;
        if ((tail || kv0 < win1) && (!two || g == 0)) {
          // Values of places that some row does not see must be finite: a weight of 0 times them is added.  What is not
          // finite is taken out, noted, and put back at the end for the rows that see it.  (Behind the wait for S, which tells that the products in front are done:
          // in front of it the place's tile before this one may still be on its way, and its barrier two phases from the one waited for.)
          const uint32_t t = t0 + 2 * b + 1;
          ok = __all_sync(0xffffffffu, ta_wait(&t_full[t % slots], (t / slots) & 1, abort_flag, a.status, 830, b));
          // eight threads a row, 16 rows a turn
          constexpr int kTurns = DV / 64;
#pragma unroll 1
          for (int row = r >> 3; ok && row < 128; row += 16) {
            const int at = kv0 + row;
            if (!(at >= min(ctx, len) || at < win1)) continue;
            const uint32_t in = at < len ? 0xffffffffu : 0u;
            uint8_t* w = ring + (t % slots) * kSlot + row * 128 + (((r ^ row) & 7) << 4);
            bool odd = false;
#pragma unroll
            for (int c = 0; c < kTurns; ++c) {
              uint4 v = *reinterpret_cast<uint4*>(w + c * 16384);
              uint32_t* x = reinterpret_cast<uint32_t*>(&v);
              bool put = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                uint32_t keep = in;
                if ((x[e] & 0x7f80u) == 0x7f80u) keep &= 0xffff0000u;
                if ((x[e] & 0x7f800000u) == 0x7f800000u) keep &= 0x0000ffffu;
                put |= keep != 0xffffffffu;
                x[e] &= keep;
              }
              if (put) *reinterpret_cast<uint4*>(w + c * 16384) = v;
              odd |= put;
            }
            const int x = at >= ctx ? at - ctx : at - win0 + 256;              // (the window's begin is cut by fewer places than there are nodes)
            if (odd && at < len && x >= (at >= ctx ? 0 : 256) && x < (at >= ctx ? 256 : 512)) atomicOr(&s_odd[x >> 5], 1 << (x & 31));
          }
          fence_proxy_async_smem();
        }
        if (!ok) break;
        tc_fence_after();
        __syncwarp();
        if (warp_live) softmax_step<DV, FOLD>(s_t, fold, first, edge, see, m, l);
        first = false;
        tc_fence_before();
        mbar_arrive(&p_ready[g]);
      }
      t0 += 2 * n;
      // ---- the segment's rows.  Two tiles: each group writes its own.  One tile: both groups (and all copies) hold a share of every row, and each group
      // writes half of the columns.
      const int own = two ? g : 0;
      const bool both = !two && n > 1;                                         // accumulator 1 holds something of this group's rows too
      float w0, w1 = 0.f, lse;                                                 // factors of the lane's accumulators
      s_m[g * 128 + r] = m;
      s_l[g * 128 + r] = l;
      ok = bar256_and(ok);                                                     // all 256 threads leave together
      if (!ok) break;
      if (two) {
        w0 = l == 0.f ? 0.f : 1.0f / l;
        lse = l == 0.f ? -INFINITY : m + log2f(l);
      } else {
        float ms[2 * FOLD], top = -INFINITY;
#pragma unroll
        for (int x = 0; x < 2 * FOLD; ++x) { ms[x] = s_m[(x / FOLD) * 128 + (x % FOLD) * (128 / FOLD) + rr]; top = fmaxf(top, ms[x]); }
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = 0.f, e0 = 0.f, e1 = 0.f;
#pragma unroll
        for (int x = 0; x < 2 * FOLD; ++x) {                                   // (2^-inf = 0)
          const float e = fast_exp2(ms[x] - ref);
          sum += e * s_l[(x / FOLD) * 128 + (x % FOLD) * (128 / FOLD) + rr];
          if (x == fold) e0 = e;
          if (x == FOLD + fold) e1 = e;
        }
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        w0 = e0 * inv;
        w1 = e1 * inv;
        lse = sum == 0.f ? -INFINITY : ref + log2f(sum);
      }
      uint32_t any_odd = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) any_odd |= (uint32_t)s_odd[i];
      if (n > 0) {
        ok = ta_wait(&o_full[own], own ? o_ph1 : o_ph0, abort_flag, a.status, 832, k);
        if (both) ok = ok && ta_wait(&o_full[1], o_ph1, abort_flag, a.status, 833, k);
        o_ph0 ^= 1;
        if (two || n > 1) o_ph1 ^= 1;
      }
      tc_fence_after();
      const long prow = ((long)s.slot * a.pair + (two ? g : 0)) * 128;         // of the parts: the tile's first
      const bool full = s.full;
      const int first_node = (s.tile + own) * tpt, n_live = min(tpt, s.q.nodes - first_node);
      const long row0 = full ? (long)(s.q.begin + first_node) * a.hq + s.kvh * G : prow;
      constexpr int kC = DV / 32;
      const int c0 = !two && g == 1 ? kC / 2 : 0, c1 = !two && g == 0 ? kC / 2 : kC;
      uint8_t* st = s_stage + g * 16384;
#pragma unroll 1
      for (int c = c0; c < c1; ++c) {
        float o[32];
        __syncwarp();
        const bool any = ok && n > 0 && warp_live;
        if (any) {
          tmem_ld_x32(tmem_base + lane_off + own * 256 + 128 + c * 32, reinterpret_cast<uint32_t*>(o));
          tc_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = any ? o[i] * w0 : 0.f;
        if (any && both) {
          uint32_t o1[32];
          tmem_ld_x32(tmem_base + lane_off + 256 + 128 + c * 32, o1);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = fmaf(__uint_as_float(o1[i]), w1, o[i]);
        }
        // Through shared memory, where the copies of a row are added up; eight lanes then store a row's 32 columns.
#pragma unroll
        for (int v = 0; v < 8; ++v) *reinterpret_cast<float4*>(st + r * 128 + ((v ^ (r & 7)) << 4)) = make_float4(o[v * 4], o[v * 4 + 1], o[v * 4 + 2], o[v * 4 + 3]);
        if (any_odd && ok && live && fold == 0) {
#pragma unroll 1
          for (int x = 0; x < 512; ++x) {
            if (!((s_odd[x >> 5] >> (x & 31)) & 1)) continue;
            const int at = x < 256 ? ctx + x : win0 + x - 256;
            if (x < 256 ? x >= a.words * 64 || !((mrow[x >> 6] >> (x & 63)) & 1) || (lo > ctx && (x >= s.q.nodes || min(a.positions[s.q.begin + x], last_pos) < lo)) : at < lo) continue;
            const long slot = (long)a.block_table[(size_t)s.seq * a.max_pages + at / a.page_size] * a.page_size + at % a.page_size;
            if (slot < 0 || slot >= a.num_slots) continue;
            const __nv_bfloat16* vr = a.v_cache + ((size_t)slot * a.hkv + s.kvh) * DV + c * 32;
#pragma unroll 1
            for (int i = 0; i < 32; ++i) {
              const float v = __bfloat162float(vr[i]);
              if (!(fabsf(v) < INFINITY)) *reinterpret_cast<float*>(st + r * 128 + (((i >> 2) ^ (r & 7)) << 4) + (i & 3) * 4) += v;
            }
          }
        }
        bar_group(g);
#pragma unroll
        for (int it = 0; it < 8 / FOLD; ++it) {
          const int row = it * 16 + (r >> 3), th = s_row[row];
          const uint8_t* from = st + row * 128 + (((r ^ row) & 7) << 4);
          float4 x = *reinterpret_cast<const float4*>(from);
#pragma unroll
          for (int f = 1; f < FOLD; ++f) {
            const float4 y = *reinterpret_cast<const float4*>(from + f * (128 / FOLD) * 128);
            x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
          }
          if (!ok || (th >> 8) >= n_live) continue;
          const int col = c * 32 + (r & 7) * 4;
          if (full) *reinterpret_cast<uint2*>(a.out + (row0 + (long)(th >> 8) * a.hq + (th & 255)) * DV + col) = make_uint2(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w));
          else *reinterpret_cast<float4*>(a.part_o + (row0 + row) * DV + col) = x;
        }
        bar_group(g);
      }
      if (live && fold == 0 && !full && c0 == 0) a.part_lse[prow + rr] = lse;
      if (any_odd) {
        bar256_and(true);
        if (threadIdx.x < 16) s_odd[threadIdx.x] = 0;
      }
      tc_fence_before();
      ok = ok && ta_wait(&g_full[(k + 1) % kTaSegs], ((k + 1) / kTaSegs) & 1, abort_flag, a.status, 834, k + 1);
      ok = bar256_and(ok);                                                     // both accumulators, s_m, s_l and the segment are free again
      if (threadIdx.x == 0) mbar_arrive(&g_empty[k % kTaSegs]);
    }
  }
  pdl_trigger();                       // a long kernel: its dependents are released at its end
  if (*abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) { tc_fence_after(); tmem_dealloc(tmem_base, 512); }
}

// Joins the parts of the items that were cut: out = sum_i 2^(lse_i - max) O_i / sum_i 2^(lse_i - max), in the order of the parts.  One warp per row: 3 us with few rows, 5 to 11 us where
// each SM leaves one or two parts of 128 or 256 rows (four rows to a warp and one load after the other: 9 to 17 us).
template <int DV>
__global__ void __launch_bounds__(256, 8)
tree_join_kernel(const TreeAttnArgs a) {
  pdl_wait();
  pdl_trigger();
  const int4 of = a.part_of[blockIdx.x];
  const int lane = threadIdx.x & 31, row = blockIdx.y * 8 + (threadIdx.x >> 5);          // of the item
  const int r = row & 127, t_local = r / a.G, node = (row >> 7) * a.tpt + t_local;
  if (of.x <= 0 || t_local >= a.tpt || node >= of.w) return;
  const int slot = of.y & 0xffff, kvh = of.y >> 16;
  constexpr int kV = DV / 32;
  auto at = [&](int i) { return (size_t)(i == 0 ? slot : 2 * ((int)blockIdx.x + i)) * (a.pair * 128) + row; };
  // four parts at a time, all their loads in flight
  float top = -INFINITY, acc[kV], den = 0.f;
#pragma unroll
  for (int v = 0; v < kV; ++v) acc[v] = 0.f;
  for (int i0 = 0; i0 < of.x; i0 += 4) {
    float lse[4], o[4][kV];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      lse[k] = -INFINITY;
#pragma unroll
      for (int v = 0; v < kV; ++v) o[k][v] = 0.f;
      if (i0 + k >= of.x) continue;
      lse[k] = a.part_lse[at(i0 + k)];
      const float* p = a.part_o + at(i0 + k) * DV + lane * kV;
      if constexpr (kV == 4) { const float4 x = *reinterpret_cast<const float4*>(p); o[k][0] = x.x; o[k][1] = x.y; o[k][2] = x.z; o[k][3] = x.w; }
      else { const float2 x = *reinterpret_cast<const float2*>(p); o[k][0] = x.x; o[k][1] = x.y; }
    }
    float m = top;
#pragma unroll
    for (int k = 0; k < 4; ++k) m = fmaxf(m, lse[k]);
    const float ref = m == -INFINITY ? 0.f : m, scale = exp2f(top - ref);      // (nothing so far: 0)
    top = m;
#pragma unroll
    for (int v = 0; v < kV; ++v) acc[v] *= scale;
    den *= scale;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float w = exp2f(lse[k] - ref);
#pragma unroll
      for (int v = 0; v < kV; ++v) acc[v] += lse[k] == -INFINITY ? 0.f : w * o[k][v];
      den += w;
    }
  }
  const float inv = den == 0.f ? 0.f : 1.0f / den;
  uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + ((size_t)(of.z + node) * a.hq + kvh * a.G + (r - t_local * a.G)) * DV + lane * kV);
#pragma unroll
  for (int v = 0; v < kV / 2; ++v) dst[v] = pack_bf16x2(acc[2 * v] * inv, acc[2 * v + 1] * inv);
}

template <int DK, int DV, int FOLD>
static int tree_attn_launch(const void* q, long q_ts, const void* k_cache, const void* v_cache, TreeAttnArgs a, int grid, cudaStream_t stream) {
  const int G = a.G, tpt = a.tpt;
  CUtensorMap tmQ, tmK, tmV;
  {
    uint64_t dims[3] = {DK, (uint64_t)a.hq, (uint64_t)a.total_tokens};
    uint64_t strides[2] = {DK * 2, (uint64_t)q_ts * 2};
    uint32_t box[3] = {64, (uint32_t)G, (uint32_t)tpt};
    if (make_tmap(&tmQ, q, TM_BF16, 3, dims, strides, box, TM_SW_128)) return -1;
  }
  {
    uint64_t dk[3] = {DK, (uint64_t)a.hkv, (uint64_t)a.num_slots}, dv[3] = {DV, (uint64_t)a.hkv, (uint64_t)a.num_slots};
    uint64_t sk[2] = {DK * 2, (uint64_t)a.hkv * DK * 2}, sv[2] = {DV * 2, (uint64_t)a.hkv * DV * 2};
    uint32_t box[3] = {64, 1, (uint32_t)a.page_size};
    if (make_tmap(&tmK, k_cache, TM_BF16, 3, dk, sk, box, TM_SW_128)) return -1;
    if (make_tmap(&tmV, v_cache, TM_BF16, 3, dv, sv, box, TM_SW_128)) return -1;
  }
  static bool attr[64];
  int dev = 0;
  GB_CUDA_OK(cudaGetDevice(&dev));
  if (dev > 63 || !attr[dev]) {
    GB_CUDA_OK(cudaFuncSetAttribute(tree_attn_kernel<DK, DV, FOLD>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTaSmem));
    if (dev < 64) attr[dev] = true;
  }
  launch_k(tree_attn_kernel<DK, DV, FOLD>, grid, kTaThreads, kTaSmem, stream, tmQ, tmK, tmV, a);
  GB_CUDA_OK(cudaGetLastError());
  if (!a.whole) {
    launch_k(tree_join_kernel<DV>, dim3(grid, a.pair * 128 / a.fold / 8), 256, 0, stream, a);
    GB_CUDA_OK(cudaGetLastError());
  }
  return 0;
}

}  // namespace gb

using namespace gb;

// Blocks of the launch, how the rows lie in a tile, and whether the items stay whole: bounds by what the host knows (at most max_pages pages and max_nodes nodes a
// sequence).
static int tree_attn_grid(int n_seqs, int max_pages, int page_size, int max_nodes, int hq, int hkv, int window, int* pair, int* fold, int* whole) {      // 0: too much work for 32-bit places
  const int G = hq / hkv;
  const long rows = (long)max_nodes * G;
  *fold = rows <= 32 ? 4 : rows <= 64 ? 2 : 1;
  const int tpt = 128 / *fold / G, tiles = (max_nodes + tpt - 1) / tpt;
  *pair = tiles > 1 ? 2 : 1;
  long blocks = std::max(1l, ((long)max_pages * page_size + 127) / 128);
  if (window > 0) blocks = std::min(blocks, ((long)window + max_nodes + 126) / 128 + 1);
  const long items = (long)n_seqs * hkv * ((tiles + *pair - 1) / *pair);
  const long idle = sm_count() - 1 - (items + sm_count() - 1) % sm_count();      // SMs without an item in the last round
  *whole = blocks <= kTaWhole || (window > 0 && blocks <= kTaWholeWindow && 2 * idle <= sm_count());
  if (items * *pair * (blocks + 8) > 1l << 30) return 0;
  return (int)std::max(1l, std::min((long)sm_count(), *whole ? items : (items * blocks + 1) / 2));
}

// Floats of the workspace that gb_tree_attn wants; 0: not for gb_tree_attn.
GB_API int gb_tree_attn_workspace(int n_seqs, int max_pages, int page_size, int max_nodes, int hq, int hkv, int dv, int window) {
  int pair, fold, whole;
  const long grid = tree_attn_grid(n_seqs, max_pages, page_size, max_nodes, hq, hkv, window, &pair, &fold, &whole);
  return grid == 0 ? 0 : whole ? 4 : (int)((grid + 1) / 2 * 8 + 2 * grid * pair * 128 * (dv + 1));          // (at most 148 * 2 * 2 * 128 rows)
}

GB_API int gb_tree_attn(const void* q, long q_ts, const void* k_cache, const void* v_cache, void* out, float* workspace, const int* cu_q, const int* kv_len,
                        const int* block_table, int max_pages, int page_size, const void* mask, int words, const int* positions, int n_seqs, long num_slots,
                        int tokens, int max_nodes, int hq, int hkv, int dk, int dv, int window, void* status, cudaStream_t stream) {
  if (tokens <= 0 || n_seqs <= 0) return 0;
  if ((dk != 64 && dk != 128) || (dv != 64 && dv != 128)) return fail("tree_attn: heads of 64 or 128 columns%s");
  if (hq < 1 || hkv < 1 || hq % hkv || hq / hkv > 128) return fail("tree_attn: bad head counts%s");
  if (page_size < 8 || page_size > 128 || 128 % page_size) return fail("tree_attn: page_size must be 8..128 and divide 128%s");
  if (max_nodes < 1 || words < 1 || max_pages < 0 || window < 0 || num_slots < 1 || hkv > 32767) return fail("tree_attn: bad sizes%s");
  if (window > 0 && positions == nullptr) return fail("tree_attn: a window needs the nodes' positions%s");
  TreeAttnArgs a;
  memset(&a, 0, sizeof(a));
  const int grid = tree_attn_grid(n_seqs, max_pages, page_size, max_nodes, hq, hkv, window, &a.pair, &a.fold, &a.whole);
  if (grid == 0) return fail("tree_attn: too much work for one call%s");
  a.cu_q = cu_q; a.kv_len = kv_len; a.block_table = block_table; a.mask = (const unsigned long long*)mask; a.positions = positions; a.n_seqs = n_seqs;
  a.max_pages = max_pages; a.page_size = page_size; a.words = words; a.window = window; a.hq = hq; a.hkv = hkv; a.total_tokens = tokens;
  a.head = a.pair == 2 ? 6 : 2;
  a.G = hq / hkv; a.tpt = 128 / a.fold / a.G;
  a.max_nodes = max_nodes; a.cap = (int)std::min((long)max_pages * page_size, 0x7fffffffl);
  a.num_slots = num_slots; a.out = (__nv_bfloat16*)out; a.v_cache = (const __nv_bfloat16*)v_cache; a.status = (KernelStatus*)status;
  if (!a.whole) {
    a.part_of = (int4*)workspace;
    a.part_o = workspace + (grid + 1) / 2 * 8;                     // on a 32-byte boundary
    a.part_lse = a.part_o + 2l * grid * a.pair * 128 * dv;
  }
#define GB_TREE(K, V, F) if (dk == K && dv == V && a.fold == F) return tree_attn_launch<K, V, F>(q, q_ts, k_cache, v_cache, a, grid, stream);
#define GB_TREE_FOLDS(K, V) GB_TREE(K, V, 1) GB_TREE(K, V, 2) GB_TREE(K, V, 4)
  GB_TREE_FOLDS(64, 64)
  GB_TREE_FOLDS(64, 128)
  GB_TREE_FOLDS(128, 64)
  GB_TREE_FOLDS(128, 128)
#undef GB_TREE_FOLDS
#undef GB_TREE
  return fail("tree_attn: no such form%s");
}

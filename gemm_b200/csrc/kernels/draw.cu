// One token per row of logits from a given uniform number, with the row's own temperature T, top-k, top-p and min-p.
//
//   w_i = 2^((x_i - max x) log2(e) / T).  In the order (x descending, id ascending): the first top_k ids; of these the ids that have less than top_p of the
//   mass in front of them; of these the ids with w_i >= min_p.  The draw is the first id, in id order, at which the mass so far exceeds u times the kept mass.
//
// All three filters cut that order at one place, so what is kept is {key > tau} and the first m ids with key = tau.  No sort: tau comes from radix searches.
//
// Masses are whole numbers: w_i is rounded to a multiple of 2^-44 (the rounding moves a border of the draw by 2^-45 of the largest weight).  A row has fewer than 2^20
// ids (eight blocks' shared memory holds no more), so a mass is below 2^64, and every sum is unsigned.  Sums are then exact in any order: the atomics of the histograms, the split over blocks and the order of the warps change nothing, and the
// draw agrees with one in 64-bit floats except where u falls within some 1e-12 of a border (32-bit sums over a vocabulary: a row in a thousand).
// 2^t: table of 2^(j/32) and a polynomial for the rest (P. T. P. Tang, "Table-driven implementation of the exponential function", 1989), in 64-bit floats.
//
// A cluster of up to eight blocks holds a row in its shared memory (bulk copies), so that HBM is read once whatever the number of passes.  Every instruction
// per logit and every step of the whole cluster counts, so most of a row's work is left to one block while the others make room for the next row:
//   top-k         the k-th largest of 4096 maxima of small groups of logits is a lower bound of the k-th largest logit; the logits above it, few more than k,
//                 go to the first block, which finishes alone: by comparing all pairs, or by radix searches if they are many;
//   top-p alone   one pass for all weights and their histogram; then the candidates go to the first block, or, if they are too many, those of the cut's step;
//   neither       one pass for the masses of chunks of ids, and a look at the chunk in which the draw falls.
// Rows that this does not settle (a large top-k, equal logits, likely tokens side by side: each block of a cluster has its share of the 2048 places for candidates, and
// 512 f32 rows of 151936 with top-k 300 take 205 us where 1500 likely tokens are spread over the ids and 880 where they are neighbours, 222 and 1458 with top-k 1000;
// bf16 130 and 398, 144 and 755) take the cluster's path: histograms over 1/16-wide steps below the maximum and over the keys of
// the step that holds the cut, exchanged through distributed shared memory.
//
// What bounds it: instructions (rows are read at a fraction of the bandwidth), and for few rows the chain of the steps.  Cycles of a row of 32003 bf16 logits in one block, another
// one beside it on the SM: load 3000, maxima 2900, top-k bound 3400 to 4300, its candidates 4300 to 8100, the comparisons 6700 or, for 1000 candidates, the searches 18000; top-p: weights and
// histogram 27000 (the weights alone 17000: ten 64-bit operations and some fourteen others a logit), the candidates 4100.  1500 such rows of all kinds: 130 us (96 MB: 15 us
// of bandwidth); 512 f32 rows of 151936: 265 us (48 us); one such row: 9.3 us.
#include "sm100.cuh"
#include "host_common.h"
#include <float.h>
#include <algorithm>

namespace gb {

constexpr int kDrList = 256;               // candidates a warp lists
constexpr int kDrCand = 2048;              // candidates of a row in the first block
constexpr int kDrPairs = 256;              // candidates that are compared with one another
constexpr int kDrPrune = 1000;             // k' at most: a half of the groups or less, so that few logits beyond the k'-th lie above the bound
constexpr int kDrMass = 44;                // fraction bits of a weight
// Rows of as many logits or fewer take half the threads, if there are more of them than fill the GPU: 30000 f32 rows of 1000 602 us, with 512 threads 914; 12000 bf16 rows of
// 2500 527 and 479; 8000 f32 rows of 4000 323 and 324.
constexpr int kDrShort = 2048;
constexpr size_t kDrSmem = 202000;         // bytes of logits that a block holds at most
static_assert(8 * kDrSmem / sizeof(__nv_bfloat16) < 1ull << (64 - kDrMass), "the mass of a row, at most 2^kDrMass for each id, fits 64 bits");

struct DrawArgs {
  const void* logits;
  long ld;
  int rows, vocab, ctas, per;              // blocks per row, ids per block
  const float* u;
  const float* temperature; const int* top_k; const float* top_p; const float* min_p;      // per row; null: the value for all rows
  float temperature_all; int top_k_all; float top_p_all, min_p_all;
  int* out; float* logprob;                // logprob: null = not wanted
  KernelStatus* status;
};

// Blocks have 512 threads, or 256 where rows are many and short.  As many steps of 1/16 below the maximum make the histogram (the last one takes all that lies further
// down), and eight times as many groups of logits have their maxima taken.
template <int kDrThreads>
struct alignas(16) DrawShared {
  static constexpr int kDrWarps = kDrThreads / 32, kDrBins = kDrThreads, kDrGroups = 8 * kDrThreads;
  unsigned count[2][kDrBins];              // histogram, by step parity
  unsigned lo[2][kDrBins], hi[2][kDrBins]; // its masses in two words
  double table[32];
  unsigned long long warp_mass[kDrWarps];
  int warp_ties[kDrWarps];
  unsigned long long scan[kDrWarps];
  unsigned long long found_before;
  int found_at;
  float red[2 * kDrWarps];
  float max_x, low_x;                      // this block's maximum and its lowest group's, read by the others
  int first_max;
  unsigned long long total[2];             // this block's kept mass, read by the others
  int ties;
  int list_n[kDrWarps];
  uint64_t bar;
  int abort_flag;
  float bound;                             // written by the first block into all
  int cand_n[8];                           // of every block, written by it into all
  int cand_own;
  int many;                                // in the steps up to the cut, about
  int cut;                                 // of top-p: its step, the mass in front of the step, and the mass in front of which it keeps (written by the first block into all)
  unsigned long long cut_before, cut_target;
  unsigned tau, last;                      // written by the first block into all: the cut
  unsigned long long block_mass[8];        // kept mass of every block, written by it into all
  union {
    float group[kDrGroups];                // first block: maxima of the groups
    uint2 cand[kDrCand];                   // first block: key and id; a share of the places for every block
    unsigned long long chunk[kDrThreads];  // masses of the block's chunks of ids
    unsigned short list[kDrWarps][kDrList];
  };
};

__device__ __forceinline__ uint32_t dr_mapa(uint32_t addr, int cta) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(cta));
  return r;
}
__device__ __forceinline__ uint32_t dr_peer32(const void* p, int cta) {
  uint32_t v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(dr_mapa(smem_u32(p), cta)) : "memory");
  return v;
}
__device__ __forceinline__ uint4 dr_peer128(const void* p, int cta) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(dr_mapa(smem_u32(p), cta)) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long dr_peer64(const void* p, int cta) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(dr_mapa(smem_u32(p), cta)) : "memory");
  return v;
}
__device__ __forceinline__ void dr_put32(void* p, int cta, uint32_t v) { asm volatile("st.shared::cluster.b32 [%0], %1;" :: "r"(dr_mapa(smem_u32(p), cta)), "r"(v) : "memory"); }
__device__ __forceinline__ void dr_put64(void* p, int cta, unsigned long long v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" :: "r"(dr_mapa(smem_u32(p), cta)), "l"(v) : "memory");
}
__device__ __forceinline__ void dr_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Order-preserving integer of a logit: larger logit, larger key.
template <typename T> struct DrawKey;
template <> struct DrawKey<float> {
  static __device__ __forceinline__ float value(float v) { return v == v ? v : -INFINITY; }              // NaN is never drawn
  static __device__ __forceinline__ unsigned of(float v) { const unsigned u = __float_as_uint(v + 0.0f); return (u & 0x80000000u) ? ~u : (u | 0x80000000u); }
};
template <> struct DrawKey<__nv_bfloat16> {
  static __device__ __forceinline__ float value(__nv_bfloat16 b) { const float v = __bfloat162float(b); return v == v ? v : -INFINITY; }
  static __device__ __forceinline__ unsigned of(float v) { return DrawKey<float>::of(v) >> 16; }         // (the value is a bf16: nothing is lost, and the order stays)
};

// 2^(d scale / 32) in units of 2^-44, for -32000 < d scale <= 0.  table[j]: 2^(44 + j / 32).
__device__ __forceinline__ unsigned long long dr_weight(double d, double scale, const double* table) {
  constexpr double kRound = 6755399441055744.0;                   // 1.5 * 2^52: the sum's low bits are the rounded number
  const double m = fma(d, scale, kRound);
  const int k = __double2loint(m);
  const double r = fma(d, scale, kRound - m);                     // |r| <= 1/2
  // 2^(r / 32) = sum (r ln 2 / 32)^n / n!, the fifth power by (20 r^3 / 4 - 5 r / 16) / 16 (its error: Chebyshev's polynomial, 8e-14 of the weight)
  constexpr double c5 = 0.0013333558146428443 / 33554432, c4 = 0.009618129107628477 / 1048576, c3 = 0.05550410866482158 / 32768 + c5 * 0.3125,
                   c2 = 0.24022650695910072 / 1024, c1 = 0.69314718055994531 / 32 - c5 * 0.01953125;
  double p = fma(r, c4, c3);
  p = fma(r, p, c2); p = fma(r, p, c1); p = fma(r, p, 1.0);
  p *= table[k & 31];
  p = __hiloint2double(__double2hiint(p) + (int)((unsigned)(k & ~31) << 15), __double2loint(p));   // times 2^(k >> 5)
  return (unsigned long long)__double_as_longlong(p + 4503599627370496.0) & 0xfffffffffffffull;    // 2^52: rounded to a whole number
}

// Exclusive position of `target` in the running sum of the threads' values: the thread with before < target <= before + v stores itself.
template <typename S>
__device__ __forceinline__ void dr_find(unsigned long long v, unsigned long long target, S& s) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned long long incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const unsigned long long x = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += x; }
  if (lane == 31) s.scan[warp] = incl;
  if (threadIdx.x == 0) { s.found_at = -1; s.found_before = 0; }
  __syncthreads();
  unsigned long long front = lane < warp ? s.scan[lane] : 0ull;    // (16 warps at most: the lanes fetch, and add up)
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) front += __shfl_xor_sync(0xffffffffu, front, o);
  incl += __shfl_sync(0xffffffffu, front, 0);
  if (v != 0 && incl - v < target && target <= incl) { s.found_at = threadIdx.x; s.found_before = incl - v; }
  __syncthreads();
}

template <typename T, int kDrThreads>
__global__ void __launch_bounds__(kDrThreads, 1024 / kDrThreads)
draw_kernel(const DrawArgs a) {
  constexpr int kDrWarps = kDrThreads / 32, kDrBins = kDrThreads, kDrGroups = 8 * kDrThreads, kDrBits = kDrThreads == 512 ? 9 : 8;
  static_assert(1 << kDrBits == kDrThreads, "a digit of the searches for each thread");
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ DrawShared<kDrThreads> s;
  using Key = DrawKey<T>;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = a.ctas;
  const int row = blockIdx.x / C, rank = blockIdx.x - row * C;     // (the cluster is C blocks along x: rank is the block's place in it)
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // here; what another block's shared memory gets in front of the first exchange waits for it
  if (tid == 0) { mbar_init(&s.bar, 1); s.abort_flag = 0; fence_barrier_init(); }
  if (tid < 32) s.table[tid] = exp2(kDrMass + (double)tid * 0.03125);
  __syncthreads();
  pdl_wait();
  pdl_trigger();

  // ---- the block's ids [i0, i0 + n) into shared memory, at the same offset from a 16-byte boundary as they have in global memory
  const int i0 = min(a.vocab, rank * a.per), n = min(a.vocab, i0 + a.per) - i0;
  const T* g = (const T*)a.logits + (size_t)row * a.ld + i0;
  const int skew = (int)((uintptr_t)g & 15) / (int)sizeof(T);
  T* x = (T*)dyn + skew;
  constexpr int kVec = 16 / sizeof(T);
  const int head = min(n, (kVec - skew) % kVec), body = (n - head) / kVec * kVec;
  if (tid == 0 && body > 0) {
    mbar_expect_tx(&s.bar, (uint32_t)(body * sizeof(T)));
    bulk_load(x + head, g + head, (uint32_t)(body * sizeof(T)), &s.bar);
  }
  if (tid < head) x[tid] = g[tid];
  if (tid < n - head - body) x[head + body + tid] = g[head + body + tid];
  const float temp = a.temperature != nullptr ? a.temperature[row] : a.temperature_all;
  const int top_k = a.top_k != nullptr ? a.top_k[row] : a.top_k_all;
  const float top_p = a.top_p != nullptr ? a.top_p[row] : a.top_p_all;
  const float min_p = a.min_p != nullptr ? a.min_p[row] : a.min_p_all;
  const float u = a.u != nullptr ? a.u[row] : 0.f;
  if (body > 0) mbar_wait(&s.bar, 0, (volatile int*)&s.abort_flag, a.status, 700, row);
  __syncthreads();

  // f(value, index in the block) for the thread's share of the block's logits: 16 bytes at a time, and the ragged ends.  Step: threads between two of a thread's turns
  const int nv = body / kVec;
  auto vec_raw = [&](int j) -> uint4 { return *reinterpret_cast<const uint4*>(x + head + j * kVec); };
  auto vec_max = [&](const uint4& r) -> float {                    // the largest (NaN only where there is nothing else)
    if constexpr (sizeof(T) == 4) return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
    else {                                                         // (two to an instruction)
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
      const float2 m = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
      return fmaxf(m.x, m.y);
    }
  };
  auto vec_of = [&](const uint4& raw, float* v) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < kVec; ++e) v[e] = sizeof(T) == 4 ? __uint_as_float(w[e & 3]) : __uint_as_float(e & 1 ? w[(e >> 1) & 3] & 0xffff0000u : w[(e >> 1) & 3] << 16);
  };
  auto ends = [&](auto f) {                                        // head and tail: a thread each
    if (tid < head) f(Key::value(x[tid]), tid);
    if (tid < n - head - body) f(Key::value(x[head + body + tid]), head + body + tid);
  };

  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  // ---- maximum, and the maxima of the groups: a thread's share of the block's logits in 8 / C pieces.  (fmaxf passes over NaN.)
  const bool has_k = top_k > 0 && top_k < a.vocab, has_p = top_p < 1.f, few_groups = has_k && top_k <= kDrThreads / 8;      // eight groups for each logit that top-k keeps
  float mx = -INFINITY, low = INFINITY;
  {
    constexpr int kPieces = kDrGroups / kDrThreads;
    const int pieces = kPieces / C;
    float gm[kPieces];                                             // eight running maxima, joined to as many as there are pieces
#pragma unroll
    for (int p = 0; p < kPieces; ++p) gm[p] = -INFINITY;
    if (2 * nv < pieces * kDrThreads) {                            // few logits: groups of single ones rather than empty groups
      for (int i = tid; i < n; i += kPieces * kDrThreads) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) if (i + p * kDrThreads < n) gm[p] = fmaxf(gm[p], Key::value(x[i + p * kDrThreads]));
      }
    } else {
      for (int j = tid; j < nv; j += kPieces * kDrThreads) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) if (j + p * kDrThreads < nv) gm[p] = fmaxf(gm[p], vec_max(vec_raw(j + p * kDrThreads)));
      }
      ends([&](float v, int) { gm[0] = fmaxf(gm[0], v); });
    }
#pragma unroll
    for (int half = kPieces / 2; half > 0; half /= 2) {
      if (pieces > half) break;
#pragma unroll
      for (int p = 0; p < half; ++p) gm[p] = fmaxf(gm[p], gm[p + half]);
    }
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      if (p >= pieces) break;
      mx = fmaxf(mx, gm[p]);
      if (gm[p] > -INFINITY) low = fminf(low, gm[p]);
    }
    auto put_group = [&](int at, float v) {                        // (a store through the cluster's network takes several times as long, to the own block too)
      if (rank == 0) s.group[at] = v;
      else dr_put32(&s.group[at], 0, __float_as_uint(v));
    };
    if (few_groups) {                                              // one for each thread of a block in all: a thread's maxima in one, and those of C threads
#pragma unroll
      for (int p = 1; p < kPieces; ++p) if (p < pieces) gm[0] = fmaxf(gm[0], gm[p]);
      for (int o = 1; o < C; o <<= 1) gm[0] = fmaxf(gm[0], __shfl_xor_sync(0xffffffffu, gm[0], o));
      if ((tid & (C - 1)) == 0) put_group(rank * (kDrThreads / C) + tid / C, gm[0]);
    } else if (has_k) {
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        if (p >= pieces) break;
        put_group((rank * pieces + p) * kDrThreads + tid, gm[p]);
      }
    }
  }
  mx = warp_max(mx);
  low = -warp_max(-low);
  if (lane == 0) { s.red[warp] = mx; s.red[kDrWarps + warp] = -low; }
  if (tid == 0) s.first_max = 0x7fffffff;
  __syncthreads();
  mx = warp_max(s.red[lane & (kDrWarps - 1)]);
  low = -warp_max(s.red[kDrWarps + (lane & (kDrWarps - 1))]);
  const bool greedy = !(temp > 0.f);
  if (greedy) {
    int at = 0x7fffffff;
    for (int i = tid; i < n; i += kDrThreads) if (Key::value(x[i]) == mx) { at = i0 + i; break; }
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0 && at != 0x7fffffff) atomicMin(&s.first_max, at);
  }
  if (tid == 0) { s.max_x = mx; s.low_x = low; }
  __syncthreads();
  dr_cluster_sync();
  low = -warp_max(lane < C ? -__uint_as_float(dr_peer32(&s.low_x, lane)) : -INFINITY);
  mx = warp_max(lane < C ? __uint_as_float(dr_peer32(&s.max_x, lane)) : -INFINITY);
  if (greedy || mx == -INFINITY) {
    // the lowest id of the maximum; a row without any logit to draw from answers 0, as the arg-max does
    if (rank == 0 && warp == 0) {
      int at = 0x7fffffff;
      if (mx > -INFINITY && lane < C && __uint_as_float(dr_peer32(&s.max_x, lane)) == mx) at = (int)dr_peer32(&s.first_max, lane);
      at = __reduce_min_sync(0xffffffffu, at);
      if (lane == 0) {
        a.out[row] = at == 0x7fffffff ? 0 : at;
        if (a.logprob != nullptr) a.logprob[row] = mx > -INFINITY ? 0.f : -INFINITY;
      }
    }
    dr_cluster_sync();                                             // nobody leaves while another one reads its shared memory
    return;
  }

  // Logits of floor_x and below (and NaN) weigh nothing: 46.5 halvings or more.  Where the next logit below the maximum lies further down than 1000 halvings, the scale is one
  // that takes it to 64 (the exponent stays in range).  Rows whose floor is no number take the cluster's path, which looks at every logit.
  const double dmx = (double)mx;
  const float floor_x = fmaxf(__fsub_rd(mx, 32.25f * temp), -FLT_MAX);
  const bool plain = mx < INFINITY && floor_x > -FLT_MAX;
  double scale = 1.4426950408889634 / (double)temp;
  if (plain && (dmx - (double)floor_x) * scale > 1000.0) scale = 64.0 / (dmx - (double)floor_x);
  const double scale32 = scale * 32.0;
  auto weight = [&](float v) -> unsigned long long { return dr_weight((double)fmaxf(v, floor_x) - dmx, scale32, s.table); };
  // and for any row: 0 from -46 on (and for NaN)
  auto weight_any = [&](float v) -> unsigned long long {
    const double t = ((double)v - dmx) * scale;
    return v == mx ? 1ull << kDrMass : t > -46.0 ? dr_weight(t, 32.0, s.table) : 0ull;
  };
  auto bin_of = [&](float v) -> int { return min(kDrBins - 1, (int)fminf((mx - v) * 16.0f, 1e6f)); };       // monotone in v (mx = inf: all in the last bin)
  const unsigned long long min_w = min_p > 0.f ? (unsigned long long)ceil(fmin((double)min_p, 1.0) * (double)(1ull << kDrMass)) : 0ull;
  auto value_of = [&](unsigned key) -> float {                     // the logit of a key
    if (sizeof(T) == 2) key = (key << 16) | ((key & 0x8000u) ? 0u : 0xffffu);
    return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
  };
  auto logprob_of = [&](float v, unsigned long long all) -> float {
    return (v == mx ? 0.f : (float)(((double)v - dmx) * scale * 0.69314718055994531)) - logf((float)((double)all * (1.0 / (double)(1ull << kDrMass))));
  };
  auto spot_of = [&](unsigned long long all) -> unsigned long long {         // u below 0 or NaN: the first id; 1 and above: the last
    const double spot = (double)u * (double)all;
    return spot > 0.0 ? min(spot >= (double)all ? all - 1 : (unsigned long long)spot, all - 1) : 0ull;
  };
  auto top_p_target = [&](unsigned long long all) -> unsigned long long {    // kept: while less than this lies in front
    const double goal = ceil((double)top_p * (double)all);
    return goal >= (double)all ? all : goal < 1.0 ? 1ull : (unsigned long long)goal;
  };

  // The block's ids in chunks, in id order: the head, the body by 32 vectors, the tail.  A warp's chunk: f(values, index of the first, chunk), with -inf where the lane has none.
  const int chunks = (nv + 31) / 32 + 2;                           // at most 397
  auto chunk_at = [&](int c, float* v) -> int {
    if (c > 0 && c < chunks - 1) {
      const int j = (c - 1) * 32 + lane;
      vec_of(vec_raw(min(j, nv - 1)), v);
      if (j >= nv) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[e] = -INFINITY;
      }
      return head + j * kVec;
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) v[e] = -INFINITY;               // (the ends have fewer than kVec ids: one a lane)
    const int i = c == 0 ? lane : head + body + lane;
    if (c == 0 ? lane < head : i < n) v[0] = Key::value(x[i]);
    return i;
  };
  auto each_vec = [&](auto f) {
    for (int c = 1 + warp; c < chunks - 1; c += kDrWarps) {
      float v[kVec];
      const int i = chunk_at(c, v);
      f(v, i, c);
    }
    if (warp < 2) {
      float v[kVec];
      const int c = warp == 0 ? 0 : chunks - 1, i = chunk_at(c, v);
      f(v, i, c);
    }
  };
  auto sum = [&](unsigned long long v) -> unsigned long long {     // over the block
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) s.scan[warp] = v;
    __syncthreads();
    v = s.scan[lane & (kDrWarps - 1)];
#pragma unroll
    for (int o = kDrWarps / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    return v;
  };

  // ---- The first block, alone, over the row's candidates: `found` of them, number q at cand_at(q).  A superset of what top-k and top-p keep; `target`: mass
  // in front of which top-p keeps (0: top-p of the candidates that top-k keeps).
  auto finish = [&](int found, unsigned long long target, auto cand_at) {
    const bool cut_k = has_k && found > top_k;
    if (found <= kDrPairs) {
      // Few: every candidate against every other one.  Its rank, the mass in front of it, and the kept mass at lower ids are plain sums.
      uint4* pair = reinterpret_cast<uint4*>(&s.lo[0][0]);         // key, id, mass (8 KB: lo and hi lie one behind the other)
      constexpr int kHalves = kDrThreads / kDrPairs;               // two threads to a candidate, or one
      const int q = tid & (kDrPairs - 1), half = tid / kDrPairs;
      const uint2 e = q < found ? cand_at(q) : make_uint2(0u, 0u);
      unsigned long long w = q < found ? weight(value_of(e.x)) : 0ull;
      if (half == 0) pair[q] = make_uint4(e.x, e.y, (unsigned)w, (unsigned)(w >> 32));
      __syncthreads();
      // (warps without a candidate sit the loops out)
      const int j0 = half ? (found + 1) / 2 : 0, j1 = (q & ~31) >= found ? j0 : half || kHalves == 1 ? found : (found + 1) / 2;
      int place = 0;
      unsigned long long front = 0;
#pragma unroll 4
      for (int j = j0; j < j1; ++j) {
        const uint4 o = pair[j];
        const bool ahead = o.x > e.x || (o.x == e.x && o.y < e.y);
        place += ahead;
        front += ahead ? (unsigned long long)o.w << 32 | o.z : 0ull;
      }
      unsigned long long* other = reinterpret_cast<unsigned long long*>(&s.count[0][0]);      // [kDrPairs], then the places
      int* other_place = (int*)(other + kDrPairs);
      if (kHalves > 1) {
        if (half) { other[q] = front; other_place[q] = place; }
        __syncthreads();
        if (!half) { front += other[q]; place += other_place[q]; }
      }
      bool keep = !half && q < found && (!cut_k || place < top_k);
      if (has_p) {
        const unsigned long long goal = target != 0 ? target : top_p_target(sum(keep ? w : 0ull));
        keep = keep && front < goal;
      }
      keep = keep && w >= min_w;
      if (!keep) w = 0;
      const unsigned long long all = sum(half ? 0ull : w), r = spot_of(all);
      if (!half) pair[q] = make_uint4(e.x, e.y, (unsigned)w, (unsigned)(w >> 32));
      __syncthreads();
      unsigned long long below = 0;
#pragma unroll 4
      for (int j = j0; j < j1; ++j) {
        const uint4 o = pair[j];
        below += o.y < e.y ? (unsigned long long)o.w << 32 | o.z : 0ull;
      }
      if (kHalves > 1) {
        if (half) other[q] = below;
        __syncthreads();
      }
      if (!half && w != 0) {
        if (kHalves > 1) below += other[q];
        if (below <= r && r < below + w) {
          a.out[row] = (int)e.y;
          if (a.logprob != nullptr) a.logprob[row] = logprob_of(value_of(e.x), all);
        }
      }
      return;
    }
    // Many: radix searches, four candidates a thread
    constexpr int kOwn = kDrCand / kDrThreads;
    unsigned key[kOwn], id[kOwn], least = 0xffffffffu;
    unsigned long long w[kOwn];
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const int q = k * kDrThreads + tid;
      const uint2 e = q < found ? cand_at(q) : make_uint2(0u, 0u); // key 0: no candidate
      key[k] = e.x; id[k] = e.y;
      w[k] = q < found ? weight(value_of(e.x)) : 0ull;
      if (q < found) least = min(least, e.x);
    }
    least = __reduce_min_sync(0xffffffffu, least);
    if (tid == 0) s.first_max = -1;
    __syncthreads();
    if (lane == 0) atomicMin((unsigned*)&s.first_max, least);
    __syncthreads();
    least = (unsigned)s.first_max;
    // Searches the numbers of(k) in [base, base + range] for the one at which the running sum of val(k), from the top down (or from the bottom up), reaches `goal`;
    // `before`: the sum in front of it.
    auto search = [&](unsigned base, unsigned range, bool up, bool mass, unsigned long long goal, unsigned long long& before, auto of, auto val) -> unsigned {
      unsigned prefix = 0;
      before = 0;
      for (int bits = 32 - __clz(range); bits > 0;) {
        const int shift = max(0, bits - kDrBits);
        s.count[0][tid] = 0;
        if (mass) { s.lo[0][tid] = 0; s.hi[0][tid] = 0; }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
          const unsigned long long v = val(k);
          const unsigned off = min(of(k) - base, range);
          if (v == 0 || (bits >= 32 ? 0u : off >> bits) != prefix) continue;
          const int d = (off >> shift) & (kDrThreads - 1);
          if (!mass) atomicAdd(&s.count[0][d], 1u);
          else {
            const unsigned l = (unsigned)v, old = atomicAdd(&s.lo[0][d], l);
            const unsigned h = (unsigned)(v >> 32) + (old + l < old ? 1u : 0u);
            if (h != 0) atomicAdd(&s.hi[0][d], h);
          }
        }
        __syncthreads();
        const int d = up ? tid : kDrThreads - 1 - tid;
        const unsigned long long v = mass ? ((unsigned long long)s.hi[0][d] << 32) + s.lo[0][d] : s.count[0][d];
        dr_find(v, goal - before, s);
        const int hit = s.found_at < 0 ? 0 : s.found_at;
        prefix = prefix << (bits - shift) | (unsigned)(up ? hit : kDrThreads - 1 - hit);
        before += s.found_before;
        bits = shift;
        __syncthreads();
      }
      return base + prefix;
    };
    const unsigned top = Key::of(mx);
    unsigned tau = 0;                                              // kept: key > tau, and the first `ties` ids of key tau
    unsigned long long ties = 0, before;
    auto key_of = [&](int k) { return key[k]; };
    auto id_of = [&](int k) { return id[k]; };
    auto strike = [&]() {                                          // takes the others out
      unsigned long long n_tie = 0;
#pragma unroll
      for (int k = 0; k < kOwn; ++k) n_tie += key[k] != 0 && key[k] == tau;
      n_tie = sum(n_tie);
      unsigned last = 0xffffffffu;
      if (n_tie > ties && ties > 0) last = search(0, (unsigned)a.vocab - 1, true, false, ties, before, id_of, [&](int k) -> unsigned long long { return key[k] != 0 && key[k] == tau; });
#pragma unroll
      for (int k = 0; k < kOwn; ++k) if (key[k] < tau || (key[k] == tau && (ties == 0 || id[k] > last))) { key[k] = 0; w[k] = 0; }
    };
    auto mass_of = [&]() {
      unsigned long long m = 0;
#pragma unroll
      for (int k = 0; k < kOwn; ++k) m += w[k];
      return sum(m);
    };
    if (cut_k) {
      tau = search(least, top - least, false, false, (unsigned long long)top_k, before, key_of, [&](int k) -> unsigned long long { return key[k] != 0; });
      ties = (unsigned long long)top_k - before;
      strike();
    }
    if (has_p) {
      const unsigned long long have = mass_of(), goal = target != 0 ? target : top_p_target(have);
      if (have > goal) {                                           // (else all are kept: min-p has left out what lies behind)
        tau = search(least, top - least, false, true, goal, before, key_of, [&](int k) -> unsigned long long { return w[k]; });
        const unsigned long long wt = weight(value_of(tau));
        ties = wt > 0 ? (goal - before + wt - 1) / wt : 0;
        strike();
      }
    }
#pragma unroll
    for (int k = 0; k < kOwn; ++k) if (w[k] < min_w) w[k] = 0;
    const unsigned long long m = mass_of();
    const unsigned token = search(0, (unsigned)a.vocab - 1, true, true, spot_of(m) + 1, before, id_of, [&](int k) -> unsigned long long { return w[k]; });
#pragma unroll
    for (int k = 0; k < kOwn; ++k)
      if (w[k] != 0 && id[k] == token) {
        a.out[row] = (int)token;
        if (a.logprob != nullptr) a.logprob[row] = logprob_of(value_of(key[k]), m);
      }
  };

  // Masses of the chunks, of what keeps(logit, id) and min-p leave; returns the thread's chunk's.
  auto weigh = [&](auto keeps) -> unsigned long long {
    each_vec([&](const float* v, int i, int c) {
      unsigned long long m = 0;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const unsigned long long w = weight(v[e]);
        m += (w >= min_w) & keeps(v[e], (unsigned)(i0 + i + e)) ? w : 0ull;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
      if (lane == 0) s.chunk[c] = m;
    });
    __syncthreads();
    return tid < chunks ? s.chunk[tid] : 0ull;
  };
  // The first id of this block at which the mass, `front` of it in front of the block and `mine` in the thread's chunk, exceeds r.
  auto locate = [&](unsigned long long mine, unsigned long long front, unsigned long long r, unsigned long long all, auto keeps) {
    dr_find(mine, r - front + 1, s);
    if (warp != 0 || s.found_at < 0) return;
    front += s.found_before;
    float v[kVec];
    const int i = chunk_at(s.found_at, v);
    unsigned long long w[kVec], m = 0;
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      w[e] = weight(v[e]);
      w[e] = w[e] >= min_w && keeps(v[e], (unsigned)(i0 + i + e)) ? w[e] : 0ull;
      m += w[e];
    }
    unsigned long long incl = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const unsigned long long y = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += y; }
    const unsigned hit = __ballot_sync(0xffffffffu, r < front + incl);
    if (hit == 0 || lane != __ffs(hit) - 1) return;
    front += incl - m;
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      if (r < front + w[e]) {
        a.out[row] = i0 + i + e;
        if (a.logprob != nullptr) a.logprob[row] = logprob_of(v[e], all);
        return;
      }
      front += w[e];
    }
  };

  // The block's candidates, into its own list: logits of `bound` and above that `wanted` takes; Few vectors hold
  // one, and few of their logits are one, so each thread goes on by itself.  Plain stores: the first block gets the list in one go.
  const int cap = kDrCand / C;                                     // a block's places in the first block's list
  auto collect = [&](float bound, int room, auto wanted) {
    auto take = [&](unsigned m, int i) {                           // logits i + the bits of m
      int q = atomicAdd(&s.cand_own, __popc(m));
      for (; m != 0; m &= m - 1, ++q) {
        const int at = i + __ffs(m) - 1;
        const float v = Key::value(x[at]);
        if (q < room) s.cand[q] = make_uint2(Key::of(v), (unsigned)(i0 + at));
      }
    };
#pragma unroll 2
    for (int j = tid; j < nv; j += kDrThreads) {
      const uint4 raw = vec_raw(j);
      if (!(vec_max(raw) >= bound)) continue;
      float v[kVec];
      vec_of(raw, v);
      unsigned m = 0;
#pragma unroll
      for (int e = 0; e < kVec; ++e) m |= (v[e] >= bound && wanted(v[e])) ? 1u << e : 0u;
      if (m != 0) take(m, head + j * kVec);
    }
    ends([&](float v, int i) { if (v >= bound && wanted(v)) take(1u, i); });
  };
  auto hand_over = [&](int many, int place) {                      // to the first block
    if (rank == 0) return;
    for (int q = tid; q < many; q += kDrThreads) dr_put64(&s.cand[place + q], 0, *reinterpret_cast<const unsigned long long*>(&s.cand[q]));
  };
  auto settle = [&](unsigned long long target) {                   // the first block finishes with the lists of all
    int found = 0;
    for (int c = 0; c < C; ++c) found += s.cand_n[c];
    finish(found, target, [&](int q) -> uint2 {
      int c = 0;
      while (q >= s.cand_n[c]) q -= s.cand_n[c++];
      return s.cand[c * cap + q];
    });
  };

  // ---- rows with a top-k: pruned.  With min-p alone the bound is known
  if (plain && (has_k ? top_k <= kDrPrune : !has_p && min_w != 0)) {
    if (tid == 0) s.cand_own = 0;
    float bound = fmaxf(mx + temp * logf(fminf(min_p, 1.0f)) - fmaf(fabsf(mx), 2.5e-7f, 1e-5f) - temp * 1e-5f, -FLT_MAX);
    if (!has_k) __syncthreads();
    if (has_k && rank == 0) {
      s.count[0][tid] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < (few_groups ? 1 : kDrGroups / kDrThreads); ++i) {
        const float v = s.group[i * kDrThreads + tid];
        if (v > mx - kDrBins / 16.0f) atomicAdd(&s.count[0][bin_of(v)], 1u);
      }
      __syncthreads();
      dr_find(s.count[0][tid], top_k, s);
      // at least top_k logits lie in the bin and above; fewer in reach: all of them count
      const float low_bound = s.found_at >= 0 && s.found_at < kDrBins - 1 ? fmaxf(mx - (s.found_at + 1) * 0.0625f - fmaf(fabsf(mx), 2.5e-7f, 1e-5f), -FLT_MAX) : -FLT_MAX;
      if (tid < C) dr_put32(&s.bound, tid, __float_as_uint(low_bound));
    }
    if (has_k) {
      __syncthreads();
      dr_cluster_sync();
      bound = s.bound;
    }
    collect(bound, cap, [](float) { return true; });
    __syncthreads();
    hand_over(min(s.cand_own, cap), rank * cap);
    if (tid < C) dr_put32(&s.cand_n[rank], tid, s.cand_own);
    dr_cluster_sync();
    bool settled = true;
    for (int c = 0; c < C; ++c) settled &= s.cand_n[c] <= cap;
    if (settled) {
      if (rank != 0) return;                                       // (nobody reads this block's shared memory any more)
      settle(0);
      return;
    }
  }
  // ---- rows with a top-p alone: one pass for all weights and their histogram, over steps that suit the row: to twice the depth of its lowest group, at most
  // 45 halvings.  The step of the cut is then known, with the mass in front of it.
  bool by_min_p = false;
  if (plain && has_p && !has_k) {
    const float depth = fminf(2.0f * (mx - low), 32.0f * temp), steps = kDrBins / depth;
    auto step_of = [&](float v) -> int { return max(0, min(kDrBins - 1, (int)((mx - v) * steps))); };      // monotone in v
    s.lo[0][tid] = 0; s.hi[0][tid] = 0;
    if (tid == 0) s.cand_own = 0;
    __syncthreads();
    each_vec([&](const float* v, int, int) {
      unsigned long long w[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) w[e] = weight(v[e]);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        if (w[e] == 0) continue;
        const int b = step_of(v[e]);
        const unsigned l = (unsigned)w[e], old = atomicAdd(&s.lo[0][b], l);
        const unsigned h = (unsigned)(w[e] >> 32) + (old + l < old ? 1u : 0u);
        if (h != 0) atomicAdd(&s.hi[0][b], h);
      }
    });
    __syncthreads();
    dr_cluster_sync();
    // min-p may cut higher up: what lies more than a step below its weight is kept by neither
    const float min_off = min_w != 0 ? -temp * logf(fminf(min_p, 1.0f)) : 0.f, slack = fmaf(fabsf(mx) + depth + min_off, 1e-6f, 1e-4f);
    const int min_step = min_w != 0 ? step_of(mx - min_off - slack) + 1 : kDrBins;         // no logit of this step or below has the weight
    const int all_step = min_w != 0 ? step_of(mx - min_off + slack) : kDrBins;             // all logits above this step have it
    // The first block adds up the histograms, four steps of one block a turn (16-byte loads; lanes 8 apart hold the same block), and tells the step of the cut.
    if (rank == 0) {
      unsigned long long at;
      if (C == 1) at = ((unsigned long long)s.hi[0][tid] << 32) + s.lo[0][tid];
      else {
        const int block = lane & 7;
        unsigned long long part[2 * 4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int quad = (tid >> 3) + k * (kDrThreads / 8);
          uint4 l4 = make_uint4(0, 0, 0, 0), h4 = l4;
          if (block < C) { l4 = dr_peer128(&s.lo[0][quad * 4], block); h4 = dr_peer128(&s.hi[0][quad * 4], block); }
          part[k * 4] = ((unsigned long long)h4.x << 32) + l4.x; part[k * 4 + 1] = ((unsigned long long)h4.y << 32) + l4.y;
          part[k * 4 + 2] = ((unsigned long long)h4.z << 32) + l4.z; part[k * 4 + 3] = ((unsigned long long)h4.w << 32) + l4.w;
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
#pragma unroll
          for (int k = 0; k < 8; ++k) part[k] += __shfl_xor_sync(0xffffffffu, part[k], o);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int b = ((tid >> 3) + (k >> 2) * (kDrThreads / 8)) * 4 + (k & 3);
          if (block == k) { s.lo[1][b] = (unsigned)part[k]; s.hi[1][b] = (unsigned)(part[k] >> 32); }
        }
        __syncthreads();
        at = (unsigned long long)s.hi[1][tid] << 32 | s.lo[1][tid];
      }
      const unsigned long long goal = top_p_target(sum(at));
      dr_find(at, goal, s);
      // About how many lie in the steps up to the cut: a step's mass by the weight in its middle (a step is a tenth of a halving or less).
      const float halvings = (float)scale * depth * (1.0f / kDrBins);
      const unsigned long long many = sum(tid <= min(s.found_at, min_step) ? (unsigned long long)((float)at * exp2f((tid + 0.5f) * halvings - kDrMass)) : 0ull);
      if (tid < C) {
        dr_put32(&s.many, tid, (uint32_t)min(many, 0x7fffffffull));
        dr_put32(&s.cut, tid, (uint32_t)s.found_at); dr_put64(&s.cut_before, tid, s.found_before); dr_put64(&s.cut_target, tid, goal);
      }
    }
    dr_cluster_sync();
    const unsigned long long target = s.cut_target, before = s.cut_before;
    const int full_cut = s.cut;
    const int cut = full_cut > 0 ? min(full_cut, min_step) : full_cut;
    if (cut >= 0 && cut < kDrBins - 1) {
      // the candidates to the first block
      const float bound = fmaxf(mx - (cut + 1) / steps - fmaf(fabsf(mx) + depth, 1e-6f, 1e-4f), -FLT_MAX);       // (a little below the step: which step a logit is of is asked anew)
      bool few = s.many <= kDrCand + kDrCand / 8;                  // (many that are not too many after all take the other way)
      if (few) {
        collect(bound, cap, [](float) { return true; });           // (with some of the next step: they lie behind the cut)
        __syncthreads();
        hand_over(min(s.cand_own, cap), rank * cap);
        if (tid < C) dr_put32(&s.cand_n[rank], tid, s.cand_own);
        dr_cluster_sync();
        for (int c = 0; c < C; ++c) few &= s.cand_n[c] <= cap;
        if (few) {
          if (rank == 0) settle(target);
          return;
        }
        dr_cluster_sync();                                         // (cand_n is written again)
      }
      by_min_p = min_step < full_cut;                              // min-p cuts first: nothing of top-p is left to do
      bool settled = !by_min_p && full_cut < all_step;             // (the second: min-p leaves all that top-p leaves)
      if (settled) {
        // too many: those of the cut's step, of which each block keeps its own too
        if (tid == 0) s.cand_own = 0;
        __syncthreads();
        collect(bound, cap, [&](float v) { return step_of(v) == cut; });
        __syncthreads();
        hand_over(min(s.cand_own, cap), rank * cap);
        if (tid < C) dr_put32(&s.cand_n[rank], tid, s.cand_own);
        dr_cluster_sync();
        for (int c = 0; c < C; ++c) settled &= s.cand_n[c] <= cap;
      }
      if (settled) {
        const int own = s.cand_own;
        // Many above the cut: the first block finds the cut in its step, every block then knows its kept mass, and the block in which the draw falls goes through
        // its logits once more.
        if (rank == 0) {
          constexpr int kOwn = kDrCand / kDrThreads;
          unsigned key[kOwn], id[kOwn], least = 0xffffffffu, most = 0;
          unsigned long long w[kOwn];
#pragma unroll
          for (int k = 0; k < kOwn; ++k) {
            const int q = k * kDrThreads + tid;                      // of the list: place q - c cap of block c
            const bool in = (q & (cap - 1)) < s.cand_n[q / cap];
            const uint2 e = in ? s.cand[q] : make_uint2(0u, 0u);
            key[k] = e.x; id[k] = e.y;
            w[k] = in ? weight(value_of(e.x)) : 0ull;
            if (in) { least = min(least, e.x); most = max(most, e.x); }
          }
          least = __reduce_min_sync(0xffffffffu, least);
          most = __reduce_max_sync(0xffffffffu, most);
          if (tid == 0) { s.first_max = -1; s.tau = 0; }
          __syncthreads();
          if (lane == 0) { atomicMin((unsigned*)&s.first_max, least); atomicMax(&s.tau, most); }
          __syncthreads();
          least = (unsigned)s.first_max; most = s.tau;
          // the key at which the mass reaches the target, and, of equal keys, the id
          unsigned found[2] = {0, 0};
          unsigned long long goal = target - before;
#pragma unroll
          for (int by_id = 0; by_id < 2; ++by_id) {
            if (by_id) {
              unsigned long long same = 0;
#pragma unroll
              for (int k = 0; k < kOwn; ++k) same += key[k] == found[0];
              if (sum(same) == 1) { found[1] = 0xffffffffu; break; }
            }
            const unsigned first = by_id ? 0u : least, range = by_id ? (unsigned)a.vocab - 1 : most - least;
            unsigned prefix = 0;
            for (int bits = 32 - __clz(range); bits > 0;) {
              const int shift = max(0, bits - kDrBits);
              __syncthreads();
              s.lo[1][tid] = 0; s.hi[1][tid] = 0;
              __syncthreads();
#pragma unroll
              for (int k = 0; k < kOwn; ++k) {
                const unsigned off = min((by_id ? id[k] : key[k]) - first, range);
                if (w[k] == 0 || (by_id && key[k] != found[0]) || (bits >= 32 ? 0u : off >> bits) != prefix) continue;
                const int d = (off >> shift) & (kDrThreads - 1);
                const unsigned l = (unsigned)w[k], old = atomicAdd(&s.lo[1][d], l);
                const unsigned h = (unsigned)(w[k] >> 32) + (old + l < old ? 1u : 0u);
                if (h != 0) atomicAdd(&s.hi[1][d], h);
              }
              __syncthreads();
              const int d = by_id ? tid : kDrThreads - 1 - tid;
              dr_find(((unsigned long long)s.hi[1][d] << 32) + s.lo[1][d], goal, s);
              const int hit = s.found_at < 0 ? 0 : s.found_at;
              prefix = prefix << (bits - shift) | (unsigned)(by_id ? hit : kDrThreads - 1 - hit);
              goal -= s.found_before;
              bits = shift;
            }
            found[by_id] = first + prefix;
          }
          __syncthreads();
          if (tid < C) { dr_put32(&s.tau, tid, found[0]); dr_put32(&s.last, tid, found[1]); }
        }
        dr_cluster_sync();
        const unsigned tau = s.tau, last = s.last;
        const float tau_x = value_of(tau);
        auto keeps = [&](float v, unsigned id) -> bool { return (v > tau_x) | ((v == tau_x) & (id <= last)); };
        unsigned long long mine = tid < cut ? ((unsigned long long)s.hi[0][tid] << 32) + s.lo[0][tid] : 0ull;
        for (int q = tid; q < own; q += kDrThreads) {
          const uint2 e = s.cand[q];
          if (keeps(value_of(e.x), e.y)) mine += weight(value_of(e.x));
        }
        mine = sum(mine);
        if (tid < C) dr_put64(&s.block_mass[rank], tid, mine);
        dr_cluster_sync();
        unsigned long long all = 0, front = 0;
        for (int c = 0; c < C; ++c) { if (c < rank) front += s.block_mass[c]; all += s.block_mass[c]; }
        const unsigned long long r = spot_of(all);
        if (r < front || r >= front + mine) return;
        locate(weigh(keeps), front, r, all, keeps);
        return;
      }
    }
  }
  // ---- rows without a limit, or with min-p alone (too many for the first block): one pass for the blocks' masses
  if (plain && !has_k && (!has_p || by_min_p)) {
    auto keeps = [](float, unsigned) { return true; };
    const unsigned long long chunk = weigh(keeps), mine = sum(chunk);
    if (tid < C) dr_put64(&s.block_mass[rank], tid, mine);
    dr_cluster_sync();
    unsigned long long all = 0, front = 0;
    for (int c = 0; c < C; ++c) { if (c < rank) front += s.block_mass[c]; all += s.block_mass[c]; }
    const unsigned long long r = spot_of(all);
    if (r < front || r >= front + mine) return;
    locate(chunk, front, r, all, keeps);
    return;
  }

  // ---- the cluster's path.  A warp owns a run of the block's ids
  const int run = (n + kDrWarps - 1) / kDrWarps, r0 = min(n, warp * run), rn = min(n, r0 + run) - r0;
  bool listed = false;
  int list_n = 0;
  // f(value, in range) for the warp's ids, or for the listed ones; all lanes take part in every turn
  auto each = [&](auto f) {
    const int m = listed ? list_n : rn;
    for (int b = 0; b < m; b += 32) {
      const int i = b + lane;
      const bool in = i < m;
      const int at = in ? (listed ? (int)s.list[warp][i] : i) : 0;
      const float v = in ? Key::value(x[r0 + at]) : -INFINITY;
      f(v, in && v > -INFINITY);
    }
  };
  int step = 1;                                                    // parity of the histogram in use (not the one that other blocks may still be reading)
  auto clear = [&](bool mass) {
    for (int i = tid; i < kDrBins; i += kDrThreads) { s.count[step & 1][i] = 0; if (mass) { s.lo[step & 1][i] = 0; s.hi[step & 1][i] = 0; } }
    __syncthreads();
  };
  auto put = [&](int b, bool in) {                                 // one more in bin b
    const int b0 = __shfl_sync(0xffffffffu, b, 0);
    if (__all_sync(0xffffffffu, in && b == b0)) { if (lane == 0) atomicAdd(&s.count[step & 1][b], 32u); }      // rows of equal logits: not 32 adds to one word
    else if (in) atomicAdd(&s.count[step & 1][b], 1u);
  };
  auto put_mass = [&](int b, unsigned long long w) {
    const unsigned l = (unsigned)w, old = atomicAdd(&s.lo[step & 1][b], l);
    const unsigned h = (unsigned)(w >> 32) + (old + l < old ? 1u : 0u);
    if (h != 0) atomicAdd(&s.hi[step & 1][b], h);
  };
  auto gather = [&](int b, bool mass) -> unsigned long long {      // the bin over all blocks
    unsigned long long v = 0;
    for (int c = 0; c < C; ++c)
      v += mass ? ((unsigned long long)dr_peer32(&s.hi[step & 1][b], c) << 32) + dr_peer32(&s.lo[step & 1][b], c) : dr_peer32(&s.count[step & 1][b], c);
    return v;
  };
  const unsigned key_none = Key::of(-INFINITY);
  unsigned tau = key_none;                                         // kept: key > tau, and the first `ties` ids of key tau
  unsigned long long ties = 0;
  // The cut in front of which `target` (ids, or mass) lies: sets tau; returns what lies above it.  extra: mass that the ids of key `extra_key` count, which the
  // passes leave out (the ties at the top-k cut: only some of them are kept).
  auto cut = [&](bool mass, unsigned long long target, unsigned extra_key, unsigned long long extra, int extra_bin) -> unsigned long long {
    // the histogram of bins is complete in all blocks
    unsigned long long v = gather(tid, mass);
    if (mass && tid == extra_bin) v += extra;
    dr_find(v, target, s);
    const int bin = s.found_at;
    unsigned long long before = s.found_before;
    __syncthreads();
    if (!listed) {                                                 // from here on only ids up to this bin matter: the warp lists them, in order
      int cnt = 0;
      for (int b = 0; b < rn; b += 32) {
        const int i = b + lane;
        const float e = i < rn ? Key::value(x[r0 + i]) : -INFINITY;
        const bool in = e > -INFINITY && bin_of(e) <= bin;
        const unsigned m = __ballot_sync(0xffffffffu, in);
        const int at = cnt + __popc(m & ((1u << lane) - 1));
        if (in && at < kDrList) s.list[warp][at] = (unsigned short)i;
        cnt += __popc(m);
      }
      __syncwarp();
      if (cnt <= kDrList) { listed = true; list_n = cnt; }
    }
    // keys of the bin lie in [k0, k1]
    const float eps = fmaf(fabsf(mx), 2.5e-7f, 1e-5f);
    const unsigned k1 = bin == 0 ? Key::of(mx) : Key::of(mx - bin * 0.0625f + eps);
    const unsigned k0 = bin == kDrBins - 1 ? Key::of(-FLT_MAX) : Key::of(mx - (bin + 1) * 0.0625f - eps);
    const unsigned range = k1 > k0 ? k1 - k0 : 0;
    unsigned prefix = 0;
    for (int bits = 32 - __clz(range); bits > 0;) {
      const int shift = max(0, bits - 8);
      ++step;
      clear(mass);
      each([&](float e, bool in) {
        const unsigned off = min(Key::of(e) - k0, range);
        in = in && bin_of(e) == bin && (bits >= 32 ? 0u : off >> bits) == prefix;
        if (!mass) put((off >> shift) & 255, in);
        else if (in && Key::of(e) > tau) { const unsigned long long w = weight_any(e); if (w) put_mass((off >> shift) & 255, w); }
      });
      __syncthreads();
      dr_cluster_sync();
      unsigned long long d = 0;
      const int digit = 255 - tid;                                 // from the largest key down
      if (tid < 256) {
        d = gather(digit, mass);
        if (mass && extra != 0 && bin == extra_bin) {
          const unsigned off = min(extra_key - k0, range);
          if ((bits >= 32 ? 0u : off >> bits) == prefix && (int)((off >> shift) & 255) == digit) d += extra;
        }
      }
      dr_find(d, target - before, s);
      prefix = prefix << (bits - shift) | (unsigned)(255 - s.found_at);
      before += s.found_before;
      bits = shift;
      __syncthreads();
    }
    tau = k0 + prefix;
    return before;
  };

  // ---- top-k
  unsigned long long tie_mass = 0;                                 // of the ids kept at tau
  int tau_bin = -1;
  if (has_k) {
    clear(false);
    each([&](float e, bool in) { put(in ? bin_of(e) : 0, in); });
    __syncthreads();
    dr_cluster_sync();
    unsigned long long mine = gather(tid, false);                  // all there are
    unsigned long long all = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (lane == 0) s.warp_mass[warp] = all;
    __syncthreads();
    all = 0;
    for (int w = 0; w < kDrWarps; ++w) all += s.warp_mass[w];
    __syncthreads();
    if (all > (unsigned long long)top_k) {
      const unsigned long long above = cut(false, (unsigned long long)top_k, 0, 0, -1);
      ties = (unsigned long long)top_k - above;
      const float vt = value_of(tau);
      tie_mass = ties * weight_any(vt);
      tau_bin = bin_of(vt);
    }
    ++step;
  }
  // ---- top-p of what is left
  if (has_p) {
    clear(true);
    each([&](float e, bool in) { const unsigned long long w = weight_any(e); if (in && Key::of(e) > tau && w) put_mass(bin_of(e), w); });
    __syncthreads();
    dr_cluster_sync();
    unsigned long long all = gather(tid, true);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (lane == 0) s.warp_mass[warp] = all;
    __syncthreads();
    all = tie_mass;
    for (int w = 0; w < kDrWarps; ++w) all += s.warp_mass[w];
    __syncthreads();
    const unsigned long long target = top_p_target(all);
    const unsigned old_tau = tau;
    const unsigned long long old_ties = ties;
    const unsigned long long above = cut(true, target, old_tau, tie_mass, tau_bin);
    const unsigned long long wt = weight_any(value_of(tau));
    ties = wt > 0 ? (target - above + wt - 1) / wt : 0;
    if (tau == old_tau) ties = min(ties, old_ties);
    ++step;
  }
  // ---- the draw, in id order: blocks, warps, sixteenths of a warp's ids, ids
  unsigned long long wt = ties > 0 ? weight_any(value_of(tau)) : 0;
  if (wt < min_w) wt = 0;
  auto kept = [&](float e, bool in, bool& tie) -> unsigned long long {       // (the whole warp)
    const unsigned k = Key::of(e);
    tie = in && k == tau;
    const unsigned long long w = weight_any(e);
    return in && k > tau && w >= min_w ? w : 0;
  };
  unsigned long long mass = 0;
  int n_tie = 0;
  each([&](float e, bool in) { bool tie; mass += kept(e, in, tie); n_tie += tie; });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
  n_tie = __reduce_add_sync(0xffffffffu, n_tie);
  if (lane == 0) { s.warp_mass[warp] = mass; s.warp_ties[warp] = n_tie; s.list_n[warp] = listed ? list_n : -1; }
  __syncthreads();
  if (tid == 0) {
    unsigned long long m = 0; int t = 0;
    for (int w = 0; w < kDrWarps; ++w) { m += s.warp_mass[w]; t += s.warp_ties[w]; }
    s.total[0] = m; s.ties = t;
  }
  __syncthreads();
  dr_cluster_sync();
  unsigned long long gt = 0, all = 0;                              // above tau: in front of this block; in all
  unsigned long long nt = 0, all_ties = 0;
  for (int c = 0; c < C; ++c) {
    const unsigned long long m = dr_peer64(&s.total[0], c);
    const unsigned t = dr_peer32(&s.ties, c);
    if (c < rank) { gt += m; nt += t; }
    all += m; all_ties += t;
  }
  all += min(all_ties, ties) * wt;
  const unsigned long long r = spot_of(all);
  // mass in front of a place with m above tau and t ties in front of it
  auto front = [&](unsigned long long m, unsigned long long t) { return m + min(t, ties) * wt; };
  const bool here = front(gt, nt) <= r && r < front(gt + s.total[0], nt + (unsigned)s.ties);
  if (here) {                                                      // the same for all threads of the block, and true in one block
    int w = 0;
    for (; w < kDrWarps - 1; ++w) {
      if (r < front(gt + s.warp_mass[w], nt + (unsigned)s.warp_ties[w])) break;
      gt += s.warp_mass[w]; nt += (unsigned)s.warp_ties[w];
    }
    const int wn = s.list_n[w], w0 = min(n, w * run), m = wn >= 0 ? wn : min(n, w0 + run) - w0;
    const int piece = (m + kDrWarps * 32 - 1) / (kDrWarps * 32) * 32;
    auto at_of = [&](int i) { return w0 + (wn >= 0 ? (int)s.list[w][i] : i); };
    __syncthreads();                                               // warp_mass and warp_ties are used again
    mass = 0; n_tie = 0;
    for (int b = warp * piece; b < min(m, (warp + 1) * piece); b += 32) {
      const int i = b + lane;
      const float e = i < m ? Key::value(x[at_of(i)]) : -INFINITY;           // (a piece is a multiple of 32)
      bool tie;
      mass += kept(e, e > -INFINITY, tie);
      n_tie += tie;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
    n_tie = __reduce_add_sync(0xffffffffu, n_tie);
    if (lane == 0) { s.warp_mass[warp] = mass; s.warp_ties[warp] = n_tie; }
    __syncthreads();
    int p = 0;
    for (; p < kDrWarps - 1; ++p) {
      if (r < front(gt + s.warp_mass[p], nt + (unsigned)s.warp_ties[p])) break;
      gt += s.warp_mass[p]; nt += (unsigned)s.warp_ties[p];
    }
    if (warp == 0) {
      bool done = false;
      const int end = min(m, (p + 1) * piece);
      for (int b = p * piece; b < end && !done; b += 32) {
        const int i = b + lane;
        const float e = i < end ? Key::value(x[at_of(i)]) : -INFINITY;
        bool tie;
        unsigned long long incl = kept(e, e > -INFINITY, tie);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const unsigned long long y = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += y; }
        const unsigned tm = __ballot_sync(0xffffffffu, tie);
        const unsigned hit = __ballot_sync(0xffffffffu, r < front(gt + incl, nt + __popc(tm & (0xffffffffu >> (31 - lane)))));
        if (hit) {
          if (lane == __ffs(hit) - 1) {
            a.out[row] = i0 + at_of(i);
            if (a.logprob != nullptr)
              a.logprob[row] = logprob_of(e, all);
          }
          done = true;
        }
        gt += __shfl_sync(0xffffffffu, incl, 31);
        nt += __popc(tm);
      }
    }
  }
  dr_cluster_sync();                                               // nobody leaves while another one reads its shared memory
}

template <typename T, int kDrThreads>
static int draw_launch(DrawArgs a, cudaStream_t stream) {
  // Blocks per row: as few as hold it with two blocks to an SM (the steps of a cluster cost every block of it: 1500 bf16 rows of 32003 in one block each 219 us, in eight 257, at the
  // time of the choice); few rows take as many as there is room for.
  int c = 1;
  while (c < 8 && ((long)((a.vocab + c - 1) / c) * (long)sizeof(T) > 90000 || (a.vocab > c * 4096 && a.rows * c * 2 <= sm_count()))) c *= 2;
  a.ctas = c;
  a.per = ((a.vocab + c - 1) / c + 15) / 16 * 16;
  const size_t smem = (size_t)a.per * sizeof(T) + 32;
  if (smem > kDrSmem) return fail("draw: the vocabulary does not fit the shared memory of eight blocks%s");
  static bool attr[64];
  int dev = 0;
  GB_CUDA_OK(cudaGetDevice(&dev));
  if (dev > 63 || !attr[dev]) {
    GB_CUDA_OK(cudaFuncSetAttribute(draw_kernel<T, kDrThreads>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kDrSmem));
    if (dev < 64) attr[dev] = true;
  }
  launch_k_cluster(draw_kernel<T, kDrThreads>, (unsigned)(a.rows * c), kDrThreads, smem, stream, (unsigned)c, a);
  GB_CUDA_OK(cudaGetLastError());
  return 0;
}

template <typename T>
static int draw_for(const DrawArgs& a, cudaStream_t stream) {
  return a.vocab <= kDrShort && a.rows > 2 * sm_count() ? draw_launch<T, 256>(a, stream) : draw_launch<T, 512>(a, stream);
}

}  // namespace gb

using namespace gb;

// dtype: 0 = f32, 1 = bf16.  temperature / top_k / top_p / min_p: one value per row (device), or null and the value for all rows.
GB_API int gb_draw(const void* logits, long ld, int dtype, int rows, int vocab, const float* u, const float* temperature, float temperature_all,
                   const int* top_k, int top_k_all, const float* top_p, float top_p_all, const float* min_p, float min_p_all, int* out, float* logprob,
                   void* status, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (vocab < 1 || ld < vocab || rows > (1 << 27)) return fail("draw: bad sizes%s");
  DrawArgs a;
  memset(&a, 0, sizeof(a));
  a.logits = logits; a.ld = ld; a.rows = rows; a.vocab = vocab; a.u = u; a.temperature = temperature; a.temperature_all = temperature_all;
  a.top_k = top_k; a.top_k_all = top_k_all; a.top_p = top_p; a.top_p_all = top_p_all; a.min_p = min_p; a.min_p_all = min_p_all; a.out = out;
  a.logprob = logprob; a.status = (KernelStatus*)status;
  return dtype == 0 ? draw_for<float>(a, stream) : draw_for<__nv_bfloat16>(a, stream);
}

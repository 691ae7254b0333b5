// Attention of drafted tree nodes over a paged KV cache, for any head sizes and element types: the path of f32 caches and of head sizes the tcgen05 kernel
// (tree_attn.cu) is not built for.
//
// Node i of a sequence with context ctx and n nodes (cached at places ctx .. ctx + n - 1) sees the places j < ctx and the nodes whose bit is set in its mask; with a
// window, those less than it in front of the node's position (ctx + its depth; a place of the context has its number for position).  o = sum_j 2^(q . k_j - m) v_j / sum_j 2^(q . k_j - m); nothing seen: 0.
// Q arrives multiplied by scale * log2(e); scores, weights and sums are f32.  A key that is not seen takes no part, whatever its rows hold.
//
// Heads of up to 256 columns: a block has 16 rows of a KV head ((node, head) pairs, in the order of the tokens), four to a warp, and goes over the keys 32 at a time, K and V through
// shared memory as f32.  What bounds it is the chain of a step: rows fetched, four dot products a lane, sums over the warp.  16 sequences of 8 nodes on 2048 places, 32 query and 4 KV
// heads of 128, f32: 668 us; bf16, heads of 96: 496 us (the tcgen05 kernel, bf16, heads of 128: 37 us).
// Wider heads: one warp per (node, query head), a key a lane (the same f32 shape with a warp per row took 5157 us: every row reads its keys from L2 again).
#include "sm100.cuh"
#include "host_common.h"

namespace gb {

struct TreeAnyArgs {
  const void* q; const void* k; const void* v; void* out;      // q [T, hq, dk] with q_ts elements from token to token; caches [slots, hkv, dk / dv]; out [T, hq, dv]
  long q_ts;
  const int* cu_q; const int* kv_len; const int* block_table; const unsigned long long* mask; const int* positions;
  int max_pages, page_size, n_seqs, words;
  long num_slots;
  int tokens, hq, hkv, dk, dv, window;
};

__device__ __forceinline__ float ldt(const float* p) { return *p; }
__device__ __forceinline__ float ldt(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void stt(float* p, float v) { *p = v; }
__device__ __forceinline__ void stt(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

// First position in the window of a node (nodes have positions ctx to ctx + nodes - 1), and whether another node lies in a window that begins at position `from`.
__device__ __forceinline__ int tree_from(const TreeAnyArgs& a, long token, int ctx, int nodes) { return max(0, min(max(a.positions[token], ctx), ctx + nodes - 1) - a.window + 1); }
__device__ __forceinline__ bool tree_near(const TreeAnyArgs& a, int token, int ctx, int nodes, int from) {
  return from <= ctx || (token < a.tokens && min(a.positions[token], ctx + nodes - 1) >= from);
}

template <typename T>
__global__ void __launch_bounds__(128)
tree_any_kernel(const TreeAnyArgs a) {
  constexpr int NV = 32;                            // dv <= 1024
  pdl_wait();
  pdl_trigger();
  extern __shared__ float s_q[];                    // [4 warps][dk]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long item = (long)blockIdx.x * 4 + warp;
  if (item >= (long)a.tokens * a.hq) return;
  const int t = (int)(item / a.hq), h = (int)(item - (long)t * a.hq);
  T* o = (T*)a.out + ((size_t)t * a.hq + h) * a.dv;
  if (t >= a.cu_q[a.n_seqs]) return;                // behind the last sequence: left as it was
  int lo = 0, hi = a.n_seqs;
  while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (a.cu_q[mid] <= t) lo = mid; else hi = mid; }
  const int seq = lo, begin = a.cu_q[seq], n_nodes = a.cu_q[seq + 1] - begin;
  const int len = min(a.kv_len[seq], (int)min((long)a.max_pages * a.page_size, 0x7fffffffl)), ctx = max(0, a.kv_len[seq] - n_nodes);
  const int kvh = h / (a.hq / a.hkv);
  float* q = s_q + warp * a.dk;
  for (int c = lane; c < a.dk; c += 32) q[c] = ldt((const T*)a.q + (size_t)t * a.q_ts + (size_t)h * a.dk + c);
  __syncwarp();
  const int from = a.window > 0 ? tree_from(a, t, ctx, n_nodes) : 0, first = min(ctx, from);      // from: the first position in the window
  const int* bt = a.block_table + (size_t)seq * a.max_pages;
  float m = -INFINITY, l = 0.f, acc[NV];
#pragma unroll
  for (int c = 0; c < NV; ++c) acc[c] = 0.f;
  for (int b = first; b < len; b += 32) {
    const int j = b + lane;
    bool live = j < len;
    if (live && j >= ctx) {
      const int x = j - ctx;
      live = x < a.words * 64 && ((a.mask[(size_t)t * a.words + (x >> 6)] >> (x & 63)) & 1) && tree_near(a, begin + x, ctx, n_nodes, from);
    }
    long slot = 0;
    float sc = -INFINITY;
    if (live) {
      slot = (long)bt[j / a.page_size] * a.page_size + j % a.page_size;
      if (slot < 0 || slot >= a.num_slots) slot = 0;
      const T* kr = (const T*)a.k + ((size_t)slot * a.hkv + kvh) * a.dk;
      float s = 0.f;
      for (int c = 0; c < a.dk; ++c) s = fmaf(q[c], ldt(kr + c), s);
      sc = s;
    }
    const float mn = fmaxf(m, warp_max(sc));
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = exp2f(m - ref);
    const float p = live ? exp2f(sc - ref) : 0.f;
    m = mn;
    l = l * alpha + warp_sum(p);
#pragma unroll
    for (int c = 0; c < NV; ++c) acc[c] *= alpha;
    for (unsigned seen = __ballot_sync(0xffffffffu, live); seen; seen &= seen - 1) {
      const int y = __ffs(seen) - 1;
      const float py = __shfl_sync(0xffffffffu, p, y);
      const long sy = __shfl_sync(0xffffffffu, slot, y);
      const T* vr = (const T*)a.v + ((size_t)sy * a.hkv + kvh) * a.dv;
#pragma unroll
      for (int c = 0; c < NV; ++c) { const int e = lane + 32 * c; if (e < a.dv) acc[c] = fmaf(py, ldt(vr + e), acc[c]); }
    }
  }
#pragma unroll
  for (int c = 0; c < NV; ++c) { const int e = lane + 32 * c; if (e < a.dv) stt(o + e, l == 0.f ? 0.f : acc[c] / l); }
}

constexpr int kTyRows = 16, kTyKeys = 32, kTyWide = 256;

template <typename T, int NV>                       // dv <= 32 * NV
__global__ void __launch_bounds__(128)
tree_tile_kernel(const TreeAnyArgs a) {
  extern __shared__ __align__(16) float smem[];
  __shared__ long s_slot[kTyKeys];
  __shared__ int s_lo[kTyRows];
  float4* s_q = reinterpret_cast<float4*>(smem);                   // [4 warps][dk] a column of the warp's four rows
  float4* s_p = s_q + 4 * a.dk;                                    // [4 warps][32 keys] weights of the four rows
  float* s_k = reinterpret_cast<float*>(s_p + 4 * kTyKeys);        // [32][dk + 1]
  float* s_v = s_k + kTyKeys * (a.dk + 1);                         // [32][dv]
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.hq / a.hkv, kvh = blockIdx.y;
  const long rows = (long)min(a.tokens, max(a.cu_q[a.n_seqs], 0)) * G, r0 = (long)blockIdx.x * kTyRows, r1 = min(r0 + kTyRows, rows);      // (behind the last sequence: left as it was)
  auto row_of = [&](int k) { return r0 + warp * 4 + k; };
  for (int c = lane; c < a.dk; c += 32) {
    float q[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long r = row_of(k), t = r / G;
      q[k] = r < r1 ? ldt((const T*)a.q + (size_t)t * a.q_ts + (size_t)(kvh * G + (int)(r - t * G)) * a.dk + c) : 0.f;
    }
    s_q[warp * a.dk + c] = make_float4(q[0], q[1], q[2], q[3]);
  }
  for (long at = r0; at < r1;) {                                   // the rows of one sequence after the other
    const int t0 = (int)(at / G);
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (a.cu_q[mid] <= t0) lo = mid; else hi = mid; }
    const int seq = lo, begin = a.cu_q[seq], n_nodes = a.cu_q[seq + 1] - begin;
    const long to = min(r1, (long)max(a.cu_q[seq + 1], t0 + 1) * G);
    const int len = min(a.kv_len[seq], (int)min((long)a.max_pages * a.page_size, 0x7fffffffl)), ctx = max(0, a.kv_len[seq] - n_nodes);
    const int* bt = a.block_table + (size_t)seq * a.max_pages;
    if (threadIdx.x < kTyRows) {
      const long r = r0 + threadIdx.x;
      s_lo[threadIdx.x] = a.window > 0 && r >= at && r < to ? tree_from(a, r / G, ctx, n_nodes) : a.window > 0 ? ctx : 0;
    }
    __syncthreads();
    int first = ctx;
    for (int k = 0; k < kTyRows; ++k) first = min(first, s_lo[k]);
    float m[4], l[4], acc[4][NV];
    int from[4];
    bool mine[4];
    const unsigned long long* mask[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long r = row_of(k);
      mine[k] = r >= at && r < to;
      from[k] = s_lo[warp * 4 + k];
      mask[k] = a.mask + (size_t)(mine[k] ? r / G : t0) * a.words;
      m[k] = -INFINITY; l[k] = 0.f;
#pragma unroll
      for (int c = 0; c < NV; ++c) acc[k][c] = 0.f;
    }
    for (int b = first; b < len; b += kTyKeys) {
      if (threadIdx.x < kTyKeys) {
        const int j = b + threadIdx.x;
        long slot = j < len ? (long)bt[j / a.page_size] * a.page_size + j % a.page_size : 0;
        if (slot < 0 || slot >= a.num_slots) slot = 0;
        s_slot[threadIdx.x] = slot;
      }
      __syncthreads();                                             // (and the tiles before have been read)
      long slot[kTyKeys / 4];                                      // a warp fetches eight rows at a time
#pragma unroll
      for (int i = 0; i < kTyKeys / 4; ++i) slot[i] = s_slot[warp + 4 * i] * a.hkv + kvh;
      auto fetch = [&](const T* from, int width, float* to, int pitch) {
        for (int c = lane; c < width; c += 32) {
          float x[kTyKeys / 4];
#pragma unroll
          for (int i = 0; i < kTyKeys / 4; ++i) x[i] = ldt(from + (size_t)slot[i] * width + c);
#pragma unroll
          for (int i = 0; i < kTyKeys / 4; ++i) to[(warp + 4 * i) * pitch + c] = x[i];
        }
      };
      fetch((const T*)a.k, a.dk, s_k, a.dk + 1);
      fetch((const T*)a.v, a.dv, s_v, a.dv);
      __syncthreads();
      const int j = b + lane;
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      for (int c = 0; c < a.dk; ++c) {
        const float x = s_k[lane * (a.dk + 1) + c];
        const float4 q = s_q[warp * a.dk + c];
        s[0] = fmaf(q.x, x, s[0]); s[1] = fmaf(q.y, x, s[1]); s[2] = fmaf(q.z, x, s[2]); s[3] = fmaf(q.w, x, s[3]);
      }
      unsigned seen[4];
      float p[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        bool live = mine[k] && j < len;
        if (live && j < ctx) live = j >= from[k];
        else if (live) {
          const int x = j - ctx;
          live = x < a.words * 64 && ((mask[k][x >> 6] >> (x & 63)) & 1) && tree_near(a, begin + x, ctx, n_nodes, from[k]);
        }
        seen[k] = __ballot_sync(0xffffffffu, live);
        const float mn = fmaxf(m[k], warp_max(live ? s[k] : -INFINITY)), ref = mn == -INFINITY ? 0.f : mn, alpha = exp2f(m[k] - ref);
        p[k] = live ? exp2f(s[k] - ref) : 0.f;
        m[k] = mn;
        l[k] = l[k] * alpha + warp_sum(p[k]);
#pragma unroll
        for (int c = 0; c < NV; ++c) acc[k][c] *= alpha;
      }
      s_p[warp * kTyKeys + lane] = make_float4(p[0], p[1], p[2], p[3]);
      __syncwarp();
      for (unsigned any = seen[0] | seen[1] | seen[2] | seen[3]; any; any &= any - 1) {
        const int y = __ffs(any) - 1;
        const float4 w = s_p[warp * kTyKeys + y];
        float v[NV];
#pragma unroll
        for (int c = 0; c < NV; ++c) { const int e = lane + 32 * c; v[c] = e < a.dv ? s_v[y * a.dv + e] : 0.f; }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (!((seen[k] >> y) & 1)) continue;                     // (its value may be no number)
          const float wk = k == 0 ? w.x : k == 1 ? w.y : k == 2 ? w.z : w.w;
#pragma unroll
          for (int c = 0; c < NV; ++c) acc[k][c] = fmaf(wk, v[c], acc[k][c]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (!mine[k]) continue;
      const long r = row_of(k), t = r / G;
      T* o = (T*)a.out + ((size_t)t * a.hq + kvh * G + (int)(r - t * G)) * a.dv;
#pragma unroll
      for (int c = 0; c < NV; ++c) { const int e = lane + 32 * c; if (e < a.dv) stt(o + e, l[k] == 0.f ? 0.f : acc[k][c] / l[k]); }
    }
    __syncthreads();
    at = to;
  }
}

template <typename T, int NV>
static int tree_tile_launch(const TreeAnyArgs& a, cudaStream_t stream) {
  const size_t smem = (size_t)(4 * a.dk + 4 * kTyKeys) * 16 + (size_t)kTyKeys * (a.dk + 1 + a.dv) * 4;
  constexpr size_t kMost = (4 * kTyWide + 4 * kTyKeys) * 16 + kTyKeys * (2 * kTyWide + 1) * 4;
  static bool attr[64];
  int dev = 0;
  GB_CUDA_OK(cudaGetDevice(&dev));
  if (dev > 63 || !attr[dev]) {
    GB_CUDA_OK(cudaFuncSetAttribute(tree_tile_kernel<T, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost));
    if (dev < 64) attr[dev] = true;
  }
  const long rows = (long)a.tokens * (a.hq / a.hkv);
  launch_k(tree_tile_kernel<T, NV>, dim3((unsigned)((rows + kTyRows - 1) / kTyRows), a.hkv), 128, smem, stream, a);
  GB_CUDA_OK(cudaGetLastError());
  return 0;
}

template <typename T>
static int tree_any_launch(const TreeAnyArgs& a, cudaStream_t stream) {
  if (a.dk <= kTyWide && a.dv <= kTyWide && a.hkv <= 65535) return a.dv <= 64 ? tree_tile_launch<T, 2>(a, stream) : a.dv <= 128 ? tree_tile_launch<T, 4>(a, stream) : tree_tile_launch<T, 8>(a, stream);
  const unsigned grid = (unsigned)(((long)a.tokens * a.hq + 3) / 4);
  const size_t smem = (size_t)4 * a.dk * sizeof(float);
  launch_k(tree_any_kernel<T>, grid, 128, smem, stream, a);
  GB_CUDA_OK(cudaGetLastError());
  return 0;
}

}  // namespace gb

using namespace gb;

GB_API int gb_tree_any(const void* q, long q_ts, const void* k, const void* v, void* out, int f32, const int* cu_q, const int* kv_len, const int* block_table,
                       int max_pages, int page_size, const void* mask, int words, const int* positions, int n_seqs, long num_slots, int tokens, int hq, int hkv,
                       int dk, int dv, int window, cudaStream_t stream) {
  if (tokens <= 0 || n_seqs <= 0) return 0;
  if (hq < 1 || hkv < 1 || hq % hkv || dk < 1 || dv < 1 || page_size < 1 || max_pages < 0 || words < 1 || window < 0) return fail("tree_any: bad sizes%s");
  if (dk > 2048 || dv > 1024) return fail("tree_any: keys of at most 2048 and values of at most 1024 features%s");
  if (window > 0 && positions == nullptr) return fail("tree_any: a window needs the nodes' positions%s");
  if (num_slots < 1) return fail("tree_any: an empty cache%s");
  TreeAnyArgs a;
  a.q = q; a.k = k; a.v = v; a.out = out; a.q_ts = q_ts; a.cu_q = cu_q; a.kv_len = kv_len; a.block_table = block_table;
  a.mask = (const unsigned long long*)mask; a.positions = positions; a.max_pages = max_pages; a.page_size = page_size; a.n_seqs = n_seqs; a.words = words;
  a.num_slots = num_slots; a.tokens = tokens; a.hq = hq; a.hkv = hkv; a.dk = dk; a.dv = dv; a.window = window;
  return f32 ? tree_any_launch<float>(a, stream) : tree_any_launch<__nv_bfloat16>(a, stream);
}

// Attention of drafted tree nodes over a paged KV cache, for any head sizes and element types, one warp per (node, query head): the path of f32 caches and of head
// sizes the tcgen05 kernel (tree_attn.cu) is not built for.
//
// Node i of a sequence with context ctx and n nodes (cached at places ctx .. ctx + n - 1) sees the places j < ctx (with a window: position - j < window, where
// the node's position is ctx + its depth) and the nodes whose bit is set in its mask.  o = sum_j 2^(q . k_j - m) v_j / sum_j 2^(q . k_j - m); nothing seen: 0.
// Q arrives multiplied by scale * log2(e); scores, weights and sums are f32.  A key that is not seen takes no part, whatever its rows hold.
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

template <typename T, int NV>                       // dv <= 32 * NV
__global__ void __launch_bounds__(128)
tree_any_kernel(const TreeAnyArgs a) {
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
  const int first = a.window > 0 ? min(ctx, max(0, a.positions[t] - a.window + 1)) : 0;
  const int* bt = a.block_table + (size_t)seq * a.max_pages;
  float m = -INFINITY, l = 0.f, acc[NV];
#pragma unroll
  for (int c = 0; c < NV; ++c) acc[c] = 0.f;
  for (int b = first; b < len; b += 32) {
    const int j = b + lane;
    bool live = j < len;
    if (live && j >= ctx) {
      const int x = j - ctx;
      live = x < a.words * 64 && ((a.mask[(size_t)t * a.words + (x >> 6)] >> (x & 63)) & 1);
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

template <typename T>
static int tree_any_launch(const TreeAnyArgs& a, cudaStream_t stream) {
  const unsigned grid = (unsigned)(((long)a.tokens * a.hq + 3) / 4);
  const size_t smem = (size_t)4 * a.dk * sizeof(float);
  if (a.dv <= 64) launch_k(tree_any_kernel<T, 2>, grid, 128, smem, stream, a);
  else if (a.dv <= 128) launch_k(tree_any_kernel<T, 4>, grid, 128, smem, stream, a);
  else if (a.dv <= 256) launch_k(tree_any_kernel<T, 8>, grid, 128, smem, stream, a);
  else launch_k(tree_any_kernel<T, 32>, grid, 128, smem, stream, a);
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

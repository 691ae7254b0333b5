// Tables of a forward pass over a paged KV cache, from the lengths of its requests: token offsets, sequence lengths, positions, cache
// slots, block table and, for trees of drafted tokens, depths and ancestor masks.
//
//   cu[s] = q[0] + .. + q[s - 1];  token i of sequence s:  place = ctx[s] + i,  slot = page(s, place / P) P + place % P,
//   position = place (tree: ctx[s] + depth),  mask = bits of the node's ancestors and of itself.
//
// One launch.  The scan over the sequences is short (a few KB of lengths, in L2 after the first block has read them), so every block makes it for itself in
// shared memory instead of waiting for another launch; behind it the tokens and the block table's columns are independent, and are dealt out evenly, not by
// sequence: one long prompt would else be one block's work.  Latency bounds it: 32 trees of 16 nodes 3.9 us, 768 sequences of up to 60 tokens with 1024 pages at most 5.7 us (the tables are
// 6 MB: 0.9 us of bandwidth), the launch's own start and end about 3 us of either.
#include "sm100.cuh"
#include "host_common.h"
#include <algorithm>

namespace gb {

constexpr int kBtThreads = 512;
constexpr int kBtTokens = 512;      // tokens per block and turn
constexpr int kBtCols = 256;        // block-table columns per warp and turn
constexpr int kBtWords = 4;         // 64-bit words of a node's mask

struct BatchTablesArgs {
  const int* q_lens; const int* ctx_lens; const int* page_ptr; const int* pages; const int* parents;
  int n_seqs, n_listed, page_size, tokens, max_pages, words, max_nodes;
  int* cu_q; int* kv_len; int* positions; int* slots; int* block_table; unsigned long long* mask;
};

__global__ void __launch_bounds__(kBtThreads)
batch_tables_kernel(const BatchTablesArgs a) {
  extern __shared__ int s_cu[];                       // [n_seqs + 1], capped at `tokens`; then [kBtTokens + max_nodes] parents
  __shared__ int s_part[kBtThreads / 32];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // scan of the lengths: every thread adds a run of them, the runs are scanned over the block
  {
    const int per = (a.n_seqs + kBtThreads - 1) / kBtThreads;
    const int i0 = min(a.n_seqs, tid * per), i1 = min(a.n_seqs, i0 + per);
    long long sum = 0;
    for (int i = i0; i < i1; ++i) sum += max(a.q_lens[i], 0);
    const int mine = (int)min(sum, (long long)a.tokens);         // (no more than `tokens` counts: the sums stay small)
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl = min(incl + x, a.tokens); }
    if (lane == 31) s_part[warp] = incl;
    __syncthreads();
    if (warp == 0) {
      int v = lane < kBtThreads / 32 ? s_part[lane] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, v, o); if (lane >= o) v = min(v + x, a.tokens); }
      if (lane < kBtThreads / 32) s_part[lane] = v;
    }
    __syncthreads();
    // exclusive: what lies in front of the thread's run
    const int before = __shfl_up_sync(0xffffffffu, incl, 1);
    int at = min((warp > 0 ? s_part[warp - 1] : 0) + (lane > 0 ? before : 0), a.tokens);
    for (int i = i0; i < i1; ++i) { s_cu[i] = at; at = (int)min((long long)at + max(a.q_lens[i], 0), (long long)a.tokens); }
    if (i1 == a.n_seqs && i0 < i1) s_cu[a.n_seqs] = at;
    if (a.n_seqs == 0 && tid == 0) s_cu[0] = 0;
  }
  __syncthreads();
  const int total = s_cu[a.n_seqs];
  if (blockIdx.x == 0) {
    for (int i = tid; i <= a.n_seqs; i += kBtThreads) {
      a.cu_q[i] = s_cu[i];
      if (i < a.n_seqs) a.kv_len[i] = a.ctx_lens[i] + (s_cu[i + 1] - s_cu[i]);
    }
  }
  // block table: a warp takes 256 columns of a row
  {
    const int parts = (a.max_pages + kBtCols - 1) / kBtCols;
    const long items = (long)a.n_seqs * parts, step = (long)gridDim.x * (kBtThreads / 32);
    for (long it = (long)blockIdx.x * (kBtThreads / 32) + warp; it < items; it += step) {
      const int s = (int)(it / parts), c0 = (int)(it - (long)s * parts) * kBtCols;
      const int lo = max(a.page_ptr[s], 0), have = min(a.page_ptr[s + 1], a.n_listed) - lo;
      int* row = a.block_table + (size_t)s * a.max_pages;
      int v[kBtCols / 32];
#pragma unroll
      for (int k = 0; k < kBtCols / 32; ++k) { const int c = c0 + k * 32 + lane; v[k] = c < have ? a.pages[lo + c] : 0; }
#pragma unroll
      for (int k = 0; k < kBtCols / 32; ++k) { const int c = c0 + k * 32 + lane; if (c < a.max_pages) row[c] = v[k]; }
    }
  }
  // tokens
  int* s_par = s_cu + a.n_seqs + 1;
  for (int t0 = blockIdx.x * kBtTokens; t0 < a.tokens; t0 += gridDim.x * kBtTokens) {
    const int t = t0 + tid;
    int first = 0;                                    // the first token whose parent is held in shared memory
    if (a.parents != nullptr) {
      first = max(0, t0 - a.max_nodes);               // (a tree has at most max_nodes nodes: the ones of t0's own tree are there)
      __syncthreads();
      for (int i = first + tid; i < min(t0 + kBtTokens, total); i += kBtThreads) s_par[i - first] = a.parents[i];
      __syncthreads();
    }
    if (t >= a.tokens) continue;
    int pos = 0, slot = -1;
    unsigned long long m[kBtWords] = {0, 0, 0, 0};
    if (t < total) {
      int lo = 0, hi = a.n_seqs;                      // the last sequence that begins at or before t (empty ones begin where the next does)
      while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (s_cu[mid] <= t) lo = mid; else hi = mid; }
      const int s = lo, begin = s_cu[s], i = t - begin, ctx = a.ctx_lens[s];
      const int place = ctx + i, pg = place / a.page_size;
      const int p0 = max(a.page_ptr[s], 0), have = min(a.page_ptr[s + 1], a.n_listed) - p0;
      if (place >= 0 && pg < have) slot = (int)((long long)a.pages[p0 + pg] * a.page_size + place % a.page_size);
      pos = place;
      if (a.parents != nullptr) {
        int depth = 0, x = i;
        while (true) {
#pragma unroll
          for (int w = 0; w < kBtWords; ++w) if ((x >> 6) == w) m[w] |= 1ull << (x & 63);
          const int at = begin + x - first;
          const int p = at >= 0 ? s_par[at] : -1;
          if (p < 0 || p >= x) break;                 // the root, or no parent of its own: parents come in front of their children
          x = p; ++depth;
        }
        pos = ctx + depth;
      }
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
    if (a.parents != nullptr) {
#pragma unroll
      for (int w = 0; w < kBtWords; ++w) if (w < a.words) a.mask[(size_t)t * a.words + w] = m[w];
    }
  }
}

}  // namespace gb

using namespace gb;

GB_API int gb_batch_tables(const int* q_lens, const int* ctx_lens, const int* page_ptr, const int* pages, int n_listed, int n_seqs, int page_size, int tokens,
                           int max_pages, const int* parents, int max_nodes, int* cu_q, int* kv_len, int* positions, int* slots, int* block_table, void* mask,
                           cudaStream_t stream) {
  if (n_seqs < 0 || n_seqs > 8192 || page_size < 1 || tokens < 0 || max_pages < 0 || n_listed < 0) return fail("batch_tables: bad sizes%s");
  if (parents != nullptr && (max_nodes < 1 || max_nodes > 64 * kBtWords || mask == nullptr)) return fail("batch_tables: trees of 1 to 256 nodes%s");
  BatchTablesArgs a;
  memset(&a, 0, sizeof(a));
  a.q_lens = q_lens; a.ctx_lens = ctx_lens; a.page_ptr = page_ptr; a.pages = pages; a.parents = parents; a.n_seqs = n_seqs; a.n_listed = n_listed;
  a.page_size = page_size; a.tokens = tokens; a.max_pages = max_pages; a.words = (max_nodes + 63) / 64; a.max_nodes = max_nodes; a.cu_q = cu_q; a.kv_len = kv_len;
  a.positions = positions; a.slots = slots; a.block_table = block_table; a.mask = (unsigned long long*)mask;
  const long by_tokens = ((long)tokens + kBtTokens - 1) / kBtTokens;
  const long by_table = ((long)n_seqs * ((max_pages + kBtCols - 1) / kBtCols) + kBtThreads / 32 - 1) / (kBtThreads / 32);
  const long grid = std::min<long>(2 * sm_count(), std::max<long>(1, std::max(by_tokens, by_table)));
  const size_t smem = (size_t)(n_seqs + 1 + (parents != nullptr ? kBtTokens + max_nodes : 0)) * sizeof(int);      // at most 36 KB
  launch_k(batch_tables_kernel, (unsigned)grid, kBtThreads, smem, stream, a);
  GB_CUDA_OK(cudaGetLastError());
  return 0;
}

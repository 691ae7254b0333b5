// End of a verification step with trees of drafted tokens: along the path of drafts that the drawn tokens confirm, the K / V rows move to
// the positions directly behind the context, in every layer's cache.
//
// Sequence s has nodes 0 (the last certain token) .. n - 1 at places ctx + 0 .. ctx + n - 1 of the cache.  The walk: from node x to its first child whose token is
// the one drawn at x, as long as there is one.  Accepted node number j goes from place ctx + path[j] to ctx + j.  Since path[j] >= j and the path ascends,
// a thread that moves one column of a row in path order has read every row before it overwrites it: no staging.
//
// 64 trees of 64 nodes, 36 layers, 8 KV heads of 128: 63 MB move in 11.7 us, 5.4 TB/s; 4 trees, 28 layers: 3.3 us, the launch.
//
// One launch for all layers: a block handles one sequence and some of the caches, and makes the (short) walk for itself in one warp: a ballot per step, tokens
// and parents in registers.  Blocks of the first column of the grid also write the results.
#include "sm100.cuh"
#include "host_common.h"
#include <algorithm>
#include <utility>
#include <vector>

namespace gb {

constexpr int kTcThreads = 128;
constexpr int kTcNodes = 256;
constexpr int kTcCaches = 224;      // caches per launch (their addresses are kernel parameters)

struct TreeCommitArgs {
  void* cache[kTcCaches];
  int row_bytes[kTcCaches];
  int n_caches, per_block;
  const int* tokens; const int* parents; const int* sampled; const int* cu_q; const int* kv_len; const int* block_table;
  int max_pages, page_size, total_tokens, max_nodes;
  long num_slots;
  int* count; int* path; int* next_token; int* new_len;      // null in the launches behind the first
};

template <typename V>
__device__ __forceinline__ void move_rows(V* base, int cols, int moves, const long* s_src, const long* s_dst, int c0, int step) {
  for (int c = c0; c < cols; c += step) {
    for (int j = 0; j < moves; j += 4) {
      V v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) if (j + k < moves) v[k] = base[s_src[j + k] * cols + c];
#pragma unroll
      for (int k = 0; k < 4; ++k) if (j + k < moves) base[s_dst[j + k] * cols + c] = v[k];
    }
  }
}

__global__ void __launch_bounds__(kTcThreads)
tree_commit_kernel(const __grid_constant__ TreeCommitArgs a) {
  __shared__ int s_path[kTcNodes];
  __shared__ long s_src[kTcNodes], s_dst[kTcNodes];
  __shared__ int s_moves;
  pdl_wait();
  pdl_trigger();
  const int s = blockIdx.y, lane = threadIdx.x & 31;
  const int begin = min(max(a.cu_q[s], 0), a.total_tokens);
  const int n = min(max(min(a.cu_q[s + 1], a.total_tokens) - begin, 0), min(a.max_nodes, kTcNodes));
  const int len = a.kv_len[s], ctx = len - max(a.cu_q[s + 1] - a.cu_q[s], 0);
  if (threadIdx.x < 32) {
    int tok[kTcNodes / 32], par[kTcNodes / 32], drawn[kTcNodes / 32];
#pragma unroll
    for (int w = 0; w < kTcNodes / 32; ++w) {
      const int i = w * 32 + lane;
      const bool in = i < n;
      tok[w] = in ? a.tokens[begin + i] : 0;
      par[w] = in ? a.parents[begin + i] : -2;
      drawn[w] = in ? a.sampled[begin + i] : -1;
    }
    int cur = 0, got = n > 0 ? 1 : 0, want = 0;
    if (lane == 0 && n > 0) s_path[0] = 0;
    while (got > 0) {
      want = 0;                                              // the token drawn at `cur`
#pragma unroll
      for (int w = 0; w < kTcNodes / 32; ++w) if ((cur >> 5) == w) want = __shfl_sync(0xffffffffu, drawn[w], cur & 31);
      int next = -1;
#pragma unroll
      for (int w = kTcNodes / 32 - 1; w >= 0; --w) {
        if (w * 32 >= n) continue;
        const unsigned hit = __ballot_sync(0xffffffffu, par[w] == cur && tok[w] == want && w * 32 + lane > cur);
        if (hit) next = w * 32 + __ffs(hit) - 1;
      }
      if (next < 0) break;
      if (lane == 0) s_path[got] = next;
      cur = next; ++got;
    }
    __syncwarp();
    if (blockIdx.x == 0 && a.count != nullptr) {
      for (int i = lane; i < a.max_nodes; i += 32) a.path[(size_t)s * a.max_nodes + i] = i < got ? s_path[i] : -1;
      if (lane == 0) { a.count[s] = got; a.next_token[s] = n > 0 ? want : -1; a.new_len[s] = ctx + got; }
    }
    // the rows that move
    const int* bt = a.block_table + (size_t)s * a.max_pages;
    int moves = 0;
    for (int b = 0; b < got; b += 32) {
      const int j = b + lane;
      long from = -1, to = -1;
      if (j < got && s_path[j] != j) {
        const int p0 = ctx + s_path[j], p1 = ctx + j;
        if (p1 >= 0 && p0 / a.page_size < a.max_pages) {
          from = (long)bt[p0 / a.page_size] * a.page_size + p0 % a.page_size;
          to = (long)bt[p1 / a.page_size] * a.page_size + p1 % a.page_size;
        }
      }
      const bool ok = from >= 0 && to >= 0 && from < a.num_slots && to < a.num_slots;
      const unsigned m = __ballot_sync(0xffffffffu, ok);
      if (ok) { const int at = moves + __popc(m & ((1u << lane) - 1)); s_src[at] = from; s_dst[at] = to; }
      moves += __popc(m);
    }
    if (lane == 0) s_moves = moves;
  }
  __syncthreads();
  const int moves = s_moves;
  if (moves == 0) return;
  const int c_end = min(a.n_caches, (int)(blockIdx.x + 1) * a.per_block);
  for (int c = blockIdx.x * a.per_block; c < c_end; ++c) {
    const int rb = a.row_bytes[c];
    const uintptr_t base = (uintptr_t)a.cache[c];
    if (((base | rb) & 15) == 0) move_rows((uint4*)base, rb / 16, moves, s_src, s_dst, threadIdx.x, kTcThreads);
    else if (((base | rb) & 3) == 0) move_rows((uint32_t*)base, rb / 4, moves, s_src, s_dst, threadIdx.x, kTcThreads);
    else move_rows((uint8_t*)base, rb, moves, s_src, s_dst, threadIdx.x, kTcThreads);
  }
}

}  // namespace gb

using namespace gb;

// caches[i]: num_slots rows, bytes[i] in all (host arrays; a cache without bytes is passed over).  No caches: the walk alone.
GB_API int gb_tree_commit(const void* const* caches, const long long* bytes, int n_caches, long num_slots, const int* tokens, const int* parents, const int* sampled,
                          const int* cu_q, const int* kv_len, const int* block_table, int max_pages, int page_size, int n_seqs, int total_tokens, int max_nodes,
                          int* count, int* path, int* next_token, int* new_len, cudaStream_t stream) {
  if (n_seqs <= 0) return 0;
  if (n_seqs > 65535 || n_caches < 0 || page_size < 1 || max_pages < 0 || total_tokens < 0 || max_nodes < 1 || max_nodes > kTcNodes) return fail("tree_commit: bad sizes%s");
  // a row moved twice, or by two blocks at once, would be read after it was written
  try {
    std::vector<std::pair<uintptr_t, long long>> at;
    at.reserve(n_caches);
    for (int i = 0; i < n_caches; ++i) if (bytes[i] > 0) at.emplace_back((uintptr_t)caches[i], bytes[i]);
    std::sort(at.begin(), at.end());
    for (size_t i = 1; i < at.size(); ++i) if (at[i - 1].first + at[i - 1].second > at[i].first) return fail("tree_commit: caches that overlap%s");
  } catch (...) { return fail("tree_commit: out of memory%s"); }
  TreeCommitArgs a;
  int done = 0;
  do {
    a.n_caches = 0;
    a.count = a.path = a.next_token = a.new_len = nullptr;
    const int n_here = std::min(n_caches - done, kTcCaches);
    for (int i = 0; i < n_here; ++i) {
      const long long row = num_slots > 0 ? bytes[done + i] / num_slots : 0;
      if (row <= 0) continue;
      if (row > (1 << 30)) return fail("tree_commit: rows of at most 2^30 bytes%s");
      a.cache[a.n_caches] = const_cast<void*>(caches[done + i]);
      a.row_bytes[a.n_caches++] = (int)row;
    }
    // enough blocks to fill the GPU a few times over, no more walks than that
    a.per_block = std::max(1, (int)((long)a.n_caches * n_seqs / (16l * sm_count())));
    a.tokens = tokens; a.parents = parents; a.sampled = sampled; a.cu_q = cu_q; a.kv_len = kv_len; a.block_table = block_table; a.max_pages = max_pages;
    a.page_size = page_size; a.total_tokens = total_tokens; a.max_nodes = max_nodes; a.num_slots = num_slots;
    if (done == 0) { a.count = count; a.path = path; a.next_token = next_token; a.new_len = new_len; }
    launch_k(tree_commit_kernel, dim3(std::max(1, (a.n_caches + a.per_block - 1) / a.per_block), n_seqs), kTcThreads, 0, stream, a);
    GB_CUDA_OK(cudaGetLastError());
    done += n_here;
  } while (done < n_caches);
  return 0;
}

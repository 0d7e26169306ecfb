// Where the drafted tokens of a speculative step sit, and which of them each one descends from (gfx950).
//
// A row drafts a tree: node 0 is the last accepted token, parents[i] < i the node that node i follows.
// anc(i) = {i} and the ancestors of its parent.  Node i's depth is |anc(i)| - 1, its position (what the
// rotary embedding takes) context_len + depth, its cache slot that of position context_len + i: nodes of
// one depth share a position but never a slot.  The reference drafts chains only and keeps no layout
// (src/inference/speculative.py).
//
// One workgroup per row, one thread per node.  anc() by pointer doubling in LDS: after round r every node
// holds its nearest 2^r ancestors as a bit set of 64-bit words and a pointer past them, so a round ORs one
// set into another and a chain of 64 takes 6 rounds instead of 64 dependent steps.  Bound by the launch:
// a row reads and writes a few hundred bytes.
#include "pa_common.hpp"
#include "pa_host.hpp"

namespace pa {

struct LayoutParams {
  const int32_t* parents;
  int64_t parents_stride;      // 0: one tree for every row
  const int32_t* context_lens;
  const int32_t* num_nodes;    // nullptr: every row drafts `nodes`
  const int32_t* block_tables; // nullptr: no slots
  int64_t bt_stride;
  int64_t* positions;
  int32_t* slots;
  uint64_t* mask;
  int nodes, table_width, block_size, num_blocks;
};

template <int T>
__global__ __launch_bounds__(T) void draft_layout_kernel(const LayoutParams p) {
  constexpr int W = T / 64;                   // words of a set
  __shared__ int next[T];                     // the nearest ancestor not yet in the set, -1: none
  __shared__ uint64_t seen[W][T];
  const int b = blockIdx.x, i = threadIdx.x;
  const int32_t* parents = p.parents + b * p.parents_stride;
  int up = -1;
  if (i < p.nodes) {
    up = parents[i];
    if (up < 0 || up >= i) up = -1;           // the root, or no tree: the node then descends from itself alone
  }
  uint64_t set[W];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    set[w] = (i >> 6) == w ? 1ull << (i & 63) : 0ull;
    seen[w][i] = set[w];
  }
  next[i] = up;
  __syncthreads();
  for (int reach = 1; reach < p.nodes; reach *= 2) {
    int past = -1;
    if (up >= 0) {
      past = next[up];
#pragma unroll
      for (int w = 0; w < W; ++w) set[w] |= seen[w][up];
    }
    __syncthreads();
    up = past;
    next[i] = up;
#pragma unroll
    for (int w = 0; w < W; ++w) seen[w][i] = set[w];
    __syncthreads();
  }
  if (i >= p.nodes) return;
  const int words = (p.nodes + 63) >> 6;
  if (p.parents_stride != 0 || b == 0) {
    uint64_t* row = p.mask + ((p.parents_stride != 0 ? (int64_t)b * p.nodes : 0) + i) * words;
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (w < words) row[w] = set[w];
  }
  int depth = -1;
#pragma unroll
  for (int w = 0; w < W; ++w) depth += __popcll(set[w]);
  const int64_t base = p.context_lens[b];
  const int real = base < 0 ? 0 : p.num_nodes ? min(p.num_nodes[b], p.nodes) : p.nodes;
  const int64_t at = (int64_t)b * p.nodes + i;
  p.positions[at] = i < real ? base + depth : 0;
  if (p.block_tables) {
    int slot = -1;
    if (i < real) {
      const int64_t pos = base + i, col = pos / p.block_size;
      if (col < p.table_width) {
        const int id = p.block_tables[b * p.bt_stride + col];
        if (id >= 0 && id < p.num_blocks) slot = (int)((int64_t)id * p.block_size + pos % p.block_size);
      }
    }
    p.slots[at] = slot;
  }
}

}  // namespace pa

using namespace pa;

extern "C" int pa_draft_layout(const int32_t* parents, int64_t parents_stride, const int32_t* context_lens,
                               const int32_t* num_nodes, const int32_t* block_tables, int64_t bt_stride,
                               int64_t table_width, int64_t* positions, int32_t* slots, uint64_t* tree_mask,
                               int64_t batch, int64_t nodes, int64_t block_size, int64_t num_blocks, void* stream) {
  if (batch < 0 || nodes < 0) return fail(PA_ERR_BAD_ARG, "pa_draft_layout: negative size");
  if (batch == 0 || nodes == 0) return PA_OK;
  if (nodes > PA_MAX_DRAFT_NODES) return fail(PA_ERR_UNSUPPORTED, "pa_draft_layout: more than 256 nodes a row");
  if (batch > 0x7fffffff) return fail(PA_ERR_UNSUPPORTED, "pa_draft_layout: batch too large");
  if (!parents || !context_lens || !positions || !tree_mask) return fail(PA_ERR_BAD_ARG, "pa_draft_layout: null pointer");
  if (parents_stride != 0 && parents_stride < nodes)
    return fail(PA_ERR_BAD_ARG, "pa_draft_layout: parents rows overlap (stride smaller than the nodes of a row)");
  if (block_tables) {
    if (!slots) return fail(PA_ERR_BAD_ARG, "pa_draft_layout: block_tables without slots");
    if (block_size <= 0 || num_blocks <= 0 || table_width <= 0 || bt_stride < table_width || table_width > 0x7fffffff)
      return fail(PA_ERR_BAD_ARG, "pa_draft_layout: block table or pool sizes out of range");
    if (num_blocks > 0x7fffffff / block_size) return fail(PA_ERR_UNSUPPORTED, "pa_draft_layout: slots beyond 32 bits");
  }
  LayoutParams p = {parents, parents_stride, context_lens, num_nodes, block_tables, bt_stride, positions, slots, tree_mask,
                    (int)nodes, (int)table_width, (int)block_size, (int)num_blocks};
  const dim3 grid((unsigned)batch);
  hipStream_t st = (hipStream_t)stream;
  if (nodes <= 64) hipLaunchKernelGGL(draft_layout_kernel<64>, grid, dim3(64), 0, st, p);
  else if (nodes <= 128) hipLaunchKernelGGL(draft_layout_kernel<128>, grid, dim3(128), 0, st, p);
  else hipLaunchKernelGGL(draft_layout_kernel<256>, grid, dim3(256), 0, st, p);
  return check_launch("pa_draft_layout");
}

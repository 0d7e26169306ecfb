// Keeping the accepted tokens of a speculative step (gfx950): the K and V rows of the accepted path move to
// consecutive cache positions, in every layer.
//
// The forward pass wrote node i's row at position context_len + i.  path[0..counts) are the nodes kept, in
// ascending order (node 0 first: path[j] >= j), so row path[j] moves to position context_len + j.  No source
// of a later move is an earlier move's target (path[k] > path[j] >= j for k > j), and a thread owns one
// 16-byte column of a row in one plane for all the row's moves: it reads kBatch sources ahead, then writes
// their targets, and needs no synchronisation with anyone.
//
// The pool is [planes][slots][row_bytes] with planes = 2 x layers (all of K, then all of V); fp8 pools carry a
// float per slot and layer beside each, moved by the first column's thread.  Bound by HBM and, for a few rows,
// by the launch and two dependent loads (table entry, row).
#include "pa_common.hpp"
#include "pa_host.hpp"

namespace pa {

typedef uint32_t piece_t __attribute__((ext_vector_type(4)));

constexpr int kCommitBatch = 8;      // rows a thread holds between reading and writing

struct CommitParams {
  uint8_t* pool;
  int64_t plane_stride;              // bytes
  float* k_scale;                    // [layers][scale_stride], nullptr: none
  float* v_scale;
  int64_t scale_stride;              // floats between layers
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* context_lens;
  const int32_t* path;
  int64_t path_stride;
  const int32_t* counts;
  int32_t* new_lens;
  int row_bytes, layers, nodes, table_width, block_size, num_blocks;
};

__global__ __launch_bounds__(256) void draft_commit_kernel(const CommitParams p) {
  const int plane = blockIdx.x, b = blockIdx.y;
  const int base = p.context_lens[b];
  const int count = base < 0 ? 0 : min(max(p.counts[b], 0), p.nodes);
  if (plane == 0 && threadIdx.x == 0) p.new_lens[b] = base + count;
  // where move j reads and writes: -1 = stays (in place already, no node of this row, outside the table or the pool)
  __shared__ int from[PA_MAX_DRAFT_NODES], to[PA_MAX_DRAFT_NODES];
  const int32_t* table = p.block_tables + b * p.bt_stride;
  auto slot_of = [&](int pos) {
    const int col = pos / p.block_size;
    const int id = col < p.table_width ? table[col] : -1;
    return id >= 0 && id < p.num_blocks ? id * p.block_size + pos % p.block_size : -1;
  };
  for (int j = threadIdx.x; j < count; j += blockDim.x) {
    const int node = p.path[b * p.path_stride + j];
    int src = -1, dst = -1;
    if (node > j && node < p.nodes && base <= 0x7fffffff - PA_MAX_DRAFT_NODES) {
      src = slot_of(base + node);
      dst = slot_of(base + j);
    }
    from[j] = dst >= 0 ? src : -1;
    to[j] = dst;
  }
  __syncthreads();
  float* scale = nullptr;
  if (p.k_scale)
    scale = plane < p.layers ? p.k_scale + plane * p.scale_stride : p.v_scale + (plane - p.layers) * p.scale_stride;
  uint8_t* rows = p.pool + plane * p.plane_stride;
  for (int col = threadIdx.x * 16; col < p.row_bytes; col += blockDim.x * 16) {
    for (int j0 = 1; j0 < count; j0 += kCommitBatch) {
      piece_t held[kCommitBatch];
      float held_scale[kCommitBatch];
      int src[kCommitBatch];
#pragma unroll
      for (int k = 0; k < kCommitBatch; ++k) {
        src[k] = j0 + k < count ? from[j0 + k] : -1;
        held[k] = piece_t{0, 0, 0, 0};
        held_scale[k] = 0.0f;
        if (src[k] >= 0) {
          held[k] = *(const piece_t*)(rows + (int64_t)src[k] * p.row_bytes + col);
          if (scale && col == 0) held_scale[k] = scale[src[k]];
        }
      }
#pragma unroll
      for (int k = 0; k < kCommitBatch; ++k)
        if (src[k] >= 0) {
          const int64_t dst = to[j0 + k];
          *(piece_t*)(rows + dst * p.row_bytes + col) = held[k];
          if (scale && col == 0) scale[dst] = held_scale[k];
        }
    }
  }
}

}  // namespace pa

using namespace pa;

extern "C" int pa_draft_commit(void* pool, int64_t layers, int64_t plane_stride_bytes, int64_t row_bytes, float* k_scale,
                               float* v_scale, int64_t scale_stride, const int32_t* block_tables, int64_t bt_stride,
                               int64_t table_width, const int32_t* context_lens, const int32_t* path,
                               int64_t path_stride, const int32_t* counts, int32_t* new_lens, int64_t batch,
                               int64_t nodes, int64_t block_size, int64_t num_blocks, void* stream) {
  if (batch < 0 || nodes < 0 || layers < 0) return fail(PA_ERR_BAD_ARG, "pa_draft_commit: negative size");
  if (batch == 0 || layers == 0) return PA_OK;
  if (nodes > PA_MAX_DRAFT_NODES) return fail(PA_ERR_UNSUPPORTED, "pa_draft_commit: more than 256 nodes a row");
  if (!pool || !block_tables || !context_lens || !path || !counts || !new_lens)
    return fail(PA_ERR_BAD_ARG, "pa_draft_commit: null pointer");
  if (new_lens == context_lens)
    return fail(PA_ERR_BAD_ARG, "pa_draft_commit: new_lens must not be context_lens (other workgroups still read them)");
  if ((k_scale == nullptr) != (v_scale == nullptr)) return fail(PA_ERR_BAD_ARG, "pa_draft_commit: one of the two scales is missing");
  if (block_size <= 0 || num_blocks <= 0 || table_width <= 0 || bt_stride < table_width || path_stride < nodes ||
      row_bytes <= 0 || block_size > 0x7fffffff || num_blocks > 0x7fffffff || table_width > 0x7fffffff || row_bytes > 0x7fffffff)
    return fail(PA_ERR_BAD_ARG, "pa_draft_commit: size or stride out of range");
  if (plane_stride_bytes / row_bytes / block_size < num_blocks || (k_scale && scale_stride / block_size < num_blocks))
    return fail(PA_ERR_BAD_ARG, "pa_draft_commit: plane stride smaller than a plane");
  if (row_bytes % 16 != 0 || plane_stride_bytes % 16 != 0 || !aligned16(pool))
    return fail(PA_ERR_UNSUPPORTED, "pa_draft_commit: rows and planes must be multiples of 16 bytes, the pool 16-byte aligned");
  if (num_blocks > 0x7fffffff / block_size) return fail(PA_ERR_UNSUPPORTED, "pa_draft_commit: slots beyond 32 bits");
  if (batch > 65535 || layers > 0x3fffffff) return fail(PA_ERR_UNSUPPORTED, "pa_draft_commit: more than 65535 rows in one launch");
  CommitParams p = {(uint8_t*)pool, plane_stride_bytes, k_scale, v_scale, scale_stride, block_tables, bt_stride, context_lens,
                    path, path_stride, counts, new_lens, (int)row_bytes, (int)layers, (int)nodes, (int)table_width,
                    (int)block_size, (int)num_blocks};
  const int64_t pieces = row_bytes / 16;
  const unsigned threads = pieces >= 256 ? 256 : (unsigned)((pieces + 63) / 64 * 64);
  hipLaunchKernelGGL(draft_commit_kernel, dim3((unsigned)(2 * layers), (unsigned)batch), dim3(threads), 0, (hipStream_t)stream, p);
  return check_launch("pa_draft_commit");
}

// Drafted-token attention: the merge over partitions, and the C entry points.
#include "draft_attention_kernel.hpp"

namespace pa {

// One wave per (node, query head) row.  out = sum_p w_p out_p / sum_p w_p with w_p = sum_p * 2^(max_p - max) over the
// partitions of the row that hold tokens; a row that saw nothing in any of them is zero, and so is a node that the row
// does not draft.
template <int D>
__global__ __launch_bounds__(256) void draft_merge_kernel(const DraftParams p) {
  constexpr int PER = D / 64;
  const int lane = threadIdx.x & 63;
  const int head = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int node = blockIdx.y, b = blockIdx.z;
  if (head >= p.num_q_heads) return;
  const int64_t o = ((int64_t)b * p.nodes + node) * p.out_stride + (int64_t)head * D + lane * PER;
  float acc[PER] = {};
  if (node < draft_nodes(p, b)) {
    const int np = min((draft_keys(p, b) + p.partition_size - 1) / p.partition_size, p.max_partitions);
    const int64_t row = (((int64_t)b * p.nodes + node) * p.num_q_heads + head) * p.max_partitions;
    float top = -INFINITY;
    for (int q = lane; q < np; q += 64) top = fmaxf(top, p.ws_max[row + q]);
    top = wave_max(top);
    if (top != -INFINITY) {
      float den = 0.0f;
#pragma unroll 4
      for (int q = 0; q < np; ++q) {
        const float w = p.ws_sum[row + q] * __builtin_amdgcn_exp2f(p.ws_max[row + q] - top);
        den += w;
#pragma unroll
        for (int d = 0; d < PER; ++d) {
          const float v = p.ws_out[(row + q) * D + lane * PER + d];
          acc[d] = w != 0.0f ? fmaf(w, v, acc[d]) : acc[d];
        }
      }
#pragma unroll
      for (int d = 0; d < PER; ++d) acc[d] /= den;
    }
  }
#pragma unroll
  for (int d = 0; d < PER; ++d) store_from_f32(p.out, o + d, p.q_dtype, acc[d]);
}

static int64_t draft_rows_bytes(int64_t rows) { return (rows * 4 + 255) / 256 * 256; }

}  // namespace pa

using namespace pa;

extern "C" int64_t pa_draft_workspace_bytes(int64_t batch, int64_t nodes, int64_t num_q_heads, int64_t head_dim,
                                            int64_t max_partitions) {
  if (batch <= 0 || nodes <= 0 || num_q_heads <= 0 || head_dim <= 0 || max_partitions <= 1) return 0;
  const int64_t rows = batch * nodes * num_q_heads * max_partitions;
  return 2 * draft_rows_bytes(rows) + rows * head_dim * 4;
}

extern "C" int pa_draft_attention(const void* q, int q_dtype, int64_t q_stride, const void* k_cache, const void* v_cache,
                                  const float* k_scale, const float* v_scale, int kv_dtype, const int32_t* block_tables,
                                  int64_t bt_stride, int64_t table_width, const int32_t* context_lens,
                                  const int32_t* num_nodes, const uint64_t* tree_mask, int64_t mask_stride, void* out,
                                  int64_t out_stride, int64_t batch, int64_t nodes, int64_t num_q_heads,
                                  int64_t num_kv_heads, int64_t head_dim, int64_t block_size, int64_t num_blocks,
                                  float scale, int64_t partition_size, int64_t max_partitions, void* workspace,
                                  int64_t workspace_bytes, int col_tiles, void* stream) {
#define DRAFT_FAIL(code, text) return fail(code, "pa_draft_attention: " text)
  if (batch < 0 || nodes < 0) DRAFT_FAIL(PA_ERR_BAD_ARG, "negative size");
  if (batch == 0 || nodes == 0) return PA_OK;
  if (!q || !k_cache || !v_cache || !block_tables || !context_lens || !tree_mask || !out) DRAFT_FAIL(PA_ERR_BAD_ARG, "null pointer");
  if (nodes > PA_MAX_DRAFT_NODES) DRAFT_FAIL(PA_ERR_UNSUPPORTED, "more than 256 nodes a row");
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0)
    DRAFT_FAIL(PA_ERR_BAD_ARG, "num_q_heads must be a positive multiple of num_kv_heads");
  if (num_q_heads > 65535 || batch > 65535) DRAFT_FAIL(PA_ERR_UNSUPPORTED, "more than 65535 rows or heads in one launch");
  if (head_dim != 64 && head_dim != 128) DRAFT_FAIL(PA_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (block_size < 8 || (block_size & (block_size - 1)) != 0 || block_size > (1 << 20))
    DRAFT_FAIL(PA_ERR_UNSUPPORTED, "block_size must be a power of two from 8 on");
  if (num_blocks <= 0 || num_blocks > 0x7fffffff || table_width <= 0 || table_width > 0x7fffffff || bt_stride < table_width)
    DRAFT_FAIL(PA_ERR_BAD_ARG, "pool or table sizes out of range");
  if (q_dtype != PA_DTYPE_F16 && q_dtype != PA_DTYPE_BF16 && q_dtype != PA_DTYPE_F32) DRAFT_FAIL(PA_ERR_UNSUPPORTED, "q must be f16, bf16 or f32");
  const int qe = q_dtype == PA_DTYPE_F32 ? 4 : 2;
  const int kvb = kv_dtype == PA_DTYPE_FP8_E4M3 ? 1 : 2;
  if (kv_dtype != PA_DTYPE_F16 && kv_dtype != PA_DTYPE_BF16 && kv_dtype != PA_DTYPE_FP8_E4M3)
    DRAFT_FAIL(PA_ERR_UNSUPPORTED, "the cache must be f16, bf16 or fp8");
  if (kv_dtype == PA_DTYPE_FP8_E4M3 && (!k_scale || !v_scale || !aligned16(k_scale) || !aligned16(v_scale)))
    DRAFT_FAIL(PA_ERR_BAD_ARG, "an fp8 cache needs 16-byte aligned k_scale and v_scale");
  if (q_stride < num_q_heads * head_dim || out_stride < num_q_heads * head_dim) DRAFT_FAIL(PA_ERR_BAD_ARG, "node stride smaller than a node's heads");
  if (!aligned16(q) || (q_stride * qe) % 16 != 0 || !aligned16(k_cache) || !aligned16(v_cache))
    DRAFT_FAIL(PA_ERR_BAD_ARG, "q rows and caches must be 16-byte aligned");
  if (num_kv_heads * head_dim * kvb > (int64_t)0x7fffffff / block_size) DRAFT_FAIL(PA_ERR_UNSUPPORTED, "a cache block beyond 2 GiB");
  const int64_t words = (nodes + 63) / 64;
  if (mask_stride != 0 && mask_stride < nodes * words) DRAFT_FAIL(PA_ERR_BAD_ARG, "mask rows overlap");
  if (!(scale > 0.0f) || !(scale < INFINITY)) DRAFT_FAIL(PA_ERR_BAD_ARG, "scale must be positive and finite");
  if (col_tiles != 0 && col_tiles != 1 && col_tiles != 2) DRAFT_FAIL(PA_ERR_BAD_ARG, "col_tiles must be 0, 1 or 2");
  if (max_partitions < 1) DRAFT_FAIL(PA_ERR_BAD_ARG, "max_partitions must be positive");
  if (max_partitions > 1) {
    if (partition_size <= 0 || partition_size % 32 != 0 || partition_size > 0x7fffff00)
      DRAFT_FAIL(PA_ERR_UNSUPPORTED, "partition_size must be a positive multiple of 32");
    if (!workspace || workspace_bytes < pa_draft_workspace_bytes(batch, nodes, num_q_heads, head_dim, max_partitions))
      DRAFT_FAIL(PA_ERR_WORKSPACE, "workspace missing or too small");
    if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) DRAFT_FAIL(PA_ERR_BAD_ARG, "workspace must be 256-byte aligned");
  }
  const int64_t gq = num_q_heads / num_kv_heads, rows = nodes * gq;
  if (col_tiles == 0) col_tiles = rows <= 16 ? 1 : 2;
  DraftParams p;
  p.q = q;
  p.q_stride = q_stride;
  p.k_cache = (const uint8_t*)k_cache;
  p.v_cache = (const uint8_t*)v_cache;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_tables = block_tables;
  p.bt_stride = bt_stride;
  p.context_lens = context_lens;
  p.num_nodes = num_nodes;
  p.mask = tree_mask;
  p.mask_stride = mask_stride;
  p.out = out;
  p.out_stride = out_stride;
  p.ws_max = p.ws_sum = p.ws_out = nullptr;
  if (max_partitions > 1) {
    const int64_t part_rows = batch * nodes * num_q_heads * max_partitions;
    p.ws_max = (float*)workspace;
    p.ws_sum = (float*)((uint8_t*)workspace + draft_rows_bytes(part_rows));
    p.ws_out = (float*)((uint8_t*)workspace + 2 * draft_rows_bytes(part_rows));
  }
  p.q_dtype = q_dtype;
  p.nodes = (int)nodes;
  p.words = (int)words;
  p.num_q_heads = (int)num_q_heads;
  p.num_kv_heads = (int)num_kv_heads;
  p.table_width = (int)table_width;
  p.bs_log2 = __builtin_ctzll((unsigned long long)block_size);
  p.num_blocks = (int)num_blocks;
  p.partition_size = (int)partition_size;
  p.max_partitions = (int)max_partitions;
  p.batch = (int)batch;
  p.row_tiles = (int)((rows + 16 * col_tiles - 1) / (16 * col_tiles));
  p.scale_log2e = scale * 1.4426950408889634f;
  const int64_t wgs = batch * max_partitions * num_kv_heads * p.row_tiles;
  if (wgs > 0x7fffffff) DRAFT_FAIL(PA_ERR_UNSUPPORTED, "too many workgroups for one launch");
#undef DRAFT_FAIL
  hipStream_t st = (hipStream_t)stream;
  int rc;
  if (kv_dtype == PA_DTYPE_F16) rc = launch_draft_f16(p, (int)head_dim, col_tiles, (unsigned)wgs, st);
  else if (kv_dtype == PA_DTYPE_FP8_E4M3) rc = launch_draft_fp8(p, (int)head_dim, col_tiles, (unsigned)wgs, st);
  else if (q_dtype == PA_DTYPE_BF16) rc = launch_draft_bf16(p, (int)head_dim, col_tiles, (unsigned)wgs, st);
  else rc = launch_draft_bf16_as_f16(p, (int)head_dim, col_tiles, (unsigned)wgs, st);
  if (rc != PA_OK) return rc;
  if (max_partitions > 1) {
    const dim3 grid((unsigned)((num_q_heads + 3) / 4), (unsigned)nodes, (unsigned)batch);
    if (head_dim == 128) hipLaunchKernelGGL(draft_merge_kernel<128>, grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL(draft_merge_kernel<64>, grid, dim3(256), 0, st, p);
  }
  return check_launch("pa_draft_attention");
}

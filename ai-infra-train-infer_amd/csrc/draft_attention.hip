// Drafted-token attention: the merge over partitions, and the C entry points.
#include "draft_attention_kernel.hpp"

namespace pa {

// out = sum_p w_p out_p / sum_p w_p with w_p = sum_p * 2^(max_p - max) over the partitions of a (node, query head) row that
// hold tokens; a partition without a maximum weighs nothing, or NaN if it met a score of NaN.  A row that saw nothing in any of
// them is zero, and so is a node that the row does not draft.
// D / 4 threads read one partial result 16 bytes each; `slots` of them side by side take the row's partitions in turn, and
// 256 / (slots x D / 4) rows share a workgroup: with few partitions a row needs few threads, with many they are read at once.
// Bound by latency: the maxima and sums, the context length that says how many of them count, and the first partial results
// are all asked for before anything is waited for (whatever lies behind the row's last partition is loaded and not used),
// and the weights meet in LDS.
constexpr int kDraftMergeThreads = 256;
constexpr int kDraftMergeAhead = 4;       // partial results per thread in flight

template <int D>
__global__ __launch_bounds__(kDraftMergeThreads) void draft_merge_kernel(const DraftParams p, const int slots, const int rows) {
  extern __shared__ float lds[];            // rows of the workgroup x (2 x max_partitions), then 256 x 4 floats
  constexpr int LPP = D / 4;
  const int np_max = p.max_partitions;
  const int group = slots * LPP, per_wg = kDraftMergeThreads / group;
  const int tid = threadIdx.x, tg = tid % group, ld = tid % LPP, slot = tg / LPP, lr = tid / group;
  const int row = min((int)blockIdx.x * per_wg + lr, rows - 1);     // a surplus group repeats the last row and does not write
  const bool writes = (int)blockIdx.x * per_wg + lr < rows;
  const int head = row % p.num_q_heads, bn = row / p.num_q_heads;
  const int node = bn % p.nodes, b = bn / p.nodes;
  const int64_t at = (int64_t)row * np_max;
  float* s_max = lds + lr * 2 * np_max;
  float* s_w = s_max + np_max;
  float4 ahead[kDraftMergeAhead];
#pragma unroll
  for (int k = 0; k < kDraftMergeAhead; ++k) {
    const int q = slot + k * slots;
    ahead[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (q < np_max) ahead[k] = *(const float4*)(p.ws_out + (at + q) * D + 4 * ld);
  }
  const bool live = node < draft_nodes(p, b);
  const int keys = draft_keys(p, b), whole = keys / p.partition_size;       // no rounding up: sizes go up to 2^31 - 256
  const int np = live ? min(whole + (keys % p.partition_size != 0 ? 1 : 0), np_max) : 0;
  for (int q = tg; q < np_max; q += group) {
    const float m = p.ws_max[at + q], w = p.ws_sum[at + q];
    s_max[q] = q < np ? m : -INFINITY;
    s_w[q] = w;
  }
  __syncthreads();
  float top = -INFINITY;
  for (int q = 0; q < np; ++q) top = fmaxf(top, s_max[q]);
  for (int q = tg; q < np; q += group)
    if (s_max[q] != -INFINITY) s_w[q] *= __builtin_amdgcn_exp2f(s_max[q] - top);
  __syncthreads();
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](int q, const float4& v) __attribute__((always_inline)) {
    const float w = q < np ? s_w[q] : 0.0f;
    if (w != 0.0f) { acc.x += w * v.x; acc.y += w * v.y; acc.z += w * v.z; acc.w += w * v.w; }
  };
#pragma unroll
  for (int k = 0; k < kDraftMergeAhead; ++k) add(slot + k * slots, ahead[k]);
#pragma unroll 4
  for (int q = slot + kDraftMergeAhead * slots; q < np; q += slots) add(q, *(const float4*)(p.ws_out + (at + q) * D + 4 * ld));
  float4* s_acc = (float4*)(lds + (per_wg * 2 * np_max + 3) / 4 * 4);
  s_acc[tid] = acc;
  __syncthreads();
  if (slot != 0 || !writes) return;
  float den = 0.0f;
  for (int q = 0; q < np; ++q) den += s_w[q];
  for (int i = 1; i < slots; ++i) {
    const float4 v = s_acc[tid + i * LPP];
    acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
  }
  const float inv = 1.0f / den;
  const int64_t o = (int64_t)bn * p.out_stride + (int64_t)head * D + 4 * ld;
  float x[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
  if (__builtin_expect(top == -INFINITY, 0)) x[0] = x[1] = x[2] = x[3] = live ? draft_unreferenced(p, b, node) : 0.0f;
  if (p.q_dtype == PA_DTYPE_F32) *(float4*)((float*)p.out + o) = make_float4(x[0], x[1], x[2], x[3]);
  else if (p.q_dtype == PA_DTYPE_F16) *(uint2*)((uint16_t*)p.out + o) = make_uint2(draft_pack<CT_F16>(x[0], x[1]), draft_pack<CT_F16>(x[2], x[3]));
  else *(uint2*)((uint16_t*)p.out + o) = make_uint2(draft_pack<CT_BF16>(x[0], x[1]), draft_pack<CT_BF16>(x[2], x[3]));
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
                                  int64_t workspace_bytes, int rows_per_workgroup, void* stream) {
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
  int tile = rows_per_workgroup;
  if (tile != 0 && tile != 16 && tile != 32 && tile != 64 && tile != 128)
    DRAFT_FAIL(PA_ERR_BAD_ARG, "rows_per_workgroup must be 0, 16, 32, 64 or 128");
  if (max_partitions < 1) DRAFT_FAIL(PA_ERR_BAD_ARG, "max_partitions must be positive");
  if (max_partitions > 1024) DRAFT_FAIL(PA_ERR_UNSUPPORTED, "more than 1024 partitions");
  if (batch * nodes * num_q_heads > 0x7fffffff) DRAFT_FAIL(PA_ERR_UNSUPPORTED, "too many rows for one launch");
  // results are written 8 (f32: 16) bytes at a time
  if ((reinterpret_cast<uintptr_t>(out) & (q_dtype == PA_DTYPE_F32 ? 15u : 7u)) != 0 || out_stride % 4 != 0)
    DRAFT_FAIL(PA_ERR_BAD_ARG, "out rows must be 8-byte aligned (f32: 16)");
  if (max_partitions > 1) {
    if (partition_size <= 0 || partition_size % 32 != 0 || partition_size > 0x7fffff00)
      DRAFT_FAIL(PA_ERR_UNSUPPORTED, "partition_size must be a positive multiple of 32");
    if (!workspace || workspace_bytes < pa_draft_workspace_bytes(batch, nodes, num_q_heads, head_dim, max_partitions))
      DRAFT_FAIL(PA_ERR_WORKSPACE, "workspace missing or too small");
    if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) DRAFT_FAIL(PA_ERR_BAD_ARG, "workspace must be 256-byte aligned");
  }
  const int64_t gq = num_q_heads / num_kv_heads, rows = nodes * gq;
  if (tile == 0) tile = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
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
  p.row_tiles = (int)((rows + tile - 1) / tile);
  p.scale_log2e = scale * 1.4426950408889634f;
  const int64_t wgs = batch * max_partitions * num_kv_heads * p.row_tiles;
  if (wgs > 0x7fffffff) DRAFT_FAIL(PA_ERR_UNSUPPORTED, "too many workgroups for one launch");
#undef DRAFT_FAIL
  hipStream_t st = (hipStream_t)stream;
  int rc;
  if (kv_dtype == PA_DTYPE_F16) rc = launch_draft_f16(p, (int)head_dim, tile, (unsigned)wgs, st);
  else if (kv_dtype == PA_DTYPE_FP8_E4M3) rc = launch_draft_fp8(p, (int)head_dim, tile, (unsigned)wgs, st);
  else if (q_dtype == PA_DTYPE_BF16) rc = launch_draft_bf16(p, (int)head_dim, tile, (unsigned)wgs, st);
  else rc = launch_draft_bf16_as_f16(p, (int)head_dim, tile, (unsigned)wgs, st);
  if (rc != PA_OK) return rc;
  if (max_partitions > 1) {
    const int64_t out_rows = batch * nodes * num_q_heads;
    const int most = (int)(kDraftMergeThreads * 4 / head_dim);              // all of a workgroup for one row
    int slots = 1;
    while (slots < most && slots * 2 <= max_partitions) slots *= 2;
    const int64_t per_wg = kDraftMergeThreads / (slots * (head_dim / 4));
    const dim3 grid((unsigned)((out_rows + per_wg - 1) / per_wg));
    const size_t lds = (size_t)((per_wg * 2 * max_partitions + 3) / 4 * 4 + kDraftMergeThreads * 4) * 4;
    if (head_dim == 128) hipLaunchKernelGGL(draft_merge_kernel<128>, grid, dim3(kDraftMergeThreads), lds, st, p, slots, (int)out_rows);
    else hipLaunchKernelGGL(draft_merge_kernel<64>, grid, dim3(kDraftMergeThreads), lds, st, p, slots, (int)out_rows);
  }
  return check_launch("pa_draft_attention");
}

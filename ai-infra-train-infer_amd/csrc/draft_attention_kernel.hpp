// Attention of a tree of drafted tokens over the paged cache, on the matrix cores (gfx950).
//
// Row b drafts n nodes; node i attends to the row's committed tokens 0 .. c - 1 and to the nodes of its mask,
// whose K and V lie at cache positions c .. c + n - 1.  All nodes of a row, and all query heads of a KV head,
// read the same K and V, so the R = n x G rows (node, head of the group) of one KV head form one matrix operand
// and a K/V row leaves HBM once for all of them: 2 G n FLOP per K/V element against 2 in a decode step, memory
// bound up to R ~ 128 and bound by the matrix pipe and the exponentials beyond that.
//
//  * One workgroup per (batch row, KV head, tile of 16 C rows, partition); wave w of its 4 walks the 32-token
//    tiles w, w + 4, ... of the partition on its own, without a barrier in the loop, and multiplies each with C
//    16-row operands: the tile's fragments are read from LDS once for all C.
//  * Loads, LDS layout and the two products are those of paged_decode_mfma_kernel.hpp: one tile of K and V in
//    flight in registers (16 bytes per lane), written to the wave's own LDS, S^T = K . Q^T and O^T += V^T . P^T
//    with 16x16x32 products, V^T through the LDS transpose read.
//  * Queries keep their own bits (no scale folded in): 16-bit caches and queries of one type are multiplied as
//    they are, everything else as fp16, and scale * log2(e) is applied to the fp32 score in the same fused
//    multiply-add that subtracts the reference maximum.  What is rounded to 16 bits is the probability, in
//    [0, 2^8] relative to the reference point.
//  * The mask is looked at only in tiles that reach the drafted tokens or the end: 32 bits a row, cut out of the
//    row's mask words.  A row that has seen nothing yet has reference -inf; one that sees nothing at all sums to
//    zero and its output is zero.
//  * NaN or infinity in the V of a node must not reach the nodes that do not see it, but a matrix product adds
//    0 * NaN.  Tiles of drafted tokens are checked for such values on their way into LDS, and a tile that holds
//    one goes through a key-by-key loop on the vector ALU that skips the zero probabilities.
//  * The waves' partial results are merged through LDS, 16 rows at a time, and written to `out` or, as maximum,
//    sum and normalised output, to the workspace.
#pragma once

#include "paged_decode_mfma_kernel.hpp"

#include <atomic>

namespace pa {

enum : int { CT_F16 = 0, CT_BF16 = 1 };   // what the products multiply

typedef __bf16 mbf8_t __attribute__((ext_vector_type(8)));
typedef __bf16 mbf2_t __attribute__((ext_vector_type(2)));
typedef uint32_t mword4_t __attribute__((ext_vector_type(4)));

constexpr int kDraftWaves = 4;

struct DraftParams {
  const void* q;
  int64_t q_stride;              // elements between nodes
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* context_lens;
  const int32_t* num_nodes;      // nullptr: all of them
  const uint64_t* mask;
  int64_t mask_stride;           // words between rows of the batch, 0: one tree
  void* out;
  int64_t out_stride;
  float* ws_max;                 // per (batch row, node, query head), partition: in log2 units
  float* ws_sum;
  float* ws_out;
  int q_dtype;
  int nodes, words;
  int num_q_heads, num_kv_heads;
  int table_width, bs_log2, num_blocks;
  int partition_size, max_partitions;
  int batch;
  int row_tiles;                 // tiles of 16 C rows per KV head
  float scale_log2e;
};

// nodes that row b drafts; 0 also for a context that is no length
__device__ __forceinline__ int draft_nodes(const DraftParams& p, int b) {
  const int ctx = p.context_lens[b];
  if (ctx < 0 || ctx > 0x7fffffff - 2 * PA_MAX_DRAFT_NODES) return 0;
  return p.num_nodes ? min(max(p.num_nodes[b], 0), p.nodes) : p.nodes;
}
// tokens of row b: committed and drafted
__device__ __forceinline__ int draft_keys(const DraftParams& p, int b) {
  const int n = draft_nodes(p, b);
  return n > 0 ? p.context_lens[b] + n : 0;
}

// Work unit u of a partitioned launch -> (row, partition), the partitions that hold tokens first: the numbering of
// unit_to_row_partition, whole partitions before the rows' last ones.
__device__ __forceinline__ bool draft_unit(const DraftParams& p, int u, int lane, int& row, int& part) {
  const int per_lane = (p.batch + 63) >> 6;
  const int first = lane * per_lane;
  auto whole_of = [&](int r) { return min(draft_keys(p, r) / p.partition_size, p.max_partitions); };
  auto live_of = [&](int r) { return min((draft_keys(p, r) + p.partition_size - 1) / p.partition_size, p.max_partitions); };
  int whole = 0, tails = 0;
  for (int i = 0; i < per_lane; ++i)
    if (first + i < p.batch) {
      const int w = whole_of(first + i);
      whole += w;
      tails += live_of(first + i) - w;
    }
  int total_whole;
  if (locate_item(whole, u, lane, per_lane, whole_of, row, part, total_whole)) return true;
  int index, total_tails;
  if (!locate_item(tails, u - total_whole, lane, per_lane, [&](int r) { return live_of(r) - whole_of(r); }, row, index, total_tails))
    return false;
  part = whole_of(row);
  return true;
}

__host__ __device__ constexpr int draft_lds_bytes(int C, int D) {
  return kDraftWaves * decode_mfma_wave_bytes(1, D) + 2 * C * kMfmaHeads * kDraftWaves * 4;
}

// 8 source elements -> 8 elements of the products' type
template <int KV, int CT>
__device__ __forceinline__ mword4_t words_to_ct(const uint32_t* w) {
  if constexpr (CT == CT_BF16) {
    static_assert(KV == KV_BF16, "only bf16 caches are multiplied as bf16");
    return mword4_t{w[0], w[1], w[2], w[3]};
  } else {
    return __builtin_bit_cast(mword4_t, words_to_f16<KV>(w));
  }
}

template <int CT>
__device__ __forceinline__ mfloat4_t draft_mfma(mword4_t a, mword4_t b, mfloat4_t c) {
  if constexpr (CT == CT_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mbf8_t, a), __builtin_bit_cast(mbf8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(mhalf8_t, a), __builtin_bit_cast(mhalf8_t, b), c, 0, 0, 0);
}

// two floats -> one word of the products' type, rounded to nearest
template <int CT>
__device__ __forceinline__ uint32_t draft_pack(float a, float b) {
  if constexpr (CT == CT_BF16) return __builtin_bit_cast(uint32_t, mbf2_t{(__bf16)a, (__bf16)b});
  else return __builtin_bit_cast(uint32_t, half2_t{(_Float16)a, (_Float16)b});
}
template <int CT>
__device__ __forceinline__ float draft_unpack(uint32_t w, int half) {
  const uint32_t h = half ? w >> 16 : w & 0xffffu;
  if constexpr (CT == CT_BF16) return bf16_bits_to_f32(h);
  else return f16_bits_to_f32(h);
}
// whether a word holds an infinity or NaN
template <int CT>
__device__ __forceinline__ bool draft_not_finite(uint32_t w) {
  constexpr uint32_t E = CT == CT_BF16 ? 0x7f80u : 0x7c00u;
  return (w & E) == E || ((w >> 16) & E) == E;
}

// C 16-row operands per wave (see the head of this file)
template <int KV, int CT, int D, int C>
__global__ __launch_bounds__(kDraftWaves * 64, C == 1 ? 2 : 1) void draft_attention_kernel(const DraftParams p) {
  using G = Geo<KV, D, 1>;
  using TileT = MfmaTile<KV, D, 1>;
  constexpr int W = kDraftWaves;
  constexpr int TILE = kMfmaTile;
  constexpr int NC = kMfmaHeads;
  constexpr int RL = TileT::RL;              // row loads of 8 tokens per tile: 4
  constexpr int CPR = D / 8;
  constexpr int ROWB = D * 2;
  constexpr int KSTEPS = D / 32;
  constexpr int MT = D / 16;
  constexpr int CPL = G::EPC / 8;
  constexpr bool LM = kLaneMajorTokens<KV>;
  constexpr float NEG_INF = -INFINITY;
  constexpr int WAVEB = decode_mfma_wave_bytes(1, D);

  extern __shared__ __align__(16) uint8_t lds_raw[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint8_t* my_lds = lds_raw + wave * WAVEB;
  float* my_scales = reinterpret_cast<float*>(my_lds + decode_mfma_tile_bytes(D));
  float (*red)[NC * D] = reinterpret_cast<float (*)[NC * D]>(lds_raw);             // [W][16 x D], over the tiles
  float (*sm)[W] = reinterpret_cast<float (*)[W]>(lds_raw + W * WAVEB);            // [16 C][W]
  float (*sl)[W] = sm + C * NC;

  const int g = lane >> 3;
  const int j = lane & 7;
  const int col = lane & 15;
  const int kg = lane >> 4;

  // ---- which rows and tokens --------------------------------------------------------------------------------
  const int inner = p.num_kv_heads * p.row_tiles;
  const int in = blockIdx.x % inner;
  int b = blockIdx.x / inner, part = 0;
  if (p.max_partitions > 1) {
    if (!draft_unit(p, blockIdx.x / inner, lane, b, part)) return;
    b = __builtin_amdgcn_readfirstlane(b);
    part = __builtin_amdgcn_readfirstlane(part);
  }
  // KV heads fastest: the row tiles of a head are num_kv_heads workgroups apart, which with 8 heads puts them on one XCD
  const int kvh = in % p.num_kv_heads;
  const int gq = p.num_q_heads / p.num_kv_heads;
  const int row0 = (in / p.num_kv_heads) * (NC * C);       // first (node, head) row of the workgroup
  const int n = draft_nodes(p, b);
  const int ctx = p.context_lens[b];
  const int live = min(n * gq - row0, NC * C);             // rows of the workgroup that a node stands behind
  const int all = min(p.nodes * gq - row0, NC * C);
  const bool direct = p.max_partitions == 1;
  auto out_at = [&](int r) { return ((int64_t)b * p.nodes + (row0 + r) / gq) * p.out_stride + (int64_t)(kvh * gq + (row0 + r) % gq) * D; };
  if (direct)                                              // nodes the row does not draft
    for (int o = threadIdx.x + max(live, 0) * D; o < all * D; o += W * 64) store_from_f32(p.out, out_at(o / D) + o % D, p.q_dtype, 0.0f);
  if (live <= 0) return;
  const int keys = ctx + n;
  int begin = 0, end = keys;
  if (!direct) {
    begin = part * p.partition_size;
    end = part == p.max_partitions - 1 ? keys : min(begin + p.partition_size, keys);
  }
  if (begin >= end) return;

  // ---- Q^T as the B operand: lane (col, kg) holds dims 32 s + 8 kg .. +7 of row 16 c + col ---------------------
  mword4_t qreg[C][KSTEPS];
  {
    auto load_q = [&](auto dt_tag) __attribute__((always_inline)) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int r = min(16 * c + col, live - 1);         // rows without a node repeat the last one; never written
        const int64_t base = ((int64_t)b * p.nodes + (row0 + r) / gq) * p.q_stride + (int64_t)(kvh * gq + (row0 + r) % gq) * D + 8 * kg;
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) {
          float x[8];
          load8_as_f32(p.q, base + 32 * s, decltype(dt_tag)::value, x);
#pragma unroll
          for (int e = 0; e < 4; ++e) qreg[c][s][e] = draft_pack<CT>(x[2 * e], x[2 * e + 1]);
        }
      }
    };
    if (p.q_dtype == PA_DTYPE_F16) load_q(std::integral_constant<int, PA_DTYPE_F16>{});
    else if (p.q_dtype == PA_DTYPE_BF16) load_q(std::integral_constant<int, PA_DTYPE_BF16>{});
    else load_q(std::integral_constant<int, PA_DTYPE_F32>{});
  }

  // ---- loads ---------------------------------------------------------------------------------------------------
  const int bs_mask = (1 << p.bs_log2) - 1;
  const uint32_t token_bytes = (uint32_t)(p.num_kv_heads * D * G::ES);
  const uint32_t block_bytes = token_bytes << p.bs_log2;
  auto token_of = [&](int r) { return LM ? g * 4 + r : r * 8 + g; };
  const uint32_t lane_off = (uint32_t)(((LM ? 0 : g) * p.num_kv_heads + kvh) * D * G::ES + j * G::LB);
  const int32_t* bt_row = p.block_tables + b * p.bt_stride;
  const int last_blk = min((end - 1) >> p.bs_log2, max(p.table_width - 1, 0));
  const int ntiles = (end - begin + TILE - 1) / TILE;

  auto load_ids = [&](int tile, int (&ids)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < 4; ++x) ids[x] = bt_row[min((begin + tile * TILE + x * 8) >> p.bs_log2, last_blk)];
  };
  auto issue_as = [&](auto stream_tag, TileT& t, int tile, const int (&ids)[4]) __attribute__((always_inline)) {
    constexpr bool STREAM = decltype(stream_tag)::value;
    if constexpr (LM) {
      int id = 0;               // by masks: a select between entries becomes an indexed array, which lives in scratch memory
#pragma unroll
      for (int x = 0; x < 4; ++x) id |= ids[x] & (g / 2 == x ? -1 : 0);
      const uint32_t phys = (uint32_t)min(max(id, 0), p.num_blocks - 1);
      const uint32_t off = (uint32_t)((begin + tile * TILE + g * 4) & bs_mask);
      const uint64_t base = (uint64_t)phys * block_bytes + off * token_bytes + lane_off;
      const uint8_t* kp = p.k_cache + base;
      const uint8_t* vp = p.v_cache + base;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int c = 0; c < G::NLD; ++c) {
          load_words<G::LB, STREAM>(kp + (r * token_bytes + c * G::LPR * G::LB), &t.k[r][c * (G::LB / 4)]);
          load_words<G::LB, STREAM>(vp + (r * token_bytes + c * G::LPR * G::LB), &t.v[r][c * (G::LB / 4)]);
        }
      }
      const uint64_t slot = ((uint64_t)phys << p.bs_log2) + off;
      const float4 k4 = *(const float4*)(p.k_scale + slot);
      const float4 v4 = *(const float4*)(p.v_scale + slot);
      t.ks[0] = k4.x; t.ks[1] = k4.y; t.ks[2] = k4.z; t.ks[3] = k4.w;
      t.vs[0] = v4.x; t.vs[1] = v4.y; t.vs[2] = v4.z; t.vs[3] = v4.w;
    } else {
#pragma unroll
      for (int r = 0; r < RL; ++r) {
        const int tok = begin + tile * TILE + r * 8;
        const uint32_t phys = (uint32_t)min(max(ids[r], 0), p.num_blocks - 1);
        const uint64_t base = (uint64_t)phys * block_bytes + (uint32_t)(tok & bs_mask) * token_bytes;
        const uint8_t* kp = p.k_cache + base;
        const uint8_t* vp = p.v_cache + base;
#pragma unroll
        for (int c = 0; c < G::NLD; ++c) {
          load_words<G::LB, STREAM>(kp + (lane_off + c * G::LPR * G::LB), &t.k[r][c * (G::LB / 4)]);
          load_words<G::LB, STREAM>(vp + (lane_off + c * G::LPR * G::LB), &t.v[r][c * (G::LB / 4)]);
        }
      }
    }
  };

  // ---- registers -> LDS; returns whether a drafted token's V (special tiles only) holds NaN or infinity ---------
  auto write_tile = [&](TileT& t, int tile, bool special) __attribute__((always_inline)) -> bool {
    bool wild = false;
#pragma unroll
    for (int r = 0; r < RL; ++r) {
      const int tk = token_of(r);
      const bool valid = !special || (begin + tile * TILE + tk) < end;
      // fp8: the power of two of 1 / v_scale goes into V here, exactly, the mantissa into the probability
      float v_pow2 = 1.0f;
      if constexpr (KV == KV_FP8) v_pow2 = __uint_as_float(__float_as_uint(__builtin_amdgcn_rcpf(t.vs[r])) & 0xff800000u);
#pragma unroll
      for (int c = 0; c < G::NLD; ++c) {
#pragma unroll
        for (int x = 0; x < CPL; ++x) {
          const int chunk = (c * 8 + j) * CPL + x;
          constexpr int wpc = (KV == KV_FP8) ? 2 : 4;
          mword4_t kf = words_to_ct<KV, CT>(&t.k[r][c * (G::LB / 4) + x * wpc]);
          mword4_t vf;
          if constexpr (KV == KV_FP8) vf = __builtin_bit_cast(mword4_t, fp8_words_to_f16_pow2(&t.v[r][c * (G::LB / 4) + x * wpc], v_pow2));
          else vf = words_to_ct<KV, CT>(&t.v[r][c * (G::LB / 4) + x * wpc]);
          if (special) {
            if (!valid) kf = vf = mword4_t{0, 0, 0, 0};     // past the end: scores masked, and 0 * V must stay 0
#pragma unroll
            for (int e = 0; e < 4; ++e) wild = wild || draft_not_finite<CT>(vf[e]);
          }
          uint8_t* dst = my_lds + tk * ROWB + ((chunk ^ lds_swz<CPR>(tk)) << 4);
          *(mword4_t*)dst = kf;
          *(mword4_t*)(dst + TILE * ROWB) = vf;
        }
      }
    }
    if constexpr (KV == KV_FP8) {
      float ik[4], mv[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool valid = !special || (begin + tile * TILE + token_of(r)) < end;
        ik[r] = valid ? __builtin_amdgcn_rcpf(t.ks[r]) : 0.0f;
        const uint32_t bits = __float_as_uint(__builtin_amdgcn_rcpf(t.vs[r]));
        mv[r] = valid ? __uint_as_float((bits & 0x007fffffu) | 0x3f800000u) : 0.0f;
      }
      *(float4*)&my_scales[token_of(0)] = make_float4(ik[0], ik[1], ik[2], ik[3]);
      *(float4*)&my_scales[TILE + token_of(0)] = make_float4(mv[0], mv[1], mv[2], mv[3]);
    }
    return wild;
  };

  // ---- LDS read addresses ----------------------------------------------------------------------------------------
  const uint8_t* k_rd[KSTEPS];
#pragma unroll
  for (int s = 0; s < KSTEPS; ++s) k_rd[s] = my_lds + col * ROWB + (((4 * s + kg) ^ lds_swz<CPR>(col)) << 4);
  const uint8_t* v_rd[MT];
  {
    const int key = 4 * kg + (col >> 2);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      v_rd[mt] = my_lds + TILE * ROWB + key * ROWB + (((2 * mt + ((col & 3) >> 1)) ^ lds_swz<CPR>(key)) << 4) + (col & 1) * 8;
  }

  // The tile's keys that row 16 c + col sees, bit k = key k of the tile (special tiles only).
  auto visible = [&](int c, int tile) __attribute__((always_inline)) -> uint32_t {
    const int r = min(16 * c + col, live - 1);
    const uint64_t* words = p.mask + b * p.mask_stride + (int64_t)((row0 + r) / gq) * p.words;
    const int off = begin + tile * TILE - ctx;             // the tile's first key as a node; negative: committed keys come first
    auto word = [&](int w) -> uint64_t { return w < p.words ? words[w] : 0ull; };
    uint32_t bits = 0;
    if (off >= 0) {
      const int w = off >> 6, sh = off & 63;
      uint64_t v = word(w) >> sh;
      if (sh > 32) v |= word(w + 1) << (64 - sh);
      bits = (uint32_t)v;
    } else if (off > -32) {
      bits = ((uint32_t)word(0) << -off) | ((1u << -off) - 1u);
    } else {
      bits = 0xffffffffu;
    }
    const int left = end - (begin + tile * TILE);          // keys of the tile that exist
    return left < 32 ? bits & ((1u << left) - 1u) : bits;
  };

  float m_ref[C], l_run[C];      // reference maximum (log2 units, the same in a row's 4 lanes), this lane's share of the sum
  mfloat4_t o[C][MT];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    m_ref[c] = NEG_INF;
    l_run[c] = 0.0f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) o[c][mt] = mfloat4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }

  auto compute = [&](int tile, bool special, bool wild) __attribute__((always_inline)) {
    mfloat4_t s[C][2];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) s[c][kb] = mfloat4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int st = 0; st < KSTEPS; ++st)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const mword4_t a = *(const mword4_t*)(k_rd[st] + kb * 16 * ROWB);
#pragma unroll
        for (int c = 0; c < C; ++c) s[c][kb] = draft_mfma<CT>(a, qreg[c][st], s[c][kb]);
      }
    mfloat4_t mvs[2];
    if constexpr (KV == KV_FP8) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const float4 a = *(const float4*)&my_scales[16 * kb + 4 * kg];
        const float4 m4 = *(const float4*)&my_scales[TILE + 16 * kb + 4 * kg];
        mvs[kb] = mfloat4_t{m4.x, m4.y, m4.z, m4.w};
#pragma unroll
        for (int c = 0; c < C; ++c) s[c][kb] *= mfloat4_t{a.x, a.y, a.z, a.w};
      }
    }
    if (special) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint32_t vis = visible(c, tile) >> (4 * kg);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[c][kb][e] = (vis >> (16 * kb + e)) & 1u ? s[c][kb][e] : NEG_INF;
      }
    }
    bool want = false;
    float top[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float mx = s[c][0][0];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[c][kb][e]);
      top[c] = mx * p.scale_log2e;                         // scale > 0
      want = want || top[c] > m_ref[c] + 8.0f;
    }
    // The reference follows a row's maximum only when that has outgrown it by 2^8: p <= 256 fits the 16-bit types,
    // and the rescale of the accumulators almost never runs.
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(want) != 0, 0)) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float rmax = fmaxf(top[c], __shfl_xor(top[c], 16));
        rmax = fmaxf(rmax, __shfl_xor(rmax, 32));
        const bool grow = rmax > m_ref[c] + 8.0f;
        const float alpha = grow ? __builtin_amdgcn_exp2f(m_ref[c] - rmax) : 1.0f;   // from -inf: 0 times nothing
        m_ref[c] = grow ? rmax : m_ref[c];
        l_run[c] *= alpha;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c][mt][e] *= alpha;
      }
    }
    // ---- P^T as B operand: contraction index 8 kg + e <-> key 4 kg + e (e < 4), 16 + 4 kg + e - 4 ------------------
    mword4_t pb[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float ref = m_ref[c] == NEG_INF ? 0.0f : m_ref[c];
      float psum = 0.0f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          float p0 = __builtin_amdgcn_exp2f(fmaf(s[c][kb][e], p.scale_log2e, -ref));
          float p1 = __builtin_amdgcn_exp2f(fmaf(s[c][kb][e + 1], p.scale_log2e, -ref));
          psum += p0 + p1;
          if constexpr (KV == KV_FP8) { p0 *= mvs[kb][e]; p1 *= mvs[kb][e + 1]; }
          pb[c][2 * kb + e / 2] = draft_pack<CT>(p0, p1);
        }
      l_run[c] += psum;
    }
    if (__builtin_expect(wild, 0)) {
      // a V row that must not be multiplied by the zeros of the rows that do not see it
#pragma unroll 1
      for (int key = 0; key < TILE; ++key) {
        const int from = ((key & 15) >> 2) * 16 + col;     // the lane of this row that holds the key's probability
        const int e = (key & 3) + 4 * (key >> 4);
        float pk[C];
        bool seen[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
          uint32_t w = 0;
#pragma unroll
          for (int x = 0; x < 4; ++x) w |= pb[c][x] & ((e >> 1) == x ? 0xffffffffu : 0u);
          pk[c] = draft_unpack<CT>(__shfl(w, from), e & 1);
          seen[c] = (visible(c, tile) >> key) & 1u;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const uint2 w = *(const uint2*)(my_lds + TILE * ROWB + key * ROWB + (((2 * mt + (kg >> 1)) ^ lds_swz<CPR>(key)) << 4) + (kg & 1) * 8);
          const mfloat4_t v = {draft_unpack<CT>(w.x, 0), draft_unpack<CT>(w.x, 1), draft_unpack<CT>(w.y, 0), draft_unpack<CT>(w.y, 1)};
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int d = 0; d < 4; ++d) o[c][mt][d] = seen[c] ? fmaf(pk[c], v[d], o[c][mt][d]) : o[c][mt][d];
        }
      }
      return;
    }
    // ---- O^T += V^T . P^T ---------------------------------------------------------------------------------------
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const mfp16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) mfp16x4_t*)(v_rd[mt]));
      const mfp16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) mfp16x4_t*)(v_rd[mt] + 16 * ROWB));
      const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
      const mword4_t a = {l2.x, l2.y, h2.x, h2.y};
#pragma unroll
      for (int c = 0; c < C; ++c) o[c][mt] = draft_mfma<CT>(a, pb[c], o[c][mt]);
    }
  };

  // ---- this wave's tiles: wave, wave + W, ... -------------------------------------------------------------------
  const int n_mine = ntiles > wave ? (ntiles - wave + W - 1) / W : 0;
  auto run_tiles = [&](auto stream_tag) __attribute__((always_inline)) {
    if (n_mine > 0) {
      TileT t;
      int ids[4], ids_next[4];
      load_ids(wave, ids);
      issue_as(stream_tag, t, wave, ids);
      if (n_mine > 1) load_ids(wave + W, ids);
      for (int i = 0; i < n_mine; ++i) {
        const int tile = wave + i * W;
        const int past = begin + (tile + 1) * TILE;
        const bool special = past > ctx || past > end;     // drafted tokens or the end inside
        if (i + 2 < n_mine) load_ids(tile + 2 * W, ids_next);
        const bool wild = write_tile(t, tile, special);
        if (i + 1 < n_mine) issue_as(stream_tag, t, tile + W, ids);
        compute(tile, special, special && __builtin_amdgcn_ballot_w64(wild) != 0);
#pragma unroll
        for (int x = 0; x < 4; ++x) ids[x] = ids_next[x];
      }
    }
  };
  // non-temporal loads where nobody else reads the range: no second row tile, no neighbour with the same blocks
  if (p.row_tiles == 1 && decode_range_is_private(bt_row, p.bt_stride, b, p.batch, min(begin >> p.bs_log2, last_blk)))
    run_tiles(std::true_type{});
  else
    run_tiles(std::false_type{});

  // ---- merge the waves ------------------------------------------------------------------------------------------
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (kg == 0) sm[16 * c + col][wave] = m_ref[c];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    __syncthreads();                 // the maxima are there; every wave is done with its tiles, or with the 16 rows before
    float mx = sm[16 * c + col][0];
#pragma unroll
    for (int i = 1; i < W; ++i) mx = fmaxf(mx, sm[16 * c + col][i]);
    const float w = m_ref[c] == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(m_ref[c] - mx);
    float lw = l_run[c] * w;
    lw += __shfl_xor(lw, 16);
    lw += __shfl_xor(lw, 32);
    if (kg == 0) sl[16 * c + col][wave] = lw;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      *(float4*)&red[wave][col * D + 16 * mt + 4 * kg] = make_float4(o[c][mt][0] * w, o[c][mt][1] * w, o[c][mt][2] * w, o[c][mt][3] * w);
    __syncthreads();
    const int rows = min(live - 16 * c, 16);
    for (int idx = threadIdx.x; idx < rows * D; idx += W * 64) {
      const int r = idx / D, d = idx % D;
      float num = 0.0f, den = 0.0f, mo = NEG_INF;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        num += red[i][idx];
        den += sl[16 * c + r][i];
        mo = fmaxf(mo, sm[16 * c + r][i]);
      }
      const float res = mo == NEG_INF ? 0.0f : num / den;  // a row that saw no key: zero
      if (direct) {
        store_from_f32(p.out, out_at(16 * c + r) + d, p.q_dtype, res);
      } else {
        const int rr = row0 + 16 * c + r;
        const int64_t at = (((int64_t)b * p.nodes + rr / gq) * p.num_q_heads + kvh * gq + rr % gq) * p.max_partitions + part;
        p.ws_out[at * D + d] = res;
        if (d == 0) {
          p.ws_max[at] = mo;
          p.ws_sum[at] = mo == NEG_INF ? 0.0f : den;
        }
      }
    }
  }
}

template <int KV, int CT, int D, int C>
int launch_draft_shape(const DraftParams& p, unsigned grid, hipStream_t st) {
  auto kern = draft_attention_kernel<KV, CT, D, C>;
  constexpr int lds = draft_lds_bytes(C, D);
  // the attribute belongs to the kernel on one device: once per instantiation and device
  static std::atomic<bool> attr_set[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return fail(PA_ERR_LAUNCH, "pa_draft_attention: cannot tell the current device");
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
      return fail(PA_ERR_LAUNCH, "pa_draft_attention: cannot raise the dynamic LDS limit");
    attr_set[dev].store(true, std::memory_order_release);
  }
  hipLaunchKernelGGL(kern, dim3(grid), dim3(kDraftWaves * 64), lds, st, p);
  return PA_OK;
}

template <int KV, int CT>
int launch_draft(const DraftParams& p, int head_dim, int col_tiles, unsigned grid, hipStream_t st) {
  if (head_dim == 128)
    return col_tiles == 1 ? launch_draft_shape<KV, CT, 128, 1>(p, grid, st) : launch_draft_shape<KV, CT, 128, 2>(p, grid, st);
  return col_tiles == 1 ? launch_draft_shape<KV, CT, 64, 1>(p, grid, st) : launch_draft_shape<KV, CT, 64, 2>(p, grid, st);
}

int launch_draft_f16(const DraftParams& p, int head_dim, int col_tiles, unsigned grid, hipStream_t st);
int launch_draft_bf16(const DraftParams& p, int head_dim, int col_tiles, unsigned grid, hipStream_t st);
int launch_draft_bf16_as_f16(const DraftParams& p, int head_dim, int col_tiles, unsigned grid, hipStream_t st);
int launch_draft_fp8(const DraftParams& p, int head_dim, int col_tiles, unsigned grid, hipStream_t st);

}  // namespace pa

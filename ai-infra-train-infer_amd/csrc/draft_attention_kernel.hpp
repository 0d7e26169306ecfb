// Attention of a tree of drafted tokens over the paged cache, on the matrix cores (gfx950).
//
// Row b drafts n nodes; node i attends to the row's committed tokens 0 .. c - 1 and to the nodes of its mask,
// whose K and V lie at cache positions c .. c + n - 1.  All nodes of a row, and all query heads of a KV head,
// read the same K and V, so the R = n x G rows (node, head of the group) of one KV head form one matrix operand
// and a K/V row leaves HBM once for all of them: 2 G n FLOP per K/V element against 2 in a decode step, memory
// bound up to R ~ 128 and bound by the matrix pipe and the exponentials beyond that.
//
//  * One workgroup of 4 or 8 waves per (batch row, KV head, tile of 16 ... 128 rows, partition).  Up to 32 rows
//    (draft_narrow_kernel, memory bound): each wave walks its own 32-token tiles without a barrier, as a decode step's
//    matrix kernel does.  More (draft_wide_kernel): the workgroup shares 64-token tiles and its waves split the rows, so
//    that a K/V byte is fetched once per 128 rows.
//  * Loads, LDS layout and the two products are those of paged_decode_mfma_kernel.hpp: tiles in flight in registers
//    (16 bytes per lane), written to LDS, S^T = K . Q^T and O^T += V^T . P^T with 16x16x32 products, V^T through the
//    LDS transpose read.
//  * Queries keep their own bits (no scale folded in): 16-bit caches and queries of one type are multiplied as
//    they are, everything else as fp16, bf16 and fp32 queries times a power of two per row that brings their largest
//    element to fp16's range.  scale * log2(e), and that power, are applied to the fp32 score in the same fused
//    multiply-add that subtracts the reference maximum.  What is rounded to 16 bits is the probability, in
//    [0, 2^8] relative to the reference point: to fp16's 11 bits, or to 8 where bf16 is multiplied, since an instruction takes
//    both operands of one type and V keeps its range only in its own.  The errors of a row's keys average out: 0.23 % of an
//    output's norm in all against 0.17 % for rounding the output alone (bf16; fp16 0.029 against 0.021 %).  fp32 queries have
//    fp16's 11 bits; two parts would have 22, in registers that 128 rows do not leave.
//  * The mask is looked at only in tiles that reach the drafted tokens or the end: 32 bits a row, cut out of the
//    row's mask words.  A row that has seen nothing yet has reference -inf; one that sees nothing at all sums to
//    zero and its output is zero.  Scores of NaN never move the reference but make the row's sum NaN, and a row that sees
//    keys and yet has no reference at the end (all of them NaN or -inf) is NaN, as its softmax is (draft_unreferenced).
//  * NaN or infinity in the V of a node must not reach the nodes that do not see it, but a matrix product adds
//    0 * NaN.  Tiles of drafted tokens enter LDS without such values; if there were any, the rows that do see them get
//    them at the end (draft_wild).
//  * Waves that took different tokens are merged through LDS; results go to `out` or, as maximum, sum and normalised
//    output, to the workspace.
#pragma once

#include "paged_decode_mfma_kernel.hpp"

#include <atomic>

namespace pa {

enum : int { CT_F16 = 0, CT_BF16 = 1 };   // what the products multiply

typedef __bf16 mbf8_t __attribute__((ext_vector_type(8)));
typedef __bf16 mbf2_t __attribute__((ext_vector_type(2)));
typedef uint32_t mword4_t __attribute__((ext_vector_type(4)));

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
  int row_tiles;                 // workgroups' worth of rows per KV head
  float scale_log2e;
};

// nodes that row b drafts; 0 also for a context that is no length, or so long that the tiles asked for ahead would pass 32 bits
__device__ __forceinline__ int draft_nodes(const DraftParams& p, int b) {
  const int ctx = p.context_lens[b];
  if (ctx < 0 || ctx > 0x7fffffff - 8 * PA_MAX_DRAFT_NODES) return 0;
  return p.num_nodes ? min(max(p.num_nodes[b], 0), p.nodes) : p.nodes;
}
// tokens of row b: committed and drafted
__device__ __forceinline__ int draft_keys(const DraftParams& p, int b) {
  const int n = draft_nodes(p, b);
  return n > 0 ? p.context_lens[b] + n : 0;
}

// Work unit u of a partitioned launch -> (row, partition), the partitions that hold tokens first: the numbering of
// unit_to_row_partition, whole partitions before the rows' last ones.  Lane l counts those of rows l * per_lane ....  Every
// workgroup waits for this before its first load.
__device__ __forceinline__ bool draft_unit(const DraftParams& p, int u, int lane, int& row, int& part) {
  if (p.batch == 1) {                // nothing to look for: a lone sequence is waited for
    row = 0;
    part = u;
    return u * (int64_t)p.partition_size < draft_keys(p, 0);
  }
  const int per_lane = (p.batch + 63) >> 6;
  const int first = lane * per_lane;
  auto count = [&](int r, int& whole, int& live) __attribute__((always_inline)) {
    const int keys = draft_keys(p, r), q = keys / p.partition_size;
    whole = min(q, p.max_partitions);
    live = min(q + (q * p.partition_size < keys ? 1 : 0), p.max_partitions);
  };
  int whole = 0, tails = 0;
  for (int i = 0; i < per_lane; ++i)
    if (first + i < p.batch) {
      int w, l;
      count(first + i, w, l);
      whole += w;
      tails += l - w;
    }
  const int whole_to = wave_scan(whole), tails_to = wave_scan(tails);
  const int total = __builtin_amdgcn_readlane(whole_to, 63);
  const bool tail = u >= total;
  const int want = tail ? u - total : u;
  const unsigned long long past = __builtin_amdgcn_ballot_w64((tail ? tails_to : whole_to) > want);
  if (past == 0) return false;
  const int owner = __builtin_ctzll(past);
  int base = __builtin_amdgcn_readlane(tail ? tails_to - tails : whole_to - whole, owner), w = __builtin_amdgcn_readlane(whole, owner);
  row = owner;
  if (per_lane > 1) {                // the owner's rows hold more than want - base, so the walk ends inside them
    for (row = owner * per_lane;; ++row) {
      int l;
      count(row, w, l);
      const int c = tail ? l - w : w;
      if (want < base + c) break;
      base += c;
    }
  }
  part = tail ? w : want - base;     // a row's last partition comes after its whole ones
  return true;
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
// Infinities and NaN become zeros; whether there were any.
template <int CT>
__device__ __forceinline__ bool draft_tame(mword4_t& v) {
  constexpr uint32_t E = CT == CT_BF16 ? 0x7f80u : 0x7c00u;
  bool wild = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool lo = (v[e] & E) == E, hi = (v[e] & (E << 16)) == (E << 16);
    v[e] = (lo ? 0u : v[e] & 0xffffu) | (hi ? 0u : v[e] & 0xffff0000u);
    wild = wild || lo || hi;
  }
  return wild;
}

template <class T>
using lds_ptr = __attribute__((address_space(3))) T*;
__device__ __forceinline__ uint32_t lds_offset(const uint8_t* p) { return (uint32_t)(uintptr_t)(lds_ptr<const uint8_t>)p; }

// LDS bytes of a 32-token tile of K, or of V
__host__ __device__ constexpr int draft_half_bytes(int D) { return kMfmaTile * D * 2; }

// What a wave keeps of its 16 C rows, and one step of them over 32 tokens in LDS.  Result layout of the products: lane
// (col, kg) holds, for row 16 c + col, keys 4 kg .. + 3 of a 16-key half (scores) or dims 16 mt + 4 kg .. + 3 (output).
// AHEAD: a step asks for V's fragments before its softmax (32 registers at head_dim 128): for the wide workgroups, which have
// them; with 16 rows it makes no difference (184 us for 64 rows of 5 nodes x 4096 tokens either way), with 32 they do not fit.
template <int KV, int CT, int D, int C, bool AHEAD>
struct DraftRows {
  static constexpr int KSTEPS = D / 32, MT = D / 16, ROWB = D * 2, CPR = D / 8;
  mword4_t q[C][KSTEPS];         // Q^T as the B operand: dims 32 s + 8 kg .. + 7 of row 16 c + col
  mfloat4_t o[C][MT];
  float scale[C];                // what a product is times to be a score in log2 units
  float m_ref[C];                // reference maximum in log2 units, the same in a row's 4 lanes; -inf: nothing seen
  float l_run[C];                // this lane's share of the row's sum
  uint32_t k_first, v_first;     // this lane's K fragment of dims 0 .. 31 and V fragment of dims 0 .. 15 in a tile
  int col, kg;

  __device__ __forceinline__ void init(int lane) {
    col = lane & 15;
    kg = lane >> 4;
    k_first = col * ROWB + ((kg ^ lds_swz<CPR>(col)) << 4);
    // V^T through the transpose read: within a block of 16 lanes lane a supplies the address of 4 dims of key 4 kg + a / 4
    const int key = 4 * kg + (col >> 2);
    v_first = key * ROWB + ((((col & 3) >> 1) ^ lds_swz<CPR>(key)) << 4) + (col & 1) * 8;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      m_ref[c] = -INFINITY;
      l_run[c] = 0.0f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[c][mt] = mfloat4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }

  // at(c): element index of row 16 c + col's query
  template <class At>
  __device__ __forceinline__ void load_q(const void* ptr, int dtype, float scale_log2e, At&& at) {
    // the dtype switch sits outside the loops: inside, it would put a branch and a wait between loads in flight
    auto load = [&](auto dt_tag) __attribute__((always_inline)) {
      constexpr int DT = decltype(dt_tag)::value;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int64_t base = at(c) + 8 * kg;
        float x[KSTEPS][8];
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) load8_as_f32(ptr, base + 32 * s, DT, x[s]);
        scale[c] = scale_log2e;
        if constexpr (CT == CT_F16 && DT != PA_DTYPE_F16) {
          // the row's largest element to 2^14 ... 2^15: no size overflows, and what is more than 2^28 below it alone loses bits
          float most = 0.0f;
#pragma unroll
          for (int s = 0; s < KSTEPS; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[s][e]));
          most = fmaxf(most, __shfl_xor(most, 16));
          most = fmaxf(most, __shfl_xor(most, 32));
          // nothing to bring anywhere in a row of zeros, and none that would help one of infinities
          const int up = most > 0.0f && most < INFINITY ? min(15 - __builtin_amdgcn_frexp_expf(most), 100) : 0;
          scale[c] = __builtin_amdgcn_ldexpf(scale_log2e, -up);
#pragma unroll
          for (int s = 0; s < KSTEPS; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[s][e] = __builtin_amdgcn_ldexpf(x[s][e], up);
        }
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s)
#pragma unroll
          for (int e = 0; e < 4; ++e) q[c][s][e] = draft_pack<CT>(x[s][2 * e], x[s][2 * e + 1]);
      }
    };
    if constexpr (CT == CT_BF16) {
      load(std::integral_constant<int, PA_DTYPE_BF16>{});
    } else {
      if (dtype == PA_DTYPE_F16) load(std::integral_constant<int, PA_DTYPE_F16>{});
      else if (dtype == PA_DTYPE_BF16) load(std::integral_constant<int, PA_DTYPE_BF16>{});
      else load(std::integral_constant<int, PA_DTYPE_F32>{});
    }
  }

  // Fragments of a 32-token tile at `tile` (of 256 bytes' alignment: a 16-byte piece's number is exclusive-ored with the row's
  // swizzle, and so may the fragment's number be with the address).  K's fragment i: dims
  // 32 (i / 2) + 8 kg .. + 7 of key 16 (i % 2) + col.
  __device__ __forceinline__ mword4_t load_k(uint32_t tile, int i) const {
    return *(lds_ptr<mword4_t>)(((tile + k_first) ^ (uint32_t)(i >> 1 << 6)) + (i & 1) * 16 * ROWB);
  }
  // V^T's: dims 16 mt + col of keys 4 kg .. + 3 and 16 + 4 kg .. + 3
  __device__ __forceinline__ mword4_t load_v(uint32_t tile, int mt) const {
    const uint32_t at = (tile + v_first) ^ (uint32_t)(mt << 5);
    const mfp16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_ptr<mfp16x4_t>)at);
    const mfp16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_ptr<mfp16x4_t>)(at + 16 * ROWB));
    const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
    return mword4_t{l2.x, l2.y, h2.x, h2.y};
  }

  // k, v: the tile in LDS; iks, mvs: per token 1 / k_scale and the mantissa of 1 / v_scale (fp8).  visible(c): bit k =
  // the row sees key k, asked for only in special tiles.
  template <class Visible>
  __device__ __forceinline__ void step(const uint8_t* k, const uint8_t* v, const float* iks, const float* mvs_lds, bool special,
                                       Visible&& visible) {
    mfloat4_t s[C][2];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) s[c][kb] = mfloat4_t{0.0f, 0.0f, 0.0f, 0.0f};
    // All of K's fragments are requested before the first product, all of V's before the softmax: left to the scheduler a
    // product waits for the read issued just before it.
    mword4_t f[MT];
    const uint32_t k_at = lds_offset(k), v_at = lds_offset(v);
#pragma unroll
    for (int i = 0; i < MT; ++i) f[i] = load_k(k_at, i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int c = 0; c < C; ++c) s[c][i & 1] = draft_mfma<CT>(f[i], q[c][i >> 1], s[c][i & 1]);
    if constexpr (AHEAD) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) f[mt] = load_v(v_at, mt);
      __builtin_amdgcn_sched_barrier(0);
    }
    mfloat4_t mvs[2];
    if constexpr (KV == KV_FP8) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const float4 a = *(const float4*)&iks[16 * kb + 4 * kg];
        const float4 m4 = *(const float4*)&mvs_lds[16 * kb + 4 * kg];
        mvs[kb] = mfloat4_t{m4.x, m4.y, m4.z, m4.w};
#pragma unroll
        for (int c = 0; c < C; ++c) s[c][kb] *= mfloat4_t{a.x, a.y, a.z, a.w};
      }
    }
    if (special) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint32_t vis = visible(c) >> (4 * kg);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[c][kb][e] = (vis >> (16 * kb + e)) & 1u ? s[c][kb][e] : -INFINITY;
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
      top[c] = mx * scale[c];                              // scale > 0
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
    // P^T as the B operand: contraction index 8 kg + e <-> key 4 kg + e (e < 4), 16 + 4 kg + e - 4
    mword4_t pb[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float ref = m_ref[c] == -INFINITY ? 0.0f : m_ref[c];
      float psum = 0.0f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          float p0 = __builtin_amdgcn_exp2f(fmaf(s[c][kb][e], scale[c], -ref));
          float p1 = __builtin_amdgcn_exp2f(fmaf(s[c][kb][e + 1], scale[c], -ref));
          psum += p0 + p1;
          if constexpr (KV == KV_FP8) { p0 *= mvs[kb][e]; p1 *= mvs[kb][e + 1]; }
          pb[c][2 * kb + e / 2] = draft_pack<CT>(p0, p1);
        }
      l_run[c] += psum;
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const mword4_t a = AHEAD ? f[mt] : load_v(v_at, mt);
#pragma unroll
      for (int c = 0; c < C; ++c) o[c][mt] = draft_mfma<CT>(a, pb[c], o[c][mt]);
    }
  }
};

// Which rows and tokens a workgroup takes.
struct DraftWork {
  int b, part, kvh, gq, row0;    // row0: first (node, head) row
  int n, ctx, live, all;         // nodes drafted, committed tokens, rows of the workgroup with a node, rows of the launch
  int begin, end;
};

// ROWS (node, head) rows per workgroup.  False: nothing to do (zeros for nodes that a row does not draft are written).
template <int ROWS, int D>
__device__ __forceinline__ bool draft_work(const DraftParams& p, DraftWork& w) {
  const int inner = p.num_kv_heads * p.row_tiles;
  const int in = blockIdx.x % inner, lane = threadIdx.x & 63;
  w.b = blockIdx.x / inner;
  w.part = 0;
  if (p.max_partitions > 1) {
    if (!draft_unit(p, blockIdx.x / inner, lane, w.b, w.part)) return false;
    w.b = __builtin_amdgcn_readfirstlane(w.b);
    w.part = __builtin_amdgcn_readfirstlane(w.part);
  }
  // KV heads fastest: the row tiles of a head are num_kv_heads workgroups apart, which with 8 heads puts them on one XCD
  w.kvh = in % p.num_kv_heads;
  w.gq = p.num_q_heads / p.num_kv_heads;
  w.row0 = in / p.num_kv_heads * ROWS;
  w.n = draft_nodes(p, w.b);
  w.ctx = p.context_lens[w.b];
  w.live = min(w.n * w.gq - w.row0, ROWS);
  w.all = min(p.nodes * w.gq - w.row0, ROWS);
  const int keys = w.ctx + w.n;
  w.begin = 0;
  w.end = keys;
  if (p.max_partitions > 1) {
    w.begin = w.part * p.partition_size;
    // no sum of a place and a size before it is known to stay below the keys
    w.end = w.part == p.max_partitions - 1 || keys - w.begin <= p.partition_size ? keys : w.begin + p.partition_size;
  }
  return w.live > 0 && w.begin < w.end;
}

__device__ __forceinline__ int64_t draft_out_at(const DraftParams& p, const DraftWork& w, int r, int D) {
  return ((int64_t)w.b * p.nodes + (w.row0 + r) / w.gq) * p.out_stride + (int64_t)(w.kvh * w.gq + (w.row0 + r) % w.gq) * D;
}

// zeros for the nodes that a row does not draft (a partitioned launch leaves them to the merge)
template <int THREADS, int D>
__device__ __forceinline__ void draft_zero_dead(const DraftParams& p, const DraftWork& w) {
  if (p.max_partitions > 1) return;
  for (int o = threadIdx.x + max(w.live, 0) * D; o < w.all * D; o += THREADS)
    store_from_f32(p.out, draft_out_at(p, w, o / D, D) + o % D, p.q_dtype, 0.0f);
}

// The keys first .. first + 31 that row r sees, bit k = key first + k.
__device__ __forceinline__ uint32_t draft_visible(const DraftParams& p, const DraftWork& w, int r, int first) {
  const uint64_t* words = p.mask + w.b * p.mask_stride + (int64_t)((w.row0 + min(r, w.live - 1)) / w.gq) * p.words;
  const int off = first - w.ctx;                           // the first key as a node; negative: committed keys come first
  auto word = [&](int i) -> uint64_t { return i < p.words ? words[i] : 0ull; };
  uint32_t bits = 0xffffffffu;
  if (off >= 0) {
    const int i = off >> 6, sh = off & 63;
    uint64_t v = word(i) >> sh;
    if (sh > 32) v |= word(i + 1) << (64 - sh);
    bits = (uint32_t)v;
  } else if (off > -32) {
    bits = ((uint32_t)word(0) << -off) | ((1u << -off) - 1u);
  }
  const int left = w.end - first;                          // keys that exist
  return left >= 32 ? bits : left > 0 ? bits & ((1u << left) - 1u) : 0u;
}

// What a row without a reference maximum holds: zero if it sees no key, NaN if what it sees are scores of NaN and -inf alone.
__device__ __forceinline__ float draft_unreferenced(const DraftParams& p, int b, int node) {
  bool sees = p.context_lens[b] > 0;
  const uint64_t* words = p.mask + b * p.mask_stride + (int64_t)node * p.words;
  const int n = draft_nodes(p, b);
  for (int i = 0; 64 * i < n; ++i) {
    const int left = n - 64 * i;
    sees = sees || (left >= 64 ? words[i] : words[i] & ((1ull << left) - 1)) != 0;
  }
  return sees ? __builtin_nanf("") : 0.0f;
}

// Writes one row's 4 dims of result, or of a partition's partial result.
__device__ __forceinline__ void draft_store4(const DraftParams& p, const DraftWork& w, int r, int d, int D, const float (&x)[4]) {
  if (p.max_partitions == 1) {
    const int64_t at = draft_out_at(p, w, r, D) + d;
    if (p.q_dtype == PA_DTYPE_F32) {
      *(float4*)((float*)p.out + at) = make_float4(x[0], x[1], x[2], x[3]);
    } else if (p.q_dtype == PA_DTYPE_F16) {
      *(uint2*)((uint16_t*)p.out + at) = make_uint2(draft_pack<CT_F16>(x[0], x[1]), draft_pack<CT_F16>(x[2], x[3]));
    } else {
      *(uint2*)((uint16_t*)p.out + at) = make_uint2(draft_pack<CT_BF16>(x[0], x[1]), draft_pack<CT_BF16>(x[2], x[3]));
    }
  } else {
    const int rr = w.row0 + r;
    const int64_t at = (((int64_t)w.b * p.nodes + rr / w.gq) * p.num_q_heads + w.kvh * w.gq + rr % w.gq) * p.max_partitions + w.part;
    *(float4*)(p.ws_out + at * D + d) = make_float4(x[0], x[1], x[2], x[3]);
  }
}
__device__ __forceinline__ void draft_store_stats(const DraftParams& p, const DraftWork& w, int r, float top, float sum) {
  const int rr = w.row0 + r;
  const int64_t at = (((int64_t)w.b * p.nodes + rr / w.gq) * p.num_q_heads + w.kvh * w.gq + rr % w.gq) * p.max_partitions + w.part;
  p.ws_max[at] = top;
  p.ws_sum[at] = sum;                // without a maximum 0, or NaN if a score was
}

// The infinities and NaN that tiles of drafted tokens were multiplied without: a row that sees one gets the sum of those
// it sees in that dim on top of its result (which earlier tiles may have made infinite or NaN already).  Rare, so it reads V
// again from the cache, 8 dims of a row per thread.
template <int KV, int CT, int D, int THREADS>
__device__ __forceinline__ void draft_wild(const DraftParams& p, const DraftWork& w) {
  constexpr int ES = KV == KV_FP8 ? 1 : 2;
  __syncthreads();                   // the finite results are written
  const int32_t* bt_row = p.block_tables + w.b * p.bt_stride;
  const int first = max(w.begin, w.ctx - 63);              // no tile with a drafted token starts earlier
  for (int item = threadIdx.x; item < w.live * (D / 8); item += THREADS) {
    const int r = item / (D / 8), d = item % (D / 8) * 8;
    float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    bool any = false;
    for (int key = first; key < w.end; ++key) {
      if (!(draft_visible(p, w, r, key) & 1u)) continue;
      const int blk = min(key >> p.bs_log2, p.table_width - 1);
      const int64_t phys = min(max(bt_row[blk], 0), p.num_blocks - 1);
      const int64_t slot = (phys << p.bs_log2) + (key & ((1 << p.bs_log2) - 1));
      const uint8_t* at = p.v_cache + ((slot * p.num_kv_heads + w.kvh) * D + d) * ES;
      mword4_t v;
      if constexpr (KV == KV_FP8) {
        const uint32_t words[2] = {((const uint32_t*)at)[0], ((const uint32_t*)at)[1]};
        const float pow2 = __uint_as_float(__float_as_uint(__builtin_amdgcn_rcpf(p.v_scale[slot])) & 0xff800000u);
        v = __builtin_bit_cast(mword4_t, fp8_words_to_f16_pow2(words, pow2));
      } else {
        const mword4_t raw = *(const mword4_t*)at;
        const uint32_t words[4] = {raw[0], raw[1], raw[2], raw[3]};
        v = words_to_ct<KV, CT>(words);
      }
      mword4_t tame = v;
      if (!draft_tame<CT>(tame)) continue;
      any = true;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = draft_unpack<CT>(v[e / 2], e & 1);
        if (!(fabsf(x) < INFINITY)) sum[e] += x;
      }
    }
    if (!any) continue;
    const int rr = w.row0 + r;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (fabsf(sum[e]) < INFINITY) continue;              // nothing wild in this dim
      if (p.max_partitions == 1) {
        const int64_t at = draft_out_at(p, w, r, D) + d + e;
        store_from_f32(p.out, at, p.q_dtype, load_as_f32(p.out, at, p.q_dtype) + sum[e]);
      } else {
        const int64_t at = (((int64_t)w.b * p.nodes + rr / w.gq) * p.num_q_heads + w.kvh * w.gq + rr % w.gq) * p.max_partitions + w.part;
        p.ws_out[at * D + d + e] += sum[e];
      }
    }
  }
}

// ---- up to 32 rows: every wave has its own tokens ----------------------------------------------------------------

// C 16-row operands, 1 or 2.  64 rows of 5 nodes x 4096 tokens of an fp8 cache: 101 us, 5.4 TB/s; one row of 5 nodes x 2048
// tokens: 7.4 us, a chain of five dependent loads (length, table, tile, partial result, merge).  (8 waves a workgroup in launches of fewer workgroups than CUs changed nothing: a lone
// workgroup is bound by what its CU can pull, about 70 GB/s, and more partitions put more CUs to work.)
constexpr int kDraftWaves = 4;

__host__ __device__ constexpr int draft_narrow_lds_bytes(int D, int C) {
  return kDraftWaves * decode_mfma_wave_bytes(1, D) + 2 * C * kMfmaHeads * kDraftWaves * 4 + 16;
}

template <int KV, int CT, int D, int C>
__global__ __launch_bounds__(kDraftWaves * 64, 2) void draft_narrow_kernel(const DraftParams p) {
  constexpr int W = kDraftWaves;
  using G = Geo<KV, D, 1>;
  using TileT = MfmaTile<KV, D, 1>;
  constexpr int TILE = kMfmaTile;
  constexpr int NC = kMfmaHeads;
  constexpr int RL = TileT::RL;              // row loads of 8 tokens per tile: 4
  constexpr int CPR = D / 8;
  constexpr int ROWB = D * 2;
  constexpr int MT = D / 16;
  constexpr int CPL = G::EPC / 8;
  constexpr bool LM = kLaneMajorTokens<KV>;
  constexpr int WAVEB = decode_mfma_wave_bytes(1, D);

  extern __shared__ __align__(256) uint8_t draft_lds[];       // fragments' addresses want it (DraftRows)
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint8_t* my_lds = draft_lds + wave * WAVEB;
  float* my_scales = reinterpret_cast<float*>(my_lds + 2 * draft_half_bytes(D));
  float (*red)[NC * D] = reinterpret_cast<float (*)[NC * D]>(draft_lds);             // [W][16 x D], over the tiles, one operand at a time
  float (*sm)[W] = reinterpret_cast<float (*)[W]>(draft_lds + W * WAVEB);            // [16 C][W]
  float (*sl)[W] = sm + C * NC;
  int* any_wild = reinterpret_cast<int*>(sl + C * NC);         // a drafted token's V holds infinities or NaN

  const int g = lane >> 3;
  const int j = lane & 7;
  DraftWork w;
  const bool some = draft_work<C * NC, D>(p, w);
  draft_zero_dead<W * 64, D>(p, w);
  if (!some) return;
  DraftRows<KV, CT, D, C, false> rows;
  rows.init(lane);
  const int col = rows.col, kg = rows.kg;

  if (threadIdx.x == 0) *any_wild = 0;
  __syncthreads();

  const int begin = w.begin, end = w.end;
  const int bs_mask = (1 << p.bs_log2) - 1;
  const uint32_t token_bytes = (uint32_t)(p.num_kv_heads * D * G::ES);
  const uint32_t block_bytes = token_bytes << p.bs_log2;
  auto token_of = [&](int r) { return LM ? g * 4 + r : r * 8 + g; };
  const uint32_t lane_off = (uint32_t)(((LM ? 0 : g) * p.num_kv_heads + w.kvh) * D * G::ES + j * G::LB);
  const int32_t* bt_row = p.block_tables + w.b * p.bt_stride;
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

  // registers -> LDS
  auto write_tile = [&](TileT& t, int tile, bool special) __attribute__((always_inline)) {
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
            wild = draft_tame<CT>(vf) || wild;
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
    if (special && wild) *any_wild = 1;
  };

  // this wave's tiles: wave, wave + W, ...
  const int n_mine = ntiles > wave ? (ntiles - wave + W - 1) / W : 0;
  auto run_tiles = [&](auto stream_tag) __attribute__((always_inline)) {
    if (n_mine > 0) {
      TileT t;
      int ids[4], ids_next[4];
      load_ids(wave, ids);
      issue_as(stream_tag, t, wave, ids);
      // The queries while the first tile is on its way.  Rows without a node repeat the last one; they are never written.
      rows.load_q(p.q, p.q_dtype, p.scale_log2e, [&](int c) {
        const int r = w.row0 + min(16 * c + col, w.live - 1);
        return ((int64_t)w.b * p.nodes + r / w.gq) * p.q_stride + (int64_t)(w.kvh * w.gq + r % w.gq) * D;
      });
      load_ids(wave + W, ids);
      for (int i = 0; i < n_mine; ++i) {
        const int tile = wave + i * W;
        const int first = begin + tile * TILE;
        const bool special = first + TILE > w.ctx || first + TILE > end;     // drafted tokens or the end inside
        load_ids(tile + 2 * W, ids_next);
        write_tile(t, tile, special);
        if (i + 1 < n_mine) issue_as(stream_tag, t, tile + W, ids);
        rows.step(my_lds, my_lds + draft_half_bytes(D), my_scales, my_scales + TILE, special, [&](int c) { return draft_visible(p, w, 16 * c + col, first); });
#pragma unroll
        for (int x = 0; x < 4; ++x) ids[x] = ids_next[x];
      }
    }
  };
  // non-temporal loads where no neighbour in the batch maps the same blocks
  if (decode_range_is_private(bt_row, p.bt_stride, w.b, p.batch, min(begin >> p.bs_log2, last_blk))) run_tiles(std::true_type{});
  else run_tiles(std::false_type{});

  // merge the waves
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (kg == 0) sm[16 * c + col][wave] = rows.m_ref[c];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    __syncthreads();                 // the maxima are there; every wave is done with its tiles, or with the operand before
    float mx = sm[16 * c + col][0];
#pragma unroll
    for (int i = 1; i < W; ++i) mx = fmaxf(mx, sm[16 * c + col][i]);
    const float f = rows.m_ref[c] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(rows.m_ref[c] - mx);
    float lw = rows.l_run[c] * f;
    lw += __shfl_xor(lw, 16);
    lw += __shfl_xor(lw, 32);
    if (kg == 0) sl[16 * c + col][wave] = lw;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) *(mfloat4_t*)&red[wave][col * D + 16 * mt + 4 * kg] = rows.o[c][mt] * f;
    __syncthreads();
    const int some_rows = min(w.live - 16 * c, 16);
    for (int idx = threadIdx.x; idx < some_rows * (D / 4); idx += W * 64) {
      const int r = idx / (D / 4), d = idx % (D / 4) * 4;
      float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, den = 0.0f, top = -INFINITY;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float4 v = *(const float4*)&red[i][r * D + d];
        x[0] += v.x; x[1] += v.y; x[2] += v.z; x[3] += v.w;
        den += sl[16 * c + r][i];
        top = fmaxf(top, sm[16 * c + r][i]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = x[e] / den;
      if (__builtin_expect(top == -INFINITY, 0)) {           // partitions: the merge decides
        const float none = p.max_partitions > 1 ? 0.0f : draft_unreferenced(p, w.b, (w.row0 + 16 * c + r) / w.gq);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = none;
      }
      draft_store4(p, w, 16 * c + r, d, D, x);
      if (p.max_partitions > 1 && d == 0) draft_store_stats(p, w, 16 * c + r, top, den);
    }
  }
  if (__builtin_expect(*any_wild, 0)) draft_wild<KV, CT, D, W * 64>(p, w);
}

// ---- more rows: the waves share the tokens -----------------------------------------------------------------------
// 32 WR rows per workgroup.  A 64-token tile of K and V is fetched by the whole workgroup and staged in LDS, double
// buffered, one barrier a tile; the next DEPTH tiles' loads are in flight in registers meanwhile.  Wave (wr, wk) takes
// rows 32 wr .. + 31 of the tile's half wk, and the halves are merged at the end.  8 waves for 128 rows: a CU then holds one workgroup with two waves per SIMD and 64 KiB of loads in flight (4 waves
// taking all 64 tokens each, one tile ahead: 32 rows of 64 nodes x 4096 tokens took 146 us; now 104, 5.2 TB/s, which is what
// the loads by themselves take).
// Two row tiles per KV head and long contexts are bound by the turn instead: 4 rows of 27 nodes x 64 heads x 16k to 32k tokens
// take 162 us (540 TFLOP/s of rows that count), of which the launch and two rounds of first loads and last stores are 44,
// products and exponentials 82, fetching and staging 36.  A turn is 1.2 us: matrix pipe 0.42, vector ALU 0.55, LDS 0.55, hardly
// overlapped.  Waves half a turn apart, a third stage with the next fragments read ahead of the barrier, and a raised wave
// priority during the products left it where it is.

constexpr int kWideTile = 64;
__host__ __device__ constexpr int draft_wide_waves(int WR) { return WR == 4 ? 8 : 4; }
__host__ __device__ constexpr int draft_wide_stage_bytes(int D, int WR) {
  const int tiles = 2 * kWideTile * D * 4, merge = WR * 32 * (D + 4) * 4;
  return tiles > merge ? tiles : merge;
}
__host__ __device__ constexpr int draft_wide_lds_bytes(int D, int WR) { return draft_wide_stage_bytes(D, WR) + 2 * 2 * kWideTile * 4 + 16; }

template <int KV, int CT, int D, int WR, bool STREAM>
__global__ __launch_bounds__(draft_wide_waves(WR) * 64, 2) void draft_wide_kernel(const DraftParams p) {
  constexpr int W = draft_wide_waves(WR), NT = W * 64;
  constexpr int TK = kWideTile;
  constexpr int DEPTH = W == 8 ? 2 : 1;
  constexpr int C = 2;                       // 16-row operands per wave
  constexpr int ES = KV == KV_FP8 ? 1 : 2;
  constexpr int LPR = D * ES / 16;           // threads per token row
  constexpr int RPI = NT / LPR < TK ? NT / LPR : TK;     // rows per load instruction of the workgroup
  constexpr int NIT = TK / RPI;       // load instructions per tile (K and V each)
  constexpr int CPT = 16 / ES / 8;           // 8-element chunks per load
  constexpr int CPR = D / 8;
  constexpr int ROWB = D * 2;
  constexpr int MT = D / 16;
  constexpr int TILEB = TK * ROWB;           // the tile's K or V

  extern __shared__ __align__(256) uint8_t draft_lds[];       // fragments' addresses want it (DraftRows)
  // stage: K, V; then per stage 1 / k_scale and the mantissa of 1 / v_scale; then any_wild
  float* scales = reinterpret_cast<float*>(draft_lds + draft_wide_stage_bytes(D, WR));
  int* any_wild = reinterpret_cast<int*>(scales + 2 * 2 * TK);        // a drafted token's V holds infinities or NaN
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  DraftWork w;
  const bool some = draft_work<32 * WR, D>(p, w);
  draft_zero_dead<NT, D>(p, w);
  if (!some) return;
  const int wr = wave >> 1, wk = wave & 1;
  const bool active = 32 * wr < w.live;      // the wave has rows (it fetches tiles in any case)
  const int row_w = 32 * wr;
  DraftRows<KV, CT, D, C, true> rows;
  rows.init(lane);
  const int col = rows.col, kg = rows.kg;

  const int begin = w.begin, end = w.end;
  const int bs_mask = (1 << p.bs_log2) - 1;
  const uint32_t token_bytes = (uint32_t)(p.num_kv_heads * D * ES);
  const uint32_t block_bytes = token_bytes << p.bs_log2;
  const int32_t* bt_row = p.block_tables + w.b * p.bt_stride;
  const int last_blk = min((end - 1) >> p.bs_log2, max(p.table_width - 1, 0));
  const int ntiles = (end - begin + TK - 1) / TK;
  const int lrow = tid / LPR;                // this thread's row of a load instruction
  const bool fetches = LPR * TK >= NT || lrow < TK;      // narrow fp8 rows need only part of the workgroup
  const uint32_t lane_off = (uint32_t)(w.kvh * D * ES + (tid % LPR) * 16);

  struct Stage {                             // a tile as loaded
    mword4_t k[NIT], v[NIT];
    float ks[NIT], vs[NIT];
  };
  Stage st[DEPTH];
  int ids[NIT];                              // table entries of the next tile to ask for, fetched a tile ahead of its loads
  auto load_ids = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NIT; ++i) ids[i] = bt_row[min((begin + tile * TK + i * RPI + lrow) >> p.bs_log2, last_blk)];
  };
  // The next tile's table entries are asked for before this tile's data: loads return in order, and a wait for entries asked
  // for behind the data would be a wait for the data.  Past the last tile everybody loads the pool's first token: a wait is for
  // a number of loads, so loads under a condition would make it one for all of them.
  auto issue = [&](Stage& t, int tile) __attribute__((always_inline)) {
    int now[NIT];
#pragma unroll
    for (int i = 0; i < NIT; ++i) now[i] = ids[i];
    load_ids(tile + 1);
    const bool real = tile < ntiles && fetches;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      const uint32_t phys = real ? (uint32_t)min(max(now[i], 0), p.num_blocks - 1) : 0u;
      const uint32_t off = real ? (uint32_t)((begin + tile * TK + i * RPI + lrow) & bs_mask) : 0u;
      const uint64_t base = (uint64_t)phys * block_bytes + off * token_bytes + (real ? lane_off : 0u);
      const mword4_t* kp = (const mword4_t*)(p.k_cache + base);
      const mword4_t* vp = (const mword4_t*)(p.v_cache + base);
      if constexpr (STREAM) {
        t.k[i] = __builtin_nontemporal_load(kp);
        t.v[i] = __builtin_nontemporal_load(vp);
      } else {
        t.k[i] = *kp;
        t.v[i] = *vp;
      }
      if constexpr (KV == KV_FP8) {
        const uint64_t slot = ((uint64_t)phys << p.bs_log2) + off;
        t.ks[i] = p.k_scale[slot];
        t.vs[i] = p.v_scale[slot];
      }
    }
  };
  auto commit = [&](Stage& t, int tile) __attribute__((always_inline)) {
    if (tile >= ntiles || !fetches) return;
    const int buf = tile & 1;
    uint8_t* kt = draft_lds + buf * 2 * TILEB;
    // Only tiles of drafted tokens are rid of infinities and NaN: what a committed token holds is every row's, and a partition
    // of 32 mod 64 tokens ends inside a tile of such, far from where draft_wild looks.  One branch for both: two cost every
    // tile (4 rows of 27 nodes 181 us instead of 168).
    const int past = begin + (tile + 1) * TK;
    const bool drafted = past > w.ctx, special = drafted || past > end;
    bool wild = false;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      const int r = i * RPI + lrow;
      const bool valid = begin + tile * TK + r < end;
      float v_pow2 = 1.0f;
      if constexpr (KV == KV_FP8) v_pow2 = __uint_as_float(__float_as_uint(__builtin_amdgcn_rcpf(t.vs[i])) & 0xff800000u);
#pragma unroll
      for (int x = 0; x < CPT; ++x) {
        const int chunk = (tid % LPR) * CPT + x;
        const uint32_t kw[4] = {t.k[i][0], t.k[i][1], t.k[i][2], t.k[i][3]};
        const uint32_t vw[4] = {t.v[i][0], t.v[i][1], t.v[i][2], t.v[i][3]};
        mword4_t kf = words_to_ct<KV, CT>(kw + 2 * x);
        mword4_t vf;
        if constexpr (KV == KV_FP8) vf = __builtin_bit_cast(mword4_t, fp8_words_to_f16_pow2(vw + 2 * x, v_pow2));
        else vf = words_to_ct<KV, CT>(vw);
        if (special) {
          if (!valid) kf = vf = mword4_t{0, 0, 0, 0};       // past the end: scores masked, and 0 * V must stay 0
          if (drafted) wild = draft_tame<CT>(vf) || wild;
        }
        uint8_t* dst = kt + r * ROWB + ((chunk ^ lds_swz<CPR>(r)) << 4);
        *(mword4_t*)dst = kf;
        *(mword4_t*)(dst + TILEB) = vf;
      }
      if constexpr (KV == KV_FP8) {
        if (tid % LPR == 0) {
          const uint32_t bits = __float_as_uint(__builtin_amdgcn_rcpf(t.vs[i]));
          scales[buf * 2 * TK + r] = valid ? __builtin_amdgcn_rcpf(t.ks[i]) : 0.0f;
          scales[buf * 2 * TK + TK + r] = valid ? __uint_as_float((bits & 0x007fffffu) | 0x3f800000u) : 0.0f;
        }
      }
    }
    if (special && wild) *any_wild = 1;
  };
  auto compute = [&](int tile) __attribute__((always_inline)) {
    const int at = wk * (TK / 2), first = begin + tile * TK + at;
    if (!active || first >= end) return;
    const uint8_t* kt = draft_lds + (tile & 1) * 2 * TILEB;
    const float* sc = scales + (tile & 1) * 2 * TK;
    const bool special = first + 32 > w.ctx || first + 32 > end;       // drafted tokens or the end inside
    rows.step(kt + at * ROWB, kt + TILEB + at * ROWB, sc + at, sc + TK + at, special,
              [&](int c) { return draft_visible(p, w, row_w + 16 * c + col, first); });
  };

  if (tid == 0) *any_wild = 0;
  load_ids(0);
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) issue(st[d], d);
  // the queries while the first tiles are on their way
  rows.load_q(p.q, p.q_dtype, p.scale_log2e, [&](int c) {
    const int r = w.row0 + min(row_w + 16 * c + col, w.live - 1);
    return ((int64_t)w.b * p.nodes + r / w.gq) * p.q_stride + (int64_t)(w.kvh * w.gq + r % w.gq) * D;
  });
  __syncthreads();
  commit(st[0], 0);
  issue(st[0], DEPTH);
  __syncthreads();
  // before a turn its tile is in LDS and tiles + 1 ... + DEPTH are on their way, tile t in st[t % DEPTH]
  auto turn = [&](Stage& next, int t) __attribute__((always_inline)) {
    compute(t);
    commit(next, t + 1);             // the other stage: its last readers passed the barrier before this tile
    issue(next, t + 1 + DEPTH);
    __syncthreads();
  };
  // no way out between the turns of a pair: where such paths meet, waits are for the fewest loads that any of them left
  for (int tile = 0; tile < ntiles; tile += DEPTH) {
    turn(st[1 % DEPTH], tile);
    if constexpr (DEPTH == 2) turn(st[0], tile + 1);
  }

  // ---- merge the halves, write --------------------------------------------------------------------------------------
  float sum[C], top[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    sum[c] = rows.l_run[c];
    sum[c] += __shfl_xor(sum[c], 16);
    sum[c] += __shfl_xor(sum[c], 32);
    top[c] = rows.m_ref[c];
  }
  float* other = reinterpret_cast<float*>(draft_lds) + wr * (32 * (D + 4));  // [32][D + 4]: output, maximum, sum
  if (active && wk == 1) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float* at = other + (16 * c + col) * (D + 4);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) *(mfloat4_t*)(at + 16 * mt + 4 * kg) = rows.o[c][mt];
      if (kg == 0) { at[D] = top[c]; at[D + 1] = sum[c]; }
    }
  }
  __syncthreads();
  if (active && wk == 0) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int r = row_w + 16 * c + col;
      const float* at = other + (16 * c + col) * (D + 4);
      const float t1 = at[D], mx = fmaxf(top[c], t1);
      const float f0 = top[c] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top[c] - mx);
      const float f1 = t1 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(t1 - mx);
      const float total = sum[c] * f0 + at[D + 1] * f1;
      if (r >= w.live) continue;
      const float inv = 1.0f / total;
      const bool none = mx == -INFINITY;
      float instead = 0.0f;                                  // partitions: the merge decides
      if (__builtin_expect(none, 0) && p.max_partitions == 1) instead = draft_unreferenced(p, w.b, (w.row0 + r) / w.gq);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const mfloat4_t v = (rows.o[c][mt] * f0 + *(const mfloat4_t*)(at + 16 * mt + 4 * kg) * f1) * inv;
        const float x[4] = {none ? instead : v[0], none ? instead : v[1], none ? instead : v[2], none ? instead : v[3]};
        draft_store4(p, w, r, 16 * mt + 4 * kg, D, x);
      }
      if (p.max_partitions > 1 && kg == 0) draft_store_stats(p, w, r, mx, total);
    }
  }
  if (__builtin_expect(*any_wild, 0)) draft_wild<KV, CT, D, NT>(p, w);
}

using DraftKernel = void (*)(DraftParams);

// `attr_set`: one flag per device, the kernel's own (the LDS limit belongs to the kernel on one device)
inline int launch_draft_kernel(DraftKernel kern, int threads, int lds, std::atomic<bool>* attr_set, const DraftParams& p, unsigned grid, hipStream_t st) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return fail(PA_ERR_LAUNCH, "pa_draft_attention: cannot tell the current device");
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
      return fail(PA_ERR_LAUNCH, "pa_draft_attention: cannot raise the dynamic LDS limit");
    attr_set[dev].store(true, std::memory_order_release);
  }
  hipLaunchKernelGGL(kern, dim3(grid), dim3(threads), lds, st, p);
  return PA_OK;
}

template <int KV, int CT, int D, int C>
int launch_draft_narrow(const DraftParams& p, unsigned grid, hipStream_t st) {
  static std::atomic<bool> attr_set[64];
  return launch_draft_kernel(draft_narrow_kernel<KV, CT, D, C>, kDraftWaves * 64, draft_narrow_lds_bytes(D, C), attr_set, p, grid, st);
}

template <int KV, int CT, int D, int WR>
int launch_draft_wide(const DraftParams& p, unsigned grid, hipStream_t st) {
  static std::atomic<bool> attr_set[2][64];
  // Non-temporal loads where no second row tile reads the same range: 104 us instead of 109 for 32 rows of 64 nodes x 4096
  // tokens, and no loss where all rows share their blocks (98 us either way).  64-row workgroups gain nothing (153 us).
  if constexpr (WR == 4)
    if (p.row_tiles == 1)
      return launch_draft_kernel(draft_wide_kernel<KV, CT, D, WR, true>, draft_wide_waves(WR) * 64, draft_wide_lds_bytes(D, WR), attr_set[1], p, grid, st);
  return launch_draft_kernel(draft_wide_kernel<KV, CT, D, WR, false>, draft_wide_waves(WR) * 64, draft_wide_lds_bytes(D, WR), attr_set[0], p, grid, st);
}

template <int KV, int CT, int D>
int launch_draft_dim(const DraftParams& p, int rows, unsigned grid, hipStream_t st) {
  switch (rows) {
    case 16: return launch_draft_narrow<KV, CT, D, 1>(p, grid, st);
    case 32: return launch_draft_narrow<KV, CT, D, 2>(p, grid, st);
    case 64: return launch_draft_wide<KV, CT, D, 2>(p, grid, st);
    default: return launch_draft_wide<KV, CT, D, 4>(p, grid, st);
  }
}

// rows: (node, head) rows per workgroup, 16, 32, 64 or 128
template <int KV, int CT>
int launch_draft(const DraftParams& p, int head_dim, int rows, unsigned grid, hipStream_t st) {
  return head_dim == 128 ? launch_draft_dim<KV, CT, 128>(p, rows, grid, st) : launch_draft_dim<KV, CT, 64>(p, rows, grid, st);
}

int launch_draft_f16(const DraftParams& p, int head_dim, int rows, unsigned grid, hipStream_t st);
int launch_draft_bf16(const DraftParams& p, int head_dim, int rows, unsigned grid, hipStream_t st);
int launch_draft_bf16_as_f16(const DraftParams& p, int head_dim, int rows, unsigned grid, hipStream_t st);
int launch_draft_fp8(const DraftParams& p, int head_dim, int rows, unsigned grid, hipStream_t st);

}  // namespace pa

// Which drafted tokens the target model accepts, and the token that follows them (gfx950).
//
// Reference: the draft / target decoder's greedy and sampled verification (src/inference/speculative.py), there
// on the host, chains only, without top-p.  Here, per row of the batch, over a tree of nodes whose logits l the
// target has produced:
//     w_j = exp((l_j - max l) / T);  with top_p < 1 a token stays while the mass of the strictly likelier ones is
//     at most top_p * sum w, the others' w becomes 0 (sample_tokens' rule);  z = sum w,  p = w / z
//     from node 0: the children of an accepted node are tried in index order,
//       point-mass drafts:     child c passes iff  u_c * (z - sum of w of the siblings refused before) < w_c
//                              (a token offered twice counts once), i.e. with the probability that is left of it
//       drafts drawn from q:   child c passes iff  u_c * q(c) * z < w_c             (one child a node)
//     the first that passes is accepted and its children come next; when none does, the next token is drawn by
//     inversion of u_0 in index order from  w without the refused children,  max(w / z - q, 0),  or w (a leaf).
//     T <= 0: a child passes iff it is its parent's first maximum, and the next token is the last node's.
// The emitted tokens are distributed as the target's own samples whatever the drafts.
//
// Everything a decision compares is a 64-bit float: with a 152k vocabulary the tokens of a broad row are 1e-6
// apart in the inverted distribution, and sums of 32-bit exponentials (1e-7 each, biased) pick a neighbour every
// few hundred draws.
//
// Launches: (1) row statistics (z, max, the smallest kept logit; greedy: the first maximum) of every node a row
// drafts, one workgroup a node; (2) the walk, by every workgroup of (row, slice of the vocabulary) for itself -
// a few hundred LDS reads - and, sampling, the slice's part of the sums the draw needs, per chunk of 2048
// entries; (3) the draw: the chunk by a scan of the sums, the token inside it.  Greedy stops after (2).
//
// (1) for 16-bit logits is a histogram, not a pass of exponentials: a row holds at most 65536 different values, a
// few thousand in practice, so the row's entries are counted by bit pattern in LDS (two 16-bit counters to a
// word: +x and -x) and exp runs once per value that occurs, times its count, in 64 bits.  The same counts, summed
// in descending order, give the top-p threshold, so a row leaves HBM once whatever top_p is.  A 16-bit counter
// that overflows (more than 65535 equal logits) shows in the total of all counters; such rows, and 32-bit logits,
// take a search over ordered bit patterns instead, 11 bits a pass.
#include "logit_row.hpp"
#include "pa_common.hpp"
#include "pa_host.hpp"

#include <math.h>

#include <atomic>

namespace pa {

constexpr int kStatThreads = 1024;
constexpr int kStatWaves = kStatThreads / 64;
constexpr int kWalkThreads = 256;
constexpr int kWalkWaves = kWalkThreads / 64;
constexpr int kChunk = 2048;                    // vocabulary entries behind one pair of stored sums
constexpr int kNodeWords = PA_MAX_DRAFT_NODES / 64;
constexpr int kBins = 2048;                     // bins of one pass of the search
constexpr int kVerifyMaxDevices = 64;

struct VerifyParams {
  const void* logits;
  int64_t row_stride, batch_stride;             // elements between nodes, between rows of the batch
  const int64_t* tokens;                        // [batch][nodes]
  const float* uniforms;                        // [batch][nodes], nullptr: greedy
  const int32_t* parents;                       // nullptr: a chain
  int64_t parents_stride;
  const int32_t* num_nodes;                     // nullptr: all of them
  const void* q;                                // [batch][nodes - 1][vocab] probabilities, nullptr: point masses
  int64_t q_row_stride, q_batch_stride;
  int q_dtype;
  double c;                                     // log2(e) / T
  double top_p;
  int nodes, vocab, chunks, chunks_per_wg;
  // workspace
  double* z;                                    // [batch][nodes]
  float* top;                                   // [batch][nodes]
  float* cut;                                   // [batch][nodes] smallest kept logit; greedy: the first maximum's index (as bits)
  double* sums;                                 // [batch][chunks][2]: the draw's weights, all kept weights
  int32_t* last;                                // [batch]: the last accepted node, -1: an empty row
  int64_t* out_tokens;
  int32_t* out_counts;
  int32_t* out_path;
};

__device__ __forceinline__ int nodes_of(const VerifyParams& p, int b) {
  return p.num_nodes ? min(max(p.num_nodes[b], 0), p.nodes) : p.nodes;
}

// w of one logit; NaN and -inf weigh nothing
__device__ __forceinline__ double logit_weight(float l, float top, double c) {
  if (l == top) return l == -INFINITY ? 0.0 : 1.0;
  return l < top ? exp2(((double)l - (double)top) * c) : 0.0;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// inclusive prefix sum over the lanes of a wave
__device__ __forceinline__ double wave_scan(double v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double up = __shfl_up(v, o);
    if (lane >= o) v += up;
  }
  return v;
}

// Sum over a workgroup of WAVES waves, the same in every thread; red holds WAVES doubles.
template <int WAVES>
__device__ __forceinline__ double group_sum(double v, double* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) s += red[w];
  return s;
}

// Inclusive prefix sum over a workgroup of WAVES waves, thread order; red holds WAVES doubles.
template <int WAVES>
__device__ __forceinline__ double group_scan(double v, double* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan(v, lane);
  __syncthreads();
  if (lane == 63) red[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v += red[w];
  return v;
}

struct StatLds {
  double seg[1024];            // mass of 64 neighbouring values, in descending order of the values
  double red[kStatWaves];
  double found[2];             // the crossing: mass above it, kept mass
  uint32_t key[2];             // its place
  uint32_t redu[3][kStatWaves];
};

struct RowStats {
  double z;
  float top, cut;
};

// Row statistics without the histogram: maximum, then the sum of all weights, then (top_p < 1) the smallest kept
// logit by a search over ordered bit patterns: the range that holds it is cut into 2048 bins, the weights of the
// range's entries are added up per bin as 64-bit fixed-point numbers (exact, so the order of the atomics does not
// matter), and the bin in which the mass above crosses top_p * z is the next range.  The first range starts at the
// smallest weight that can be kept: tokens lighter than (1 - top_p) z / vocab weigh less than 1 - top_p together.
// A pass costs one read of the row from the L2 and an exponential per entry in range: 3 passes on 32-bit logits.
template <int DT>
__device__ RowStats search_row(const void* ptr, const VerifyParams& p, uint64_t* bins, StatLds& s) {
  const int tid = threadIdx.x;
  RowStats r;
  float best = -INFINITY;
  for_each_logit<DT, kStatThreads>(ptr, p.vocab, [&](int, float x) __attribute__((always_inline)) { best = fmaxf(best, x); });   // fmaxf drops NaN
  best = wave_max(best);
  __syncthreads();
  if ((tid & 63) == 0) s.redu[0][tid >> 6] = __float_as_uint(best);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kStatWaves; ++w) best = fmaxf(best, __uint_as_float(s.redu[0][w]));
  r.top = best + 0.0f;
  r.cut = -INFINITY;
  if (best == -INFINITY) { r.z = 0.0; return r; }
  double mine = 0.0;
  for_each_logit<DT, kStatThreads>(ptr, p.vocab, [&](int, float x) __attribute__((always_inline)) { mine += logit_weight(x, best, p.c); });
  r.z = group_sum<kStatWaves>(mine, s.red);
  if (!(p.top_p < 1.0) || best == INFINITY) return r;
  const double limit = p.top_p * r.z;
  const int log_vocab = 32 - __builtin_clz((uint32_t)p.vocab);
  const double unit = ldexp(1.0, 62 - log_vocab), back = 1.0 / unit;     // a row's weights sum to at most `vocab`
  const float low = (float)((double)best + log2((1.0 - p.top_p) * r.z / p.vocab * 0.5) / p.c);
  uint32_t lo = ordered_key32(low < best ? low : best), hi = ordered_key32(r.top);
  double above = 0.0;
  for (;;) {
    const uint32_t span = hi - lo;
    const int shift = span < kBins ? 0 : 21 - __builtin_clz(span);       // span >> shift < 2048
    for (int i = tid; i < kBins; i += kStatThreads) bins[i] = 0;
    __syncthreads();
    for_each_logit<DT, kStatThreads>(ptr, p.vocab, [&](int, float x) __attribute__((always_inline)) {
      const uint32_t off = ordered_key32(x + 0.0f) - lo;                   // -0 counts as +0; NaN lies beyond every finite key
      if (off <= span)
        __hip_atomic_fetch_add(&bins[off >> shift], (uint64_t)(logit_weight(x, best, p.c) * unit + 0.5), __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_WORKGROUP);
    });
    __syncthreads();
    // bins from the top: thread t takes bins 2047 - 2t and 2046 - 2t
    const double m0 = (double)bins[kBins - 1 - 2 * tid] * back, m1 = (double)bins[kBins - 2 - 2 * tid] * back;
    const double upto = above + group_scan<kStatWaves>(m0 + m1, s.red), before = upto - (m0 + m1);
    if (tid == 0) s.key[0] = kBins;
    __syncthreads();
    if (upto > limit) __hip_atomic_fetch_min(&s.key[0], (uint32_t)tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    __syncthreads();
    const uint32_t crossing = s.key[0];                                     // the first thread past the limit
    if ((uint32_t)tid == crossing) {
      const bool second = before + m0 <= limit;
      s.key[1] = kBins - 1 - 2 * tid - (second ? 1 : 0);
      s.found[0] = second ? before + m0 : before;
      s.found[1] = second ? upto : before + m0;
    }
    __syncthreads();
    const uint32_t bin = s.key[1];
    if (crossing == kBins) {             // rounding left the total at the limit: the whole range is kept
      r.z = limit > 0.0 ? limit : r.z;
      r.cut = key_value32(lo);
      break;
    }
    above = s.found[0];
    const uint32_t next = lo + (bin << shift);
    if (shift == 0) {
      r.cut = key_value32(next);
      r.z = s.found[1];
      break;
    }
    const uint32_t size = (1u << shift) - 1;
    hi = hi - next < size ? hi : next + size;
    lo = next;
    __syncthreads();                      // everyone has read the bins
  }
  return r;
}

// One workgroup per node.  16-bit logits: LDS holds 32768 words of two counters, then StatLds.
template <int DT>
__global__ __launch_bounds__(kStatThreads) void draft_row_stats_kernel(const VerifyParams p) {
  extern __shared__ __align__(16) uint8_t lds_raw[];
  const int node = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (node >= nodes_of(p, b)) return;
  constexpr bool COUNTS = DT != PA_DTYPE_F32;
  constexpr int WORDS = 32768;
  uint32_t* hist = (uint32_t*)lds_raw;
  StatLds& s = *(StatLds*)(lds_raw + (COUNTS ? WORDS * 4 : kBins * 8));
  const void* ptr = (const uint8_t*)p.logits + (b * p.batch_stride + node * p.row_stride) * (COUNTS ? 2 : 4);
  const int64_t at = (int64_t)b * p.nodes + node;
  RowStats r;
  bool counted = false;
  if constexpr (COUNTS) {
    constexpr uint32_t INF = DT == PA_DTYPE_F16 ? 0x7c00u : 0x7f80u;
    for (int i = tid; i < WORDS / 4; i += kStatThreads) ((uint4*)hist)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for_each_logit_bits<DT, kStatThreads>(ptr, p.vocab, [&](int, uint32_t bits) __attribute__((always_inline)) {
      __hip_atomic_fetch_add(&hist[bits & 0x7fffu], (bits & 0x8000u) ? 0x10000u : 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    });
    __syncthreads();
    // the largest value (NaN left out), and the number of entries counted
    uint32_t pos = 0, neg = 0xffffffffu, count = 0;       // largest m with +m (plus 1), smallest m with -m
#pragma unroll 4
    for (int i = tid; i < WORDS; i += kStatThreads) {
      const uint32_t v = hist[i];
      count += (v & 0xffffu) + (v >> 16);
      if ((uint32_t)i <= INF) {
        if ((v & 0xffffu) || (i == 0 && v)) pos = i + 1;
        if ((v >> 16) && neg == 0xffffffffu) neg = i;
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      pos = max(pos, (uint32_t)__shfl_xor(pos, o));
      neg = min(neg, (uint32_t)__shfl_xor(neg, o));
      count += __shfl_xor(count, o);
    }
    if (lane == 0) { s.redu[0][wave] = pos; s.redu[1][wave] = neg; s.redu[2][wave] = count; }
    __syncthreads();
    pos = 0; neg = 0xffffffffu; count = 0;
#pragma unroll
    for (int w = 0; w < kStatWaves; ++w) {
      pos = max(pos, s.redu[0][w]);
      neg = min(neg, s.redu[1][w]);
      count += s.redu[2][w];
    }
    counted = count == (uint32_t)p.vocab;
    if (counted) {
      r.top = pos ? logit_value<DT>(pos - 1) : neg < INF ? logit_value<DT>(neg | 0x8000u) : -INFINITY;
      r.cut = -INFINITY;
      // masses of 64 neighbouring values; segments 0..511: positive values, largest first; 512..1023: negative ones
      auto masses = [&](int m, double& up, double& down) __attribute__((always_inline)) {
        const uint32_t v = hist[m];
        uint32_t a = v & 0xffffu, d = v >> 16;
        if (m == 0) { a += d; d = 0; }                     // -0 and +0 are one value
        if ((uint32_t)m > INF) a = d = 0;                  // NaN
        up = a ? a * logit_weight(logit_value<DT>(m), r.top, p.c) : 0.0;
        down = d && (uint32_t)m != INF ? d * logit_weight(logit_value<DT>(m | 0x8000u), r.top, p.c) : 0.0;
      };
      for (int g = wave; g < WORDS / 64; g += kStatWaves) {
        const int m = 64 * g + lane;
        double up = 0.0, down = 0.0;
        if (__builtin_amdgcn_ballot_w64(hist[m] != 0)) {
          masses(m, up, down);
          up = wave_sum(up);
          down = wave_sum(down);
        }
        if (lane == 0) { s.seg[511 - g] = up; s.seg[512 + g] = down; }
      }
      __syncthreads();
      const double mass = s.seg[tid];
      const double upto = group_scan<kStatWaves>(mass, s.red);
      if (tid == kStatThreads - 1) s.found[0] = upto;
      if (tid == 0) s.key[0] = kStatThreads;
      __syncthreads();
      r.z = s.found[0];
      if (p.top_p < 1.0 && r.top != INFINITY && r.top != -INFINITY) {
        const double limit = p.top_p * r.z;
        if (upto > limit) __hip_atomic_fetch_min(&s.key[0], (uint32_t)tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        __syncthreads();
        const uint32_t o = s.key[0];                       // the first segment past the limit
        if ((uint32_t)tid == o) s.found[0] = upto - mass;
        __syncthreads();
        if (o < kStatThreads) {
          // inside the segment, lanes in descending order of the values
          const int m = o < 512 ? 64 * (511 - (int)o) + 63 - lane : 64 * ((int)o - 512) + lane;
          double up, down;
          masses(m, up, down);
          const double here = o < 512 ? up : down;
          const double to = s.found[0] + wave_scan(here, lane);
          unsigned long long hit = __builtin_amdgcn_ballot_w64(here > 0.0 && to > limit);
          const unsigned long long some = __builtin_amdgcn_ballot_w64(here > 0.0);
          // the first value whose mass crosses the limit; by rounding none: the segment's last
          const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some | 1ull);
          r.z = __shfl(to, l);
          const uint32_t mb = __shfl(m, l);
          r.cut = logit_value<DT>(o < 512 ? mb : mb | 0x8000u);
        }
      }
    }
  }
  if (!counted) {
    __syncthreads();
    r = search_row<DT>(ptr, p, (uint64_t*)lds_raw, s);
  }
  if (tid == 0) {
    p.z[at] = r.z;
    p.top[at] = r.top;
    p.cut[at] = r.cut;
  }
}

// Greedy: the index of the first maximum of every node's row (0 if every entry is NaN or -inf).
template <int DT>
__global__ __launch_bounds__(kStatThreads) void draft_row_argmax_kernel(const VerifyParams p) {
  __shared__ float redv[kStatWaves];
  __shared__ int redi[kStatWaves];
  const int node = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  if (node >= nodes_of(p, b)) return;
  const void* ptr = (const uint8_t*)p.logits + (b * p.batch_stride + node * p.row_stride) * (DT == PA_DTYPE_F32 ? 4 : 2);
  float best = -INFINITY;
  int best_i = p.vocab;
  auto take = [&](int i, float x) __attribute__((always_inline)) {
    if (x > best || (x == best && i < best_i)) { best = x; best_i = i; }
  };
  for_each_logit<DT, kStatThreads>(ptr, p.vocab, take);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float x = __shfl_xor(best, o);
    const int i = __shfl_xor(best_i, o);
    take(i, x);
  }
  if ((tid & 63) == 0) { redv[tid >> 6] = best; redi[tid >> 6] = best_i; }
  __syncthreads();
  if (tid == 0) {
    for (int w = 0; w < kStatWaves; ++w) take(redi[w], redv[w]);
    p.cut[(int64_t)b * p.nodes + node] = __int_as_float(best_i < p.vocab ? best_i : 0);
  }
}

struct WalkLds {
  double w[PA_MAX_DRAFT_NODES];      // the node's weight in its parent's row; drafts drawn from q: its weight / q
  double red[2][kWalkWaves];
  int parent[PA_MAX_DRAFT_NODES];
  int token[PA_MAX_DRAFT_NODES];
  float u[PA_MAX_DRAFT_NODES];
  int path[PA_MAX_DRAFT_NODES];
  uint64_t skip[kChunk / 64];        // entries of the chunk that the draw leaves out
};

// The walk of one row.  Every wave does the same from the same LDS values, so its result is uniform; lane l
// stands for nodes l, 64 + l, ...  Returns the last accepted node; s.path and `count` hold the way there, `refused`
// the children of that node (all of them refused).
template <bool GREEDY>
__device__ __forceinline__ int walk(const VerifyParams& p, WalkLds& s, int b, int n, int& count, uint64_t (&refused)[kNodeWords]) {
  const int lane = threadIdx.x & 63;
  const int words = (n + 63) >> 6;
  int cur = 0;
  count = 1;
  if (threadIdx.x == 0) s.path[0] = 0;
  for (;;) {
    const double z = GREEDY ? 0.0 : p.z[(int64_t)b * p.nodes + cur];
    double left = z;
    int next = -1;
#pragma unroll
    for (int w = 0; w < kNodeWords; ++w) refused[w] = 0;
    for (int w = 0; w < words && next < 0; ++w) {
      const int mine = 64 * w + lane;
      unsigned long long kids = __builtin_amdgcn_ballot_w64(mine > 0 && mine < n && s.parent[mine] == cur);
      while (kids) {
        const int j = 64 * w + __builtin_ctzll(kids);
        kids &= kids - 1;
        const int tok = s.token[j];
        double wj = s.w[j];
        if (p.q == nullptr) {
          // offered before under this node: nothing of it is left
          bool again = false;
#pragma unroll
          for (int x = 0; x < kNodeWords; ++x)
            again = again || (((refused[x] >> lane) & 1ull) && s.token[64 * x + lane] == tok);
          if (__builtin_amdgcn_ballot_w64(again)) wj = 0.0;
        }
        const bool good = GREEDY ? wj > 0.0 : (double)s.u[j] * (p.q ? z : left) < wj;
        if (good) { next = j; break; }
#pragma unroll
        for (int x = 0; x < kNodeWords; ++x)
          if (x == (j >> 6)) refused[x] |= 1ull << (j & 63);
        left -= wj;
      }
    }
    if (next < 0) return cur;
    if (threadIdx.x == 0) s.path[count] = next;
    ++count;
    cur = next;
  }
}

__device__ __forceinline__ float draft_prob(const VerifyParams& p, int b, int node, int64_t token) {
  return load_as_f32(p.q, b * p.q_batch_stride + node * p.q_row_stride + token, p.q_dtype);
}

// One workgroup per (slice of the vocabulary, row): the walk, the row's outputs (slice 0) and the slice's sums.
template <int DT, bool GREEDY>
__global__ __launch_bounds__(kWalkThreads) void draft_walk_kernel(const VerifyParams p) {
  __shared__ WalkLds s;
  constexpr int ES = DT == PA_DTYPE_F32 ? 4 : 2;
  const int b = blockIdx.y, tid = threadIdx.x;
  const int n = nodes_of(p, b);
  const int64_t at = (int64_t)b * p.nodes;
  if (n == 0) {
    if (blockIdx.x == 0) {
      for (int i = tid; i < p.nodes; i += kWalkThreads) { p.out_tokens[at + i] = -1; p.out_path[at + i] = -1; }
      if (tid == 0) { p.out_counts[b] = 0; if (!GREEDY) p.last[b] = -1; }
    }
    return;
  }
  const uint8_t* rows = (const uint8_t*)p.logits + b * p.batch_stride * ES;
  {
    const int i = tid;                    // kWalkThreads == PA_MAX_DRAFT_NODES
    int up = -1, tok = -1;
    double w = 0.0;
    if (i > 0 && i < n) {
      up = p.parents ? p.parents[b * p.parents_stride + i] : i - 1;
      if (up < 0 || up >= i) up = -1;
      const int64_t t = p.tokens[at + i];
      if (t >= 0 && t < p.vocab) tok = (int)t;
      if (up >= 0 && tok >= 0) {
        if constexpr (GREEDY) {
          w = __float_as_int(p.cut[at + up]) == tok ? 1.0 : 0.0;
        } else {
          const float l = load_as_f32(rows + up * p.row_stride * ES, tok, DT);
          if (l >= p.cut[at + up]) w = logit_weight(l, p.top[at + up], p.c);
          if (p.q) {
            // u * q * z < w  <=>  u * z < w / q; a token that the draft cannot draw passes if it has any weight
            const double qv = draft_prob(p, b, up, tok);
            w = qv > 0.0 ? w / qv : w > 0.0 ? (double)INFINITY : 0.0;
          }
        }
      }
    }
    s.parent[i] = up;
    s.token[i] = tok;
    s.w[i] = w;
    s.u[i] = !GREEDY && i < n ? p.uniforms[at + i] : 0.0f;
  }
  __syncthreads();
  int count;
  uint64_t refused[kNodeWords];
  const int last = walk<GREEDY>(p, s, b, n, count, refused);
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = tid; i < p.nodes; i += kWalkThreads) {
      p.out_path[at + i] = i < count ? s.path[i] : -1;
      // the drawn token's place is the third launch's (greedy: this one's)
      if (i + 1 < count) p.out_tokens[at + i] = p.tokens[at + s.path[i + 1]];
      else if (i >= count) p.out_tokens[at + i] = -1;
      else if (GREEDY) p.out_tokens[at + i] = __float_as_int(p.cut[at + last]);
    }
    if (tid == 0) { p.out_counts[b] = count; if (!GREEDY) p.last[b] = last; }
  }
  if constexpr (!GREEDY) {
    bool any = false;
#pragma unroll
    for (int x = 0; x < kNodeWords; ++x) any = any || refused[x] != 0;
    const float top = p.top[at + last], cut = p.cut[at + last];
    const double z = p.z[at + last];
    const uint8_t* row = rows + last * p.row_stride * ES;
    const int first = blockIdx.x * p.chunks_per_wg, end = min(first + p.chunks_per_wg, p.chunks);
    for (int chunk = first; chunk < end; ++chunk) {
      const int base = chunk * kChunk;
      __syncthreads();
      if (any && !p.q) {
        for (int i = tid; i < kChunk / 64; i += kWalkThreads) s.skip[i] = 0;
        __syncthreads();
        uint64_t mine = 0;
#pragma unroll
        for (int x = 0; x < kNodeWords; ++x)
          if (x == (tid >> 6)) mine = refused[x];
        if ((mine >> (tid & 63)) & 1ull) {
          const int off = s.token[tid] - base;
          if (off >= 0 && off < kChunk) __hip_atomic_fetch_or(&s.skip[off >> 6], 1ull << (off & 63), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
        __syncthreads();
      }
      double drawn = 0.0, all = 0.0;
#pragma unroll
      for (int k = 0; k < kChunk / kWalkThreads; ++k) {
        const int off = k * kWalkThreads + tid, i = base + off;
        if (i < p.vocab) {
          const float l = load_as_f32(row, i, DT);
          const double w = l >= cut ? logit_weight(l, top, p.c) : 0.0;
          all += w;
          if (any) {
            if (p.q) drawn += fmax(w / z - (double)draft_prob(p, b, last, i), 0.0);
            else if (!((s.skip[off >> 6] >> (off & 63)) & 1ull)) drawn += w;
          }
        }
      }
      drawn = wave_sum(drawn);
      all = wave_sum(all);
      if ((tid & 63) == 0) { s.red[0][tid >> 6] = drawn; s.red[1][tid >> 6] = all; }
      __syncthreads();
      if (tid == 0) {
        double d = 0.0, a = 0.0;
#pragma unroll
        for (int w = 0; w < kWalkWaves; ++w) { d += s.red[0][w]; a += s.red[1][w]; }
        double* out = p.sums + ((int64_t)b * p.chunks + chunk) * 2;
        out[0] = any ? d : a;
        out[1] = a;
      }
    }
  }
}

// One workgroup per row: the token drawn after the last accepted node.
template <int DT>
__global__ __launch_bounds__(kWalkThreads) void draft_draw_kernel(const VerifyParams p) {
  __shared__ double red[kWalkWaves];
  __shared__ double run;                 // weight before the chunk
  __shared__ int where, tail;
  __shared__ uint64_t skip[kChunk / 64];
  constexpr int ES = DT == PA_DTYPE_F32 ? 4 : 2;
  constexpr int PER = kChunk / kWalkThreads;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int last = p.last[b];
  if (last < 0) return;
  const int64_t at = (int64_t)b * p.nodes;
  const int n = nodes_of(p, b);
  const double* sums = p.sums + (int64_t)b * p.chunks * 2;
  // what is left after the refused children, or all that is kept if nothing is
  double mine[2] = {0.0, 0.0};
  for (int i = tid; i < p.chunks; i += kWalkThreads) { mine[0] += sums[2 * i]; mine[1] += sums[2 * i + 1]; }
  const double left = group_sum<kWalkWaves>(mine[0], red);
  const double kept = group_sum<kWalkWaves>(mine[1], red);
  const int side = left > 0.0 ? 0 : 1;
  const double target = (double)p.uniforms[at] * (side == 0 ? left : kept);
  // the first chunk in which the running sum passes the target; the last that holds any weight if none does
  if (tid == 0) { where = p.chunks; tail = 0; }
  __syncthreads();
  double before = 0.0;
  for (int base = 0; base < p.chunks; base += kWalkThreads) {
    const int i = base + tid;
    const double v = i < p.chunks ? sums[2 * i + side] : 0.0;
    const double upto = before + group_scan<kWalkWaves>(v, red);
    if (v > 0.0) {
      atomicMax(&tail, i);
      if (upto > target) atomicMin(&where, i);
    }
    __syncthreads();
    if (where < p.chunks) {
      if (i == where) run = upto - v;
      break;
    }
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < kWalkWaves; ++w) all += red[w];
    before += all;
    __syncthreads();
  }
  __syncthreads();
  const bool crossed = where < p.chunks;
  const int chunk = crossed ? where : tail;
  const int base = chunk * kChunk;
  // children of the last node: refused every one, their tokens are left out
  for (int i = tid; i < kChunk / 64; i += kWalkThreads) skip[i] = 0;
  __syncthreads();
  int up = -1;
  if (tid > 0 && tid < n) {
    up = p.parents ? p.parents[b * p.parents_stride + tid] : tid - 1;
    if (up >= tid) up = -1;
  }
  const bool any = __syncthreads_or(up == last);
  if (up == last && !p.q) {
    const int64_t off = p.tokens[at + tid] - base;
    if (off >= 0 && off < kChunk) __hip_atomic_fetch_or(&skip[off >> 6], 1ull << (off & 63), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  }
  __syncthreads();
  const float top = p.top[at + last], cut = p.cut[at + last];
  const double z = p.z[at + last];
  const uint8_t* row = (const uint8_t*)p.logits + (b * p.batch_stride + last * p.row_stride) * ES;
  // index order: thread t holds entries PER t ... of the chunk
  double w[PER], sum = 0.0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int off = tid * PER + k, i = base + off;
    w[k] = 0.0;
    if (i < p.vocab) {
      const float l = load_as_f32(row, i, DT);
      w[k] = l >= cut ? logit_weight(l, top, p.c) : 0.0;
      if (side == 0 && any) {
        if (p.q) w[k] = fmax(w[k] / z - (double)draft_prob(p, b, last, i), 0.0);
        else if ((skip[off >> 6] >> (off & 63)) & 1ull) w[k] = 0.0;
      }
    }
    sum += w[k];
  }
  if (tid == 0) { where = kChunk; tail = -1; }
  double upto = (crossed ? run : 0.0) + group_scan<kWalkWaves>(sum, red) - sum;
  int hit = kChunk, some = -1;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    upto += w[k];
    if (w[k] > 0.0) {
      some = tid * PER + k;
      if (crossed && upto > target && hit == kChunk) hit = tid * PER + k;
    }
  }
  __syncthreads();
  if (hit < kChunk) atomicMin(&where, hit);
  if (some >= 0) atomicMax(&tail, some);
  __syncthreads();
  if (tid == 0) {
    // rounding left the target at or above the chunk's sum: its last entry with any weight
    const int off = where < kChunk ? where : max(tail, 0);
    p.out_tokens[at + p.out_counts[b] - 1] = min(base + off, p.vocab - 1);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------

static int64_t align_up(int64_t n) { return (n + 255) / 256 * 256; }

struct VerifyLayout {
  int64_t z, top, cut, sums, last, total;
};
static VerifyLayout verify_layout(int64_t batch, int64_t nodes, int64_t vocab) {
  const int64_t rows = batch * nodes, chunks = (vocab + kChunk - 1) / kChunk;
  VerifyLayout l;
  l.z = 0;
  l.top = align_up(rows * 8);
  l.cut = l.top + align_up(rows * 4);
  l.sums = l.cut + align_up(rows * 4);
  l.last = l.sums + align_up(batch * chunks * 16);
  l.total = l.last + align_up(batch * 4);
  return l;
}

template <int DT>
static int launch_verify(const VerifyParams& p, int64_t batch, bool greedy, hipStream_t st) {
  const dim3 rows((unsigned)p.nodes, (unsigned)batch);
  if (greedy) {
    hipLaunchKernelGGL(draft_row_argmax_kernel<DT>, rows, dim3(kStatThreads), 0, st, p);
    hipLaunchKernelGGL((draft_walk_kernel<DT, true>), dim3(1, (unsigned)batch), dim3(kWalkThreads), 0, st, p);
    return check_launch("pa_verify_drafts");
  }
  auto kern = draft_row_stats_kernel<DT>;
  const size_t lds = (DT == PA_DTYPE_F32 ? (size_t)kBins * 8 : (size_t)32768 * 4) + sizeof(StatLds);
  // the attribute belongs to the kernel on one device: once per instantiation and device
  static std::atomic<bool> attr_set[kVerifyMaxDevices];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kVerifyMaxDevices)
    return fail(PA_ERR_LAUNCH, "pa_verify_drafts: cannot tell the current device");
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
      return fail(PA_ERR_LAUNCH, "pa_verify_drafts: cannot raise the dynamic LDS limit");
    attr_set[dev].store(true, std::memory_order_release);
  }
  hipLaunchKernelGGL(kern, rows, dim3(kStatThreads), lds, st, p);
  const unsigned slices = (unsigned)((p.chunks + p.chunks_per_wg - 1) / p.chunks_per_wg);
  hipLaunchKernelGGL((draft_walk_kernel<DT, false>), dim3(slices, (unsigned)batch), dim3(kWalkThreads), 0, st, p);
  hipLaunchKernelGGL(draft_draw_kernel<DT>, dim3((unsigned)batch), dim3(kWalkThreads), 0, st, p);
  return check_launch("pa_verify_drafts");
}

}  // namespace pa

using namespace pa;

extern "C" int64_t pa_verify_workspace_bytes(int64_t batch, int64_t nodes, int64_t vocab) {
  if (batch <= 0 || nodes <= 0 || vocab <= 0) return 0;
  return verify_layout(batch, nodes, vocab).total;
}

extern "C" int pa_verify_drafts(const void* logits, int dtype, int64_t row_stride, int64_t batch_stride,
                                const int64_t* tokens, const float* uniforms, const int32_t* parents,
                                int64_t parents_stride, const int32_t* num_nodes, const void* draft_probs,
                                int draft_dtype, int64_t draft_row_stride, int64_t draft_batch_stride,
                                double temperature, double top_p, int64_t batch, int64_t nodes, int64_t vocab,
                                int64_t* out_tokens, int32_t* out_counts, int32_t* out_path, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  if (batch < 0 || nodes < 0 || vocab <= 0) return fail(PA_ERR_BAD_ARG, "pa_verify_drafts: negative size or no vocabulary");
  if (batch == 0) return PA_OK;
  if (nodes == 0) return fail(PA_ERR_BAD_ARG, "pa_verify_drafts: a row has at least the last accepted token's node");
  if (nodes > PA_MAX_DRAFT_NODES) return fail(PA_ERR_UNSUPPORTED, "pa_verify_drafts: more than 256 nodes a row");
  if (batch > 65535) return fail(PA_ERR_UNSUPPORTED, "pa_verify_drafts: more than 65535 rows in one launch");
  if (vocab > (1 << 24)) return fail(PA_ERR_UNSUPPORTED, "pa_verify_drafts: vocabulary beyond 2^24");
  if (!logits || !tokens || !out_tokens || !out_counts || !out_path) return fail(PA_ERR_BAD_ARG, "pa_verify_drafts: null pointer");
  if (row_stride < vocab || batch_stride < 0) return fail(PA_ERR_BAD_ARG, "pa_verify_drafts: logits stride smaller than the vocabulary");
  if (parents && parents_stride != 0 && parents_stride < nodes)
    return fail(PA_ERR_BAD_ARG, "pa_verify_drafts: parents rows overlap (stride smaller than the nodes of a row)");
  if (!(temperature == temperature)) return fail(PA_ERR_BAD_ARG, "pa_verify_drafts: temperature is not a number");
  const bool greedy = temperature <= 0.0;
  if (!greedy) {
    if (!uniforms) return fail(PA_ERR_BAD_ARG, "pa_verify_drafts: sampling needs one uniform number per node");
    if (!(top_p > 0.0)) return fail(PA_ERR_BAD_ARG, "pa_verify_drafts: top_p must be positive");
    if (!(temperature >= 1e-6 && temperature <= 1e6))
      return fail(PA_ERR_UNSUPPORTED, "pa_verify_drafts: temperature outside 1e-6 ... 1e6");
  }
  if (draft_probs && parents) return fail(PA_ERR_UNSUPPORTED, "pa_verify_drafts: draft probabilities go with chains only");
  if (draft_probs && draft_row_stride < vocab && nodes > 1)
    return fail(PA_ERR_BAD_ARG, "pa_verify_drafts: draft probability rows overlap");
  if (draft_probs && draft_dtype != PA_DTYPE_F16 && draft_dtype != PA_DTYPE_BF16 && draft_dtype != PA_DTYPE_F32)
    return fail(PA_ERR_UNSUPPORTED, "pa_verify_drafts: draft probabilities are f16, bf16 or f32");
  const VerifyLayout l = verify_layout(batch, nodes, vocab);
  if (!workspace || workspace_bytes < l.total) return fail(PA_ERR_WORKSPACE, "pa_verify_drafts: workspace missing or too small");
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return fail(PA_ERR_BAD_ARG, "pa_verify_drafts: workspace must be 256-byte aligned");
  uint8_t* ws = (uint8_t*)workspace;
  VerifyParams p;
  p.logits = logits;
  p.row_stride = row_stride;
  p.batch_stride = batch_stride;
  p.tokens = tokens;
  p.uniforms = uniforms;
  p.parents = parents;
  p.parents_stride = parents_stride;
  p.num_nodes = num_nodes;
  p.q = greedy ? nullptr : draft_probs;
  p.q_row_stride = draft_row_stride;
  p.q_batch_stride = draft_batch_stride;
  p.q_dtype = draft_dtype;
  p.c = greedy ? 0.0 : 1.4426950408889634074 / temperature;
  p.top_p = top_p;
  p.nodes = (int)nodes;
  p.vocab = (int)vocab;
  p.chunks = (int)((vocab + kChunk - 1) / kChunk);
  // about 512 workgroups of the second launch, at least one chunk each
  const int64_t want = (512 + batch - 1) / batch;
  p.chunks_per_wg = (int)((p.chunks + want - 1) / want);
  p.z = (double*)(ws + l.z);
  p.top = (float*)(ws + l.top);
  p.cut = (float*)(ws + l.cut);
  p.sums = (double*)(ws + l.sums);
  p.last = (int32_t*)(ws + l.last);
  p.out_tokens = out_tokens;
  p.out_counts = out_counts;
  p.out_path = out_path;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case PA_DTYPE_F16: return launch_verify<PA_DTYPE_F16>(p, batch, greedy, st);
    case PA_DTYPE_BF16: return launch_verify<PA_DTYPE_BF16>(p, batch, greedy, st);
    case PA_DTYPE_F32: return launch_verify<PA_DTYPE_F32>(p, batch, greedy, st);
    default: return fail(PA_ERR_UNSUPPORTED, "pa_verify_drafts: logits are f16, bf16 or f32");
  }
}

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
// a few hundred LDS reads - and, sampling, the slice's part of the sums the draw needs, per chunk of 512
// entries; (3) the draw, a wave a row: the chunk by a scan of the sums, the token inside it.  Greedy stops after (2).
//
// (1) for 16-bit logits is a histogram, not a pass of exponentials: a row holds at most 65536 different values, a
// few thousand in practice, so the row's entries are counted by bit pattern in LDS (two 16-bit counters to a word: all
// entries of +x or -x, and those of -x) and exp runs three times per 16 neighbouring patterns that occur, whose weights are
// geometric sequences, times the counts, in 64 bits.  The same counts, summed in descending order, give the top-p
// threshold, so a row leaves HBM once whatever top_p is.  A 16-bit counter that overflows (more than 65535 equal logits)
// shows in the total of all counters; such rows, and 32-bit logits, take a search over ordered bit patterns instead, 11
// bits a pass.  Short rows of which top_p keeps all are summed entry by entry.
//
// One row of 152k 16-bit logits takes (1) 19.5 us: 8 us of LDS atomics, 5 us to get at the row and clear the counters, 5 us of
// masses.  64 rows of a chain of 5 with draft probabilities: 22 + 21 + 6 us, 16 rows of a tree of 64: 94 (3.3 TB/s) + 11 + 6 us;
// 5 rows of 32-bit logits: 105 to 150 us the whole call with top_p 0.9, the broader the rows the more exponentials, 49 without;
// greedy 23 (5 rows of fp16) and 80 (16 rows of 64 nodes, bf16, 4.5 TB/s).
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
constexpr int kChunk = 512;                     // vocabulary entries behind one pair of stored sums: a wave's, 8 a lane
constexpr int kNodeWords = PA_MAX_DRAFT_NODES / 64;
constexpr int kBins = 2048;                     // bins of one pass of the search
constexpr int kVerifyMaxDevices = 64;
constexpr int kSumVocab = 16384;                // 16-bit rows up to here are summed entry by entry where top_p keeps all

typedef short i16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

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
  int nodes, vocab, chunks, slices;             // slices: workgroups of the second launch per row
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

// 2^x for x <= 0 to 2^-51: x = n + f with |f| <= 1/2, the series of e^(f ln 2) to the 12th power (its rest is below
// (ln 2 / 2)^13 / 13! = 2^-52.2) and the exponent added.  0 for NaN and -inf, by the clamp.  Half the instructions of the library's exp2, which
// also takes every other argument; the row statistics and the sums of the draw are bound by them.
__device__ __forceinline__ double exp2_down(double x) {
  // (ln 2)^k / k!, held in scalar registers: as literals each costs two moves into the accumulator of its multiply-add
  double c12 = 2.5678435993488196e-11;
  double c11 = 4.44553827187081e-10;
  double c10 = 7.054911620801121e-09;
  double c9 = 1.0178086009239696e-07;
  double c8 = 1.3215486790144305e-06;
  double c7 = 1.5252733804059838e-05;
  double c6 = 0.00015403530393381606;
  double c5 = 0.0013333558146428441;
  double c4 = 0.009618129107628477;
  double c3 = 0.055504108664821576;
  double c2 = 0.2402265069591007;
  double c1 = 0.6931471805599453;
  asm("" : "+s"(c12), "+s"(c11), "+s"(c10), "+s"(c9), "+s"(c8), "+s"(c7));
  asm("" : "+s"(c6), "+s"(c5), "+s"(c4), "+s"(c3), "+s"(c2), "+s"(c1));
  x = fmax(x, -2000.0);
  const double n = __builtin_rint(x), f = x - n;
  double r = fma(c12, f, c11);
  r = fma(r, f, c10);
  r = fma(r, f, c9);
  r = fma(r, f, c8);
  r = fma(r, f, c7);
  r = fma(r, f, c6);
  r = fma(r, f, c5);
  r = fma(r, f, c4);
  r = fma(r, f, c3);
  r = fma(r, f, c2);
  r = fma(r, f, c1);
  r = fma(r, f, 1.0);
  return __builtin_amdgcn_ldexp(r, (int)n);
}

// w of one logit of a row with a finite maximum; NaN and -inf weigh nothing
__device__ __forceinline__ double finite_weight(float l, double top, double c) { return exp2_down(((double)l - top) * c); }

// The same for any maximum: under an infinite one everything else weighs nothing.
__device__ __forceinline__ double logit_weight(float l, float top, double c) {
  return l == top ? (l > -INFINITY ? 1.0 : 0.0) : finite_weight(l, top, c);
}

// One lane's value in every lane.
__device__ __forceinline__ double wave_at(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)u, lane), hi = __builtin_amdgcn_readlane((uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

__device__ __forceinline__ double wave_sum(double v) { return wave_at(wave_scan(v), 63); }

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
  v = wave_scan(v);
  __syncthreads();
  if (lane == 63) red[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v += red[w];
  return v;
}

struct StatLds {
  double seg[128];             // masses of 512 neighbouring values, in descending order of the values
  double red[kStatWaves];
  double found[2];             // the crossing: mass above it, kept mass
  uint32_t key[2];             // its place
  uint32_t redu[3][kStatWaves];
};

struct RowStats {
  double z;
  float top, cut;
};

// Row statistics without the histogram: maximum, the sum of all weights and, where top_p < 1, the smallest kept
// logit by a search over ordered bit patterns: the range that holds it is cut into 2048 bins, the weights of the
// range's entries are added up per bin as 64-bit fixed-point numbers (exact, so the order of the atomics does not
// matter), and the bin in which the mass above crosses top_p * z is the next range.  The first range starts below the
// smallest weight that can be kept: tokens lighter than (1 - top_p) z / vocab weigh less than 1 - top_p together, and
// z >= 1.  The first of the 3 passes (32-bit logits) adds up z as well; the later ones need an exponential per entry
// in range only.  Bound by the exponentials, a row to a CU.
// A bin counts in units of its own, 2^-(62 - log2 vocab) of a power of two above its largest weight, so that `vocab` entries
// of it fit and yet each is held to 2^-45 of the bin's largest for 152k entries, to 2^-38 for 2^24.  Units of the row's
// largest weight would round many equal small ones all the same way: of 4 million of 2^-40 each would weigh twice what it
// does, visible to a 24-bit uniform number.  5 rows of 152k entries take 150 us with the bins' units, 143 with the row's; the
// kept weights summed as 64-bit floats in the last pass instead took 206.
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
  if (best == INFINITY) {
    for_each_logit<DT, kStatThreads>(ptr, p.vocab, [&](int, float x) __attribute__((always_inline)) { mine += x == INFINITY ? 1.0 : 0.0; });
    r.z = group_sum<kStatWaves>(mine, s.red);
    return r;
  }
  if (!(p.top_p < 1.0)) {
    for_each_logit<DT, kStatThreads>(ptr, p.vocab, [&](int, float x) __attribute__((always_inline)) { mine += finite_weight(x, best, p.c); });
    r.z = group_sum<kStatWaves>(mine, s.red);
    return r;
  }
  const int log_vocab = 32 - __builtin_clz((uint32_t)p.vocab);
  const float c = (float)p.c;
  const int bits = min(62 - log_vocab, 51);
  const float low = (float)((double)best + log2((1.0 - p.top_p) / p.vocab * 0.5) / p.c);
  uint32_t lo = ordered_key32(low < best ? low : best), hi = ordered_key32(r.top);
  double above = 0.0, limit = 0.0;
  for (bool first = true;; first = false) {
    const uint32_t span = hi - lo;
    const int shift = span < kBins ? 0 : 21 - __builtin_clz(span);       // span >> shift < 2048
    // fraction bits of the bin that `off` is in: a bound of its weights from its largest value, in 32 bits, the same for all of it
    const uint32_t rest = (1u << shift) - 1;
    auto fraction = [&](uint32_t off) __attribute__((always_inline)) {
      const uint32_t k = lo + min(off | rest, span);
      const float largest = __uint_as_float(k ^ (~(uint32_t)((int32_t)k >> 31) | 0x80000000u));
      return bits - (int)__builtin_amdgcn_fmed3f(ceilf((largest - best) * c), -900.0f, 0.0f);
    };
    for (int i = tid; i < kBins; i += kStatThreads) bins[i] = 0;
    __syncthreads();
    for_each_logit<DT, kStatThreads>(ptr, p.vocab, [&](int, float x) __attribute__((always_inline)) {
      const uint32_t off = ordered_key32(x + 0.0f) - lo;                   // -0 counts as +0; NaN lies beyond every finite key
      if (!first && off > span) return;
      const double w = finite_weight(x, best, p.c);
      if (first) mine += w;
      if (off <= span) {                                                   // to a whole number in the low bits of 2^52 + it
        const uint64_t n = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ldexp(w, fraction(off)) + 0x1p52) & 0xfffffffffffffull;
        __hip_atomic_fetch_add(&bins[off >> shift], n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
    });
    if (first) {
      r.z = group_sum<kStatWaves>(mine, s.red);
      limit = p.top_p * r.z;
    }
    __syncthreads();
    // bins from the top: thread t takes bins 2047 - 2t and 2046 - 2t
    auto mass = [&](uint32_t i) __attribute__((always_inline)) { return __builtin_amdgcn_ldexp((double)bins[i], -fraction(i << shift)); };
    const double m0 = mass(kBins - 1 - 2 * tid), m1 = mass(kBins - 2 - 2 * tid);
    const double upto = above + group_scan<kStatWaves>(m0 + m1, s.red), before = upto - (m0 + m1);
    if (tid == 0) s.key[0] = kBins;
    if (tid == kStatThreads - 1) s.found[0] = upto;
    __syncthreads();
    const double total = s.found[0];
    if (upto > limit) __hip_atomic_fetch_min(&s.key[0], (uint32_t)tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    __syncthreads();
    const uint32_t crossing = s.key[0];                                     // the first thread past the limit
    if (crossing == kBins) {             // rounding left the total at the limit: the whole range is kept
      r.z = total;
      r.cut = key_value32(lo);
      break;
    }
    if ((uint32_t)tid == crossing) {
      const bool second = before + m0 <= limit;
      s.key[1] = kBins - 1 - 2 * tid - (second ? 1 : 0);
      s.found[0] = second ? before + m0 : before;
      s.found[1] = second ? upto : before + m0;
    }
    __syncthreads();
    const uint32_t bin = s.key[1];
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

// One workgroup per node.  16-bit logits: LDS holds 32768 words, the entries of bit pattern m in the low half of word m, those
// of -m (the same with the sign bit) counted in the high half and in the low half too; then StatLds.  Without COUNTS (32-bit
// logits, short rows that top_p leaves whole): the bins of the search, then StatLds.
template <int DT, bool COUNTS>
__global__ __launch_bounds__(kStatThreads) void draft_row_stats_kernel(const VerifyParams p) {
  extern __shared__ __align__(16) uint8_t lds_raw[];
  const int node = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (node >= nodes_of(p, b)) return;
  static_assert(!COUNTS || DT != PA_DTYPE_F32, "32-bit patterns are too many to count");
  constexpr int WORDS = 32768;
  constexpr int INF = DT == PA_DTYPE_F16 ? 0x7c00 : 0x7f80;
  uint32_t* hist = (uint32_t*)lds_raw;
  StatLds& s = *(StatLds*)(lds_raw + (COUNTS ? WORDS * 4 : kBins * 8));
  const void* ptr = (const uint8_t*)p.logits + (b * p.batch_stride + node * p.row_stride) * (DT == PA_DTYPE_F32 ? 4 : 2);
  const int64_t at = (int64_t)b * p.nodes + node;
  if constexpr (COUNTS) {
    // 2374 atomics a wave and 64 entries for 152k logits, about 8 clocks each at the LDS whatever their addresses: 8 us a row.
    // In their shadow the largest pattern as a signed number (the maximum, if it is positive) and the smallest as an
    // unsigned one (the maximum's pattern if all are negative).
    auto add = [&](uint32_t byte, uint32_t inc) __attribute__((always_inline)) {
      __hip_atomic_fetch_add((uint32_t*)__builtin_assume_aligned(lds_raw + byte, 4), inc, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    };
    i16x2_t most = {-32768, -32768};
    u16x2_t least = {65535, 65535};
    auto note = [&](uint32_t w) __attribute__((always_inline)) {
      most = __builtin_elementwise_max(most, __builtin_bit_cast(i16x2_t, w));
      least = __builtin_elementwise_min(least, __builtin_bit_cast(u16x2_t, w));
    };
    for_each_logit_pair<DT, kStatThreads, 8>(
        ptr, p.vocab,
        [&](uint32_t w) __attribute__((always_inline)) {
          add((w << 2) & 0x1fffcu, ((w & 0x8000u) << 1) | 1u);
          add((w >> 14) & 0x1fffcu, ((w >> 15) & 0x10000u) | 1u);
          note(w);
        },
        [&](uint32_t h) __attribute__((always_inline)) {
          add((h << 2) & 0x1fffcu, ((h & 0x8000u) << 1) | 1u);
          note(h | h << 16);
        },
        [&]() __attribute__((always_inline)) {       // while the first pieces are on their way
          for (int i = tid; i < WORDS / 4; i += kStatThreads) ((uint4*)hist)[i] = make_uint4(0, 0, 0, 0);
          __syncthreads();
        });
    int high = max(most[0], most[1]);
    uint32_t low = min(least[0], least[1]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      high = max(high, __shfl_xor(high, o));
      low = min(low, (uint32_t)__shfl_xor(low, o));
    }
    if (lane == 0) { s.redu[0][wave] = (uint32_t)high; s.redu[1][wave] = low; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kStatWaves; ++w) {
      high = max(high, (int)s.redu[0][w]);
      low = min(low, s.redu[1][w]);
    }
    if (high < 0 && low == 0x8000u) high = 0;                // -0 and +0 are one value
    if (high < 0 && low >= 0x8000u + INF) {                  // all -inf or NaN of that sign: nothing weighs anything
      if (tid == 0) { p.z[at] = 0.0; p.top[at] = p.cut[at] = -INFINITY; }
      return;
    }
    // A positive NaN hides the maximum, an infinite one makes every other weight 0: both are left to the search.
    if (high < INF) {
      // A wave takes blocks of 512 neighbouring m (wave, 16 + wave, ...), 8 consecutive ones a lane.  Most blocks are empty
      // and cost a read and a test.
      constexpr int BLOCKS = WORDS / 512, MINE = BLOCKS / kStatWaves;
      auto words = [&](int m0, uint32_t (&v)[8]) __attribute__((always_inline)) {
        const uint4 x = ((const uint4*)hist)[m0 / 4], y = ((const uint4*)hist)[m0 / 4 + 1];
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
      };
      // entries of +m and of -m that weigh anything
      auto weighing = [&](uint32_t word, int m, uint32_t& plus, uint32_t& minus) __attribute__((always_inline)) {
        minus = word >> 16;
        plus = (word & 0xffffu) - minus;
        if (m == 0) { plus += minus; minus = 0; }            // -0 and +0 are one value
        if (m >= INF) minus = 0;                             // -inf
        if (m > INF) plus = 0;                               // NaN
      };
      auto value = [](int m) { return logit_value<DT>(m); };
      const int top_up = high, top_down = high >= 0 ? 0 : (int)(low & 0x7fffu);        // top_up -1 or less: no positive value
      const float top = high >= 0 ? value(high) : -value(top_down);
      // Masses of a lane's 8 values of one sign, largest value first.  They are evenly spaced (a binade has 128 values or
      // more), so their weights are a geometric sequence from that of the largest one not above the maximum.
      auto masses_up = [&](int m0, double (&mass)[8]) __attribute__((always_inline)) {
        uint32_t w8[8];
        words(m0, w8);
        const double fall = exp2_down(-(double)(value(m0 + 1) - value(m0)) * p.c);
        double w = logit_weight(value(min(m0 + 7, max(top_up, 0))), top, p.c);
#pragma unroll
        for (int j = 7; j >= 0; --j) {
          uint32_t plus, minus;
          weighing(w8[j], m0 + j, plus, minus);
          const bool real = m0 + j <= top_up && m0 < INF;
          mass[7 - j] = real ? plus * w : 0.0;
          w = real ? w * fall : w;
        }
      };
      auto masses_down = [&](int m0, double (&mass)[8]) __attribute__((always_inline)) {
        uint32_t w8[8];
        words(m0, w8);
        const double fall = exp2_down(-(double)(value(m0 + 1) - value(m0)) * p.c);
        double w = logit_weight(-value(max(m0, top_down)), top, p.c);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t plus, minus;
          weighing(w8[j], m0 + j, plus, minus);
          const bool real = m0 + j >= top_down && m0 < INF;
          mass[j] = real ? minus * w : 0.0;
          w = real ? w * fall : w;
        }
      };
      auto sum8 = [](const double (&x)[8]) { return ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7])); };
      // block g's mass of positive values to seg[63 - g], of negative ones to seg[64 + g]: descending order of the values
      uint32_t count = 0;
#pragma unroll
      for (int k = 0; k < MINE; ++k) {
        const int g = wave + kStatWaves * k, m0 = g * 512 + lane * 8;
        double up = 0.0, down = 0.0;
        uint32_t v[8], any = 0;
        words(m0, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          any |= v[j];
          count += v[j] & 0xffffu;
        }
        if (__builtin_amdgcn_ballot_w64(any != 0) != 0) {
          if (g > 0 && g < INF / 512 && top_down <= g * 512 && (top_up < g * 512 || top_up >= g * 512 + 511)) {
            // neither zero nor infinity nor the maximum inside: the polynomials in `fall`, nothing to leave out
            const double fall = exp2_down(-(double)(value(m0 + 1) - value(m0)) * p.c);
            double a = 0.0, d = 0.0;
#pragma unroll
            for (int j = 0; j < 8; ++j) a = fma(a, fall, (double)((v[j] & 0xffffu) - (v[j] >> 16)));
#pragma unroll
            for (int j = 7; j >= 0; --j) d = fma(d, fall, (double)(v[j] >> 16));
            // above the maximum there is nothing to weigh
            up = top_up < g * 512 ? 0.0 : a * exp2_down(((double)value(m0 + 7) - (double)top) * p.c);
            down = d * exp2_down((-(double)value(m0) - (double)top) * p.c);
          } else {
            double mass[8];
            masses_up(m0, mass);
            up = sum8(mass);
            masses_down(m0, mass);
            down = sum8(mass);
          }
          up = wave_scan(up);
          down = wave_scan(down);
        }
        if (lane == 63) { s.seg[BLOCKS - 1 - g] = up; s.seg[BLOCKS + g] = down; }
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) count += __shfl_xor(count, o);
      if (lane == 0) s.redu[2][wave] = count;
      __syncthreads();
      count = 0;
#pragma unroll
      for (int w = 0; w < kStatWaves; ++w) count += s.redu[2][w];
      // a counter that wrapped shows in the total
      if (count == (uint32_t)p.vocab) {
        // every wave: the block past which the mass exceeds top_p of all
        const double first = s.seg[2 * lane], second = s.seg[2 * lane + 1];
        const double upto = wave_scan(first + second);
        const double z = wave_at(upto, 63), limit = p.top_p * z;
        const unsigned long long past = p.top_p < 1.0 ? __builtin_amdgcn_ballot_w64(upto > limit) : 0;
        if (!past) {                                         // everything stays
          if (tid == 0) { p.z[at] = z; p.top[at] = top; p.cut[at] = -INFINITY; }
          return;
        }
        const int l = __builtin_ctzll(past);
        double above = wave_at(upto, l) - wave_at(first, l) - wave_at(second, l);
        int o = 2 * l;
        if (above + wave_at(first, l) <= limit) { above += wave_at(first, l); ++o; }
        const bool positive = o < BLOCKS;
        const int g = positive ? BLOCKS - 1 - o : o - BLOCKS;
        if (g % kStatWaves != wave) return;
        // the wave that holds the block: its masses in descending order, lanes from 63 down for positive values
        double mass[8];
        const int m0 = g * 512 + lane * 8;
        if (positive) masses_up(m0, mass);
        else masses_down(m0, mass);
        const double own = sum8(mass), scan = wave_scan(own);
        double run = above + (positive ? wave_at(scan, 63) - scan : scan - own);       // mass above this lane's values
        int cross = 8, some = -1;
        double kept = 0.0, kept_some = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          run += mass[j];
          if (mass[j] > 0.0) {
            some = j;
            kept_some = run;
            if (cross == 8 && run > limit) { cross = j; kept = run; }
          }
        }
        const unsigned long long hit = __builtin_amdgcn_ballot_w64(cross < 8), any = __builtin_amdgcn_ballot_w64(some >= 0);
        // the first value past the limit; where rounding leaves none, the block's last
        const int who = hit ? (positive ? 63 - __builtin_clzll(hit) : __builtin_ctzll(hit))
                            : (positive ? __builtin_ctzll(any | 1ull << 63) : 63 - __builtin_clzll(any | 1ull));
        if (lane == who) {
          const int j = hit ? cross : max(some, 0);
          p.z[at] = hit ? kept : some >= 0 ? kept_some : run;
          p.top[at] = top;
          p.cut[at] = positive ? value(m0 + 7 - j) : -value(m0 + j);
        }
        return;
      }
    }
  }
  __syncthreads();
  const RowStats r = search_row<DT>(ptr, p, (uint64_t*)lds_raw, s);
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
    // without a maximum above -inf: a NaN before the first -inf counts as one, too
    p.cut[(int64_t)b * p.nodes + node] = __int_as_float(best > -INFINITY ? best_i : 0);
  }
}

struct WalkLds {
  double z[PA_MAX_DRAFT_NODES];      // the nodes' row statistics
  float top[PA_MAX_DRAFT_NODES];
  float cut[PA_MAX_DRAFT_NODES];
  double w[PA_MAX_DRAFT_NODES];      // the node's weight in its parent's row; drafts drawn from q: its weight / q
  int parent[PA_MAX_DRAFT_NODES];
  int token[PA_MAX_DRAFT_NODES];
  float u[PA_MAX_DRAFT_NODES];
  int path[PA_MAX_DRAFT_NODES];
};

// Entries i0 ... i0 + 7 of a row as floats (beyond its end: `beyond`), in 16-byte loads where they are aligned.
__device__ __forceinline__ void load_entries(const void* row, int dtype, int i0, int vocab, float beyond, float (&x)[8]) {
  const int es = dtype == PA_DTYPE_F32 ? 4 : 2;
  if (i0 >= vocab) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = beyond;
  } else if (i0 + 8 <= vocab && ((reinterpret_cast<uintptr_t>(row) + (uintptr_t)i0 * es) & 15u) == 0) {
    load8_as_f32(row, i0, dtype, x);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = i0 + e < vocab ? load_as_f32(row, i0 + e, dtype) : beyond;
  }
}

// The weights with which the token after node `last` is drawn, of 8 entries of logits l, and all kept weights.
// drop: bit e leaves entry e out (a refused child's token).  from_q: drafts drawn from q were refused; inv_z: 1 / z then.
__device__ __forceinline__ void draw_weights(const VerifyParams& p, float (&l)[8], const float (&q)[8], bool from_q, float top,
                                             float cut, double inv_z, uint32_t drop, double (&drawn)[8], double (&all)[8]) {
  if (__builtin_expect(top == INFINITY, 0)) {              // such a row keeps all of its infinities
#pragma unroll
    for (int e = 0; e < 8; ++e) l[e] = l[e] == INFINITY ? 0.0f : -INFINITY;
    top = 0.0f;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    all[e] = 0.0;
    // with top_p few entries are kept, and in most places none of a wave's: 11 us against 12 for 16 rows of 152k
    if (__builtin_amdgcn_ballot_w64(l[e] >= cut) != 0) all[e] = finite_weight(l[e] >= cut ? l[e] : -INFINITY, top, p.c);
    if (from_q) drawn[e] = fmax(fma(all[e], inv_z, -(double)q[e]), 0.0);
    else drawn[e] = (drop >> e) & 1u ? 0.0 : all[e];
  }
}

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
    const double z = GREEDY ? 0.0 : s.z[cur];
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
        left = fmax(left - wj, 0.0);         // rounding must not leave a negative rest, which any u would pass under
      }
    }
    if (next < 0) return cur;
    if (threadIdx.x == 0) s.path[count] = next;
    ++count;
    cur = next;
  }
}

__device__ __forceinline__ const void* draft_probs_row(const VerifyParams& p, int b, int node) {
  return (const uint8_t*)p.q + (b * p.q_batch_stride + node * p.q_row_stride) * (p.q_dtype == PA_DTYPE_F32 ? 4 : 2);
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
    if (i < n) {
      if (!GREEDY) { s.z[i] = p.z[at + i]; s.top[i] = p.top[at + i]; }
      s.cut[i] = p.cut[at + i];
    }
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
            const double qv = load_as_f32(draft_probs_row(p, b, up), tok, p.q_dtype);
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
      else if (GREEDY) p.out_tokens[at + i] = __float_as_int(s.cut[last]);
    }
    if (tid == 0) { p.out_counts[b] = count; if (!GREEDY) p.last[b] = last; }
  }
  if constexpr (!GREEDY) {
    const int lane = tid & 63;
    bool any = false;
    int gone[kNodeWords];                    // this lane's refused children of the last node: their tokens
#pragma unroll
    for (int x = 0; x < kNodeWords; ++x) {
      any = any || refused[x] != 0;
      gone[x] = (refused[x] >> lane) & 1ull ? s.token[64 * x + lane] : -1;
    }
    const float top = s.top[last], cut = s.cut[last];
    const void* row = rows + last * p.row_stride * ES;
    const void* q_row = any && p.q ? draft_probs_row(p, b, last) : nullptr;
    const double inv_z = q_row ? 1.0 / s.z[last] : 0.0;
    // a wave takes chunks of 512 entries by itself, 8 consecutive ones a lane, the next chunk's on their way
    const int waves = gridDim.x * kWalkWaves;
    float l[8], q[8] = {};
    auto load = [&](int chunk) __attribute__((always_inline)) {
      const int i0 = chunk < p.chunks ? chunk * kChunk + lane * 8 : p.vocab;
      load_entries(row, DT, i0, p.vocab, -INFINITY, l);
      if (q_row) load_entries(q_row, p.q_dtype, i0, p.vocab, 0.0f, q);
    };
    int chunk = blockIdx.x * kWalkWaves + (tid >> 6);
    load(chunk);
    for (; chunk < p.chunks; chunk += waves) {
      const int base = chunk * kChunk;
      uint32_t drop = 0;
      if (any && !p.q) {
#pragma unroll
        for (int x = 0; x < kNodeWords; ++x) {
          unsigned long long here = __builtin_amdgcn_ballot_w64(gone[x] >= base && gone[x] < base + kChunk);
          while (here) {
            const int off = __builtin_amdgcn_readlane(gone[x], __builtin_ctzll(here)) - base;
            here &= here - 1;
            if ((off >> 3) == lane) drop |= 1u << (off & 7);
          }
        }
      }
      float l_now[8], q_now[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) { l_now[e] = l[e]; q_now[e] = q[e]; }
      load(chunk + waves);
      double d = 0.0, a = 0.0, drawn[8], all[8];
      draw_weights(p, l_now, q_now, q_row != nullptr, top, cut, inv_z, drop, drawn, all);
#pragma unroll
      for (int e = 0; e < 8; ++e) { d += drawn[e]; a += all[e]; }
      d = wave_sum(d);
      a = wave_sum(a);
      if (lane == 0) {
        double* out = p.sums + ((int64_t)b * p.chunks + chunk) * 2;
        out[0] = d;
        out[1] = a;
      }
    }
  }
}

// One wave per row: the token drawn after the last accepted node.
template <int DT>
__global__ __launch_bounds__(64) void draft_draw_kernel(const VerifyParams p) {
  constexpr int ES = DT == PA_DTYPE_F32 ? 4 : 2;
  const int b = blockIdx.x, lane = threadIdx.x;
  const int64_t at = (int64_t)b * p.nodes;
  const int last = p.last[b], count = p.out_counts[b];
  if (last < 0) return;
  const int n = nodes_of(p, b);
  const float top = p.top[at + last], cut = p.cut[at + last];
  const double z = p.z[at + last], u = (double)p.uniforms[at];
  const double2* sums = (const double2*)(p.sums + (int64_t)b * p.chunks * 2);
  // what is left after the refused children, or all that is kept if nothing is: lane l adds up chunks l * per ...
  const int per = (p.chunks + 63) / 64;
  double left = 0.0, kept = 0.0;
  for (int i = lane * per; i < min((lane + 1) * per, p.chunks); ++i) {
    const double2 v = sums[i];
    left += v.x;
    kept += v.y;
  }
  const double left_to = wave_scan(left), kept_to = wave_scan(kept);
  const double left_all = wave_at(left_to, 63);
  const bool rest = left_all > 0.0;
  const double target = u * (rest ? left_all : wave_at(kept_to, 63));
  const double mine = rest ? left : kept, to = rest ? left_to : kept_to;
  // the first chunk in which the running sum passes the target; by rounding none: the last that holds any weight
  const unsigned long long some = __builtin_amdgcn_ballot_w64(mine > 0.0);
  unsigned long long hit = __builtin_amdgcn_ballot_w64(mine > 0.0 && to > target);
  if (!some) {                               // nothing at all (a row without a finite logit): the first token
    if (lane == 0) p.out_tokens[at + count - 1] = 0;
    return;
  }
  const int owner = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some);
  double run = wave_at(to, owner) - wave_at(mine, owner);      // weight before the chunk
  int chunk = -1, tail = owner * per;
  double before = run;
  for (int i0 = owner * per; i0 < min((owner + 1) * per, p.chunks) && chunk < 0; i0 += 64) {
    const int i = i0 + lane;
    double m = 0.0;
    if (i < min((owner + 1) * per, p.chunks)) m = rest ? sums[i].x : sums[i].y;
    const double upto = before + wave_scan(m);
    const unsigned long long weight = __builtin_amdgcn_ballot_w64(m > 0.0);
    const unsigned long long past = __builtin_amdgcn_ballot_w64(m > 0.0 && upto > target);
    if (past || weight) {
      const int l = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(weight);
      run = wave_at(upto, l) - wave_at(m, l);
      tail = i0 + l;
      if (past) chunk = tail;
    }
    before = wave_at(upto, 63);
  }
  if (chunk < 0) chunk = tail;
  // inside the chunk: lane l holds entries 8 l ... of it
  const int base = chunk * kChunk;
  uint32_t drop = 0;
  bool any = false;
  for (int c0 = 0; c0 < n; c0 += 64) {
    const int c = c0 + lane;
    int gone = -1;
    if (c > 0 && c < n) {
      const int up = p.parents ? p.parents[b * p.parents_stride + c] : c - 1;
      if (up == last) {                      // < c: `last` is one of the row's nodes, and a parent past the node is none
        any = any || last < c;
        const int64_t t = p.tokens[at + c];
        if (last < c && t >= base && t < base + kChunk) gone = (int)t - base;
      }
    }
    unsigned long long here = __builtin_amdgcn_ballot_w64(gone >= 0);
    while (here) {
      const int off = __builtin_amdgcn_readlane(gone, __builtin_ctzll(here));
      here &= here - 1;
      if ((off >> 3) == lane) drop |= 1u << (off & 7);
    }
  }
  any = __builtin_amdgcn_ballot_w64(any) != 0;
  const void* row = (const uint8_t*)p.logits + (b * p.batch_stride + last * p.row_stride) * ES;
  const void* q_row = any && p.q ? draft_probs_row(p, b, last) : nullptr;
  double drawn[8], all[8], sum = 0.0;
  const int i0 = base + lane * 8;
  float l[8], q[8] = {};
  load_entries(row, DT, i0, p.vocab, -INFINITY, l);
  if (q_row) load_entries(q_row, p.q_dtype, i0, p.vocab, 0.0f, q);
  draw_weights(p, l, q, q_row != nullptr, top, cut, q_row ? 1.0 / z : 0.0, drop, drawn, all);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    drawn[e] = rest ? drawn[e] : all[e];
    sum += drawn[e];
  }
  double upto = run + (wave_scan(sum) - sum);
  int first = 8, final = -1;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    upto += drawn[e];
    if (drawn[e] > 0.0) {
      final = e;
      if (upto > target && first == 8) first = e;
    }
  }
  hit = __builtin_amdgcn_ballot_w64(first < 8);
  const unsigned long long any_weight = __builtin_amdgcn_ballot_w64(final >= 0);
  // rounding left the target at or above the chunk's sum: its last entry with any weight
  const int from = hit ? __builtin_ctzll(hit) : any_weight ? 63 - __builtin_clzll(any_weight) : 0;
  const int off = from * 8 + max(__builtin_amdgcn_readlane(hit ? first : final, from), 0);
  if (lane == 0) p.out_tokens[at + count - 1] = min(base + off, p.vocab - 1);
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
  // Clearing and reading 128 KiB of counters takes 7 us a row: not for a short row of which only the sum is wanted (the whole
  // call, 16 rows of 64 nodes: 33 us with 8000 entries each, 46 with counters; 71 and 55 with 32000).
  const bool counts = DT != PA_DTYPE_F32 && !(p.top_p >= 1.0 && p.vocab <= kSumVocab);
  auto kern = counts ? draft_row_stats_kernel<DT, DT != PA_DTYPE_F32> : draft_row_stats_kernel<DT, false>;
  const size_t lds = (counts ? (size_t)32768 * 4 : (size_t)kBins * 8) + sizeof(StatLds);
  // the attribute belongs to the kernel on one device: once per instantiation and device
  static std::atomic<bool> attr_sets[2][kVerifyMaxDevices];
  auto& attr_set = attr_sets[counts];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kVerifyMaxDevices)
    return fail(PA_ERR_LAUNCH, "pa_verify_drafts: cannot tell the current device");
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
      return fail(PA_ERR_LAUNCH, "pa_verify_drafts: cannot raise the dynamic LDS limit");
    attr_set[dev].store(true, std::memory_order_release);
  }
  hipLaunchKernelGGL(kern, rows, dim3(kStatThreads), lds, st, p);
  hipLaunchKernelGGL((draft_walk_kernel<DT, false>), dim3((unsigned)p.slices, (unsigned)batch), dim3(kWalkThreads), 0, st, p);
  hipLaunchKernelGGL(draft_draw_kernel<DT>, dim3((unsigned)batch), dim3(64), 0, st, p);
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
  // A wave's chunks are a long chain of loads, exponentials and sums: as many workgroups as the GPU holds at once, six a CU, though
  // each of a row repeats its walk.  The whole call with 1536, 768 and 512 of them, rows of 152k entries: 64 chains of 5 with draft
  // probabilities 48, 51 and 56 us; 64 trees of 8 nodes 75, 78 and 82; 16 trees of 64 nodes 113, 113 and 114.
  const int64_t want = (1536 + batch - 1) / batch, most = (p.chunks + kWalkWaves - 1) / kWalkWaves;
  p.slices = (int)(want < most ? want : most);
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

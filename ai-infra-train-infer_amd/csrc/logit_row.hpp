// Walking a row of logits with one workgroup.
#pragma once

#include "pa_common.hpp"

namespace pa {

// fp32 -> unsigned key with the same order (no NaN), and back
__device__ __forceinline__ uint32_t ordered_key32(float f) {
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value32(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}

template <int DT>
__device__ __forceinline__ float logit_value(uint32_t bits) {
  if constexpr (DT == PA_DTYPE_F32) return __uint_as_float(bits);
  else if constexpr (DT == PA_DTYPE_F16) return f16_bits_to_f32(bits);
  else return bf16_bits_to_f32(bits);
}

// The row's entries in 16-byte pieces, the workgroup's THREADS threads taking pieces in turn with UNROLL in flight each and as
// many asked for ahead of them; the entries before the first 16-byte boundary and after the last one by themselves (rows of an
// odd vocabulary start anywhere).  piece(first index, its 4 words), one(index); first(): called once by every thread after its
// first pieces have been asked for and before anything else.
template <int ES, int THREADS, int UNROLL, class Piece, class One, class First>
__device__ __forceinline__ void walk_row(const void* row, int vocab, Piece&& piece, One&& one, First&& first) {
  constexpr int PER = 16 / ES;
  const int head = min((int)((16u - (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / ES, vocab);
  const uint4* wide = (const uint4*)((const uint8_t*)row + head * ES);
  const int pieces = (vocab - head) / PER;
  uint4 w[UNROLL], next[UNROLL];
  auto ask = [&](int c, uint4 (&to)[UNROLL]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) to[u] = c + u * THREADS < pieces ? wide[c + u * THREADS] : make_uint4(0, 0, 0, 0);
  };
  int c = threadIdx.x;
  ask(c, w);
  first();
  for (; c < pieces; c += UNROLL * THREADS) {
    ask(c + UNROLL * THREADS, next);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
      if (c + u * THREADS < pieces) piece(head + (c + u * THREADS) * PER, w[u]);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) w[u] = next[u];
  }
  for (int i = threadIdx.x; i < head; i += THREADS) one(i);
  for (int i = head + pieces * PER + threadIdx.x; i < vocab; i += THREADS) one(i);
}

// f(index, value) for every entry of the row
template <int DT, int THREADS, class F>
__device__ __forceinline__ void for_each_logit(const void* row, int vocab, F&& f) {
  walk_row<DT == PA_DTYPE_F32 ? 4 : 2, THREADS, 4>(
      row, vocab,
      [&](int i, const uint4& v) __attribute__((always_inline)) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (DT == PA_DTYPE_F32) {
            f(i + k, logit_value<DT>(w[k]));
          } else {
            f(i + 2 * k, logit_value<DT>(w[k] & 0xffffu));
            f(i + 2 * k + 1, logit_value<DT>(w[k] >> 16));
          }
        }
      },
      [&](int i) __attribute__((always_inline)) { f(i, load_as_f32(row, i, DT)); }, []() {});
}

// 16-bit rows: pair(two entries) or one(an entry), as raw bits in any order, for all entries; first() as above
template <int DT, int THREADS, int UNROLL, class Pair, class One, class First>
__device__ __forceinline__ void for_each_logit_pair(const void* row, int vocab, Pair&& pair, One&& one, First&& first) {
  walk_row<2, THREADS, UNROLL>(
      row, vocab,
      [&](int, const uint4& v) __attribute__((always_inline)) { pair(v.x); pair(v.y); pair(v.z); pair(v.w); },
      [&](int i) __attribute__((always_inline)) { one((uint32_t)((const uint16_t*)row)[i]); }, first);
}

}  // namespace pa

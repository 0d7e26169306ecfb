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

// f(index, raw bits) for every entry of the row, the workgroup's THREADS threads taking 16-byte pieces in turn,
// four in flight each (the entries before the first 16-byte boundary and after the last one by themselves: rows
// of an odd vocabulary start anywhere).
template <int DT, int THREADS, class F>
__device__ __forceinline__ void for_each_logit_bits(const void* row, int vocab, F&& f) {
  constexpr int ES = DT == PA_DTYPE_F32 ? 4 : 2;
  constexpr int PER = 16 / ES;
  constexpr int UNROLL = 4;
  auto one = [&](int i) __attribute__((always_inline)) {
    if constexpr (DT == PA_DTYPE_F32) f(i, ((const uint32_t*)row)[i]);
    else f(i, (uint32_t)((const uint16_t*)row)[i]);
  };
  const int head = min((int)((16u - (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / ES, vocab);
  const uint4* wide = (const uint4*)((const uint8_t*)row + head * ES);
  const int pieces = (vocab - head) / PER;
  auto apply = [&](int c, const uint4& w) __attribute__((always_inline)) {
    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
    const int i = head + c * PER;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (DT == PA_DTYPE_F32) {
        f(i + k, ww[k]);
      } else {
        f(i + 2 * k, ww[k] & 0xffffu);
        f(i + 2 * k + 1, ww[k] >> 16);
      }
    }
  };
  int c = threadIdx.x;
  for (; c + (UNROLL - 1) * THREADS < pieces; c += UNROLL * THREADS) {
    uint4 w[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) w[u] = wide[c + u * THREADS];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) apply(c + u * THREADS, w[u]);
  }
  for (; c < pieces; c += THREADS) apply(c, wide[c]);
  for (int i = threadIdx.x; i < head; i += THREADS) one(i);
  for (int i = head + pieces * PER + threadIdx.x; i < vocab; i += THREADS) one(i);
}

// the same with the entry's value
template <int DT, int THREADS, class F>
__device__ __forceinline__ void for_each_logit(const void* row, int vocab, F&& f) {
  for_each_logit_bits<DT, THREADS>(row, vocab, [&](int i, uint32_t bits) __attribute__((always_inline)) { f(i, logit_value<DT>(bits)); });
}

}  // namespace pa

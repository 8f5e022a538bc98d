// Rows of router logits spread over the lanes of a wave: their loads and stores and the exchanges
// between a token's lanes, for the routing and for the losses that keep it balanced.
#pragma once

#include "common.h"

namespace strata {

constexpr int ROUTE_MAX_E = 512;

template <typename T>
__device__ __forceinline__ float route_load(const void* p, int64_t i) {
  return (float)((const T*)p)[i];
}
template <typename T>
__device__ __forceinline__ void route_store(void* p, int64_t i, float v) {
  ((T*)p)[i] = (T)v;
}
__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < __builtin_inff(); }

// EPL consecutive elements from i on; VEC: as 16-byte (or one shorter) runs.
template <typename T, int EPL, bool VEC>
__device__ __forceinline__ void route_row(const void* p, int64_t i, int left, float other, float (&v)[EPL]) {
  if constexpr (VEC && EPL >= 4) {
    if (left >= EPL) {
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < EPL / 4; ++k) {
          const f32x4 x = *(const f32x4*)((const float*)p + i + 4 * k);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * k + e] = x[e];
        }
      } else {
#pragma unroll
        for (int k = 0; k < EPL / 4; ++k) {
          const u32x2 x = *(const u32x2*)((const bf16*)p + i + 4 * k);
          v[4 * k] = bf16_lo(x[0]);
          v[4 * k + 1] = bf16_hi(x[0]);
          v[4 * k + 2] = bf16_lo(x[1]);
          v[4 * k + 3] = bf16_hi(x[1]);
        }
      }
      return;
    }
  }
#pragma unroll
  for (int k = 0; k < EPL; ++k) v[k] = k < left ? route_load<T>(p, i + k) : other;
}

// The value of the lane d away in a butterfly over lanes that agree in groups of d: moves
// inside a row of 16 lanes, an exchange through LDS beyond.
template <int D>
__device__ __forceinline__ uint32_t swap_word(uint32_t v) {
  if constexpr (D == 1) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true);        // quad 1 0 3 2
  else if constexpr (D == 2) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true);   // quad 2 3 0 1
  else if constexpr (D == 4) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true);  // half row mirrored
  else if constexpr (D == 8) return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true);  // row mirrored
  else return (uint32_t)__shfl_xor((int)v, D);
}
template <int D>
__device__ __forceinline__ float swap_lane(float v) { return __uint_as_float(swap_word<D>(__float_as_uint(v))); }
template <int D>
__device__ __forceinline__ int swap_lane(int v) { return (int)swap_word<D>((uint32_t)v); }
template <int D>
__device__ __forceinline__ double swap_lane(double v) {
  const u32x2 w = __builtin_bit_cast(u32x2, v);
  return __builtin_bit_cast(double, (u32x2){swap_word<D>(w[0]), swap_word<D>(w[1])});
}
// f(integral_constant<int, d>) for d = 1, 2, 4 .. L / 2
template <int L, typename F>
__device__ __forceinline__ void butterfly(F f) {
  if constexpr (L > 1) f(std::integral_constant<int, 1>{});
  if constexpr (L > 2) f(std::integral_constant<int, 2>{});
  if constexpr (L > 4) f(std::integral_constant<int, 4>{});
  if constexpr (L > 8) f(std::integral_constant<int, 8>{});
  if constexpr (L > 16) f(std::integral_constant<int, 16>{});
  if constexpr (L > 32) f(std::integral_constant<int, 32>{});
}
template <int L, typename V>
__device__ __forceinline__ V group_max(V v) {
  butterfly<L>([&](auto d) {
    const V o = swap_lane<decltype(d)::value>(v);
    v = o > v ? o : v;
  });
  return v;
}
template <int L, typename V>
__device__ __forceinline__ V group_sum(V v) {
  butterfly<L>([&](auto d) { v += swap_lane<decltype(d)::value>(v); });
  return v;
}

}  // namespace strata

// Reductions over a few lanes of a wave, and the staging of V rows of a wave that has them in 32-byte slots: of the decode kernels
// (flash_decode.hip) and of those over pages.
#pragma once
#include <type_traits>

#include "common.hpp"

namespace LLMHIP_NS {

// Maximum / sum over the four lanes that hold one column (they differ in bits 4 and 5 of the lane index):
// v_permlane16_swap and v_permlane32_swap, no LDS crossbar.
template <typename F> __device__ __forceinline__ float quad_reduce(float x, F f) {
  typedef __attribute__((ext_vector_type(2))) unsigned u2;
  unsigned u = __builtin_bit_cast(unsigned, x);
  u2 r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  unsigned r0 = r[0], r1 = r[1];
  u = __builtin_bit_cast(unsigned, f(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1)));
  r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  r0 = r[0];
  r1 = r[1];
  return f(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
}
__device__ __forceinline__ float quad_max(float x) {
  return quad_reduce(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float quad_sum(float x) {
  return quad_reduce(x, [](float a, float b) { return a + b; });
}

// V staging swizzle for the 16x16x32 transposed reads: one instruction touches
// 8 rows x 32 bytes per half-wave, so the 32-byte slot index is XORed with
// row%8.
__device__ __forceinline__ int v_swizzle32_off(int row, int granule) {
  return row * kRowBytes + ((((granule >> 1) ^ (row & 7)) << 5) | ((granule & 1) << 4));
}

// Maximum over each N = 2, 4 or 8 lanes.
template <int N> __device__ __forceinline__ float max_of_lanes(float x) {
  auto with = [&](auto control) {
    const int i = __builtin_bit_cast(int, x);
    x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, decltype(control)::value, 0xf, 0xf, false)));
  };
  with(std::integral_constant<int, 0xB1>());                     // quad_perm: lane ^ 1
  if (N >= 4) with(std::integral_constant<int, 0x4E>());         // quad_perm: lane ^ 2
  if (N == 8) with(std::integral_constant<int, 0x141>());        // row_half_mirror: the other quad
  return x;
}

}  // namespace LLMHIP_NS

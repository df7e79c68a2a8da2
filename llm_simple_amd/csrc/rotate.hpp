// The rotation of 8 pairs by one thread, of the kernels that append to a cache.  For files compiled with -ffp-contract=off.
#pragma once
#include "common.hpp"

namespace LLMHIP_NS {

// The 8 pairs of one thread: a = elements of the first 16-byte chunk, b = of the second.  NEOX: pair i
// = (a[i], b[i]) (dims f, f + 64); interleaved: pair i = elements 2i, 2i+1 of the 16 contiguous ones.
// Arithmetic of src/llama2_layer_cpu.cpp:835-856: every product and sum rounded on its own.
template <typename T, bool NEOX>
__device__ __forceinline__ void rotate8(u32x4_t &va, u32x4_t &vb, const f32x4_t (&cs)[4]) {
  using E = Elem<T>;
  float r0[8], r1[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint16_t xa, xb;
    if (NEOX) {
      xa = (uint16_t)(va[i >> 1] >> ((i & 1) * 16));
      xb = (uint16_t)(vb[i >> 1] >> ((i & 1) * 16));
    } else {
      const uint32_t w = (i < 4) ? va[i] : vb[i - 4];
      xa = (uint16_t)w;
      xb = (uint16_t)(w >> 16);
    }
    const float a = E::widen(xa), b = E::widen(xb);
    const float c = cs[i >> 1][2 * (i & 1)], d = cs[i >> 1][2 * (i & 1) + 1];
    r0[i] = a * c - b * d;
    r1[i] = a * d + b * c;
  }
  if (NEOX) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      va[j] = E::pack2(r0[2 * j], r0[2 * j + 1]);
      vb[j] = E::pack2(r1[2 * j], r1[2 * j + 1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      va[j] = E::pack2(r0[j], r1[j]);
      vb[j] = E::pack2(r0[j + 4], r1[j + 4]);
    }
  }
}

}  // namespace LLMHIP_NS

// The rotation of q and k by their positions, in 32 bits (paged_append.hip, paged_append_int4.hip's q). Not part of
// the C ABI.
#pragma once

#include "paged.h"

namespace ldk {

// cos and sin of pos * freq.
__device__ __forceinline__ void angle(int64_t pos, float freq, float* c, float* s) {
  const double t = (double)pos * (double)freq * 0.15915494309189533577;  // turns
  sincospif(2.0f * (float)(t - __builtin_rint(t)), s, c);
}

// Rotates 8 pairs (x0[e], x1[e]) by the angles whose cos and sin are c[0..7], s[0..7].
template <typename E>
__device__ __forceinline__ void rotate8(u32x4& x0, u32x4& x1, const float* c, const float* s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2_t a = unpack2<E>(x0[i]), b = unpack2<E>(x1[i]);
    float r0[2], r1[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      r0[j] = a[j] * c[2 * i + j] - b[j] * s[2 * i + j];
      r1[j] = b[j] * c[2 * i + j] + a[j] * s[2 * i + j];
    }
    x0[i] = pack2<E>(r0[0], r0[1]);
    x1[i] = pack2<E>(r1[0], r1[1]);
  }
}

}  // namespace ldk

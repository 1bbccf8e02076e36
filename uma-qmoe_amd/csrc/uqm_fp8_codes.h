// Device-side pieces of the e4m3 codes and scales (definitions in uqm_fp8.h) that
// the row operators and the key-value cache share.
#pragma once

#include "uqm_device.h"

namespace uqm {

constexpr float kFp8Max = 448.0f;

// Four values as e4m3 bytes, to nearest even (NaN stays NaN).
__device__ __forceinline__ uint32_t pack_fp8x4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}

// Bits of max|v|: as unsigned numbers magnitudes order like the floats, and a
// NaN above every other value, which fmaxf would drop.
__device__ __forceinline__ uint32_t magnitude8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  return m;
}
template <int O>
__device__ __forceinline__ uint32_t max_step(uint32_t m) {
  return max(m, __float_as_uint(xor_partner<O>(__uint_as_float(m))));
}
// Maximum over the 16 lanes of a group.
__device__ __forceinline__ uint32_t group_max(uint32_t m) {
  m = max_step<8>(m);
  m = max_step<4>(m);
  m = max_step<2>(m);
  return max_step<1>(m);
}
__device__ __forceinline__ float scale_of(uint32_t bits) {
  const float d = __uint_as_float(bits) / kFp8Max;
  return bits == 0u ? 1.0f : (d < 0x1p-126f ? 0x1p-126f : d);
}

}  // namespace uqm

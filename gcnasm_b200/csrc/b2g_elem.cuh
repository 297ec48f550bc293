// b2g_elem.cuh -- element conversions shared by the quantisers and the 4-bit cache.
#pragma once

#include <cuda_bf16.h>

#include <cstdint>

namespace b2g {

// MXFP4 element: round to nearest with ties to the even code onto the e2m1 grid
// {0, 0.5, 1, 1.5, 2, 3, 4, 6} (the midpoints are exact fp32 values), saturating
// at 6; sign from the sign bit of x; NaN -> 7 | sign.  Nibble code, bit 3 = sign.
__device__ __forceinline__ uint32_t f32_to_e2m1(float x) {
  const uint32_t sign = (__float_as_uint(x) >> 28) & 8u;
  const float a = fabsf(x);
  uint32_t c = (a <= 0.25f) ? 0u : (a < 0.75f) ? 1u : (a <= 1.25f) ? 2u : (a < 1.75f) ? 3u
             : (a <= 2.5f) ? 4u : (a < 3.5f) ? 5u : (a <= 5.0f) ? 6u : 7u;
  if (a != a) c = 7u;
  return sign | c;
}

// eight consecutive input elements as fp32 (bf16 widens exactly); 16-byte aligned
__device__ __forceinline__ void load8_f32(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p));
  const float4 b = __ldg(reinterpret_cast<const float4*>(p + 4));
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8_f32(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 t = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(w[j] << 16);
    v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
  }
}

}  // namespace b2g

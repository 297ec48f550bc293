// b2g_kv4_weights.cuh -- the attention weight that each token of the 4-bit cache gathers.
#pragma once

#include "b2g_kv4_decode.cuh"

namespace b2g {

template <int D>
__device__ __forceinline__ void kv4_load_q(const Kv4Queries& q, int row, int head, int lane, float (&x)[D / 32]) {
#pragma unroll
  for (int j = 0; j < D / 32; j += 2) {
    const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(q.q + row * q.q_row + head * q.q_head + lane * (D / 32) + j));
    x[j] = __uint_as_float(w << 16);
    x[j + 1] = __uint_as_float(w & 0xFFFF0000u);
  }
}

// the lane's D / 32 consecutive channels of a token's K or V
template <int D>
__device__ __forceinline__ void kv4_load_token(const uint8_t* codes, const uint8_t* scales, long long at, int lane,
                                               float (&x)[D / 32]) {
  const float s = kv4_scale_value(__ldg(scales + at * (D / 32) + lane * (D / 32) / 32));
#pragma unroll
  for (int j = 0; j < D / 64; ++j) {
    const uint32_t n = __ldg(codes + at * (D / 2) + lane * (D / 64) + j);
    x[2 * j] = kv4_code_value(n) * s;
    x[2 * j + 1] = kv4_code_value(n >> 4) * s;
  }
}

template <int D>
__device__ __forceinline__ float kv4_dot(const float (&a)[D / 32], const float (&b)[D / 32]) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < D / 32; ++j) s = fmaf(a[j], b[j], s);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// One warp per (cached token, kv head): the sum over the sequence's rows and the group's heads.
template <int D>
__global__ void __launch_bounds__(128)
b2g_kv4_weights_kernel(Kv4Cache c, Kv4Batch bt, Kv4Mask mask, Kv4Queries q, const float* __restrict__ lse,
                       const float* w_in, float* w_out, int* status) {
  constexpr int kE = D / 32;
  const int h = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x & 31;
  int first, end;
  kv4_rows(bt, b, first, end);
  const int len = kv4_len(bt, b, c.page_log2);
  for (int j = blockIdx.x * 4 + (threadIdx.x >> 5); j < len; j += gridDim.x * 4) {
    const long long at = kv4_token(c, bt.table + static_cast<long long>(b) * bt.width, h, j, status);
    if (at < 0) continue;
    float t[kE], x[kE], sum = 0.f;
    kv4_load_token<D>(c.k, c.ks, at, lane, t);
    for (int row = first; row < end; ++row) {
      int lo, hi;
      kv4_visible(mask, len - (end - row), len, lo, hi);
      if (j < lo || j >= hi) continue;
      for (int g = 0; g < q.group; ++g) {
        const int head = h * q.group + g;
        kv4_load_q<D>(q, row, head, lane, x);
        float s = kv4_dot<D>(x, t) * mask.scale;
        if (mask.softcap > 0.f) s = kv4_cap(s, mask.softcap, 2.f * kLog2e / mask.softcap);
        sum += __expf(s - __ldg(lse + static_cast<long long>(row) * q.heads + head));
      }
    }
    if (lane == 0) w_out[at] = w_in[at] + sum;
  }
}

}  // namespace b2g

// b2g_kv4_attn.cuh -- attention over the 4-bit key/value cache, and the attention weight
// that each cached token gathers.
#pragma once

#include "b2g_kv4.cuh"

namespace b2g {

struct Kv4Mask {
  float scale, softcap;
  int causal, window;
};

struct Kv4Queries {
  const __nv_bfloat16* q;
  long long q_row, q_head;
  int heads, group;
};

// Tokens [lo, hi) that the query at position p of a sequence of `len` tokens sees.
__device__ __forceinline__ void kv4_visible(const Kv4Mask& m, int p, int len, int& lo, int& hi) {
  hi = m.causal ? min(max(p + 1, 0), len) : len;
  lo = m.window > 0 ? max(p - m.window + 1, 0) : 0;
}

// c tanh(s / c), by tanh x = 1 - 2 / (e^2x + 1): exact limits at both ends.
__device__ __forceinline__ float kv4_cap(float s, float cap) {
  return cap * (1.f - 2.f / (__expf(2.f * s / cap) + 1.f));
}

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

// One CTA of four warps per (row, head); the warps take tokens in turn, each with its own
// running maximum, sum and output, joined at the end.
template <int D>
__global__ void __launch_bounds__(128)
b2g_kv4_attention_kernel(Kv4Cache c, Kv4Batch bt, Kv4Mask mask, Kv4Queries q, __nv_bfloat16* __restrict__ out,
                         long long out_row, long long out_head, float* __restrict__ lse, int* status) {
  constexpr int kE = D / 32;
  __shared__ float s_m[4], s_l[4], s_o[4][D];
  const int row = blockIdx.x / q.heads, head = blockIdx.x % q.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = kv4_seq_of_row(bt, row);
  int first, end;
  kv4_rows(bt, b, first, end);
  const int len = kv4_len(bt, b, c.page_log2);
  int lo, hi;
  kv4_visible(mask, len - (end - row), len, lo, hi);
  if (row < first || row >= end) hi = 0;
  float x[kE], t[kE], o[kE] = {};
  kv4_load_q<D>(q, row, head, lane, x);
  float m = -INFINITY, l = 0.f;
  const int* pages = bt.table + static_cast<long long>(b) * bt.width;
  for (int j = lo + warp; j < hi; j += 4) {
    const long long at = kv4_token(c, pages, head / q.group, j, status);
    if (at < 0) continue;
    kv4_load_token<D>(c.k, c.ks, at, lane, t);
    float s = kv4_dot<D>(x, t) * mask.scale;
    if (mask.softcap > 0.f) s = kv4_cap(s, mask.softcap);
    kv4_load_token<D>(c.v, c.vs, at, lane, t);
    const float mn = fmaxf(m, s);
    const float f = m == -INFINITY ? 0.f : __expf(m - mn), p = __expf(s - mn);
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < kE; ++i) o[i] = o[i] * f + p * t[i];
    m = mn;
  }
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
  for (int i = 0; i < kE; ++i) s_o[warp][lane * kE + i] = o[i];
  __syncthreads();
  const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float sum = 0.f, f[4];
  for (int w = 0; w < 4; ++w) {
    f[w] = s_m[w] == -INFINITY ? 0.f : __expf(s_m[w] - top);
    sum += f[w] * s_l[w];
  }
  for (int d = threadIdx.x; d < D; d += 128) {
    float v = 0.f;
    for (int w = 0; w < 4; ++w) v += f[w] * s_o[w][d];
    out[row * out_row + head * out_head + d] = __float2bfloat16(sum > 0.f ? v / sum : 0.f);
  }
  if (threadIdx.x == 0) lse[static_cast<long long>(row) * q.heads + head] = sum > 0.f ? top + logf(sum) : -INFINITY;
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
        if (mask.softcap > 0.f) s = kv4_cap(s, mask.softcap);
        sum += __expf(s - __ldg(lse + static_cast<long long>(row) * q.heads + head));
      }
    }
    if (lane == 0) w_out[at] = w_in[at] + sum;
  }
}

}  // namespace b2g

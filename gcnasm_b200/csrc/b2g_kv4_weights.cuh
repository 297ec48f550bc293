// b2g_kv4_weights.cuh -- the attention weight that each token of the 4-bit cache gathers:
//   w_j += sum over query rows i and the group's heads of exp(s_ij - lse_i).
//
// The column sums of the attention matrix, which the attention itself cannot give: they need
// the final lse.  K is read once more, V not at all.  A CTA has 256 tokens of a kv head,
// four tiles of 16 for each warp, and goes through the query rows 64 at a time: with K Q^T as
// in the decode kernel (f16, block sums times their scale), rows lie along the
// fragment's columns, so a thread adds what it has of a token and one exchange among four
// lanes ends the sum.  No atomics: each token belongs to one thread, and the order is fixed.
//
// Bound: for a decode step K's bytes and the weights' (D / 2 + D / 32 + 8 per token and head);
// for many rows the instructions between the products (exp2, the block scales).
#pragma once

#include "b2g_kv4_decode.cuh"

namespace b2g {

constexpr int kWeightTokens = 256;

template <int D>
struct WeightsCfg {
  static constexpr int kChunks = D / 32;
  static constexpr int kNT = 8;  // tiles of eight rows in shared memory at once
  static constexpr int kRows = 8 * kNT;
  static constexpr int kK = kWeightTokens * (D / 2);
  static constexpr int kScaleBytes = kWeightTokens * kChunks;
  static constexpr int kQ = (D / 16) * kNT * 256;
  static constexpr int kFixed = kK + kScaleBytes + kQ + 3 * kRows * 4;
};

template <int D>
__global__ void __launch_bounds__(128)
b2g_kv4_weights_kernel(Kv4Cache c, Kv4Batch bt, Kv4Mask mask, Kv4Queries q, const float* __restrict__ lse,
                       const float* w_in, float* w_out, int* status) {
  using Cfg = WeightsCfg<D>;
  constexpr int kChunks = Cfg::kChunks, kNT = Cfg::kNT, kRows = Cfg::kRows;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* s_k = smem;
  uint8_t* s_ks = smem + Cfg::kK;
  uint2* s_q = reinterpret_cast<uint2*>(s_ks + Cfg::kScaleBytes);
  float* s_rs = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(s_q) + Cfg::kQ);
  float* s_lse = s_rs + kRows;
  int* s_top = reinterpret_cast<int*>(s_lse + kRows);
  long long* s_pre = reinterpret_cast<long long*>(smem + ((Cfg::kFixed + 15) & ~15));
  __shared__ long long s_scan[4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;

  griddep_wait();
  kv4_scan(bt.seqs, s_pre, s_scan, [&](int b) {
    return static_cast<long long>((kv4_len(bt, b, c.page_log2) + kWeightTokens - 1) / kWeightTokens) * c.heads;
  });
  const long long total = s_pre[bt.seqs];
  const long long u0 = total * blockIdx.x / gridDim.x, u1 = total * (blockIdx.x + 1) / gridDim.x;
  if (u0 >= u1) return;
  if (tid < kRows) s_top[tid] = 0;
  const float cap_k = mask.softcap > 0.f ? 2.f * kLog2e / mask.softcap : 0.f;
  const float s_scale = mask.softcap > 0.f ? mask.scale : mask.scale * kLog2e;
  const int lm_tok = (lane & 7) + (lane & 8), lm_ch = lane >> 4;
  const int lm_swz = D == 256 ? lm_tok & 7 : D == 128 ? (lm_tok >> 1) & 3 : (lm_tok >> 2) & 1;
  int b = kv4_seq_of_unit(s_pre, bt.seqs, u0);
  for (long long u = u0; u < u1; ++u) {
    while (u >= s_pre[b + 1]) ++b;
    int first, end;
    kv4_rows(bt, b, first, end);
    const int rows = end - first, len = kv4_len(bt, b, c.page_log2), group_rows = rows * q.group;
    const int chunks = (len + kWeightTokens - 1) / kWeightTokens;
    const int in_seq = static_cast<int>(u - s_pre[b]);
    const int h = in_seq / chunks, tok0 = (in_seq - h * chunks) * kWeightTokens;
    // tokens that some row sees
    int see_lo, see_hi, unused;
    kv4_visible(mask, len - rows, len, see_lo, unused);
    kv4_visible(mask, len - 1, len, unused, see_hi);
    const bool any = rows > 0 && see_lo < tok0 + kWeightTokens && see_hi > tok0;
    const int* pages = bt.table + static_cast<long long>(b) * bt.width;
    const int mine = tok0 + warp * 64;
    __syncthreads();  // the last unit's K and Q have been read
    unsigned there = 0;  // bit i: the warp's tile i is there
#pragma unroll
    for (int tile = 0; tile < 4; ++tile) {
      const int token = mine + tile * 16;
      const long long at = token < len ? kv4_token(c, pages, h, token, status) : -1;
      if (at >= 0) there |= 1u << tile;
      if (any) {
        const uint32_t dst = smem_u32(s_k) + (warp * 64 + tile * 16) * (D / 2);
        const uint8_t* src = c.k + (at < 0 ? 0 : at) * (D / 2) + lane * 16;
#pragma unroll
        for (int j = 0; j < kChunks / 2; ++j) {
          const int tau = (j * 32 + lane) / kChunks, ch = (j * 32 + lane) % kChunks;
          const int swz = D == 256 ? tau & 7 : D == 128 ? (tau >> 1) & 3 : (tau >> 2) & 1;
          cp_async16(dst + tau * (D / 2) + (ch ^ swz) * 16, src + j * 512, at >= 0);
        }
        if (lane < kChunks)
          cp_async16(smem_u32(s_ks) + (warp * 64 + tile * 16) * kChunks + lane * 16, c.ks + (at < 0 ? 0 : at) * kChunks + lane * 16, at >= 0);
      }
    }
    cp_async_commit();
    float sum[4][2] = {};
    if (any) {
      for (int n0 = 0; n0 < group_rows; n0 += kRows) {
        const int n1 = min(n0 + kRows, group_rows);
        int lo0, hi0, lo1, hi1;  // what the first and the last of these rows see
        kv4_visible(mask, len - rows + n0 / q.group, len, lo0, hi0);
        kv4_visible(mask, len - rows + (n1 - 1) / q.group, len, lo1, hi1);
        if (lo0 >= tok0 + kWeightTokens || hi1 <= tok0) continue;
        if (n0) __syncthreads();
        kv4_stage_q<D, kNT, 128>(q, first, h, n0, group_rows, s_scale, s_q, s_top, s_rs);
        if (tid < kRows) {
          const int n = n0 + tid;
          float x = INFINITY;  // what gives weight zero: rows that are not there, or see nothing
          if (n < group_rows) {
            const float v = __ldg(lse + static_cast<long long>(first + n / q.group) * q.heads + h * q.group + n % q.group);
            if (v != -INFINITY) x = v * kLog2e;
          }
          s_lse[tid] = x;
          s_top[tid] = 0;
        }
        cp_async_wait<0>();
        __syncthreads();
        const int tiles_n = (n1 - n0 + 7) / 8;
#pragma unroll
        for (int tile = 0; tile < 4; ++tile) {
          const int tb = mine + tile * 16;
          if (!((there >> tile) & 1) || lo0 >= tb + 16 || hi1 <= tb) continue;
          const bool masked = lo1 > tb || hi0 < tb + 16;
          // K of the tile: f16 codes and fp32 scales of tokens g and g + 8
          uint32_t kf[kChunks][2][4];
          float f0[kChunks], f1[kChunks];
          const uint32_t k_at = smem_u32(s_k) + (warp * 64 + tile * 16 + lm_tok) * (D / 2);
          const uint8_t* sr = s_ks + (warp * 64 + tile * 16 + g) * kChunks;
#pragma unroll
          for (int pair = 0; pair < kChunks / 2; ++pair) {
            uint32_t kw[4];
            ldmatrix_x4(kw, k_at + (((2 * pair + lm_ch) ^ lm_swz) * 16));
#pragma unroll
            for (int i = 0; i < 4; ++i) e2m1x8_to_f16(kw[i], kf[2 * pair + (i >> 1)][i & 1]);
          }
#pragma unroll
          for (int i = 0; i < kChunks; ++i) {
            f0[i] = kv4_scale_value(sr[i]);
            f1[i] = kv4_scale_value(sr[8 * kChunks + i]);
          }
#pragma unroll 2
          for (int nt = 0; nt < tiles_n; ++nt) {
            float s[4];
#pragma unroll
            for (int blk = 0; blk < kChunks; ++blk) {
              const uint2 b0 = s_q[(2 * blk * kNT + nt) * 32 + lane], b1 = s_q[((2 * blk + 1) * kNT + nt) * 32 + lane];
              float x[4] = {0.f, 0.f, 0.f, 0.f};
              mma_f16_16816(x, kf[blk][0][0], kf[blk][1][0], kf[blk][0][1], kf[blk][1][1], b0.x, b0.y);
              mma_f16_16816(x, kf[blk][0][2], kf[blk][1][2], kf[blk][0][3], kf[blk][1][3], b1.x, b1.y);
#pragma unroll
              for (int j = 0; j < 4; ++j) s[j] = blk ? fmaf(x[j], j < 2 ? f0[blk] : f1[blk], s[j]) : x[j] * (j < 2 ? f0[0] : f1[0]);
            }
            const float2 rs = *reinterpret_cast<const float2*>(s_rs + nt * 8 + 2 * t);
            const float2 ls = *reinterpret_cast<const float2*>(s_lse + nt * 8 + 2 * t);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float x = s[j] * ((j & 1) ? rs.y : rs.x);
              if (mask.softcap > 0.f) x = kv4_cap(x, mask.softcap, cap_k) * kLog2e;
              x -= (j & 1) ? ls.y : ls.x;
              if (masked) {
                int lo, hi;
                kv4_visible(mask, len - rows + (n0 + nt * 8 + 2 * t + (j & 1)) / q.group, len, lo, hi);
                const int token = tb + g + (j >> 1) * 8;
                if (token < lo || token >= hi) x = -INFINITY;
              }
              sum[tile][j >> 1] += ex2(x);
            }
          }
        }
      }
    }
    cp_async_wait<0>();
#pragma unroll
    for (int tile = 0; tile < 4; ++tile)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float x = sum[tile][half];
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        x += __shfl_xor_sync(0xffffffffu, x, 2);
        const int token = mine + tile * 16 + half * 8 + g;
        if (t == 0 && ((there >> tile) & 1) && token < len) {
          const long long at = kv4_token(c, pages, h, token, status);
          w_out[at] = w_in[at] + x;
        }
      }
  }
}

}  // namespace b2g

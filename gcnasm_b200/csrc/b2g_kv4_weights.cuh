// b2g_kv4_weights.cuh -- the attention weight that each token of the 4-bit cache gathers:
//   w_j += sum over query rows i and the group's heads of exp(s_ij - lse_i).
//
// The column sums of the attention matrix, which the attention itself cannot give: they need
// the final lse.  K is read once more, V not at all.  A CTA has 256 tokens of a kv head at a
// time, four tiles of 16 for each warp, and goes through the query rows 128 (D = 256: 64) at a time.  K becomes
// bf16 as the decode kernel's V does (times 2^-64, exact; once per tile, for all rows) and
// stays in registers; Q comes from shared memory, in the order of channels in which the codes
// of a word are taken out, 0 4 1 5 2 6 3 7.  In K Q^T a token is a fragment's row, so a thread
// adds what it has of a token and one exchange among four lanes ends the sum.  No atomics: each
// token belongs to one thread, and the order is fixed.
//
// Bound: for a decode step K's bytes and the weights' (D / 2 + D / 32 + 8 per token and head):
// the next 256 tokens are fetched while these are worked on, and Q stays where they share it.  For
// many rows the warp-level products, 8 clocks each on a scheduler.  Measured, one row of 32 ragged
// sequences of up to 4096 tokens, 32 heads, 8 kv heads, D = 128 (51 MB): 35 us, 1.4 TB/s.  Half of the issue
// slots are used, by 12 warps on an SM: turning codes into fragments and each unit's own
// steps (its place, pages, lse) bind it, not the memory.
#pragma once

#include "b2g_kv4_decode.cuh"

namespace b2g {

constexpr int kWeightTokens = 256;

template <int D>
struct WeightsCfg {
  static constexpr int kChunks = D / 32;
  static constexpr int kNT = D == 256 ? 8 : 16;  // tiles of eight rows in shared memory at once
  static constexpr int kRows = 8 * kNT;
  static constexpr int kTT = D == 256 ? 1 : 2;  // token tiles that share what is read of Q
  static constexpr int kK = kWeightTokens * (D / 2);
  static constexpr int kStage = kK + kWeightTokens * kChunks;
  static constexpr int kQ = (D / 16) * kNT * 256;
  static constexpr int kFixed = 2 * kStage + kQ + kRows * 4 + kWeightTokens * 4;
};

template <int D>
__global__ void __launch_bounds__(128)
b2g_kv4_weights_kernel(Kv4Cache c, Kv4Batch bt, Kv4Mask mask, Kv4Queries q, const float* __restrict__ lse,
                       const float* w_in, float* w_out, int* status) {
  using Cfg = WeightsCfg<D>;
  constexpr int kChunks = Cfg::kChunks, kNT = Cfg::kNT, kRows = Cfg::kRows, kTT = Cfg::kTT;
  extern __shared__ __align__(128) uint8_t smem[];
  uint2* s_q = reinterpret_cast<uint2*>(smem + 2 * Cfg::kStage);
  float* s_lse = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(s_q) + Cfg::kQ);
  float* s_sum = s_lse + kRows + (threadIdx.x >> 5) * 64;  // of the warp's 64 tokens
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
  const float cap_k = mask.softcap > 0.f ? 2.f * kLog2e / mask.softcap : 0.f;
  const float s_scale = mask.softcap > 0.f ? mask.scale * kTwo64 : mask.scale * kTwo64 * kLog2e;
  const int lm_tok = (lane & 7) + (lane & 8), lm_ch = lane >> 4;
  const int lm_swz = D == 256 ? lm_tok & 7 : D == 128 ? (lm_tok >> 1) & 3 : (lm_tok >> 2) & 1;

  struct Unit {
    int b, h, tok0, first, rows, len;
    bool any;         // some row sees some of its tokens
    int page[4];      // of the warp's tiles, -2 past the end
    unsigned there;   // bit i: tile i has a page
    long long at[4];  // the tile's first token among all
  };
  // where unit u is, a unit after x's; its page numbers are on the way
  auto locate = [&](Unit& x, long long u) {
    while (u >= s_pre[x.b + 1]) ++x.b;
    int end;
    kv4_rows(bt, x.b, x.first, end);
    x.rows = end - x.first;
    x.len = kv4_len(bt, x.b, c.page_log2);
    const int chunks = (x.len + kWeightTokens - 1) / kWeightTokens;
    const long long in_seq = u - s_pre[x.b];
    x.h = static_cast<int>(in_seq / chunks);
    x.tok0 = static_cast<int>(in_seq - static_cast<long long>(x.h) * chunks) * kWeightTokens;
    int lo, hi, unused;
    kv4_visible(mask, x.len - x.rows, x.len, lo, unused);
    kv4_visible(mask, x.len - 1, x.len, unused, hi);
    x.any = x.rows > 0 && lo < x.tok0 + kWeightTokens && hi > x.tok0;
#pragma unroll
    for (int tile = 0; tile < 4; ++tile) {
      const int token = x.tok0 + warp * 64 + tile * 16;
      x.page[tile] = token < x.len ? __ldg(bt.table + static_cast<long long>(x.b) * bt.width + (token >> c.page_log2)) : -2;
    }
  };
  // its K on the way to stage `st`
  auto fetch = [&](Unit& x, int st) {
    const uint32_t to = smem_u32(smem) + st * Cfg::kStage;
    x.there = 0;
#pragma unroll
    for (int tile = 0; tile < 4; ++tile) {
      const int token = x.tok0 + warp * 64 + tile * 16;
      const bool ok = static_cast<unsigned>(x.page[tile]) < static_cast<unsigned>(c.pages);
      if (!ok && x.page[tile] != -2) atomicCAS(status, 0, kDevBadPage);
      x.there |= ok ? 1u << tile : 0u;
      x.at[tile] = ok ? ((static_cast<long long>(x.page[tile]) * c.heads + x.h) << c.page_log2) + (token & ((1 << c.page_log2) - 1)) : 0;
    }
    if (x.any) {
#pragma unroll
      for (int tile = 0; tile < 4; ++tile) {
        const bool ok = (x.there >> tile) & 1;
        const uint32_t dst = to + (warp * 64 + tile * 16) * (D / 2);
        const uint8_t* src = c.k + x.at[tile] * (D / 2) + lane * 16;
#pragma unroll
        for (int j = 0; j < kChunks / 2; ++j) {
          const int tau = (j * 32 + lane) / kChunks, ch = (j * 32 + lane) % kChunks;
          const int swz = D == 256 ? tau & 7 : D == 128 ? (tau >> 1) & 3 : (tau >> 2) & 1;
          cp_async16(dst + tau * (D / 2) + (ch ^ swz) * 16, src + j * 512, ok);
        }
        if (lane < kChunks) cp_async16(to + Cfg::kK + (warp * 64 + tile * 16) * kChunks + lane * 16, c.ks + x.at[tile] * kChunks + lane * 16, ok);
      }
    }
    cp_async_commit();
  };

  Unit now, next, after;
  now.b = kv4_seq_of_unit(s_pre, bt.seqs, u0);
  locate(now, u0);
  fetch(now, 0);
  next = now;
  if (u0 + 1 < u1) locate(next, u0 + 1);
  int q_b = -1, q_h = -1;  // whose first rows are in shared memory
  for (long long u = u0; u < u1; ++u, now = next, next = after) {
    const int st = static_cast<int>(u - u0) & 1;
    if (u + 1 < u1) fetch(next, st ^ 1);
    else cp_async_commit();
    after = next;
    if (u + 2 < u1) locate(after, u + 2);
    // two tokens a lane: what they have gathered so far
    const int tile_a = lane >> 4;
    const long long at_a = (tile_a ? now.at[1] : now.at[0]) + (lane & 15), at_b = (tile_a ? now.at[3] : now.at[2]) + (lane & 15);
    const int token_a = now.tok0 + warp * 64 + lane;
    const bool has_a = ((now.there >> tile_a) & 1) && token_a < now.len, has_b = ((now.there >> (tile_a + 2)) & 1) && token_a + 32 < now.len;
    const float w_a = has_a ? w_in[at_a] : 0.f, w_b = has_b ? w_in[at_b] : 0.f;
    s_sum[lane] = s_sum[lane + 32] = 0.f;
    const int group_rows = now.rows * q.group, mine = now.tok0 + warp * 64;
    cp_async_wait<1>();
    __syncwarp();
    if (now.any) {
      for (int n0 = 0; n0 < group_rows; n0 += kRows) {
        const int n1 = min(n0 + kRows, group_rows), tiles_n = (n1 - n0 + 7) / 8;
        int lo0, hi0, lo1, hi1;  // what the first and the last of these rows see
        kv4_visible(mask, now.len - now.rows + n0 / q.group, now.len, lo0, hi0);
        kv4_visible(mask, now.len - now.rows + (n1 - 1) / q.group, now.len, lo1, hi1);
        if (lo0 >= now.tok0 + kWeightTokens || hi1 <= now.tok0) continue;
        if (q_b != now.b || q_h != now.h || group_rows > kRows) {
          __syncthreads();  // what was there has been read
          for (int i = tid; i < (D / 32) * tiles_n * 32; i += 128) {
            const int ln = i & 31, nt = (i >> 5) % tiles_n, blk = (i >> 5) / tiles_n;
            const int n = n0 + nt * 8 + (ln >> 2);
            uint4 x = make_uint4(0, 0, 0, 0);
            if (n < group_rows)
              x = __ldg(reinterpret_cast<const uint4*>(q.q + (now.first + n / q.group) * q.q_row +
                                                       (now.h * q.group + n % q.group) * q.q_head + 32 * blk + 8 * (ln & 3)));
            s_q[(2 * blk * kNT + nt) * 32 + ln] = make_uint2(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632));
            s_q[((2 * blk + 1) * kNT + nt) * 32 + ln] = make_uint2(__byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
          }
          if (tid < tiles_n * 8) {
            const int n = n0 + tid;
            float x = INFINITY;  // what gives weight zero: rows that are not there, or see nothing
            if (n < group_rows) {
              const float v = __ldg(lse + static_cast<long long>(now.first + n / q.group) * q.heads + now.h * q.group + n % q.group);
              if (v != -INFINITY) x = v * kLog2e;
            }
            s_lse[tid] = x;
          }
          __syncthreads();
          q_b = now.b;
          q_h = now.h;
        }
#pragma unroll 1
        for (int tile0 = 0; tile0 < 4; tile0 += kTT) {
          const int tb = mine + tile0 * 16;
          if (!((now.there >> tile0) & ((1u << kTT) - 1u)) || lo0 >= tb + 16 * kTT || hi1 <= tb) continue;
          const bool masked = lo1 > tb || hi0 < tb + 16 * kTT || ((now.there >> tile0) & ((1u << kTT) - 1u)) != (1u << kTT) - 1u;
          float sum[kTT][2] = {};
          // K of the tiles as A fragments: tokens g and g + 8
          uint32_t kf[kTT][kChunks][2][4];
#pragma unroll
          for (int tt = 0; tt < kTT; ++tt) {
            const int row = warp * 64 + (tile0 + tt) * 16;
            const uint32_t k_at = smem_u32(smem) + st * Cfg::kStage + (row + lm_tok) * (D / 2);
            const uint8_t* sr = smem + st * Cfg::kStage + Cfg::kK + (row + g) * kChunks;
            uint32_t f[2][kChunks];
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int i = 0; i < kChunks; i += 4) {
                uint32_t even, odd;
                const uint8_t* at = sr + half * 8 * kChunks + i;
                if constexpr (D == 64) kv4_scales_bf16<62>(*reinterpret_cast<const uint16_t*>(at), even, odd);
                else kv4_scales_bf16<62>(*reinterpret_cast<const uint32_t*>(at), even, odd);
                f[half][i] = __byte_perm(even, 0, 0x1010);
                f[half][i + 1] = __byte_perm(odd, 0, 0x1010);
                if constexpr (D > 64) {
                  f[half][i + 2] = __byte_perm(even, 0, 0x3232);
                  f[half][i + 3] = __byte_perm(odd, 0, 0x3232);
                }
              }
#pragma unroll
            for (int pair = 0; pair < kChunks / 2; ++pair) {
              uint32_t kw[4];
              ldmatrix_x4(kw, k_at + (((2 * pair + lm_ch) ^ lm_swz) * 16));
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int blk = 2 * pair + (i >> 1), half = i & 1;
                kf[tt][blk][half][0] = mul_bf16x2(kv4_raw<0>(kw[i]), f[half][blk]);
                kf[tt][blk][half][1] = mul_bf16x2(kv4_raw<1>(kw[i]), f[half][blk]);
                kf[tt][blk][half][2] = mul_bf16x2(kv4_raw<2>(kw[i]), f[half][blk]);
                kf[tt][blk][half][3] = mul_bf16x2(kv4_raw<3>(kw[i]), f[half][blk]);
              }
            }
          }
#pragma unroll 2
          for (int nt = 0; nt < tiles_n; ++nt) {
            float s[kTT][4];
#pragma unroll
            for (int tt = 0; tt < kTT; ++tt)
#pragma unroll
              for (int j = 0; j < 4; ++j) s[tt][j] = 0.f;
#pragma unroll
            for (int blk = 0; blk < kChunks; ++blk) {
              const uint2 b0 = s_q[(2 * blk * kNT + nt) * 32 + lane], b1 = s_q[((2 * blk + 1) * kNT + nt) * 32 + lane];
#pragma unroll
              for (int tt = 0; tt < kTT; ++tt) {
                mma_bf16_16816(s[tt], kf[tt][blk][0][0], kf[tt][blk][1][0], kf[tt][blk][0][1], kf[tt][blk][1][1], b0.x, b0.y);
                mma_bf16_16816(s[tt], kf[tt][blk][0][2], kf[tt][blk][1][2], kf[tt][blk][0][3], kf[tt][blk][1][3], b1.x, b1.y);
              }
            }
            const float2 ls = *reinterpret_cast<const float2*>(s_lse + nt * 8 + 2 * t);
#pragma unroll
            for (int tt = 0; tt < kTT; ++tt)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                float x;
                if (mask.softcap > 0.f) x = fmaf(kv4_cap(s[tt][j] * s_scale, mask.softcap, cap_k), kLog2e, (j & 1) ? -ls.y : -ls.x);
                else x = fmaf(s[tt][j], s_scale, (j & 1) ? -ls.y : -ls.x);
                if (masked) {
                  int lo, hi;
                  kv4_visible(mask, now.len - now.rows + (n0 + nt * 8 + 2 * t + (j & 1)) / q.group, now.len, lo, hi);
                  const int token = tb + tt * 16 + g + (j >> 1) * 8;
                  if (token < lo || token >= hi || !((now.there >> (tile0 + tt)) & 1)) x = -INFINITY;
                }
                sum[tt][j >> 1] += ex2(x);
              }
          }
#pragma unroll
          for (int tt = 0; tt < kTT; ++tt)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float x = sum[tt][half];
              x += __shfl_xor_sync(0xffffffffu, x, 1);
              x += __shfl_xor_sync(0xffffffffu, x, 2);
              if (t == 0) s_sum[(tile0 + tt) * 16 + half * 8 + g] += x;
            }
        }
      }
    }
    __syncwarp();  // sums are complete; K of this unit has been read: its stage takes the unit after the next
    if (has_a) w_out[at_a] = w_a + s_sum[lane];
    if (has_b) w_out[at_b] = w_b + s_sum[lane + 32];
  }
  cp_async_wait<0>();
}

}  // namespace b2g

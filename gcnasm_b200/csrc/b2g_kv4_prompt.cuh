// b2g_kv4_prompt.cuh -- attention of many query rows over the 4-bit cache, on tcgen05.
//
// A CTA has kNQ tiles of 128 query rows of one kv head (row = query token x heads of the
// group, so that the group's heads share what is read of the cache) and walks the cached
// tokens kN at a time:
//   S = Q K^T        tcgen05.mma, both operands in shared memory, S in TMEM
//   P = 2^(S - m)    one thread per row; P as two bf16 terms over S in TMEM
//   O += P V         tcgen05.mma, P from TMEM, V in shared memory with channels along its rows
// Warps: one softmax warpgroup per query tile, four warps that turn codes into bf16 tiles, one
// that issues the products.
//
// What bounds it: for D = 128 the products of a step take 3072 clocks at 4096 multiplications a
// clock, its 2 x 128 x 128 exponentials 2048 at 16 a clock, decoding 32768 codes ~700 issue slots a
// scheduler.  Hence two query tiles: while one's S is being exponentiated the other's products
// run, and what a step decodes serves 256 rows.  D = 256 leaves TMEM for one query tile, whose S
// has two buffers instead.
//
// Codes become bf16 as in the decode kernel (times 2^-64, exact), in the order 0 4 1 5 2 6 3 7 of
// each eight channels: Q is stored in the same order, O's columns are put back when written.
// What weights refer to, m, is a score of the row and moves only when weights become large (a
// chunk's sum above 2^20), so that O is rescaled in TMEM a few times per row, not once per step.
// A weight is the sum of two bf16 numbers, to 2^-17: rounded to one it would add as much error to
// the output as the output's own rounding.  That is a third of the products' time.
#pragma once

#include "b2g_kv4_decode.cuh"

namespace b2g {

template <int D>
struct PromptCfg {
  static constexpr int kNQ = D == 256 ? 1 : 2;
  static constexpr int kN = D == 256 ? 64 : 128;  // cached tokens of a step
  static constexpr int kSB = D == 256 ? 2 : 1;    // buffers of a query tile's S
  static constexpr int kRows = 128 * kNQ;
  static constexpr int kThreads = kNQ * 128 + 128 + 32;
  static constexpr int kQBytes = 128 * D * 2;
  static constexpr int kKBytes = kN * D * 2;
  static constexpr int kOffK = kNQ * kQBytes;
  static constexpr int kOffV = kOffK + 2 * kKBytes;
  static constexpr int kOffBar = kOffV + 2 * kKBytes;
  static constexpr int kBars = 1 + 8 + 2 * kNQ * kSB + 2 * kNQ + 1;
  static constexpr int kSmem = kOffBar + kBars * 8 + 16 + 1024;  // and room to align to 1024
  static constexpr uint32_t kColO = 256;  // S at column (tile * kSB + buffer) * kN, O here
};

// kind::f16 with bf16 operands, fp32 sums; b_mn: B's rows are along N (not K)
__host__ __device__ constexpr uint32_t idesc_bf16(uint32_t M, uint32_t N, uint32_t b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn << 16) | ((N >> 3) << 17) | ((M >> 4) << 24);
}

__device__ __forceinline__ void mma_bf16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_bf16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// packed fp32: (a0, a1) = (a0, a1) * k + c; (a0, a1) += (b0, b1); (a0, a1) -= (b0, b1)
__device__ __forceinline__ void fma2(float& a0, float& a1, float k, float c) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tmov.b64 c, {%3, %3};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(k), "f"(c));
}
__device__ __forceinline__ void add2(float& a0, float& a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "add.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(b0), "f"(b1));
}
__device__ __forceinline__ void sub2(float& a0, float& a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "sub.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(b0), "f"(b1));
}

__device__ __forceinline__ void mul2(float& a0, float& a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "mul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(b0), "f"(b1));
}
// (a0, a1) = (a0 * b0 + c0, a1 * b1 + c1)
__device__ __forceinline__ void fma2(float& a0, float& a1, float b0, float b1, float c0, float c1) {
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tmov.b64 c, {%4, %5};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}

// tanh x for |x| < 0.4 by the odd series (as kv4_cap), and by 1 - 2 / (e^2x + 1): to 2^-22
// absolutely, exact at both ends.  The series takes no special function, which bound the kernel.
__device__ __forceinline__ float kv4_tanh_near(float x) {
  const float y = x * x;
  float p = fmaf(y, -1382.f / 155925.f, 62.f / 2835.f);
  p = fmaf(y, p, -17.f / 315.f);
  p = fmaf(y, p, 2.f / 15.f);
  p = fmaf(y, p, -1.f / 3.f);
  return fmaf(x * y, p, x);
}
__device__ __forceinline__ void kv4_tanh_near2(float& x0, float& x1) {
  float y0 = x0, y1 = x1, p0 = -1382.f / 155925.f, p1 = p0;
  mul2(y0, y1, x0, x1);
  fma2(p0, p1, y0, y1, 62.f / 2835.f, 62.f / 2835.f);
  fma2(p0, p1, y0, y1, -17.f / 315.f, -17.f / 315.f);
  fma2(p0, p1, y0, y1, 2.f / 15.f, 2.f / 15.f);
  fma2(p0, p1, y0, y1, -1.f / 3.f, -1.f / 3.f);
  mul2(y0, y1, x0, x1);
  fma2(p0, p1, y0, y1, x0, x1);
  x0 = p0, x1 = p1;
}
__device__ __forceinline__ float kv4_tanh_far(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(ex2(x * (2.f * kLog2e)) + 1.f));
  return fmaf(r, -2.f, 1.f);
}

// bits [a, b) of a word
__device__ __forceinline__ uint32_t kv4_bits(int a, int b) {
  a = min(max(a, 0), 32);
  b = min(max(b, 0), 32);
  const uint32_t below_b = b == 32 ? 0xFFFFFFFFu : (1u << b) - 1u;
  const uint32_t below_a = a == 32 ? 0xFFFFFFFFu : (1u << a) - 1u;
  return below_b & ~below_a;
}

template <int D, bool kCap>
__global__ void __launch_bounds__(PromptCfg<D>::kThreads, 1)
b2g_kv4_prompt_kernel(Kv4Cache c, Kv4Batch bt, Kv4Mask mask, Kv4Queries q, Kv4Out out, uint64_t timeout_ns, int* status) {
  using Cfg = PromptCfg<D>;
  constexpr int kNQ = Cfg::kNQ, kN = Cfg::kN, kSB = Cfg::kSB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;
  uint64_t* k_empty = bars + 3;
  uint64_t* v_full = bars + 5;
  uint64_t* v_empty = bars + 7;
  uint64_t* s_full = bars + 9;                // [tile][buffer]
  uint64_t* p_full = s_full + kNQ * kSB;
  uint64_t* o_done = p_full + kNQ * kSB;      // [tile]: a step's O
  uint64_t* o_last = o_done + kNQ;            // [tile]: the last step's
  uint64_t* fin = o_last + kNQ;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + Cfg::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kDecodeWarp = 4 * kNQ, kMmaWarp = kDecodeWarp + 4;

  griddep_wait();
  const int h = blockIdx.x, b = blockIdx.y;
  int first, end;
  kv4_rows(bt, b, first, end);
  const int rows = end - first, len = kv4_len(bt, b, c.page_log2), group_rows = rows * q.group;
  // the last blocks see most: they come first
  const int blk = (group_rows + Cfg::kRows - 1) / Cfg::kRows - 1 - static_cast<int>(blockIdx.z);
  if (blk < 0) return;
  const int r0 = blk * Cfg::kRows, r1 = min(r0 + Cfg::kRows, group_rows) - 1;
  int lo0, hi1, unused;
  kv4_visible(mask, len - rows + r0 / q.group, len, lo0, unused);
  kv4_visible(mask, len - rows + r1 / q.group, len, unused, hi1);
  const int j0 = lo0 / kN, steps = max(0, (hi1 + kN - 1) / kN - j0);
  const int* pages = bt.table + static_cast<long long>(b) * bt.width;

  if (threadIdx.x == 0) {
    mbar_init(q_full, kNQ * 128);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 128);
      mbar_init(&v_full[i], 128);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < kNQ * kSB; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
    }
    for (int i = 0; i < kNQ; ++i) {
      mbar_init(&o_done[i], 1);
      mbar_init(&o_last[i], 1);
    }
    mbar_init(fin, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) tmem_alloc<512>(tmem_holder);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp < kDecodeWarp) {
    // ---------------------------------------------------------------- softmax: one thread per row
    const int tile = warp >> 2, in_tile = threadIdx.x & 127;
    const int r = r0 + tile * 128 + in_tile;
    const bool real = r < group_rows;
    const int row = first + r / q.group, head = h * q.group + r % q.group;
    {  // Q, in the codes' channel order; a negative scale goes to its signs
      const uint32_t flip = mask.scale < 0.f ? 0x80008000u : 0u;
      uint8_t* dst = smem + tile * Cfg::kQBytes + in_tile * 128;
      const uint4* src = reinterpret_cast<const uint4*>(q.q + row * q.q_row + head * q.q_head);
#pragma unroll 8
      for (int i = 0; i < D / 8; ++i) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (real) x = __ldg(src + i);
        x = make_uint4(__byte_perm(x.x, x.z, 0x5410) ^ flip, __byte_perm(x.x, x.z, 0x7632) ^ flip,
                       __byte_perm(x.y, x.w, 0x5410) ^ flip, __byte_perm(x.y, x.w, 0x7632) ^ flip);
        *reinterpret_cast<uint4*>(dst + (i >> 3) * (128 * 128) + (((i & 7) ^ (in_tile & 7)) << 4)) = x;
      }
      fence_proxy_async_smem();
      mbar_arrive(q_full);
    }
    int lo, hi;
    kv4_visible(mask, len - rows + r / q.group, len, lo, hi);
    const float scale = fabsf(mask.scale) * kTwo64;
    // with a cap: tanh's argument.  Not zero, so that -inf stays that
    const float s_scale = fmaxf(kCap ? scale / mask.softcap : scale * kLog2e, 1.2e-38f);
    const float cap2 = kCap ? mask.softcap * kLog2e : 0.f;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    float m = -1e30f, l0 = 0.f, l1 = 0.f;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {  // all lanes go on, or none: what follows is the warp's
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, kDevTimeoutEpilogue, timeout_ns)) != 0;
    };
    for (int i = 0; i < steps && ok; ++i) {
      const int tb = (j0 + i) * kN;
      // which groups of 16 tokens have a page
      uint32_t there;
      {
        const int token = tb + lane * 16;
        bool t = false;
        if (lane < kN / 16 && token < len) t = static_cast<unsigned>(__ldg(pages + (token >> c.page_log2))) < static_cast<unsigned>(c.pages);
        there = __ballot_sync(0xffffffffu, t);
      }
      const int buf = kSB == 2 ? i & 1 : 0;
      const uint32_t parity = kSB == 2 ? (i >> 1) & 1 : i & 1;
      const uint32_t s_at = tmem + lanes + (tile * kSB + buf) * kN;
      const uint32_t o_at = tmem + lanes + Cfg::kColO + tile * D;
      const bool masked = __any_sync(0xffffffffu, tb < lo || tb + kN > hi) || there != (1u << (kN / 16)) - 1u;
      if (!(ok = wait(&s_full[tile * kSB + buf], parity))) break;
      tc_fence_after();
      auto seen = [&](int col) {  // bits of 32 columns from col
        const uint32_t pages16 = ((there >> (col >> 4)) & 1u ? 0xFFFFu : 0u) | ((there >> ((col >> 4) + 1)) & 1u ? 0xFFFF0000u : 0u);
        return kv4_bits(lo - tb - col, hi - tb - col) & pages16;
      };
      // S is read once, 32 columns ahead of the ones worked on; a chunk whose weights sum to more than
      // 2^20 moves m and is done again.
      // What is rare (and the two halves' loop) stays rolled: three kinds of warps share the
      // instruction cache.
      auto raise = [&](float top, bool need, int upto) {  // columns before `upto` hold weights already
        // m moves by a whole number, so that weights are rescaled exactly
        const bool fresh = m < -1e29f;
        const float up = fresh || !need ? 0.f : ceilf(top - m);
        const float f = fresh && need ? 0.f : __int_as_float(max(127 - static_cast<int>(fminf(up, 127.f)), 0) << 23);
        m = fresh && need ? top : m + up;
        l0 *= f;
        l1 *= f;
        // one buffer of S: step i's products came after step i - 1's in the pipe.  Two: they may have
        // come before, but after step i - 2's, so the barrier is in phase i - 1 or just past it
        if (kSB == 2 && i > 0 && !(ok = wait(&o_done[tile], (i - 1) & 1))) return;
        tc_fence_after();
#pragma unroll 1
        for (int col = 0; i > 0 && col < D; col += 32) {
          uint32_t x[32];
          tmem_ld_32x32b_x32(o_at + col, x);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
          tmem_st_32x32b_x32(o_at + col, x);
        }
        tc_wait_st();
#pragma unroll 1
        for (int col = 0; col < upto; col += 32) {
          uint32_t x[32];
          tmem_ld_32x32b_x32(s_at + col, x);
          tc_wait_ld();
          const uint32_t f2 = __byte_perm(__float_as_uint(f), 0, 0x3232);  // a power of two: exact as bf16
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = mul_bf16x2(x[e], f2);
          tmem_st_32x32b_x32(s_at + col, x);
        }
      };
      auto chunk = [&](uint32_t (&x)[32], int col) {
        uint32_t bits = 0;
        if (masked) {
          bits = seen(col);
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = (bits >> e) & 1u ? x[e] : 0xFF800000u;
        }
        if (kCap) {
          float far = 0.f;
#pragma unroll
          for (int e = 0; e < 32; ++e) far = fmaxf(far, fabsf(__uint_as_float(x[e])));
          const bool near = __all_sync(0xffffffffu, far * s_scale < 0.4f);  // the series serves (a NaN is not near)
          if (near) {
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float y0 = __uint_as_float(x[e]), y1 = __uint_as_float(x[e + 1]);
              mul2(y0, y1, s_scale, s_scale);
              kv4_tanh_near2(y0, y1);
              x[e] = __float_as_uint(y0), x[e + 1] = __float_as_uint(y1);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              x[e] = __float_as_uint(kv4_tanh_far(__uint_as_float(x[e]) * s_scale));
              if (masked && !((bits >> e) & 1u)) x[e] = 0xFF800000u;
            }
          }
        }
        const float k = kCap ? cap2 : s_scale;
        uint32_t pk[32];
        float c0, c1;
        // weights of the chunk, first terms to its first 16 columns, second terms to the others
        auto weigh = [&]() {
          c0 = c1 = 0.f;
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float y0 = __uint_as_float(x[e]), y1 = __uint_as_float(x[e + 1]);
            fma2(y0, y1, k, -m);
            y0 = ex2(y0);
            y1 = ex2(y1);
            add2(c0, c1, y0, y1);
            const uint32_t p = pack_bf16x2(y0, y1);
            sub2(y0, y1, __uint_as_float(p << 16), __uint_as_float(p & 0xFFFF0000u));
            pk[e >> 1] = p;
            pk[16 + (e >> 1)] = pack_bf16x2(y0, y1);
          }
        };
        weigh();
        // the sum tells, without a maximum for each element, that a weight has become too large
        if (__any_sync(0xffffffffu, c0 + c1 > 1048576.f)) {
          float top = -INFINITY;
#pragma unroll
          for (int e = 0; e < 32; ++e) top = fmaxf(top, __uint_as_float(x[e]));
          raise(top * k, top * k > m, col);
          weigh();
        }
        add2(l0, l1, c0, c1);
        tmem_st_32x32b_x32(s_at + col, pk);  // over the columns just read
      };
      uint32_t xa[32], xb[32];
      tmem_ld_32x32b_x32(s_at, xa);
#pragma unroll 1
      for (int col = 0; col < kN && ok; col += 64) {
        tc_wait_ld();
        tmem_ld_32x32b_x32(s_at + col + 32, xb);
        chunk(xa, col);
        tc_wait_ld();
        if (col + 64 < kN) tmem_ld_32x32b_x32(s_at + col + 64, xa);
        chunk(xb, col + 32);
      }
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[tile * kSB + buf]);
    }
    // ---- output
    const float l = l0 + l1;
    if (steps > 0 && ok) ok = wait(&o_last[tile], 0);
    if (ok) {
      tc_fence_after();
      const float f = l == 0.f ? 0.f : kTwo64 / l;
      uint8_t* dst = reinterpret_cast<uint8_t*>(out.out + row * out.row + head * out.head);
#pragma unroll 1
      for (int col = 0; col < D; col += 32) {
        uint32_t x[32];
        if (steps > 0) {
          tmem_ld_32x32b_x32(tmem + lanes + Cfg::kColO + tile * D + col, x);
          tc_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = l == 0.f ? 0u : __float_as_uint(__uint_as_float(x[e]) * f);
        if (real) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // columns 0 .. 7 hold channels 0 4 1 5 2 6 3 7
            auto two = [&](int a, int d) { return pack_bf16x2(__uint_as_float(x[8 * i + a]), __uint_as_float(x[8 * i + d])); };
            *reinterpret_cast<uint4*>(dst + (col + 8 * i) * 2) = make_uint4(two(0, 2), two(4, 6), two(1, 3), two(5, 7));
          }
        }
      }
      if (real) out.lse[static_cast<long long>(row) * q.heads + head] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
    }
  } else if (warp < kMmaWarp) {
    // ---------------------------------------------------------------- codes to bf16 tiles
    // K of a step, then V, by the same code: halves are fetched one ahead, page numbers a step ahead
    constexpr int kWords = D == 64 ? 8 : 16;  // a thread's words of a half
    const int dt = threadIdx.x - kDecodeWarp * 32, tok = dt % kN, part = dt / kN;  // a warp's lanes: consecutive tokens
    auto page_of = [&](int i) {
      const int token = (j0 + i) * kN + tok;
      return i < steps && token < len ? __ldg(pages + (token >> c.page_log2)) : -2;
    };
    // a step's token among all, -1 where it is not there
    auto token_of = [&](int i, int page) {
      const bool there = static_cast<unsigned>(page) < static_cast<unsigned>(c.pages);
      if (!there && page != -2) atomicCAS(status, 0, kDevBadPage);
      const int token = (j0 + i) * kN + tok;
      return there ? ((static_cast<long long>(page) * c.heads + h) << c.page_log2) + (token & ((1 << c.page_log2) - 1)) : -1ll;
    };
    auto fetch = [&](uint4 (&x)[kWords / 4], uint32_t& scales, const uint8_t* codes, const uint8_t* bytes, long long at) {
      scales = 0;
#pragma unroll
      for (int n = 0; n < kWords / 4; ++n) x[n] = make_uint4(0, 0, 0, 0);
      if (at < 0) return;
#pragma unroll
      for (int n = 0; n < kWords / 4; ++n) x[n] = *(reinterpret_cast<const uint4*>(codes + at * (D / 2) + part * 64) + n);
      if constexpr (D == 64) scales = *reinterpret_cast<const uint16_t*>(bytes + at * 2);
      else scales = *(reinterpret_cast<const uint32_t*>(bytes + at * (D / 32)) + part);
    };
    bool ok = true;
    uint4 now[kWords / 4], next[kWords / 4];
    uint32_t now_s, next_s;
    int page = page_of(0);
    long long at = steps > 0 ? token_of(0, page) : -1;
    fetch(now, now_s, c.k, c.ks, at);
    page = page_of(1);
#pragma unroll 1
    for (int i2 = 0; i2 < 2 * steps && ok; ++i2) {
      const int i = i2 >> 1, st = i & 1;
      const bool is_v = i2 & 1;
      if (is_v) {
        at = i + 1 < steps ? token_of(i + 1, page) : -1;
        page = page_of(i + 2);
      }
      fetch(next, next_s, is_v ? c.k : c.v, is_v ? c.ks : c.vs, at);
      uint64_t* empty = is_v ? &v_empty[st] : &k_empty[st];
      if (!mbar_wait(empty, ((i >> 1) & 1) ^ 1, abort_flag, status, kDevTimeoutProducer, timeout_ns)) { ok = false; break; }
      // a thread's channels of one token: words of eight codes to 16-byte pieces of 128-byte swizzled rows
      uint8_t* tile = smem + (is_v ? Cfg::kOffV : Cfg::kOffK) + st * Cfg::kKBytes + tok * 128;
      uint32_t even, odd;
      kv4_scales_bf16<62>(now_s, even, odd);
#pragma unroll
      for (int n = 0; n < kWords / 4; ++n) {
        const uint32_t f = __byte_perm(n & 1 ? odd : even, 0, n & 2 ? 0x3232 : 0x1010);
        const uint32_t w[4] = {now[n].x, now[n].y, now[n].z, now[n].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int piece = part * 16 + n * 4 + e;
          *reinterpret_cast<uint4*>(tile + (piece >> 3) * (kN * 128) + (((piece & 7) ^ (tok & 7)) << 4)) =
              make_uint4(mul_bf16x2(kv4_raw<0>(w[e]), f), mul_bf16x2(kv4_raw<1>(w[e]), f), mul_bf16x2(kv4_raw<2>(w[e]), f),
                         mul_bf16x2(kv4_raw<3>(w[e]), f));
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(is_v ? &v_full[st] : &k_full[st]);
#pragma unroll
      for (int n = 0; n < kWords / 4; ++n) now[n] = next[n];
      now_s = next_s;
    }
  } else {
    // ---------------------------------------------------------------- products
    if (lane == 0 && steps > 0) {
      constexpr uint32_t kIdQK = idesc_bf16(128, kN, 0), kIdPV = idesc_bf16(128, D, 1);
      auto qk = [&](int tile, int i) {
        const uint32_t d = tmem + (tile * kSB + (kSB == 2 ? i & 1 : 0)) * kN;
        const uint32_t a = smem_u32(smem + tile * Cfg::kQBytes), bk = smem_u32(smem + Cfg::kOffK + (i & 1) * Cfg::kKBytes);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_bf16_ss(d, desc_kmajor_sw128(a + (k >> 2) * (128 * 128) + (k & 3) * 32),
                      desc_kmajor_sw128(bk + (k >> 2) * (kN * 128) + (k & 3) * 32), kIdQK, k > 0);
      };
      auto pv = [&](int tile, int i) {
        const uint32_t a = tmem + (tile * kSB + (kSB == 2 ? i & 1 : 0)) * kN, d = tmem + Cfg::kColO + tile * D;
        const uint32_t bv = smem_u32(smem + Cfg::kOffV + (i & 1) * Cfg::kKBytes);
        // channels along the rows: 64 of them in 128 bytes, the next 64 kN rows on; eight tokens a kilobyte.
        // P: 32 tokens' first terms in 16 columns, their second terms in the next 16
#pragma unroll
        for (int k = 0; k < kN / 16; ++k) {
          const uint64_t bd = smem_desc(bv + k * 2048, kN * 128, 1024, kLayoutSW128);
          const uint32_t ak = a + (k >> 1) * 32 + (k & 1) * 8;
          mma_bf16_ts(d, ak, bd, kIdPV, i > 0 || k > 0);
          mma_bf16_ts(d, ak + 16, bd, kIdPV, 1);
        }
      };
      auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, abort_flag, status, kDevTimeoutMma, timeout_ns); };
      bool ok = wait(q_full, 0) && wait(&k_full[0], 0);
      if (ok) {
        for (int tile = 0; tile < kNQ; ++tile) {
          qk(tile, 0);
          tc_commit(&s_full[tile * kSB]);
        }
        tc_commit(&k_empty[0]);
      }
      for (int i = 0; i < steps && ok; ++i) {
        const int st = i & 1, nx = (i + 1) & 1;
        const bool more = i + 1 < steps;
        if (kSB == 2 && more) {
          if (!(ok = wait(&k_full[nx], ((i + 1) >> 1) & 1))) break;
          qk(0, i + 1);
          tc_commit(&s_full[nx]);
          tc_commit(&k_empty[nx]);
        }
        if (!(ok = wait(&v_full[st], (i >> 1) & 1))) break;
        for (int tile = 0; tile < kNQ; ++tile) {
          if (!(ok = wait(&p_full[tile * kSB + (kSB == 2 ? st : 0)], kSB == 2 ? (i >> 1) & 1 : i & 1))) break;
          tc_fence_after();
          pv(tile, i);
          tc_commit(more ? &o_done[tile] : &o_last[tile]);
          if (tile == kNQ - 1) tc_commit(&v_empty[st]);
          if (kSB == 1 && more) {
            if (tile == 0 && !(ok = wait(&k_full[nx], ((i + 1) >> 1) & 1))) break;
            qk(tile, i + 1);
            tc_commit(&s_full[tile]);
            if (tile == kNQ - 1) tc_commit(&k_empty[nx]);
          }
        }
      }
      // nothing may be in flight when TMEM is given back
      tc_commit(fin);
      volatile int no_abort = 0;
      mbar_wait(fin, 0, &no_abort, status, kDevTimeoutDrain, 1000000000ull);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc<512>(tmem);
}

}  // namespace b2g

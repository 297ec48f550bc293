// b2g_kv4.cuh -- the 4-bit key/value cache: addressing, appending, reading back and
// eviction.  K and V are MXFP4 (E2M1 codes, one UE8M0 scale per 32 channels) in pages.
#pragma once

#include <cuda_bf16.h>

#include <cstdint>
#include <type_traits>

#include "b2g_elem.cuh"
#include "b2g_ptx.cuh"

namespace b2g {

constexpr int kDevBadPage = 5;    // B2G_DEV_BAD_PAGE
constexpr int kKv4ScaleMin = 67;  // B2G_KV4_SCALE_MIN: 2^-60
constexpr int kKv4ScaleMax = 192;  // B2G_KV4_SCALE_MAX: 2^65

struct Kv4Cache {
  uint8_t* k;
  uint8_t* v;
  uint8_t* ks;
  uint8_t* vs;
  int pages, heads, page_log2;
};

struct Kv4Batch {
  const int* table;
  const int* lens;
  const int* cu;  // null: row b belongs to sequence b
  int seqs, width, rows;
};

// Rows [first, end) of sequence b, cut to the rows there are.
__device__ __forceinline__ void kv4_rows(const Kv4Batch& bt, int b, int& first, int& end) {
  if (!bt.cu) {
    first = b;
    end = b + 1;
    return;
  }
  first = min(max(__ldg(bt.cu + b), 0), bt.rows);
  end = min(max(__ldg(bt.cu + b + 1), first), bt.rows);
}

// Cached tokens of sequence b, cut to what its page table can hold.
__device__ __forceinline__ int kv4_len(const Kv4Batch& bt, int b, int page_log2) {
  return static_cast<int>(min(static_cast<long long>(max(__ldg(bt.lens + b), 0)),
                              static_cast<long long>(bt.width) << page_log2));
}

// The sequence that row r belongs to: the last b with cu[b] <= r.
__device__ __forceinline__ int kv4_seq_of_row(const Kv4Batch& bt, int r) {
  if (!bt.cu) return r;
  int lo = 0, hi = bt.seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(bt.cu + mid) <= r) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Index of (page, head, slot) among all tokens of the cache, -1 where the table names no
// page of the cache (the status word says so then).  64 bits: a cache passes 2^31 tokens x heads.
__device__ __forceinline__ long long kv4_token(const Kv4Cache& c, const int* table_row, int head, int token,
                                               int* status) {
  const int page = __ldg(table_row + (token >> c.page_log2));
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(c.pages)) {
    atomicCAS(status, 0, kDevBadPage);
    return -1;
  }
  return ((static_cast<long long>(page) * c.heads + head) << c.page_log2) + (token & ((1 << c.page_log2) - 1));
}

// Least power of two s with 6 s >= amax, as a UE8M0 byte clamped to the cache's range.
// amax = 1.m x 2^E: s = 2^(E - 2) when 1.m <= 1.5, else 2^(E - 1); zeros, subnormals and
// infinity land on the clamps.
__device__ __forceinline__ int kv4_scale_byte(float amax) {
  const int bits = __float_as_int(amax) & 0x7FFFFFFF;
  const int byte = (bits >> 23) - 2 + ((bits & 0x7FFFFF) > 0x400000 ? 1 : 0);
  return min(max(byte, kKv4ScaleMin), kKv4ScaleMax);
}

// ---------------------------------------------------------------------------
// append: one thread per 8 channels, four threads per scale block.  A row of a batch is
// K and V of every head: 2 * heads * D / 8 threads, so a warp reads 512 consecutive bytes
// (bf16) and writes 128.  Bound by the input's bytes (bf16: 4 of the 5.06 bytes moved per value pair).
// ---------------------------------------------------------------------------
template <typename In, int D>
__global__ void __launch_bounds__(256)
b2g_kv4_append_kernel(Kv4Cache c, Kv4Batch bt, const In* __restrict__ k, const In* __restrict__ v, long long k_row,
                      long long k_head, long long v_row, long long v_head, float* __restrict__ weights,
                      int* status) {
  constexpr int kPer = D / 8;  // threads of one head's K or V
  const int per_row = 2 * c.heads * kPer;
  const long long total = static_cast<long long>(bt.rows) * per_row;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i - (threadIdx.x & 31) < total; i += gridDim.x * 256ll) {
    const bool live = i < total;
    const int row = live ? static_cast<int>(i / per_row) : 0;
    const int in = static_cast<int>(i - static_cast<long long>(row) * per_row);
    const int hv = in / kPer, g = in % kPer;
    const bool is_v = hv >= c.heads;
    const int head = is_v ? hv - c.heads : hv;
    float x[8] = {};
    if (live) load8_f32((is_v ? v + row * v_row + head * v_head : k + row * k_row + head * k_head) + g * 8, x);
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[j]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    if (!live) continue;
    const int b = kv4_seq_of_row(bt, row);
    int first, end;
    kv4_rows(bt, b, first, end);
    const int len = kv4_len(bt, b, c.page_log2);
    const int token = __ldg(bt.lens + b) - (end - row);
    if (row < first || row >= end || token < 0 || token >= len) continue;
    const long long at = kv4_token(c, bt.table + static_cast<long long>(b) * bt.width, head, token, status);
    if (at < 0) continue;
    const int byte = kv4_scale_byte(amax);
    const float inv = __int_as_float((254 - byte) << 23);  // 2^(127 - byte), exact
    uint32_t pk = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) pk |= f32_to_e2m1(x[j] * inv) << (4 * j);
    *reinterpret_cast<uint32_t*>((is_v ? c.v : c.k) + at * (D / 2) + g * 4) = pk;
    if ((g & 3) == 0) (is_v ? c.vs : c.ks)[at * (D / 32) + (g >> 2)] = static_cast<uint8_t>(byte);
    if (weights && !is_v && g == 0) weights[at] = 0.f;
  }
}

// Value of code `n` (its low four bits): 2^(e - 1) (1 + m / 2), or m / 2 for e = 0.
__device__ __forceinline__ float kv4_code_value(uint32_t n) {
  // e and m placed as an fp32 exponent and top mantissa bit: the value times 2^-126 (a
  // subnormal for e = 0), which the multiplication makes exact and normal again
  return __uint_as_float(((n & 8u) << 28) | ((n & 7u) << 22)) * __int_as_float((126 + 127) << 23);
}

__device__ __forceinline__ float kv4_scale_value(int byte) {
  return __int_as_float(min(max(byte, kKv4ScaleMin), kKv4ScaleMax) << 23);
}

// read: one thread per 8 channels of K or V.  The output's bf16 values are the bound
// (4 of 5.06 bytes per value pair).
template <int D>
__global__ void __launch_bounds__(256)
b2g_kv4_read_kernel(Kv4Cache c, Kv4Batch bt, const int* __restrict__ start, __nv_bfloat16* __restrict__ k,
                    __nv_bfloat16* __restrict__ v, int* status) {
  constexpr int kPer = D / 8;
  const long long per_kv = static_cast<long long>(bt.rows) * c.heads * kPer;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < 2 * per_kv; i += gridDim.x * 256ll) {
    const bool is_v = i >= per_kv;
    const long long o = is_v ? i - per_kv : i;
    const int g = static_cast<int>(o % kPer);
    const long long rh = o / kPer;
    const int row = static_cast<int>(rh / c.heads), head = static_cast<int>(rh - static_cast<long long>(row) * c.heads);
    const int b = kv4_seq_of_row(bt, row);
    int first, end;
    kv4_rows(bt, b, first, end);
    const long long token = static_cast<long long>(__ldg(start + b)) + row - first;
    long long at = -1;
    if (row >= first && row < end && token >= 0 && token < (static_cast<long long>(bt.width) << c.page_log2))
      at = kv4_token(c, bt.table + static_cast<long long>(b) * bt.width, head, static_cast<int>(token), status);
    uint32_t w[4] = {};
    if (at >= 0) {
      const uint32_t codes = __ldg(reinterpret_cast<const uint32_t*>((is_v ? c.v : c.k) + at * (D / 2)) + g);
      const float s = kv4_scale_value(__ldg((is_v ? c.vs : c.ks) + at * (D / 32) + (g >> 2)));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = pack_bf16x2(kv4_code_value(codes >> (8 * j)) * s, kv4_code_value(codes >> (8 * j + 4)) * s);
    }
    *reinterpret_cast<uint4*>((is_v ? v : k) + o * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ---------------------------------------------------------------------------
// evict, first half: the tokens that stay, per sequence and kv head.
// ---------------------------------------------------------------------------
// Order of weights as unsigned numbers: NaN lowest, -0 = +0.
__device__ __forceinline__ uint32_t kv4_rank(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kEvictThreads = 1024;

// One CTA per (sequence, kv head).  Radix selection over the weights of the tokens between
// the first `sink` and the last `recent`: three passes of 11, 11 and 10 bits find the rank
// `cut` of the last one kept and how many of that rank are, then a pass in token order
// writes the kept numbers.
__global__ void __launch_bounds__(kEvictThreads)
b2g_kv4_select_kernel(Kv4Cache c, Kv4Batch bt, const float* __restrict__ weights, int budget, int sink, int recent,
                      int* __restrict__ kept, int* status) {
  __shared__ int hist[2048];
  __shared__ int warp_sum[32], warp_sum2[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int h = blockIdx.x % c.heads, b = blockIdx.x / c.heads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = kv4_len(bt, b, c.page_log2);
  const int* row = bt.table + static_cast<long long>(b) * bt.width;
  int* out = kept + (static_cast<long long>(b) * c.heads + h) * budget;
  if (len <= budget) {
    for (int i = tid; i < budget; i += kEvictThreads) out[i] = i < len ? i : -1;
    return;
  }
  const int lo = sink, hi = len - recent;  // sink + recent <= budget < len
  int need = budget - sink - recent;
  uint32_t prefix = 0;  // the bits of `cut` found so far
  if (need > 0) {
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const int bits = pass == 2 ? 10 : 11;
      for (int i = tid; i < 2048; i += kEvictThreads) hist[i] = 0;
      __syncthreads();
      for (int j = lo + tid; j < hi; j += kEvictThreads) {
        const long long at = kv4_token(c, row, h, j, status);
        const uint32_t r = at < 0 ? 0u : kv4_rank(weights[at]);
        if (pass == 0 || (r >> (shift + bits)) == prefix) atomicAdd(&hist[(r >> shift) & ((1 << bits) - 1)], 1);
      }
      __syncthreads();
      // two bins a thread, from the top: how many lie above
      const int n_bins = 1 << bits;
      const int top = n_bins - 1 - 2 * tid;
      const int c0 = top >= 1 ? hist[top] : 0, c1 = top >= 1 ? hist[top - 1] : 0;
      int sum = c0 + c1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += t;
      }
      if (lane == 31) warp_sum[warp] = sum;
      __syncthreads();
      int above = sum - c0 - c1;
      for (int w = 0; w < warp; ++w) above += warp_sum[w];
      if (top >= 1) {
        if (above < need && above + c0 >= need) {
          s_prefix = (prefix << bits) | static_cast<uint32_t>(top);
          s_need = need - above;
        } else if (above + c0 < need && above + c0 + c1 >= need) {
          s_prefix = (prefix << bits) | static_cast<uint32_t>(top - 1);
          s_need = need - above - c0;
        }
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;
    }
  }
  const uint32_t cut = prefix;
  const bool any = budget - sink - recent > 0;
  // in token order: kept is what ranks above `cut`, and the first `need` of rank `cut`
  int n_kept = 0, n_tied = 0;
  for (int base = 0; base < len; base += kEvictThreads) {
    const int j = base + tid;
    bool keep = false, tied = false;
    if (j < len) {
      if (j < lo || j >= hi) {
        keep = true;
      } else if (any) {
        const long long at = kv4_token(c, row, h, j, status);
        const uint32_t r = at < 0 ? 0u : kv4_rank(weights[at]);
        keep = r > cut;
        tied = r == cut;
      }
    }
    const uint32_t below = (1u << lane) - 1u;
    const uint32_t tm = __ballot_sync(0xffffffffu, tied);
    if (lane == 0) warp_sum2[warp] = __popc(tm);
    __syncthreads();
    int before = n_tied, all = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) before += warp_sum2[w];
      all += warp_sum2[w];
    }
    n_tied += all;
    if (tied && before + __popc(tm & below) < need) keep = true;
    const uint32_t km = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) warp_sum[warp] = __popc(km);
    __syncthreads();
    int at_out = n_kept;
    all = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) at_out += warp_sum[w];
      all += warp_sum[w];
    }
    n_kept += all;
    if (keep) out[at_out + __popc(km & below)] = j;
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// evict, second half: the kept tokens move to tokens 0, 1, ... of the output pages.
// A token is D / 16 pieces of 16 bytes (K, then V) and one piece with its scales and weight.
// ---------------------------------------------------------------------------
template <int D>
struct Kv4Piece {
  uint4 codes;
  uint64_t ks, vs;
  float w;
  __device__ __forceinline__ void load(const Kv4Cache& c, const float* weights, long long at, int piece) {
    constexpr int kHalf = D / 32;
    if (piece < kHalf) codes = *reinterpret_cast<const uint4*>(c.k + at * (D / 2) + piece * 16);
    else if (piece < 2 * kHalf) codes = *reinterpret_cast<const uint4*>(c.v + at * (D / 2) + (piece - kHalf) * 16);
    else {
      using S = typename std::conditional<D == 64, uint16_t, typename std::conditional<D == 128, uint32_t, uint64_t>::type>::type;
      ks = *reinterpret_cast<const S*>(c.ks + at * (D / 32));
      vs = *reinterpret_cast<const S*>(c.vs + at * (D / 32));
      w = weights[at];
    }
  }
  __device__ __forceinline__ void store(const Kv4Cache& c, float* weights, long long at, int piece) const {
    constexpr int kHalf = D / 32;
    if (piece < kHalf) *reinterpret_cast<uint4*>(c.k + at * (D / 2) + piece * 16) = codes;
    else if (piece < 2 * kHalf) *reinterpret_cast<uint4*>(c.v + at * (D / 2) + (piece - kHalf) * 16) = codes;
    else {
      using S = typename std::conditional<D == 64, uint16_t, typename std::conditional<D == 128, uint32_t, uint64_t>::type>::type;
      *reinterpret_cast<S*>(c.ks + at * (D / 32)) = static_cast<S>(ks);
      *reinterpret_cast<S*>(c.vs + at * (D / 32)) = static_cast<S>(vs);
      weights[at] = w;
    }
  }
};

// To other pages: any order, one thread per piece.
template <int D>
__global__ void __launch_bounds__(256)
b2g_kv4_move_kernel(Kv4Cache c, Kv4Batch bt, float* weights, int budget, const int* __restrict__ out_table,
                    int out_width, const int* __restrict__ kept, int* new_lens, int* status) {
  constexpr int kPieces = D / 16 + 1;
  const long long total = static_cast<long long>(bt.seqs) * c.heads * budget * kPieces;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long t = i / kPieces;
    const int piece = static_cast<int>(i - t * kPieces);
    const long long bh = t / budget;
    const int slot = static_cast<int>(t - bh * budget);
    const int b = static_cast<int>(bh / c.heads), h = static_cast<int>(bh - static_cast<long long>(b) * c.heads);
    if (slot == 0 && piece == 0 && h == 0) new_lens[b] = min(kv4_len(bt, b, c.page_log2), budget);
    const int j = __ldg(kept + t);
    if (j < 0) continue;
    const long long from = kv4_token(c, bt.table + static_cast<long long>(b) * bt.width, h, j, status);
    const long long to = kv4_token(c, out_table + static_cast<long long>(b) * out_width, h, slot, status);
    if (from < 0 || to < 0) continue;
    Kv4Piece<D> p;
    p.load(c, weights, from, piece);
    p.store(c, weights, to, piece);
  }
}

// In place: one CTA per (sequence, kv head) moves the tokens in order, a batch at a time.
// Token i comes from kept[i] >= i, and kept ascends: when a batch's sources have been read,
// its destinations hold nothing that is still to be read.
template <int D>
__global__ void __launch_bounds__(1024)
b2g_kv4_move_in_place_kernel(Kv4Cache c, Kv4Batch bt, float* weights, int budget, const int* __restrict__ kept,
                             int* new_lens, int* status) {
  constexpr int kPieces = D / 16 + 1;
  constexpr int kTokens = 1024 / kPieces;
  const int h = blockIdx.x % c.heads, b = blockIdx.x / c.heads;
  const int* row = bt.table + static_cast<long long>(b) * bt.width;
  const int* mine = kept + (static_cast<long long>(b) * c.heads + h) * budget;
  const int piece = threadIdx.x % kPieces, sub = threadIdx.x / kPieces;
  for (int base = 0; base < budget; base += kTokens) {
    const int slot = base + sub;
    long long from = -1, to = -1;
    Kv4Piece<D> p;
    if (sub < kTokens && slot < budget) {
      const int j = __ldg(mine + slot);
      if (j > slot) {
        from = kv4_token(c, row, h, j, status);
        to = kv4_token(c, row, h, slot, status);
      }
      if (from >= 0 && to >= 0) p.load(c, weights, from, piece);
    }
    __syncthreads();
    if (from >= 0 && to >= 0) p.store(c, weights, to, piece);
    __syncthreads();
  }
  // lens may be new_lens: this thread alone reads and writes it
  if (threadIdx.x == 0 && h == 0) new_lens[b] = min(kv4_len(bt, b, c.page_log2), budget);
}

}  // namespace b2g

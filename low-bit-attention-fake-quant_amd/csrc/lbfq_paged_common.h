// What the kernels of attention over the paged cache share: a sequence's extent and masks, conversions and products, the
// end of the two decode kernels, and copies into LDS and a query's terms for the cache in 4 bits.
#pragma once

#include <algorithm>
#include <limits>
#include <type_traits>

#include "lbfq_common.h"
#include "../../include/lbfq.h"

namespace lbfq {
namespace paged {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Args {
  lbfq_paged_params p;
  int G;          // query heads of a key head
  int splits;     // parts of the keys
  int least;      // key tiles of a part, at least
  int slots;      // chunk: places for row tiles, over all sequences
  uint32_t piece;   // chunk: neighbouring slots that go to one XCD
  uint32_t share;   // chunk in 4 bits: of 2^16, what the first of two unequal parts has of the keys (0: equal parts)
  uint32_t combos;  // decode: sequences x key heads; chunk: key heads x parts
  int64_t main;   // workgroups that attend (the others fill)
  float sml2;     // sm_scale * log2(e)
  float2* ml;     // (splits, T * Hq): maximum (log2 units) and sum of a part
  float* acc;     // (splits, T * Hq, D): a part's average of the values
};

// One sequence, clamped to what the tensors hold.
struct Seq {
  int n, len, start;
  bool causal;
  int window;
  // keys [lo, hi) of query i
  __device__ __forceinline__ int hi(int i) const {
    if (!causal) return len;
    const int h = len - n + i + 1;
    return h < 0 ? 0 : h;  // i < n: never above len
  }
  __device__ __forceinline__ int lo(int i) const {
    if (!window) return 0;
    const int l = len - n + i + 1 - window;
    return l < 0 ? 0 : l;
  }
};

__device__ __forceinline__ Seq sequence(const lbfq_paged_params& p, int64_t b) {
  Seq s;
  const int T = static_cast<int>(p.T);
  int s0 = p.query_starts[b], s1 = p.query_starts[b + 1];
  s0 = s0 < 0 ? 0 : s0 > T ? T : s0;
  s1 = s1 < s0 ? s0 : s1 > T ? T : s1;
  s.start = s0;
  s.n = s1 - s0;
  const int cap = static_cast<int>(p.table_cols << p.page_shift);
  const int len = p.seq_lens[b];
  s.len = len < 0 ? 0 : len > cap ? cap : len;
  s.causal = p.causal != 0;
  s.window = static_cast<int>(p.window);
  return s;
}

// The chunk kernel's row tiles have 128 rows.  Sequence b has the slots from slot_of(b) up to slot_of(b + 1), one more
// than its rows need at the most: where a tile belongs follows from query_starts alone, and hardly a workgroup comes
// for nothing.
constexpr int kChunkRows = 128;
__device__ __forceinline__ int slot_of(const lbfq_paged_params& p, int G, int b) {
  const int T = static_cast<int>(p.T), s0 = p.query_starts[b];
  return (s0 < 0 ? 0 : s0 > T ? T : s0) * G / kChunkRows + b;
}
// The last sequence whose slots start at or before `slot`: 64 places looked at at a time.
__device__ __forceinline__ int sequence_at(const lbfq_paged_params& p, int G, int slot) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  for (int n = static_cast<int>(p.B); n > 1;) {
    const int step = (n + 63) / 64, i = lane * step;
    const uint64_t before = __ballot(i < n && slot_of(p, G, lo + (i < n ? i : 0)) <= slot);
    const int k = before ? 63 - __builtin_clzll(before) : 0;
    lo += k * step;
    n = step < n - k * step ? step : n - k * step;
  }
  return lo;
}

// Rows of the token dimension that no sequence has: zero (a new output), lse -inf.
template <int D>
__device__ void fill_rest(const lbfq_paged_params& p, int64_t wg, int64_t wgs) {
  int s0 = p.query_starts[0], s1 = p.query_starts[p.B];
  const int T = static_cast<int>(p.T);
  s0 = s0 < 0 ? 0 : s0 > T ? T : s0;
  s1 = s1 < s0 ? s0 : s1 > T ? T : s1;
  const int rest = T - (s1 - s0);
  for (int64_t k = wg; k < rest; k += wgs) {
    const int64_t t = k < s0 ? k : k - s0 + s1;
    for (int i = threadIdx.x; p.fill_rest && i < p.Hq * (D / 8); i += blockDim.x) {
      const int h = i / (D / 8), d = i % (D / 8);
      reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + t * p.out_t + h * p.out_h)[d] = make_uint4(0, 0, 0, 0);
    }
    if (p.lse)
      for (int h = threadIdx.x; h < p.Hq; h += blockDim.x) p.lse[t * p.Hq + h] = -INFINITY;
  }
}

// The larger, NaN if either is: v_maximum3_f32, three operands an instruction, where fmaxf would first quiet each
// MFMA result with an instruction of its own
__device__ __forceinline__ float vmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float vmin(float a, float b) { return __builtin_elementwise_minimum(a, b); }  // (likewise)

// v of the lanes 16 and 32 away (v_permlane16_swap / v_permlane32_swap of v with
// itself leave it and the partner's value in the two results)
__device__ __forceinline__ float max_x32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return vmax(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_x32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_x16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return vmax(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_x16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const f32x2 v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const f32x2 v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}
template <int DT>
__device__ __forceinline__ uint32_t pack_dt(float a, float b) {
  if constexpr (DT == kBF16) return pack_bf16(a, b);
  else return pack_f16(a, b);
}

// Eight fp16 values as two bf16 terms each: eight bits and the other three, exact
__device__ __forceinline__ void split_f16(const uint4& x, uint4& hi, uint4& lo) {
  const uint32_t in[4] = {x.x, x.y, x.z, x.w};
  uint32_t h[4], r[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float a = f16_bits_to_f32(static_cast<uint16_t>(in[e])), b = f16_bits_to_f32(static_cast<uint16_t>(in[e] >> 16));
    h[e] = pack_bf16(a, b);
    r[e] = pack_bf16(a - __uint_as_float(h[e] << 16), b - __uint_as_float(h[e] & 0xffff0000u));
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(r[0], r[1], r[2], r[3]);
}

// The pair I of the codes from w on (two in 16 bits, or in 8) times 2^e as 16-bit values; sc: 2^e as fp32.
template <int BITS>
__device__ __forceinline__ uint32_t cvt_bf16(const uint32_t* w, int i, float sc) {
  if constexpr (BITS == 8) {
    return __builtin_bit_cast(uint32_t, i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i >> 1], sc, true)
                                              : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i >> 1], sc, false));
  } else {
    const uint32_t x = w[i >> 2];
    switch (i & 3) {  // (known once the loops are unrolled)
      case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, sc, 0));
      case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, sc, 1));
      case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, sc, 2));
      default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, sc, 3));
    }
  }
}
template <int BITS>
__device__ __forceinline__ uint32_t cvt_f16(const uint32_t* w, int i, float sc) {
  if constexpr (BITS == 8) {
    return __builtin_bit_cast(uint32_t, i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i >> 1], sc, true)
                                              : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i >> 1], sc, false));
  } else {
    const uint32_t x = w[i >> 2];
    switch (i & 3) {
      case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, sc, 0));
      case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, sc, 1));
      case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, sc, 2));
      default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x, sc, 3));
    }
  }
}

// N bytes from p on, in words
template <int N>
__device__ __forceinline__ void load_bytes(const uint8_t* p, uint32_t* w) {
  if constexpr (N == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (N == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else if constexpr (N == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  }
}

__device__ __forceinline__ v4f mfma16_bf16(const uint4& a, const uint4& b, const v4f& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                  0);
}
__device__ __forceinline__ v16f mfma32_bf16(const uint4& a, const uint4& b, const v16f& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                  0);
}
__device__ __forceinline__ v16f mfma32_f16(const uint4& a, const uint4& b, const v16f& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Whether a row's sum has anything in it (a NaN has: a row whose query holds one comes out as NaN, not as empty)
__device__ __forceinline__ bool filled(float l) { return l != 0.0f; }

// lse of a row (natural logarithm) from what its sum is relative to, in log2 units, and the sum
__device__ __forceinline__ float row_lse(float m, float l) {
  return filled(l) ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
}

// The unit of V's sums in the decode kernels, for each block of 32 columns: scale bytes (E8M0) are taken up by `up`, so that
// sums over small values keep fp32's precision down to 2^-127.  A byte may come out at kTop: 2^30 values of 448 2^(kTop - 127)
// add up to less than 2^127.  kUp does for scales of up to 2^32; where a block's are larger, the unit follows the largest so
// far, as a row's maximum does, and bytes that would be negative (2^-kTop of the largest) count as 0.
constexpr int kTop = 215, kUp = 56;

constexpr int kDecodeRows = 16;

template <int D>
struct alignas(16) DecodeLds {
  float acc[4][kDecodeRows][D + 4];
  float m[4][kDecodeRows], l[4][kDecodeRows];
  int up[4][D / 32];
};

__device__ __forceinline__ float two_to(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }  // e: -126 .. 127

// The unit brought down for scale bytes of up to `top`.  Lane (n, g) has up and top for V's columns (D/16) n .., and rows
// 4 g + i of acc, which are columns (D/16) (4 g + i) + nb.
template <int D>
__device__ __forceinline__ void lower_unit(int top, int& up, v4f (&acc)[D / 16]) {
  constexpr int NB = D / 16, PER = 16 / (D / 32);  // lanes n of a block
  const int g = (threadIdx.x & 63) >> 4;
  int now = kTop - top < up ? kTop - top : up;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    if (i >= PER && i < 16) continue;
    const int o = __shfl_xor(now, i, 64);
    now = o < now ? o : now;
  }
  const int from = PER * (g * (D / 32) / 4);  // a lane that has the block of these rows of acc
  const float f = two_to(__shfl(now, from, 64) - __shfl(up, from, 64));
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[nb][i] *= f;
  up = now;
}

// The four waves' rows r0 .. of one part joined by their maxima: into the output, or the part's place of the workspace.
// Lane (n, g): row n's maximum m, its own share l of the sum, and columns (D/16) (4 g + i) + nb of the average times the
// sum and 2^up (its lanes' up: lower_unit).
template <int DT, int D>
__device__ __forceinline__ void join_waves(const Args& a, const Seq& s, v4f (&acc)[D / 16], float m, float l, int up,
                                           DecodeLds<D>& x, int r0, int rows, int split, int kvh) {
  constexpr int NB = D / 16, NW = 4;
  const lbfq_paged_params& p = a.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4, G = a.G;
  const int64_t R = p.T * p.Hq;
  l = add_x32(add_x16(l));
  if (g == 0) {
    x.m[wave][n] = m;
    x.l[wave][n] = l;
    if (n % (16 / (D / 32)) == 0) x.up[wave][n / (16 / (D / 32))] = up;
  }
  __syncthreads();
  auto unit = [&](int block) {  // the least of the waves'
    int u = x.up[0][block];
#pragma unroll
    for (int w = 1; w < NW; ++w) u = x.up[w][block] < u ? x.up[w][block] : u;
    return u;
  };
  {
    const int block = g * (D / 32) / 4, less = unit(block) - x.up[wave][block];
    if (__any(less != 0)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nb][i] *= two_to(less);
    }
  }
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < NW; ++w) M = vmax(M, x.m[w][n]);
  const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int nb = 0; nb < NB; nb += 4)
      *reinterpret_cast<float4*>(&x.acc[wave][n][(4 * g + i) * NB + nb]) =
          make_float4(acc[nb][i] * f, acc[nb + 1][i] * f, acc[nb + 2][i] * f, acc[nb + 3][i] * f);
  __syncthreads();
  {
    int part = threadIdx.x & 15;
    asm volatile("" : "+v"(part));  // (here: an output address formed before the loops would wait in memory)
    const int row = threadIdx.x >> 4;
    float MM = -INFINITY, L = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) MM = vmax(MM, x.m[w][row]);
#pragma unroll
    for (int w = 0; w < NW; ++w)
      L += filled(x.l[w][row]) ? x.l[w][row] * __builtin_amdgcn_exp2f(x.m[w][row] - MM) : 0.0f;
    if (r0 + row < rows) {
      float o[NB];
#pragma unroll
      for (int k = 0; k < NB; k += 4) {
        float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float4 v = *reinterpret_cast<const float4*>(&x.acc[w][row][part * NB + k]);
          t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w;
        }
        o[k] = t.x; o[k + 1] = t.y; o[k + 2] = t.z; o[k + 3] = t.w;
      }
      const int qq = (r0 + row) / G, hh = kvh * G + (r0 + row - qq * G);
      const int64_t tok = s.start + qq;
      const float inv = filled(L) ? two_to(-unit(part * NB / 32)) / L : 0.0f;
      if (a.splits == 1) {
        uint32_t w[NB / 2];
#pragma unroll
        for (int k = 0; k < NB / 2; ++k) w[k] = pack_dt<DT>(o[2 * k] * inv, o[2 * k + 1] * inv);
        uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(p.out) + tok * p.out_t + hh * p.out_h +
                                                    part * NB);
        if constexpr (NB == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
        if (p.lse && part == 0) p.lse[tok * p.Hq + hh] = row_lse(MM, L);
      } else {
        const int64_t at = split * R + tok * p.Hq + hh;
        if (part == 0) a.ml[at] = make_float2(MM, L);
        if (filled(L)) {
#pragma unroll
          for (int k = 0; k < NB; k += 4)
            *reinterpret_cast<float4*>(a.acc + at * D + part * NB + k) =
                make_float4(o[k] * inv, o[k + 1] * inv, o[k + 2] * inv, o[k + 3] * inv);
        }
      }
    }
  }
}

// ---- the chunk kernels

// Key of K row i of a 32-key block (bits 2 and 3 of i exchanged): a lane's scores are
// then of consecutive keys, eight at a time.
__device__ __forceinline__ int key_of_32(int i) { return (i & 0x13) | ((i & 4) << 1) | ((i & 8) >> 1); }

// Largest (low half) and 255 - smallest (high half) of the scale bytes so far and of word v.
__device__ __forceinline__ uint32_t span_join(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
template <int N>  // N bytes of v
__device__ __forceinline__ uint32_t span_add(uint32_t span, uint32_t v) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t b = (v >> (8 * i)) & 0xffu;
    span = span_join(span, b | ((255u - b) << 16));
  }
  return span;
}

// What the values of a part's K or V are multiplied by, 2^(134 - E), on their way to fp16, so that the largest
// code lands at 57344.  The smallest one, 2^-9, with a scale 2^-22 of the largest is then fp16's smallest step: within
// that span every value is exact.  A part whose scales are further apart is `wide`: bf16, as they are.
//
// A wide part's V is taken to where each block's (of 32 columns) largest scale byte is wide_top: weights of up to 2^15 times
// the part's `keys` (a power of two above them) values of up to 2^(wide_top - 118) add up to less than 2^127.  Scales 2^-wide_top
// of the largest count as that.
//
// E2M1's largest code, 6, lands at 49152 with 2^(140 - E), and its smallest, 1/2, stays exact 36 powers of two below.
constexpr int span_of(int bits) { return bits == 8 ? 22 : 36; }
constexpr int unit_of(int bits) { return bits == 8 ? 134 : 140; }
__device__ __forceinline__ int wide_top(int keys) { return 198 + __builtin_clz(keys); }  // 2^30 keys: 200
struct Unit {
  int E;
  bool wide;
};

// Each block's largest scale byte of V over keys k0 .. k1 - 1 of a sequence (pages that are not there left out), for all of a
// workgroup's threads: byte b is that of block b (D = 64: of block b & 1).  red: a word for each wave and half.
template <int D, int NT>
__device__ __forceinline__ uint32_t block_tops(const lbfq_paged_params& p, const int32_t* table, int kvh, int k0, int k1,
                                               uint32_t* red) {
  const int cols = static_cast<int>(p.table_cols);
  uint32_t even = 0, odd = 0;
  for (int key = k0 + static_cast<int>(threadIdx.x); key < k1; key += NT) {
    const int idx = key >> p.page_shift, page = idx < cols ? table[idx] : -1;
    if (page < 0 || page >= p.num_pages) continue;
    const int64_t row = ((page * p.Hk + kvh) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
    uint32_t w;
    load_bytes<D / 32>(p.v_scale + row * (D / 32), &w);
    even = span_join(even, w & 0x00ff00ffu);
    odd = span_join(odd, w >> 8 & 0x00ff00ffu);
  }
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    even = span_join(even, __shfl_xor(even, i, 64));
    odd = span_join(odd, __shfl_xor(odd, i, 64));
  }
  constexpr int NW = NT / 64;
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = even;
    red[NW + (threadIdx.x >> 6)] = odd;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    even = span_join(even, red[w]);
    odd = span_join(odd, red[NW + w]);
  }
  __syncthreads();
  const uint32_t tops = __builtin_amdgcn_readfirstlane(even | odd << 8);
  return D == 128 ? tops : (tops & 0xffffu) * 0x10001u;
}

// Workgroups of a CU: three where the registers do for that, at the price of a few that go to memory (1560 tokens over 32760
// keys, 40 heads of 64, bf16: 818 us with two, 765 with three; fp16 queries need more of them: 745 with two, 1075).
constexpr int chunk_groups(int dt, int64_t d) { return d == 64 && dt == kBF16 ? 3 : 2; }
constexpr int decode4_groups(int64_t d) { return d == 64 ? 3 : 2; }
constexpr int chunk4_groups(int64_t d) { return d == 64 ? 3 : 2; }  // (the 4-bit cache's kernel: 168 registers, none in memory)

// ---- the kernels of the cache in 4 bits

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x32 __attribute__((ext_vector_type(32)));

// Asynchronous copies into LDS: lane i's 16 (4) bytes go to lds + 16 (4) i.  In assembly, so that the compiler does not put
// a wait for all of them before the next LDS read (wait_for does that); an LDS copy right behind a write of M0 needs one
// wait state.  NT, for what nobody reads a second time (one token of 48 sequences of 8000 to 16000 keys, 135 -> 124 us).
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)));
}
__device__ __forceinline__ void copy_to(uint32_t lds) { asm volatile("s_mov_b32 m0, %0\n\ts_nop 0" ::"s"(lds) : "memory", "m0"); }
template <int OFF, bool NT>  // OFF: of both the source and the place in LDS
__device__ __forceinline__ void copy16(const uint8_t* base, uint32_t at) {
  if constexpr (NT) asm volatile("global_load_lds_dwordx4 %0, %1 offset:%2 nt" ::"v"(at), "s"(base), "i"(OFF) : "memory");
  else asm volatile("global_load_lds_dwordx4 %0, %1 offset:%2" ::"v"(at), "s"(base), "i"(OFF) : "memory");
}
template <bool NT>
__device__ __forceinline__ void copy4(const uint8_t* base, uint32_t at) {
  if constexpr (NT) asm volatile("global_load_lds_dword %0, %1 nt" ::"v"(at), "s"(base) : "memory");
  else asm volatile("global_load_lds_dword %0, %1" ::"v"(at), "s"(base) : "memory");
}
__device__ __forceinline__ void copy16v(const uint8_t* at) {
  asm volatile("global_load_lds_dwordx4 %0, off nt" ::"v"(at) : "memory");
}
__device__ __forceinline__ void copy4v(const uint8_t* at) {
  asm volatile("global_load_lds_dword %0, off nt" ::"v"(at) : "memory");
}
// Until no more than N copies are under way (they end in their order)
template <int N>
__device__ __forceinline__ void wait_for() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}

// The 16-byte piece of row r (of 16) that lies at place c of its D / 32 in LDS, and the place of piece c: so that 16 lanes
// that read one piece of 16 rows each are on distinct banks.
template <int D>
__device__ __forceinline__ int piece_of(int r, int c) {
  return D == 128 ? c ^ (r >> 2 & 3) : c ^ (r >> 3 & 1);
}

// 32 values over 2^e to E2M3, to nearest, and back; sc: 2^e.  In assembly for the &: the instructions write their results
// before they have read all operands, and the builtins let the compiler lay the one over the other.
__device__ __forceinline__ u32x6 to_e2m3(const f32x16& even, const f32x16& odd, float sc) {
  u32x6 w;
  asm("v_cvt_scalef32_2xpk16_fp6_f32 %0, %1, %2, %3\n\ts_nop 4" : "=&v"(w) : "v"(even), "v"(odd), "v"(sc));
  return w;
}
__device__ __forceinline__ f32x32 from_e2m3(const u32x6& w, float sc) {
  f32x32 v;
  asm("v_cvt_scalef32_pk32_f32_fp6 %0, %1, %2\n\ts_nop 4" : "=&v"(v) : "v"(w), "v"(sc));
  return v;
}

// 32 columns of a query in four E2M3 terms, and their E8M0 scales in the bytes of e: 255 (not a number) where a column is
// infinite or NaN.  They hold each column to 2^-19 of the largest (2^-129, if that is less than 2^-109).
//
// REST: what the four terms leave in four more, down to 2^-39 of the largest (2^-130).  Calls take those where the first four
// would keep fewer than nine bits, what bf16 has, of much of a block: *more, eight columns or more (not 0) that are below 2^-10
// of the largest.  Random columns do not come to that; one of 1000 times the others does.  (With such queries and without, us:
// one token of 48 sequences of 8000 to 16000 keys, 32 / 8 heads of 128, 148 and 123; a prompt of 8192, 778 and 526, in the
// chunk kernel's plain loop.  To look for them costs 1 us of four chunks' 96, 2 of the prompt.)
struct Terms {
  u32x6 w[4];
  uint32_t e;
};
struct Columns {
  uint32_t w[16];  // as they lie in memory
};
__device__ __forceinline__ Columns load_columns(const uint16_t* q) {
  Columns x;
#pragma unroll
  for (int i = 0; i < 4; ++i) load_bytes<16>(reinterpret_cast<const uint8_t*>(q) + 16 * i, x.w + 4 * i);
  return x;
}
template <int DT, bool REST = false>
__device__ __forceinline__ Terms split_query(const Columns& q, bool* more = nullptr) {
  f32x16 even, odd;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    even[i] = DT == kBF16 ? __uint_as_float(q.w[i] << 16) : f16_bits_to_f32(static_cast<uint16_t>(q.w[i]));
    odd[i] = DT == kBF16 ? __uint_as_float(q.w[i] & 0xffff0000u) : f16_bits_to_f32(static_cast<uint16_t>(q.w[i] >> 16));
  }
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = vmax(vmax(m, fabsf(even[i])), fabsf(odd[i]));
  const uint32_t top = __float_as_uint(m) >> 23;  // m is not negative, or a NaN of either sign
  const bool bad = (top & 0xffu) == 255u;
  // 2^(e - 127): the largest column is in 2 ... 4 of it, what a term leaves at most 4 of the next one's, E2M3 reaches 7.5
  uint32_t e = bad ? 100u : (top > 18u ? top : 18u) - 1u;
  if constexpr (!REST) {
    const float few = m * 0x1p-10f;
    // Eight columns are of two groups of four at least: the second smallest of the groups' smallest says where to count.
    float least = INFINITY, second = INFINITY;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float x = vmin(vmin(fabsf(even[i]), fabsf(odd[i])), vmin(fabsf(even[i + 1]), fabsf(odd[i + 1])));
      second = __builtin_amdgcn_fmed3f(least, second, x);
      least = vmin(least, x);
    }
    *more = false;
    if (__any(second < few)) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        n += (even[i] != 0.0f && fabsf(even[i]) < few) + (odd[i] != 0.0f && fabsf(odd[i]) < few);
      *more = !bad && n >= 8;
    }
  }
  Terms x;
#pragma unroll
  for (int t = REST ? -4 : 0; t < 4; ++t) {
    if (REST && t == 0) e = (e > 36u ? e : 36u) - 20u;
    const int at = t < 0 ? t + 4 : t;
    const float sc = __uint_as_float((e - 5u * at) << 23);
    x.w[at] = to_e2m3(even, odd, sc);
    if (t < 3) {
      const f32x32 back = from_e2m3(x.w[at], sc);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        even[i] -= back[2 * i];
        odd[i] -= back[2 * i + 1];
      }
    }
  }
  x.e = bad ? 0xffffffffu : e * 0x01010101u - 0x0f0a0500u;
  return x;
}

void launch_decode4(const Args& a, unsigned grid, hipStream_t stream);  // lbfq_paged4.hip
void launch_chunk4(const Args& a, unsigned grid, hipStream_t stream);   // lbfq_paged4_chunk.hip

}  // namespace paged
}  // namespace lbfq

// The quantised paged K/V cache: rows written as they come, also rotated on the way, and read back.
//
// A cache holds num_pages pages of `page` tokens.  Per page and head the codes
// of its tokens are rows of D bytes, (pages, H, page, D), and their scales rows
// of D/32 bytes, (pages, H, page, D/32): what attention reads of a head is one
// stretch.  The format is the package's MXFP8 for Q and K (lbfq_rowtile,
// LBFQ_Q_MX_QK, 32 columns a scale), the same codes and scales bit for bit:
//   e = ceil(log2(max(amax, 1e-4) / 448)),  code = e4m3(x 2^-e),
// but for e <= 119: from 2^128 on (where the value would be infinite) the largest
// is kept instead, 448 2^119.  The cache then holds finite values only, and a key
// that a row does not see adds 0 times something finite to it.
//
// In 4 bits rows of codes have D/2 bytes, the even column in the low half of each:
//   e = ceil(log2(max(amax, 1e-4) / 6)) <= 125,  code = e2m1(x 2^-e).
//
// All directions are bound by memory.  D/8 lanes hold a row, eight values each.  The
// 8-bit cache's write and read: a workgroup takes 64 consecutive tokens of one head
// of K or of V, so that the scales of its rows, four bytes each, fill whole lines from
// one workgroup, and a thread's rows (four at D = 128) are all on their way before the
// first is used.  Writing 32760 tokens x 40 heads x 128 from bf16: 196 us, 5.2 TB/s of
// bytes read and written (a copy of 1 GiB reaches 5.1 to 5.5).  Reading 8 sequences of
// up to 16384 x 8 heads to bf16: 147 us, 4.7 TB/s (what only writes reaches 5.3).  A
// few tokens: 3.0 and 4.6 us, a launch's own time.
//
// Everything else goes by tokens, four heads of 16 at a time: 32760 tokens rotated and
// appended, 40 / 40 heads of 128, to 4 bits 263 us, 5.9 TB/s, to 8 bits 285 us, 6.0; written
// in 4 bits 149 us, 5.7; 8 sequences of up to 16384 x 8 heads read from 4 bits 97 us, 6.3.
#include <algorithm>

#include "lbfq_common.h"
#include "../../include/lbfq.h"

using namespace lbfq;

namespace {

constexpr int kRows = 64;  // tokens of a workgroup

template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t i, float (&x)[8]) {
  if constexpr (DT == kF32) {
    const float4* s = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + i);
    const float4 u = s[0], v = s[1];
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + i);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[2 * k] = DT == kBF16 ? __uint_as_float(w[k] << 16) : f16_bits_to_f32(static_cast<uint16_t>(w[k]));
      x[2 * k + 1] = DT == kBF16 ? __uint_as_float(w[k] & 0xffff0000u) : f16_bits_to_f32(static_cast<uint16_t>(w[k] >> 16));
    }
  }
}

// NT: marked as not read again soon.  Where each instruction of a wave fills whole lines, that is faster (append of 32760
// tokens, 40 / 40 heads, when each store was made so: 295 -> 281 us with Q's, 289 with the codes'; reading them from 4 bits
// 148 -> 141); fp32's two stores a lane leave holes (8000 tokens, 8 heads: 16 -> 25).
template <typename T, bool NT>
__device__ __forceinline__ void put(void* at, const T& v) {
  if constexpr (NT) __builtin_nontemporal_store(v, static_cast<T*>(at));
  else *static_cast<T*>(at) = v;
}
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <int DT, bool NT = false>
__device__ __forceinline__ void store8(void* base, int64_t i, const float (&v)[8]) {
  if constexpr (DT == kF32) {
    float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + i);
    d[0] = make_float4(v[0], v[1], v[2], v[3]);
    d[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t lo = DT == kBF16 ? f32_to_bf16_bits(v[2 * k]) : f32_to_f16_bits(v[2 * k]);
      const uint32_t hi = DT == kBF16 ? f32_to_bf16_bits(v[2 * k + 1]) : f32_to_f16_bits(v[2 * k + 1]);
      w[k] = lo | (hi << 16);
    }
    put<u32x4, NT>(reinterpret_cast<uint16_t*>(base) + i, u32x4{w[0], w[1], w[2], w[3]});
  }
}

// The 2^e of a block of 32 columns whose largest value is amax
template <int BITS>
__device__ __forceinline__ float block_scale(float amax) {
  const float r = fmaxf(amax, kAmaxFloor);
  if constexpr (BITS == 8) return fminf(mx_scale_from_amax(r), 0x1p119f);
  // 6 = 1.5 2^2: r / 6 <= 2^(E - 2) for r = (1 + f) 2^E with 1 + f <= 1.5, from r's bits; no quotient is rounded
  const uint32_t u = __float_as_uint(r), e = (u >> 23) - 2 + ((u & 0x7fffffu) > 0x400000u ? 1 : 0);
  return __uint_as_float((e < 252 ? e : 252u) << 23);
}

// Row `row` of a cache tensor from the eight values that each of its lanes (lane part lp) holds.  All lanes of a wave
// take part; `live`: whether this one's row is stored.
template <int BITS, int D, bool NT>
__device__ __forceinline__ void encode_row(const float (&x)[8], uint8_t* codes, uint8_t* scale, int64_t row, int lp,
                                           bool live) {
  float m = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(x[k]));
  m = fmaxf(m, __shfl_xor(m, 1, 64));
  m = fmaxf(m, __shfl_xor(m, 2, 64));
  const float sc = block_scale<BITS>(m);
  const float inv = 1.0f / sc;  // exact: 2^-e
  if (!live) return;
  float q[8];
  if constexpr (BITS == 8) {
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = clamp448(x[k] * inv);
    put<u32x2, NT>(codes + row * D + 8 * lp, u32x2{cvt4_e4m3(q), cvt4_e4m3(q + 4)});
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = clamp6(x[k] * inv);
    put<uint32_t, NT>(codes + row * (D / 2) + 4 * lp, cvt8_e2m1(q));
  }
  if ((lp & 3) == 0) scale[row * (D / 32) + lp / 4] = static_cast<uint8_t>(__float_as_uint(sc) >> 23);
}

// workgroup: (which, head) fastest, then the block of tokens
template <int DT, int D>
__global__ void __launch_bounds__(256) kv_write_kernel(const lbfq_kv_write_params p) {
  constexpr int LPR = D / 8, RPI = 256 / LPR, U = kRows / RPI;  // rows at once, and in turn
  const int H = static_cast<int>(p.H);
  const int which_head = static_cast<int>(blockIdx.x % (2 * H));
  const int64_t t0 = static_cast<int64_t>(blockIdx.x / (2 * H)) * kRows;
  const bool isv = which_head >= H;
  const int h = isv ? which_head - H : which_head;
  const int r = threadIdx.x / LPR, lp = threadIdx.x % LPR;
  const void* src = isv ? p.v : p.k;
  const int64_t st = isv ? p.v_t : p.k_t, sh = isv ? p.v_h : p.k_h;
  uint8_t* codes = isv ? p.v_codes : p.k_codes;
  uint8_t* scale = isv ? p.v_scale : p.k_scale;
  const int64_t slots = p.num_pages << p.page_shift;
  float x[U][8];
  int64_t slot[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int64_t t = t0 + i * RPI + r;
    slot[i] = t < p.T ? p.slots[t] : -1;
    load8<DT>(src, (t < p.T ? t : p.T - 1) * st + h * sh + 8 * lp, x[i]);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    // (a slot outside the cache is padding)
    const int64_t row = ((slot[i] >> p.page_shift) * H + h) * (int64_t{1} << p.page_shift) +
                        (slot[i] & ((int64_t{1} << p.page_shift) - 1));
    encode_row<8, D, false>(x[i], codes, scale, row, lp, slot[i] >= 0 && slot[i] < slots);
  }
}

// ---- rotation, then into the cache

// Eight values as they lie in memory
template <int DT>
struct Raw {
  uint4 w[DT == kF32 ? 2 : 1];
};

template <int DT>
__device__ __forceinline__ Raw<DT> load_raw(const void* base, int64_t i) {
  Raw<DT> r;
  if constexpr (DT == kF32) {
    const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(base) + i);
    r.w[0] = s[0];
    r.w[1] = s[1];
  } else {
    r.w[0] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + i);
  }
  return r;
}

template <int DT>
__device__ __forceinline__ void widen(const Raw<DT>& r, float (&x)[8]) {
#pragma unroll
  for (int c = 0; c < (DT == kF32 ? 2 : 1); ++c) {
    const uint32_t w[4] = {r.w[c].x, r.w[c].y, r.w[c].z, r.w[c].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == kF32) {
        x[4 * c + i] = __uint_as_float(w[i]);
      } else if constexpr (DT == kBF16) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        x[2 * i] = f16_bits_to_f32(static_cast<uint16_t>(w[i]));
        x[2 * i + 1] = f16_bits_to_f32(static_cast<uint16_t>(w[i] >> 16));
      }
    }
  }
}

constexpr int kHeads = 4;  // of a workgroup of the kernels that go token by token

struct AppendArgs {
  lbfq_kv_append_params p;
  uint32_t groups;  // of kHeads heads of a token
};

enum Rotation { kNone, kAdjacent, kHalves };

// A workgroup takes four heads of 16 (D = 64: 32) tokens, the heads of Q, of K and of V being one list: a KiB of a token
// that lies together where Q, K and V are one projection's output.  (Longer stretches of a token's heads, which read its
// cos and sin less often, are slower: 32760 tokens, 40 / 40 heads to 4 bits, 4 / 8 / 12 / 16 / 48 heads: 263 / 267 / 275 / 320 /
// 318 us; 32 / 8 heads 121 / 126 / 131 / 130 / 143.)  Every product and the sum are rounded, so what is
// quantised is defined to the bit.  kNone: writing without a rotation, in 4 bits.
template <int DT, int D, int BITS, Rotation ROT>
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendArgs a) {
  constexpr int LPR = D / 8, RPI = 256 / LPR;
  constexpr bool HALVES = ROT == kHalves;
  const lbfq_kv_append_params& p = a.p;
  const int Hq = static_cast<int>(p.Hq), Hk = static_cast<int>(p.Hk), heads = Hq + 2 * Hk;
  const int r = threadIdx.x / LPR, lp = threadIdx.x % LPR, lane = threadIdx.x & 63, d0 = 8 * lp;
  const uint32_t block = blockIdx.x / a.groups;
  const int h0 = static_cast<int>(blockIdx.x - block * a.groups) * kHeads;
  const int64_t t = static_cast<int64_t>(block) * RPI + r, tok = t < p.T ? t : p.T - 1;
  Raw<DT> raw[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int g = h0 + i < heads ? h0 + i : heads - 1;
    const bool isq = g < Hq, isk = g < Hq + Hk;
    raw[i] = load_raw<DT>(isq ? p.q : isk ? p.k : p.v,
                          tok * (isq ? p.q_t : isk ? p.k_t : p.v_t) +
                              (isq ? g * p.q_h : isk ? (g - Hq) * p.k_h : (g - Hq - Hk) * p.v_h) + d0);
  }
  const int64_t slot = t < p.T ? p.slots[tok] : -1;
  const int half = p.rot / 2;
  bool past = false, turned = false;
  int partner = lane;
  float c[8], s[8];
  if (ROT != kNone && h0 < Hq + Hk) {
    // the rotation of this thread's columns
    const int64_t pos = p.positions_i64 ? reinterpret_cast<const int64_t*>(p.positions)[tok * p.pos_t]
                                        : reinterpret_cast<const int32_t*>(p.positions)[tok * p.pos_t];
    past = pos >= p.table_len;
    turned = d0 < p.rot && pos >= 0;
    constexpr int N = HALVES ? 8 : 4;
    const int i0 = HALVES ? (d0 < half ? d0 : d0 - half) : d0 / 2;
    if (HALVES && d0 < p.rot) partner = d0 < half ? lane + half / 8 : lane - half / 8;
    float cc[N], ss[N];
#pragma unroll
    for (int k = 0; k < N; ++k) cc[k] = ss[k] = __builtin_nanf("");
    if (turned && !past) {
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        const float4 cv = *reinterpret_cast<const float4*>(p.cos + pos * half + i0 + k);
        const float4 sv = *reinterpret_cast<const float4*>(p.sin + pos * half + i0 + k);
        cc[k] = cv.x; cc[k + 1] = cv.y; cc[k + 2] = cv.z; cc[k + 3] = cv.w;
        ss[k] = sv.x; ss[k + 1] = sv.y; ss[k + 2] = sv.z; ss[k + 3] = sv.w;
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      c[k] = cc[HALVES ? k : k / 2];
      const float sn = ss[HALVES ? k : k / 2];
      s[k] = (HALVES ? d0 < half : (k & 1) == 0) ? -sn : sn;  // the sign of the partner's term
    }
  } else if (ROT != kNone) {
    past = (p.positions_i64 ? reinterpret_cast<const int64_t*>(p.positions)[tok * p.pos_t]
                            : reinterpret_cast<const int32_t*>(p.positions)[tok * p.pos_t]) >= p.table_len;
  }
  const int64_t slots = p.num_pages << p.page_shift;
  const bool live = slot >= 0 && slot < slots && !past;
  const int64_t page_row = (slot >> p.page_shift) * Hk, in_page = slot & ((int64_t{1} << p.page_shift) - 1);
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int g = h0 + i;
    if (g >= heads) break;
    float x[8];
    widen<DT>(raw[i], x);
    if (ROT != kNone && g < Hq + Hk) {
      float o[8];  // the partners' values, exchanged as they lie in memory
      if constexpr (HALVES) {
        Raw<DT> other;
#pragma unroll
        for (int k = 0; k < (DT == kF32 ? 2 : 1); ++k)
          other.w[k] = make_uint4(__shfl(raw[i].w[k].x, partner, 64), __shfl(raw[i].w[k].y, partner, 64),
                                  __shfl(raw[i].w[k].z, partner, 64), __shfl(raw[i].w[k].w, partner, 64));
        widen<DT>(other, o);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = x[k ^ 1];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float y = as_f32(x[k] * c[k] + o[k] * s[k]);
        x[k] = turned ? y : x[k];
      }
    }
    if (g < Hq) {
      if (t < p.T) store8<DT, true>(p.q_out, (t * Hq + g) * D + d0, x);
    } else {
      const bool isv = g >= Hq + Hk;
      const int64_t row = ((page_row + g - (isv ? Hq + Hk : Hq)) << p.page_shift) + in_page;
      encode_row<BITS, D, true>(x, isv ? p.v_codes : p.k_codes, isv ? p.v_scale : p.k_scale, row, lp, live);
    }
  }
}

// Reading 4-bit codes is mostly writing: four heads of a few tokens to a workgroup, as above (head by head, as the 8-bit
// kernel does it, 32760 tokens x 40 heads came out at 204 us, 3.3 TB/s of writes).
struct ReadArgs {
  lbfq_kv_read_params p;
  uint32_t groups, blocks;  // of kHeads heads of K and V; of tokens of a sequence
};
template <int DT, int D>
__global__ void __launch_bounds__(256) kv_read4_kernel(const ReadArgs a) {
  constexpr int LPR = D / 8, RPI = 256 / LPR;
  const lbfq_kv_read_params& p = a.p;
  const int H = static_cast<int>(p.H), r = threadIdx.x / LPR, lp = threadIdx.x % LPR;
  const uint32_t block = blockIdx.x / a.groups, b = block / a.blocks;
  const int h0 = static_cast<int>(blockIdx.x - block * a.groups) * kHeads;
  const int64_t t = static_cast<int64_t>(block - b * a.blocks) * RPI + r, cap = p.table_cols << p.page_shift;
  const int64_t len = p.seq_lens[b] < cap ? p.seq_lens[b] : cap;
  int page = -1;
  if (t < len && t < p.max_len) page = p.block_table[b * p.table_stride + (t >> p.page_shift)];
  const bool there = page >= 0 && page < p.num_pages;
  const int64_t page_row = static_cast<int64_t>(there ? page : 0) * H, in_page = t & ((int64_t{1} << p.page_shift) - 1);
  uint32_t c[kHeads], e[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int g = h0 + i < 2 * H ? h0 + i : 2 * H - 1;
    const int64_t row = ((page_row + (g < H ? g : g - H)) << p.page_shift) + in_page;
    c[i] = *reinterpret_cast<const uint32_t*>((g < H ? p.k_codes : p.v_codes) + row * (D / 2) + 4 * lp);
    e[i] = (g < H ? p.k_scale : p.v_scale)[row * (D / 32) + lp / 4];
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int g = h0 + i;
    if (g >= 2 * H || t >= p.max_len) break;
    const float sc = __uint_as_float(e[i] == 255 ? 0x7fc00000u : e[i] ? e[i] << 23 : 0x00400000u);
    float v[8];
    values8_e2m1(c[i], v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = there ? as_f32(v[k] * sc) : 0.0f;  // the fp32 product, then the one rounding
    store8<DT, true>(g < H ? p.k_out : p.v_out, ((b * p.max_len + t) * H + (g < H ? g : g - H)) * D + 8 * lp, v);
  }
}

template <int DT, int D>
__global__ void __launch_bounds__(256) kv_read_kernel(const lbfq_kv_read_params p, int blocks) {
  constexpr int LPR = D / 8, RPI = 256 / LPR, U = kRows / RPI;
  const int H = static_cast<int>(p.H);
  const int which_head = static_cast<int>(blockIdx.x % (2 * H));
  const int64_t rest = blockIdx.x / (2 * H);
  const int64_t b = rest / blocks;
  const int t0 = static_cast<int>(rest - b * blocks) * kRows;
  const bool isv = which_head >= H;
  const int h = isv ? which_head - H : which_head;
  const int r = threadIdx.x / LPR, lp = threadIdx.x % LPR;
  const uint8_t* codes = isv ? p.v_codes : p.k_codes;
  const uint8_t* scale = isv ? p.v_scale : p.k_scale;
  void* out = isv ? p.v_out : p.k_out;
  const int64_t cap = p.table_cols << p.page_shift;
  const int64_t len = p.seq_lens[b] < cap ? p.seq_lens[b] : cap;
  uint2 c[U];
  uint32_t e[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int t = t0 + i * RPI + r;
    c[i] = make_uint2(0, 0);
    e[i] = 127;
    if (t < len) {
      const int page = p.block_table[b * p.table_stride + (t >> p.page_shift)];
      if (page >= 0 && page < p.num_pages) {
        const int64_t row = ((static_cast<int64_t>(page) * H + h) << p.page_shift) + (t & ((1 << p.page_shift) - 1));
        c[i] = *reinterpret_cast<const uint2*>(codes + row * D + 8 * lp);
        e[i] = scale[row * (D / 32) + lp / 4];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int64_t t = t0 + i * RPI + r;
    if (t >= p.max_len) continue;
    const float sc = __uint_as_float(e[i] == 255 ? 0x7fc00000u : e[i] ? e[i] << 23 : 0x00400000u);
    float v[8];
    v[0] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c[i].x), 0);
    v[1] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c[i].x), 1);
    v[2] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c[i].x), 2);
    v[3] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c[i].x), 3);
    v[4] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c[i].y), 0);
    v[5] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c[i].y), 1);
    v[6] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c[i].y), 2);
    v[7] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(c[i].y), 3);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = as_f32(v[k] * sc);  // the fp32 product, then the one rounding
    store8<DT>(out, ((b * p.max_len + t) * H + h) * D + 8 * lp, v);
  }
}

// bits of a code: 4, or 8 (also as 0, what a cleared struct of before has in that place, its padding)
bool four(int bits) { return bits == 4; }

int check_cache(const char* who, int bits, int64_t num_pages, int page_shift, int64_t H, int64_t D, const void* kc,
                const void* ks, const void* vc, const void* vs) {
  LBFQ_CHECK_ARG(bits == 0 || bits == 4 || bits == 8, "%s: codes have 4 or 8 bits", who);
  LBFQ_CHECK_ARG(D == 64 || D == 128, "%s: D must be 64 or 128", who);
  LBFQ_CHECK_ARG(page_shift >= 4 && page_shift <= 10, "%s: pages hold 16 to 1024 tokens, a power of two", who);
  LBFQ_CHECK_ARG(num_pages > 0 && num_pages < (int64_t{1} << 31), "%s: bad number of pages", who);
  LBFQ_CHECK_ARG(H > 0 && H < (1 << 16), "%s: bad number of heads", who);
  LBFQ_CHECK_ARG(kc && ks && vc && vs, "%s: missing cache tensor", who);
  LBFQ_CHECK_ARG(((reinterpret_cast<uint64_t>(kc) | reinterpret_cast<uint64_t>(vc)) & 15) == 0 &&
                     ((reinterpret_cast<uint64_t>(ks) | reinterpret_cast<uint64_t>(vs)) & 15) == 0,
                 "%s: cache tensors must be 16-byte aligned", who);
  return 0;
}

template <int DT, int D>
void launch_append_as(const AppendArgs& a, Rotation rot, dim3 grid, hipStream_t st) {
  const dim3 block(256);
  if (rot == kNone) {
    hipLaunchKernelGGL((kv_append_kernel<DT, D, 4, kNone>), grid, block, 0, st, a);
  } else if (four(a.p.bits)) {
    if (rot == kHalves) hipLaunchKernelGGL((kv_append_kernel<DT, D, 4, kHalves>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((kv_append_kernel<DT, D, 4, kAdjacent>), grid, block, 0, st, a);
  } else {
    if (rot == kHalves) hipLaunchKernelGGL((kv_append_kernel<DT, D, 8, kHalves>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((kv_append_kernel<DT, D, 8, kAdjacent>), grid, block, 0, st, a);
  }
}

int launch_append(const char* who, const lbfq_kv_append_params& p, Rotation rot, hipStream_t st) {
  AppendArgs a{};
  a.p = p;
  a.groups = static_cast<uint32_t>((p.Hq + 2 * p.Hk + kHeads - 1) / kHeads);
  const int64_t per = 256 / (p.D / 8), blocks = (p.T + per - 1) / per;
  LBFQ_CHECK_ARG(blocks < (int64_t{1} << 24) / a.groups, "%s: problem too large", who);  // (a launch has fewer than 2^32 threads)
  const dim3 grid(static_cast<unsigned>(blocks * a.groups));
  const bool d128 = p.D == 128;
  if (p.dtype == kBF16) d128 ? launch_append_as<kBF16, 128>(a, rot, grid, st) : launch_append_as<kBF16, 64>(a, rot, grid, st);
  else if (p.dtype == kF16) d128 ? launch_append_as<kF16, 128>(a, rot, grid, st) : launch_append_as<kF16, 64>(a, rot, grid, st);
  else d128 ? launch_append_as<kF32, 128>(a, rot, grid, st) : launch_append_as<kF32, 64>(a, rot, grid, st);
  LBFQ_LAUNCH_CHECK(who);
  return 0;
}

}  // namespace

extern "C" int lbfq_kv_write(const lbfq_kv_write_params* p, lbfq_stream_t stream) {
  LBFQ_CHECK_ARG(p, "lbfq_kv_write: null params");
  if (int rc = check_cache("lbfq_kv_write", p->bits, p->num_pages, p->page_shift, p->H, p->D, p->k_codes, p->k_scale,
                           p->v_codes, p->v_scale))
    return rc;
  LBFQ_CHECK_ARG(p->dtype >= kF32 && p->dtype <= kBF16, "lbfq_kv_write: bad dtype %d", p->dtype);
  LBFQ_CHECK_ARG(p->T > 0 && p->T < (int64_t{1} << 40), "lbfq_kv_write: bad number of tokens");
  LBFQ_CHECK_ARG(p->k && p->v && p->slots, "lbfq_kv_write: missing tensor");
  const int64_t s[4] = {p->k_t, p->k_h, p->v_t, p->v_h};
  for (int64_t v : s)
    LBFQ_CHECK_ARG(v % (p->dtype == kF32 ? 4 : 8) == 0, "lbfq_kv_write: rows must be 16-byte aligned");
  LBFQ_CHECK_ARG(((reinterpret_cast<uint64_t>(p->k) | reinterpret_cast<uint64_t>(p->v)) & 15) == 0,
                 "lbfq_kv_write: rows must be 16-byte aligned");
  if (four(p->bits)) {  // by tokens, as with a rotation
    lbfq_kv_append_params x{};
    x.k = p->k; x.v = p->v; x.dtype = p->dtype;
    x.T = p->T; x.Hk = p->H; x.D = p->D;
    x.k_t = p->k_t; x.k_h = p->k_h; x.v_t = p->v_t; x.v_h = p->v_h;
    x.slots = p->slots;
    x.k_codes = p->k_codes; x.k_scale = p->k_scale; x.v_codes = p->v_codes; x.v_scale = p->v_scale;
    x.num_pages = p->num_pages; x.page_shift = p->page_shift; x.bits = p->bits;
    return launch_append("lbfq_kv_write", x, kNone, static_cast<hipStream_t>(stream));
  }
  const int64_t wgs = (p->T + kRows - 1) / kRows * 2 * p->H;
  LBFQ_CHECK_ARG(wgs < (int64_t{1} << 24), "lbfq_kv_write: problem too large");  // (a launch has fewer than 2^32 threads)
  const dim3 grid(static_cast<unsigned>(wgs)), block(256);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define LBFQ_KW(DT)                                                                           \
  do {                                                                                        \
    if (p->D == 128) hipLaunchKernelGGL((kv_write_kernel<DT, 128>), grid, block, 0, st, *p);  \
    else hipLaunchKernelGGL((kv_write_kernel<DT, 64>), grid, block, 0, st, *p);               \
  } while (0)
  if (p->dtype == kBF16) LBFQ_KW(kBF16);
  else if (p->dtype == kF16) LBFQ_KW(kF16);
  else LBFQ_KW(kF32);
#undef LBFQ_KW
  LBFQ_LAUNCH_CHECK("lbfq_kv_write");
  return 0;
}

extern "C" int lbfq_kv_append(const lbfq_kv_append_params* p, lbfq_stream_t stream) {
  const char* who = "lbfq_kv_append";
  LBFQ_CHECK_ARG(p, "%s: null params", who);
  if (int rc = check_cache(who, p->bits, p->num_pages, p->page_shift, p->Hk, p->D, p->k_codes, p->k_scale, p->v_codes,
                           p->v_scale))
    return rc;
  LBFQ_CHECK_ARG(p->dtype >= kF32 && p->dtype <= kBF16, "%s: bad dtype %d", who, p->dtype);
  LBFQ_CHECK_ARG(p->T > 0 && p->T < (int64_t{1} << 40), "%s: bad number of tokens", who);
  LBFQ_CHECK_ARG(p->Hq >= 0 && p->Hq < (1 << 16), "%s: bad number of heads", who);
  LBFQ_CHECK_ARG(p->k && p->v && p->slots && p->positions && (p->table_len == 0 || (p->cos && p->sin)) &&
                     (p->Hq == 0 || (p->q && p->q_out)),
                 "%s: missing tensor", who);
  LBFQ_CHECK_ARG(p->rot > 0 && p->rot <= p->D && p->rot % 16 == 0, "%s: rot must be a multiple of 16 up to D", who);
  LBFQ_CHECK_ARG(p->table_len >= 0 && p->table_len < (int64_t{1} << 40), "%s: bad table", who);
  const int64_t s[6] = {p->q_t, p->q_h, p->k_t, p->k_h, p->v_t, p->v_h};
  for (int64_t v : s) LBFQ_CHECK_ARG(v % (p->dtype == kF32 ? 4 : 8) == 0, "%s: rows must be 16-byte aligned", who);
  uint64_t at = 0;
  for (const void* x : {p->q, p->k, p->v, static_cast<const void*>(p->q_out), static_cast<const void*>(p->cos),
                        static_cast<const void*>(p->sin)})
    at |= reinterpret_cast<uint64_t>(x);
  LBFQ_CHECK_ARG((at & 15) == 0, "%s: rows and tables must be 16-byte aligned", who);
  return launch_append(who, *p, p->halves ? kHalves : kAdjacent, static_cast<hipStream_t>(stream));
}

extern "C" int lbfq_kv_read(const lbfq_kv_read_params* p, lbfq_stream_t stream) {
  LBFQ_CHECK_ARG(p, "lbfq_kv_read: null params");
  if (int rc = check_cache("lbfq_kv_read", p->bits, p->num_pages, p->page_shift, p->H, p->D, p->k_codes, p->k_scale,
                           p->v_codes, p->v_scale))
    return rc;
  LBFQ_CHECK_ARG(p->dtype >= kF32 && p->dtype <= kBF16, "lbfq_kv_read: bad dtype %d", p->dtype);
  LBFQ_CHECK_ARG(p->B > 0 && p->max_len > 0 && p->max_len <= (int64_t{1} << 30), "lbfq_kv_read: bad number of tokens");
  LBFQ_CHECK_ARG((p->block_table || p->table_cols == 0) && p->seq_lens && p->k_out && p->v_out,
                 "lbfq_kv_read: missing tensor");
  LBFQ_CHECK_ARG(p->table_cols >= 0 && p->table_cols < (int64_t{1} << 40), "lbfq_kv_read: bad block table");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 block(256);
  if (four(p->bits)) {
    ReadArgs a{};
    a.p = *p;
    const int64_t per = 256 / (p->D / 8), blocks = (p->max_len + per - 1) / per;
    a.groups = static_cast<uint32_t>((2 * p->H + kHeads - 1) / kHeads);
    a.blocks = static_cast<uint32_t>(blocks);
    LBFQ_CHECK_ARG(p->B < (int64_t{1} << 24) / (blocks * a.groups), "lbfq_kv_read: problem too large");
    const dim3 grid(static_cast<unsigned>(p->B * blocks * a.groups));
#define LBFQ_KR4(DT)                                                                          \
  do {                                                                                        \
    if (p->D == 128) hipLaunchKernelGGL((kv_read4_kernel<DT, 128>), grid, block, 0, st, a);   \
    else hipLaunchKernelGGL((kv_read4_kernel<DT, 64>), grid, block, 0, st, a);                \
  } while (0)
    if (p->dtype == kBF16) LBFQ_KR4(kBF16);
    else if (p->dtype == kF16) LBFQ_KR4(kF16);
    else LBFQ_KR4(kF32);
#undef LBFQ_KR4
    LBFQ_LAUNCH_CHECK("lbfq_kv_read");
    return 0;
  }
  const int64_t blocks = (p->max_len + kRows - 1) / kRows;
  LBFQ_CHECK_ARG(p->B < (int64_t{1} << 24) / (blocks * 2 * p->H), "lbfq_kv_read: problem too large");
  const dim3 grid(static_cast<unsigned>(p->B * blocks * 2 * p->H));
#define LBFQ_KR(DT)                                                                                                    \
  do {                                                                                                                 \
    if (p->D == 128) hipLaunchKernelGGL((kv_read_kernel<DT, 128>), grid, block, 0, st, *p, static_cast<int>(blocks));  \
    else hipLaunchKernelGGL((kv_read_kernel<DT, 64>), grid, block, 0, st, *p, static_cast<int>(blocks));               \
  } while (0)
  if (p->dtype == kBF16) LBFQ_KR(kBF16);
  else if (p->dtype == kF16) LBFQ_KR(kF16);
  else LBFQ_KR(kF32);
#undef LBFQ_KR
  LBFQ_LAUNCH_CHECK("lbfq_kv_read");
  return 0;
}

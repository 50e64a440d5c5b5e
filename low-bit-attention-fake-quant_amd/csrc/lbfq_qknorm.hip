// RMS norm of each query and key head's row and the position rotation, in one
// pass over Q and K, forward and backward.
//
// Row x (D values), r = 1 / sqrt(mean(x^2) + eps), n = x r w; the first `rot`
// columns are rotated in pairs (a, b) by the angle of the row's position:
//   y_a = n_a cos - n_b sin,  y_b = n_a sin + n_b cos,
// pairs (2i, 2i + 1) or (i, i + rot / 2).  Backward, with g = R^T dy (the
// rotation by the negative angle) and xhat = x r:
//   dw = sum over rows of g xhat,
//   dx = r (g w - xhat mean(g w xhat)) = r (g w) - x r^3 mean(g w x).
// r is formed again from x: one more sum beside the one the backward needs,
// instead of 4 bytes a row written and read.
//
// All arithmetic is fp32, one rounding to the tensor's dtype at the end.
// Bound by memory: D/8 lanes hold a row, eight values each (one 16-byte load of
// 16-bit data), so a wave covers four (D = 128) or eight (D = 64) heads of one
// token.  The heads of Q and K of a token are one list; a wave walks a stretch of
// it with the rotation's cos and sin and both weights in registers.  32760 tokens x
// 24 heads x 128 bf16: 80 us, 5.0 TB/s (a copy of 1 GiB: 5.1 to 5.5).  Backward, 8002
// tokens x 40 heads x 128: 48 + 4 us, 5.1 TB/s.  A few tokens: 3.9 us.
#include "lbfq_common.h"
#include "../../include/lbfq.h"

using namespace lbfq;

namespace {

struct Args {
  lbfq_qk_norm_params p;
  uint32_t units;  // (token, stretch of head groups); below 2^31
  uint32_t per_token;  // stretches of a token
  int stretch;     // head groups of a stretch
  int groups;      // head groups of a token
};

// A unit's token and head groups (32-bit divisions: 64-bit ones are a hundred instructions each)
struct Place {
  uint32_t tok, b, t;
  int g0, g1;
};
__device__ __forceinline__ Place place(const Args& a, uint32_t unit) {
  Place x;
  const uint32_t S = static_cast<uint32_t>(a.p.S);
  x.tok = unit / a.per_token;
  x.g0 = static_cast<int>(unit - x.tok * a.per_token) * a.stretch;
  x.g1 = x.g0 + a.stretch < a.groups ? x.g0 + a.stretch : a.groups;
  x.b = x.tok / S;
  x.t = x.tok - x.b * S;
  return x;
}

struct GradArgs {
  Args a;
  lbfq_qk_norm_grads g;
};

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

template <int DT>
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
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(base) + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// v of the lane that DPP pattern CTRL names, within the lane's row of 16
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}

// The sum over a row's 16 or 8 lanes, in each of them: partners at distance 1, 2
// (quad_perm), then the mirror images of halves (row_half_mirror) and rows (row_mirror).
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
  v += dpp<0xB1>(v);
  v += dpp<0x4E>(v);
  v += dpp<0x141>(v);
  if constexpr (LPR == 16) v += dpp<0x140>(v);
  return v;
}

// 1 / sqrt(v), v >= 0.  The instruction takes a number below the normal ones for 0.
__device__ __forceinline__ float rsqrt_any(float v) {
  const bool low = v < 0x1p-100f;
  const float r = __builtin_amdgcn_rsqf(low ? v * 0x1p64f : v);
  return low ? r * 0x1p32f : r;
}

// What a lane needs of its token's rotation: whether its eight columns are rotated, their c and s, and the lane their
// partners are in (HALVES).
struct Turn {
  float c[8], s[8];
  int partner;
  bool on;
};

template <int LPR, bool HALVES>
__device__ __forceinline__ Turn make_turn(const lbfq_qk_norm_params& p, int64_t b, int64_t t, int lane) {
  const int lp = lane % LPR, d0 = 8 * lp, rot = p.rot, half = rot / 2;
  int64_t pos = t;
  if (p.positions) {
    const int64_t at = b * p.pos_b + t * p.pos_s;
    pos = p.positions_i64 ? reinterpret_cast<const int64_t*>(p.positions)[at]
                          : reinterpret_cast<const int32_t*>(p.positions)[at];
  }
  Turn u;
  u.partner = lane;
  u.on = false;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    u.c[k] = 1.0f;
    u.s[k] = 0.0f;
  }
  if (d0 >= rot) return u;
  if constexpr (HALVES) u.partner = d0 < half ? lane + half / 8 : lane - half / 8;
  if (pos < 0) return u;  // padding: not rotated
  u.on = true;
  if (pos >= p.table_len) {  // no such angle: loud, not out of bounds
#pragma unroll
    for (int k = 0; k < 8; ++k) u.c[k] = u.s[k] = __builtin_nanf("");
    return u;
  }
  constexpr int N = HALVES ? 8 : 4;
  const int i0 = HALVES ? (d0 < half ? d0 : d0 - half) : d0 / 2;
  float c[N], s[N];
#pragma unroll
  for (int k = 0; k < N; k += 4) {
    const float4 cv = *reinterpret_cast<const float4*>(p.cos + pos * half + i0 + k);
    const float4 sv = *reinterpret_cast<const float4*>(p.sin + pos * half + i0 + k);
    c[k] = cv.x; c[k + 1] = cv.y; c[k + 2] = cv.z; c[k + 3] = cv.w;
    s[k] = sv.x; s[k + 1] = sv.y; s[k + 2] = sv.z; s[k + 3] = sv.w;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    u.c[k] = c[HALVES ? k : k / 2];
    // the sign of the partner's term
    const float sn = s[HALVES ? k : k / 2];
    const bool first = HALVES ? d0 < half : (k & 1) == 0;
    u.s[k] = first ? -sn : sn;
  }
  return u;
}

// v rotated by the row's angle, or by its negative (BACK)
template <bool HALVES, bool BACK>
__device__ __forceinline__ void turn(const Turn& u, float (&v)[8]) {
  float o[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k] = HALVES ? __shfl(v[k], u.partner, 64) : v[k ^ 1];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    // (a choice, not a rotation by 0: that would carry a neighbour's infinity or NaN over)
    const float r = fmaf(v[k], u.c[k], o[k] * (BACK ? -u.s[k] : u.s[k]));
    v[k] = u.on ? r : v[k];
  }
}

// A lane's eight weights (ones without any); a weight vector may start anywhere.
__device__ __forceinline__ void load_weight(const void* w, int dt, int d0, float (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = 1.0f;
  if (!w) return;
  if (reinterpret_cast<uint64_t>(w) & 15) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = load_as_f32(w, d0 + k, dt);
  } else if (dt == kF32) {
    widen<kF32>(load_raw<kF32>(w, d0), v);
  } else if (dt == kBF16) {
    widen<kBF16>(load_raw<kBF16>(w, d0), v);
  } else {
    widen<kF16>(load_raw<kF16>(w, d0), v);
  }
}

template <int DT, int D, bool HALVES>
__global__ void __launch_bounds__(256) qk_norm_kernel(const Args a) {
  constexpr int LPR = D / 8, RPW = 64 / LPR, U = 4;
  const lbfq_qk_norm_params& p = a.p;
  const int lane = threadIdx.x & 63, sub = lane / LPR, d0 = 8 * (lane % LPR);
  const int Hq = static_cast<int>(p.Hq), H = Hq + static_cast<int>(p.Hk);
  float wq[8], wk[8];
  load_weight(p.q_weight, p.q_weight_dtype, d0, wq);
  load_weight(p.k_weight, p.k_weight_dtype, d0, wk);
  for (uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); unit < a.units;
       unit += gridDim.x * 4) {
    const Place pl = place(a, unit);
    const int g0 = pl.g0, g1 = pl.g1;
    const int64_t tok = pl.tok, b = pl.b, t = pl.t;
    const int64_t qin = b * p.q_b + t * p.q_s + d0, kin = b * p.k_b + t * p.k_s + d0;
    const Turn u = make_turn<LPR, HALVES>(p, b, t, lane);
    for (int g = g0; g < g1; g += U) {
      Raw<DT> raw[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        int h = (g + i) * RPW + sub;
        h = h < H ? h : H - 1;  // every lane takes part in the row sums; rows past the last are not stored
        raw[i] = load_raw<DT>(h < Hq ? p.q : p.k, h < Hq ? qin + h * p.q_h : kin + (h - Hq) * p.k_h);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (g + i >= g1) break;
        const int h = (g + i) * RPW + sub;
        const bool isq = h < Hq;
        float x[8], ss = 0.0f;
        widen<DT>(raw[i], x);
#pragma unroll
        for (int k = 0; k < 8; ++k) ss = fmaf(x[k], x[k], ss);
        const float r = rsqrt_any(fmaf(row_sum<LPR>(ss), 1.0f / D, p.eps));
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = x[k] * r * (isq ? wq[k] : wk[k]);
        turn<HALVES, false>(u, x);
        if (h < H)
          store8<DT>(isq ? p.q_out : p.k_out, (isq ? tok * p.Hq + h : tok * p.Hk + h - Hq) * D + d0, x);
      }
    }
  }
}

// Backward: the waves walk the units with both weights' gradient sums in
// registers; a workgroup adds its waves' up in LDS and writes one row of
// `partial`.  No atomics: the order of every sum is fixed by the sizes.
template <int DT, int D, bool HALVES>
__global__ void __launch_bounds__(256) qk_norm_bwd_kernel(const GradArgs ga) {
  constexpr int LPR = D / 8, RPW = 64 / LPR, U = 2;
  const Args& a = ga.a;
  const lbfq_qk_norm_params& p = a.p;
  const lbfq_qk_norm_grads& gr = ga.g;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, sub = lane / LPR, d0 = 8 * (lane % LPR);
  const int Hq = static_cast<int>(p.Hq), H = Hq + static_cast<int>(p.Hk);
  float wq[8], wk[8], sq[8], sk[8];
  load_weight(p.q_weight, p.q_weight_dtype, d0, wq);
  load_weight(p.k_weight, p.k_weight_dtype, d0, wk);
#pragma unroll
  for (int k = 0; k < 8; ++k) sq[k] = sk[k] = 0.0f;
  for (uint32_t unit = blockIdx.x * 4 + wave; unit < a.units; unit += gridDim.x * 4) {
    const Place pl = place(a, unit);
    const int g0 = pl.g0, g1 = pl.g1;
    const int64_t tok = pl.tok, b = pl.b, t = pl.t;
    const Turn u = make_turn<LPR, HALVES>(p, b, t, lane);
    const int64_t qin = b * p.q_b + t * p.q_s + d0, kin = b * p.k_b + t * p.k_s + d0;
    const int64_t gq = b * gr.dyq_b + t * gr.dyq_s + d0, gk = b * gr.dyk_b + t * gr.dyk_s + d0;
    for (int g = g0; g < g1; g += U) {
      Raw<DT> rx[U], ry[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        int h = (g + i) * RPW + sub;
        h = h < H ? h : H - 1;
        const bool isq = h < Hq;
        rx[i] = load_raw<DT>(isq ? p.q : p.k, isq ? qin + h * p.q_h : kin + (h - Hq) * p.k_h);
        ry[i] = load_raw<DT>(isq ? gr.dyq : gr.dyk, isq ? gq + h * gr.dyq_h : gk + (h - Hq) * gr.dyk_h);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (g + i >= g1) break;
        const int h = (g + i) * RPW + sub;
        const bool isq = h < Hq, live = h < H;
        float x[8], y[8], ss = 0.0f, sx = 0.0f, gw[8];
        widen<DT>(rx[i], x);
        widen<DT>(ry[i], y);
        turn<HALVES, true>(u, y);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          gw[k] = y[k] * (isq ? wq[k] : wk[k]);
          ss = fmaf(x[k], x[k], ss);
          sx = fmaf(gw[k], x[k], sx);
        }
        ss = row_sum<LPR>(ss);
        sx = row_sum<LPR>(sx);
        const float r = rsqrt_any(fmaf(ss, 1.0f / D, p.eps));
        const float c = sx * (1.0f / D) * r * r;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float dw = y[k] * (x[k] * r);
          sq[k] += live && isq ? dw : 0.0f;
          sk[k] += live && !isq ? dw : 0.0f;
          x[k] = r * fmaf(-x[k], c, gw[k]);
        }
        if (live) {
          if (isq) store8<DT>(gr.dq, (tok * p.Hq + h) * D + d0, x);
          else store8<DT>(gr.dk, (tok * p.Hk + h - Hq) * D + d0, x);
        }
      }
    }
  }
  if (!gr.partial) return;
  __shared__ float red[4][2][D];
#pragma unroll
  for (int k = 0; k < 8; ++k)
#pragma unroll
    for (int o = LPR; o < 64; o <<= 1) {
      sq[k] += __shfl_xor(sq[k], o, 64);
      sk[k] += __shfl_xor(sk[k], o, 64);
    }
  if (sub == 0) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      red[wave][0][d0 + k] = sq[k];
      red[wave][1][d0 + k] = sk[k];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * D; c += 256) {
    const float* s = &red[0][0][0] + c;
    gr.partial[static_cast<int64_t>(blockIdx.x) * 2 * D + c] = (s[0] + s[2 * D]) + (s[4 * D] + s[6 * D]);
  }
}

// The rows of `partial` added up in 64 bits: 16 columns by 64 slices a workgroup
// (1024 rows: 4.1 us; 64 columns by 16 slices, 4 workgroups: 5.4).
__global__ void __launch_bounds__(1024) qk_norm_dw_kernel(const float* partial, int rows, int D, void* dwq, int dtq,
                                                          void* dwk, int dtk) {
  const int c = threadIdx.x & 15, slice = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  double s = 0.0;
#pragma unroll 8
  for (int r = slice; r < rows; r += 64) s += partial[static_cast<int64_t>(r) * 2 * D + col];
  __shared__ double red[64][16];
  red[slice][c] = s;
  __syncthreads();
  if (slice) return;
  s = 0.0;
#pragma unroll 8
  for (int i = 0; i < 64; ++i) s += red[i][c];
  if (col < D) {
    if (dwq) store_from_f32(dwq, col, dtq, static_cast<float>(s));
  } else if (dwk) {
    store_from_f32(dwk, col - D, dtk, static_cast<float>(s));
  }
}

int check(const char* who, const lbfq_qk_norm_params* p) {
  LBFQ_CHECK_ARG(p, "%s: null params", who);
  LBFQ_CHECK_ARG(p->D == 64 || p->D == 128, "%s: D must be 64 or 128", who);
  LBFQ_CHECK_ARG(p->dtype >= kF32 && p->dtype <= kBF16, "%s: bad dtype %d", who, p->dtype);
  LBFQ_CHECK_ARG(p->B > 0 && p->S > 0 && p->Hq > 0 && p->Hk > 0, "%s: empty problem", who);
  LBFQ_CHECK_ARG(p->Hq + p->Hk < (1 << 20) && p->B < (int64_t{1} << 31) / p->S &&
                     p->B * p->S < (int64_t{1} << 31) / ((p->Hq + p->Hk + 3) / 4),
                 "%s: problem too large", who);
  LBFQ_CHECK_ARG(p->q && p->k && p->cos && p->sin, "%s: missing tensor", who);
  LBFQ_CHECK_ARG(p->rot > 0 && p->rot <= p->D && p->rot % 16 == 0, "%s: rot must be a multiple of 16 up to D", who);
  LBFQ_CHECK_ARG(p->positions || p->S <= p->table_len, "%s: the table has %lld positions, S is %lld", who,
                 static_cast<long long>(p->table_len), static_cast<long long>(p->S));
  const int64_t s[6] = {p->q_b, p->q_s, p->q_h, p->k_b, p->k_s, p->k_h};
  const uint64_t al = p->dtype == kF32 ? 4 : 8;
  for (int64_t v : s) LBFQ_CHECK_ARG(v % static_cast<int64_t>(al) == 0, "%s: rows must be 16-byte aligned", who);
  LBFQ_CHECK_ARG(((reinterpret_cast<uint64_t>(p->q) | reinterpret_cast<uint64_t>(p->k) |
                   reinterpret_cast<uint64_t>(p->cos) | reinterpret_cast<uint64_t>(p->sin)) & 15) == 0,
                 "%s: rows must be 16-byte aligned", who);
  return 0;
}

// A wave takes all heads of a token (cos, sin and the division of its index serve
// the most rows) where there are 4096 tokens; of fewer, so many stretches of
// each that there are that many waves.
void plan(const lbfq_qk_norm_params* p, Args& a) {
  a.p = *p;
  const int rpw = p->D == 128 ? 4 : 8;
  a.groups = static_cast<int>((p->Hq + p->Hk + rpw - 1) / rpw);
  const int64_t tokens = p->B * p->S;
  int64_t per = (4096 + tokens - 1) / tokens;
  per = per < a.groups ? per : a.groups;
  a.stretch = static_cast<int>((a.groups + per - 1) / per);
  a.per_token = static_cast<uint32_t>((a.groups + a.stretch - 1) / a.stretch);
  a.units = static_cast<uint32_t>(tokens * a.per_token);
}

// Workgroups of a launch, at most.  Forward: a wave per token up to 32768 of them (us for 32760 tokens x 24 heads x 128
// bf16, 1024 / 2048 / 4096 / 8192 workgroups: 89 / 92 / 84 / 80).  Backward: four per CU, whose weight sums the second
// launch adds up (8002 tokens x 40 heads, 512 / 1024 / 2048: 65 + 4, 47 + 4, 48 + 10 us).
constexpr int64_t kForwardGroups = 8192, kGradGroups = 1024;

}  // namespace

#define LBFQ_QKN(KERNEL, DT, grid, arg)                                                                    \
  do {                                                                                                     \
    if (p->D == 128 && p->halves) hipLaunchKernelGGL((KERNEL<DT, 128, true>), grid, dim3(256), 0, st, arg); \
    else if (p->D == 128) hipLaunchKernelGGL((KERNEL<DT, 128, false>), grid, dim3(256), 0, st, arg);        \
    else if (p->halves) hipLaunchKernelGGL((KERNEL<DT, 64, true>), grid, dim3(256), 0, st, arg);            \
    else hipLaunchKernelGGL((KERNEL<DT, 64, false>), grid, dim3(256), 0, st, arg);                          \
  } while (0)

#define LBFQ_QKN_DT(KERNEL, grid, arg)                       \
  do {                                                       \
    if (p->dtype == kBF16) LBFQ_QKN(KERNEL, kBF16, grid, arg); \
    else if (p->dtype == kF16) LBFQ_QKN(KERNEL, kF16, grid, arg); \
    else LBFQ_QKN(KERNEL, kF32, grid, arg);                  \
  } while (0)

extern "C" int lbfq_qk_norm_rope(const lbfq_qk_norm_params* p, lbfq_stream_t stream) {
  if (int rc = check("lbfq_qk_norm_rope", p)) return rc;
  LBFQ_CHECK_ARG(p->q_out && p->k_out, "lbfq_qk_norm_rope: missing output");
  Args a{};
  plan(p, a);
  const int64_t wgs = (static_cast<int64_t>(a.units) + 3) / 4;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(wgs < kForwardGroups ? wgs : kForwardGroups));
  LBFQ_QKN_DT(qk_norm_kernel, grid, a);
  LBFQ_LAUNCH_CHECK("lbfq_qk_norm_rope");
  return 0;
}

extern "C" int64_t lbfq_qk_norm_rope_bwd_rows(const lbfq_qk_norm_params* p) {
  if (!p || p->B <= 0 || p->S <= 0 || p->Hq <= 0 || p->Hk <= 0) return 0;
  Args a{};
  plan(p, a);
  const int64_t wgs = (static_cast<int64_t>(a.units) + 3) / 4;
  return wgs < kGradGroups ? wgs : kGradGroups;
}

extern "C" int lbfq_qk_norm_rope_bwd(const lbfq_qk_norm_params* p, const lbfq_qk_norm_grads* g, lbfq_stream_t stream) {
  if (int rc = check("lbfq_qk_norm_rope_bwd", p)) return rc;
  LBFQ_CHECK_ARG(g && g->dyq && g->dyk && g->dq && g->dk, "lbfq_qk_norm_rope_bwd: missing gradient");
  LBFQ_CHECK_ARG(g->partial || (!g->dq_weight && !g->dk_weight), "lbfq_qk_norm_rope_bwd: missing workspace");
  const int64_t s[6] = {g->dyq_b, g->dyq_s, g->dyq_h, g->dyk_b, g->dyk_s, g->dyk_h};
  for (int64_t v : s)
    LBFQ_CHECK_ARG(v % (p->dtype == kF32 ? 4 : 8) == 0, "lbfq_qk_norm_rope_bwd: rows must be 16-byte aligned");
  LBFQ_CHECK_ARG(((reinterpret_cast<uint64_t>(g->dyq) | reinterpret_cast<uint64_t>(g->dyk)) & 15) == 0,
                 "lbfq_qk_norm_rope_bwd: rows must be 16-byte aligned");
  GradArgs ga{};
  plan(p, ga.a);
  ga.g = *g;
  if (!g->dq_weight && !g->dk_weight) ga.g.partial = nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int rows = static_cast<int>(lbfq_qk_norm_rope_bwd_rows(p));
  const dim3 grid(static_cast<unsigned>(rows));
  LBFQ_QKN_DT(qk_norm_bwd_kernel, grid, ga);
  LBFQ_LAUNCH_CHECK("lbfq_qk_norm_rope_bwd");
  if (ga.g.partial) {
    hipLaunchKernelGGL(qk_norm_dw_kernel, dim3(static_cast<unsigned>(2 * p->D / 16)), dim3(1024), 0, st, g->partial,
                       rows, static_cast<int>(p->D), g->dq_weight, p->q_weight_dtype, g->dk_weight, p->k_weight_dtype);
    LBFQ_LAUNCH_CHECK("lbfq_qk_norm_rope_bwd (weights)");
  }
  return 0;
}

// Attention of new tokens over the quantised paged K/V cache (lbfq_kv_write):
//
//   O_i = sum_j p_ij V_j / sum_j p_ij,  p_ij = exp(sm_scale q_i . K_j - m_i)
//
// over the keys j that query i sees, K_j and V_j = code * 2^e.  Sequence b has n_b
// queries (rows query_starts[b] ..) and seq_lens[b] keys in the cache; its query
// i stands at position len - n + i.  causal: j <= position; window w: j >
// position - w.  A row that sees nothing is 0 with lse -inf.
//
// The G = Hq / Hk query heads that share a key head are rows of one problem:
// row r is query r / G, head kvh G + r % G, so a key tile that is in the
// chip serves all of them.  Scores are formed transposed, S^T = K Q^T, and the
// output as O^T = V^T P^T: a lane's scores are of one query, and P goes into the
// second product from the registers that the first left it in.
//
// Two kernels.
//
// decode (up to 16 rows: one token of a sequence, 16x16x32 MFMA).  Bound by
// reading the cache, 2 D (1 + 1/32) bytes a key and head.  A wave takes 32 keys at
// a time straight into registers, the next ones on their way; a workgroup's
// four waves take turns, workgroups split the keys, and the parts are joined by
// their maxima (in LDS, then by the combine kernel).  Operands are bf16, which
// holds code * 2^e exactly (four significant bits); fp16 queries are two bf16
// terms (eleven bits, exact); P is two bf16 terms (16 bits).
//
// chunk (more rows).  A workgroup of NW waves has 32 NW rows; 64-key tiles are
// read once, converted to 16 bits and staged in LDS, double-buffered, one
// barrier a tile.  V is fp16 times a power of two (2^(7 - E), E the largest
// scale exponent so far, so that the largest code lands at 57344): exact unless
// a block's scale is 2^25 below the largest, and then off by 2^-40 of the largest
// V.  So P can be fp16: 11 bits, where bf16's 8 would cost as much as the output's
// own rounding.  K is bf16 (exact) for bf16 queries, and for fp16 ones fp16 with the
// tile's own E.
#include "lbfq_common.h"
#include "../../include/lbfq.h"

using namespace lbfq;

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Args {
  lbfq_paged_params p;
  int G;          // query heads of a key head
  int tiles;      // row tiles of a sequence that the grid has
  int splits;     // parts of the keys
  int64_t main;   // workgroups that attend (the others fill)
  float sml2;     // sm_scale * log2(e)
  float2* ml;     // (splits, T * Hq): maximum (log2 units) and sum of a part
  float* acc;     // (splits, T * Hq, D)
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

// Rows of the token dimension that no sequence has: zero (a new output), lse -inf.
__device__ void fill_rest(const lbfq_paged_params& p, int64_t wg, int64_t wgs) {
  int s0 = p.query_starts[0], s1 = p.query_starts[p.B];
  const int T = static_cast<int>(p.T);
  s0 = s0 < 0 ? 0 : s0 > T ? T : s0;
  s1 = s1 < s0 ? s0 : s1 > T ? T : s1;
  const int rest = T - (s1 - s0);
  for (int64_t k = wg; k < rest; k += wgs) {
    const int64_t t = k < s0 ? k : k - s0 + s1;
    for (int i = threadIdx.x; p.fill_rest && i < p.Hq * p.D / 2; i += blockDim.x) {
      const int h = i / static_cast<int>(p.D / 2), d = i % static_cast<int>(p.D / 2);
      reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(p.out) + t * p.out_t + h * p.out_h)[d] = 0;
    }
    if (p.lse)
      for (int h = threadIdx.x; h < p.Hq; h += blockDim.x) p.lse[t * p.Hq + h] = -INFINITY;
  }
}

// v of the lanes 16 and 32 away (v_permlane16_swap / v_permlane32_swap of v with
// itself leave it and the partner's value in the two results)
__device__ __forceinline__ float max_x32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_x32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_x16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
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

// Two codes of a word (HI: the upper two) times 2^e as 16-bit values; sc: 2^e as fp32.
template <bool HI>
__device__ __forceinline__ uint32_t cvt_bf16(uint32_t w, float sc) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, sc, HI));
}
template <bool HI>
__device__ __forceinline__ uint32_t cvt_f16(uint32_t w, float sc) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, sc, HI));
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

// lse of a row (natural logarithm) from its maximum in log2 units and its sum
__device__ __forceinline__ float row_lse(float m, float l) {
  return l > 0.0f ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
}

// ---- decode ------------------------------------------------------------------

// A wave's 32 keys in registers: key t 16 + n of K for lane (n, g) = (lane % 16,
// lane / 16), columns 64 c + 16 g ..; rows t 16 + 4 g + i of V, columns (D/16) n ..
template <int D>
struct Tile {
  uint4 k[2][D / 64];
  uint32_t ks[2];
  uint32_t v[2][4][D / 64];
  uint32_t vs[2][D / 32];  // the scales of its four V rows
  bool ok[2];               // the page is there
};

template <int D>
__device__ __forceinline__ void load_tile(const lbfq_paged_params& p, const int32_t* table, int kvh, int kb, int n,
                                          int g, Tile<D>& x) {
  constexpr int NB = D / 16;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int key = kb + 16 * t, idx = key >> p.page_shift;
    int page = idx < p.table_cols ? table[idx] : -1;
    x.ok[t] = page >= 0 && page < p.num_pages;
    page = x.ok[t] ? page : 0;
    const int64_t row = ((static_cast<int64_t>(page) * p.Hk + kvh) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
    const uint8_t* kr = p.k_codes + (row + n) * D + 16 * g;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) x.k[t][c] = *reinterpret_cast<const uint4*>(kr + 64 * c);
    const uint8_t* vr = p.v_codes + (row + 4 * g) * D + NB * n;
    if constexpr (D == 128) {
      x.ks[t] = *reinterpret_cast<const uint32_t*>(p.k_scale + (row + n) * 4);
      const uint4 s = *reinterpret_cast<const uint4*>(p.v_scale + (row + 4 * g) * 4);
      x.vs[t][0] = s.x; x.vs[t][1] = s.y; x.vs[t][2] = s.z; x.vs[t][3] = s.w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint2 v = *reinterpret_cast<const uint2*>(vr + i * D);
        x.v[t][i][0] = v.x; x.v[t][i][1] = v.y;
      }
    } else {
      x.ks[t] = *reinterpret_cast<const uint16_t*>(p.k_scale + (row + n) * 2);
      const uint2 s = *reinterpret_cast<const uint2*>(p.v_scale + (row + 4 * g) * 2);
      x.vs[t][0] = s.x; x.vs[t][1] = s.y;
#pragma unroll
      for (int i = 0; i < 4; ++i) x.v[t][i][0] = *reinterpret_cast<const uint32_t*>(vr + i * D);
    }
  }
}

template <int DT, int D>
__global__ void __launch_bounds__(256) paged_decode_kernel(const Args a) {
  constexpr int NC = D / 64, NB = D / 16, NW = 4;
  const lbfq_paged_params& p = a.p;
  if (static_cast<int64_t>(blockIdx.x) >= a.main) {
    fill_rest(p, blockIdx.x - a.main, gridDim.x - a.main);
    return;
  }
  __shared__ __align__(16) float acc_s[NW][16][D + 4];
  __shared__ float m_s[NW][16], l_s[NW][16];
  const int split = static_cast<int>(blockIdx.x % a.splits);
  int64_t rest = blockIdx.x / a.splits;
  const int kvh = static_cast<int>(rest % p.Hk);
  rest /= p.Hk;
  const int tile0 = static_cast<int>(rest % a.tiles);
  const int64_t b = rest / a.tiles;
  const Seq s = sequence(p, b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int32_t* table = p.block_table + b * p.table_stride;
  const int64_t R = p.T * p.Hq, rows = static_cast<int64_t>(s.n) * a.G;
  for (int64_t r0 = static_cast<int64_t>(tile0) * 16; r0 < rows; r0 += static_cast<int64_t>(a.tiles) * 16) {
    // this lane's query; rows past the last repeat it and are not stored
    const int64_t rr = r0 + n < rows ? r0 + n : rows - 1;
    const int qi = static_cast<int>(rr / a.G), h = kvh * a.G + static_cast<int>(rr % a.G);
    const int lo_r = s.lo(qi), hi_r = s.hi(qi);
    const int first = static_cast<int>(r0 / a.G);
    const int last = static_cast<int>(((r0 + 16 < rows ? r0 + 16 : rows) - 1) / a.G);
    const int lo = s.lo(first), hi = s.hi(last);          // keys that some row sees
    const int lo_all = s.lo(last), hi_all = s.hi(first);  // keys that every row sees
    uint4 q[NC][2], q2[DT == kF16 ? NC : 1][2];
    {
      const uint16_t* qr = reinterpret_cast<const uint16_t*>(p.q) + (s.start + qi) * p.q_t + h * p.q_h + 16 * g;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint4 w = *reinterpret_cast<const uint4*>(qr + 64 * c + 8 * u);
          if constexpr (DT == kBF16) {
            q[c][u] = w;
          } else {
            const uint32_t in[4] = {w.x, w.y, w.z, w.w};
            uint32_t hi2[4], lo2[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = f16_bits_to_f32(static_cast<uint16_t>(in[e]));
              const float y = f16_bits_to_f32(static_cast<uint16_t>(in[e] >> 16));
              hi2[e] = pack_bf16(x, y);
              lo2[e] = pack_bf16(x - __uint_as_float(hi2[e] << 16), y - __uint_as_float(hi2[e] & 0xffff0000u));
            }
            q[c][u] = make_uint4(hi2[0], hi2[1], hi2[2], hi2[3]);
            q2[c][u] = make_uint4(lo2[0], lo2[1], lo2[2], lo2[3]);
          }
        }
    }
    v4f acc[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[nb][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    const int kt0 = lo / 32, nt = hi > lo ? (hi + 31) / 32 - kt0 : 0;
    const int per = (nt + a.splits - 1) / a.splits;
    const int begin = kt0 + split * per;
    const int end = begin + per < kt0 + nt ? begin + per : kt0 + nt;
    Tile<D> x;
    if (begin + wave < end) load_tile<D>(p, table, kvh, 32 * (begin + wave), n, g, x);
    for (int kt = begin + wave; kt < end; kt += NW) {
      const int kb = 32 * kt;
      Tile<D> nx;
      if (kt + NW < end) load_tile<D>(p, table, kvh, 32 * (kt + NW), n, g, nx);
      // S^T: lane (n, g) has query n, keys 16 t + 4 g + i
      float sc[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        v4f d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float e = __uint_as_float(((x.ks[t] >> (16 * c + 8 * (g >> 1))) & 0xffu) << 23);
          const uint32_t w[4] = {x.k[t][c].x, x.k[t][c].y, x.k[t][c].z, x.k[t][c].w};
          const uint4 k0 = make_uint4(cvt_bf16<false>(w[0], e), cvt_bf16<true>(w[0], e), cvt_bf16<false>(w[1], e),
                                      cvt_bf16<true>(w[1], e));
          const uint4 k1 = make_uint4(cvt_bf16<false>(w[2], e), cvt_bf16<true>(w[2], e), cvt_bf16<false>(w[3], e),
                                      cvt_bf16<true>(w[3], e));
          d = mfma16_bf16(k0, q[c][0], d);
          d = mfma16_bf16(k1, q[c][1], d);
          if constexpr (DT == kF16) {
            d = mfma16_bf16(k0, q2[c][0], d);
            d = mfma16_bf16(k1, q2[c][1], d);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[t][i] = d[i];
      }
      if (!(x.ok[0] && x.ok[1] && kb >= lo_all && kb + 32 <= hi_all)) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = kb + 16 * t + 4 * g + i;
            if (!x.ok[t] || key < lo_r || key >= hi_r) sc[t][i] = -INFINITY;
            // nothing that lies in the place of a key that no row sees may reach the product
            if (!x.ok[t] || key < lo || key >= hi) {
#pragma unroll
              for (int c = 0; c < NC; ++c) x.v[t][i][c] = 0;
              // (four scale bytes of the row at D = 128, two at D = 64)
              if constexpr (D == 128) x.vs[t][i] = 0x7f7f7f7fu;
              else x.vs[t][i / 2] = (x.vs[t][i / 2] & (i & 1 ? 0x0000ffffu : 0xffff0000u)) | (i & 1 ? 0x7f7f0000u : 0x7f7fu);
            }
          }
      }
      float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                       fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
      mx = max_x32(max_x16(mx)) * a.sml2;
      if (__any(mx > m)) {
        const float mn = fmaxf(m, mx);
        const float al = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= al;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[nb][i] *= al;
      }
      const float ms = m == -INFINITY ? 0.0f : m;
      uint32_t ph[4], pl[4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[t][i], a.sml2, -ms));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[t][i + 1], a.sml2, -ms));
          l += p0 + p1;
          const uint32_t w = pack_bf16(p0, p1);
          ph[2 * t + i / 2] = w;
          pl[2 * t + i / 2] = pack_bf16(p0 - __uint_as_float(w << 16), p1 - __uint_as_float(w & 0xffff0000u));
        }
      const uint4 pb = make_uint4(ph[0], ph[1], ph[2], ph[3]), pc = make_uint4(pl[0], pl[1], pl[2], pl[3]);
      // V^T: for product nb lane (n, g) has row NB n + nb, its eight keys in P's order
      uint32_t vv[8][NB / 2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t by;
          if constexpr (D == 128) by = x.vs[t][i] >> (8 * (n >> 2));
          else by = x.vs[t][i / 2] >> (16 * (i & 1) + 8 * (n >> 3));
          const float e = __uint_as_float((by & 0xffu) << 23);
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            vv[4 * t + i][2 * c] = cvt_bf16<false>(x.v[t][i][c], e);
            vv[4 * t + i][2 * c + 1] = cvt_bf16<true>(x.v[t][i][c], e);
          }
        }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const uint32_t sel = nb & 1 ? 0x07060302u : 0x05040100u;  // upper or lower halves of (second, first)
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __builtin_amdgcn_perm(vv[2 * j + 1][nb / 2], vv[2 * j][nb / 2], sel);
        const uint4 va = make_uint4(w[0], w[1], w[2], w[3]);
        acc[nb] = mfma16_bf16(va, pb, acc[nb]);
        acc[nb] = mfma16_bf16(va, pc, acc[nb]);
      }
      x = nx;
    }
    // join the waves
    l = add_x32(add_x16(l));
    if (g == 0) {
      m_s[wave][n] = m;
      l_s[wave][n] = l;
    }
    __syncthreads();
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, m_s[w][n]);
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int nb = 0; nb < NB; nb += 4)
        *reinterpret_cast<float4*>(&acc_s[wave][n][(4 * g + i) * NB + nb]) =
            make_float4(acc[nb][i] * f, acc[nb + 1][i] * f, acc[nb + 2][i] * f, acc[nb + 3][i] * f);
    __syncthreads();
    {
      const int row = threadIdx.x >> 4, part = threadIdx.x & 15;
      float MM = -INFINITY, L = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) MM = fmaxf(MM, m_s[w][row]);
#pragma unroll
      for (int w = 0; w < NW; ++w)
        L += m_s[w][row] == -INFINITY ? 0.0f : l_s[w][row] * __builtin_amdgcn_exp2f(m_s[w][row] - MM);
      if (r0 + row < rows) {
        float o[NB];
#pragma unroll
        for (int k = 0; k < NB; k += 4) {
          float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
          for (int w = 0; w < NW; ++w) {
            const float4 v = *reinterpret_cast<const float4*>(&acc_s[w][row][part * NB + k]);
            t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w;
          }
          o[k] = t.x; o[k + 1] = t.y; o[k + 2] = t.z; o[k + 3] = t.w;
        }
        const int64_t r = r0 + row;
        const int64_t tok = s.start + r / a.G;
        const int hh = kvh * a.G + static_cast<int>(r % a.G);
        if (a.splits == 1) {
          const float inv = L > 0.0f ? 1.0f / L : 0.0f;
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
          if (L > 0.0f) {
#pragma unroll
            for (int k = 0; k < NB; k += 4)
              *reinterpret_cast<float4*>(a.acc + at * D + part * NB + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
          }
        }
      }
    }
    __syncthreads();  // the next rows use the same LDS
  }
}

// ---- chunk -------------------------------------------------------------------

template <int D>
struct Lds {
  static constexpr int KP = 2 * D + 16;    // pitch of a K row: the eight rows of a ds_read phase on distinct banks
  static constexpr int VP = 2 * 64 + 16;   // pitch of a V^T row
  static constexpr int KBYTES = 64 * KP;
  static constexpr int BUF = KBYTES + D * VP;
};

// Key of K row i of a 32-key block (bits 2 and 3 of i exchanged): a lane's scores are
// then of consecutive keys, eight at a time.
__device__ __forceinline__ int key_of(int i) { return (i & 0x13) | ((i & 4) << 1) | ((i & 8) >> 1); }

// The largest byte of v over the wave, the same in every lane.
__device__ __forceinline__ int wave_max_byte(uint32_t v) {
  uint32_t x = v & 0xffu, y = (v >> 8) & 0xffu;
  x = x > y ? x : y;
  y = (v >> 16) & 0xffu;
  x = x > y ? x : y;
  y = v >> 24;
  x = x > y ? x : y;
#define LBFQ_ROR(c)                                                                                             \
  do {                                                                                                          \
    y = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), c, 0xf, 0xf, true));                \
    x = x > y ? x : y;                                                                                          \
  } while (0)
  LBFQ_ROR(0x128);  // row_ror:8, 4, 2, 1
  LBFQ_ROR(0x124);
  LBFQ_ROR(0x122);
  LBFQ_ROR(0x121);
#undef LBFQ_ROR
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = r[0] > r[1] ? r[0] : r[1];
  const auto r2 = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = r2[0] > r2[1] ? r2[0] : r2[1];
  return __builtin_amdgcn_readfirstlane(x);
}

// 2^(byte - E + 7) as fp32 (0 far below)
__device__ __forceinline__ float rel_scale(uint32_t byte, int E) {
  const int e = static_cast<int>(byte) - E + 134;
  return __uint_as_float(static_cast<uint32_t>(e < 0 ? 0 : e) << 23);
}

template <int DT, int D, int NW>
__global__ void __launch_bounds__(NW * 64, 2) paged_chunk_kernel(const Args a) {
  constexpr int NT = NW * 64, NKS = D / 16, NDB = D / 32, CH = D / 32;
  constexpr int KT = 64 * CH, VT = 8 * (D / 4);     // threads that K and V take, 32 codes each
  constexpr bool BOTH = NT < KT + VT;               // every thread does both
  static_assert(BOTH ? NT == KT && NT == VT : true, "a tile's threads");
  using L = Lds<D>;
  const lbfq_paged_params& p = a.p;
  if (static_cast<int64_t>(blockIdx.x) >= a.main) {
    fill_rest(p, blockIdx.x - a.main, gridDim.x - a.main);
    return;
  }
  __shared__ __align__(16) uint8_t lds[2 * L::BUF];
  // Workgroups go to the eight XCDs in turn: neighbours in `id` are on one
  // XCD, so the row tiles of a head share that XCD's L2.
  int64_t id = blockIdx.x;
  {
    const int64_t q8 = a.main / 8, r8 = a.main % 8, x = id % 8;
    id = x * q8 + (x < r8 ? x : r8) + id / 8;
  }
  // the last rows first: under a causal mask they take longest
  const int tile0 = a.tiles - 1 - static_cast<int>(id % a.tiles);
  int64_t rest = id / a.tiles;
  const int split = static_cast<int>(rest % a.splits);
  rest /= a.splits;
  const int kvh = static_cast<int>(rest % p.Hk);
  const int64_t b = rest / p.Hk;
  const Seq s = sequence(p, b);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 31, g = lane >> 5;
  const int32_t* table = p.block_table + b * p.table_stride;
  const int64_t R = p.T * p.Hq, rows = static_cast<int64_t>(s.n) * a.G;
  constexpr int QB = 32 * NW;
  const bool krole = BOTH || tid < KT, vrole = BOTH || (tid >= KT && tid < KT + VT);
  const int kid = tid, vid = BOTH ? tid : tid - KT;
  const int kkey = kid / CH, kch = kid % CH;          // K: a key's 32 columns
  const int vkg = vid / (D / 4), vdq = vid % (D / 4);  // V: eight keys by four columns

  for (int64_t r0 = static_cast<int64_t>(tile0) * QB; r0 < rows; r0 += static_cast<int64_t>(a.tiles) * QB) {
    const int64_t rw = r0 + wave * 32;
    const int64_t rr = rw + li < rows ? rw + li : rows - 1;
    const int qi = static_cast<int>(rr / a.G), h = kvh * a.G + static_cast<int>(rr % a.G);
    const int lo_r = s.lo(qi), hi_r = s.hi(qi);
    const int first = static_cast<int>(r0 / a.G);
    const int last = static_cast<int>(((r0 + QB < rows ? r0 + QB : rows) - 1) / a.G);
    const int lo = s.lo(first), hi = s.hi(last);
    // the same of the wave's rows
    const int64_t w0 = rw < rows ? rw : rows - 1, w1 = rw + 31 < rows ? rw + 31 : rows - 1;
    const int wf = __builtin_amdgcn_readfirstlane(static_cast<int>(w0 / a.G));
    const int wl = __builtin_amdgcn_readfirstlane(static_cast<int>(w1 / a.G));
    const int wlo = s.lo(wf), whi = rw < rows ? s.hi(wl) : 0, wlo_all = s.lo(wl), whi_all = s.hi(wf);

    uint4 q[NKS];
    {
      const uint16_t* qr = reinterpret_cast<const uint16_t*>(p.q) + (s.start + qi) * p.q_t + h * p.q_h + 8 * g;
#pragma unroll
      for (int k = 0; k < NKS; ++k) q[k] = *reinterpret_cast<const uint4*>(qr + 16 * k);
    }
    v16f acc[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[db][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    const int kt0 = lo / 64, nt = hi > lo ? (hi + 63) / 64 - kt0 : 0;
    const int per = (nt + a.splits - 1) / a.splits;
    const int begin = kt0 + split * per;
    const int end = begin + per < kt0 + nt ? begin + per : kt0 + nt;

    // staging registers of the next tile
    uint4 kc[2];
    uint32_t kse = 127, vc[8], vse[8 * CH / 4], vw = 0, kw = 0;
    bool vok = false;
    // exponents (bytes) of the tile in LDS and of acc; from 2^-63 on, so that no factor made of them underflows
    int E = 64, Ek = 64, Eacc = 64;

    auto row_of = [&](int key, bool& ok) -> int64_t {
      const int idx = key >> p.page_shift;
      int page = idx < p.table_cols ? table[idx] : -1;
      ok = page >= 0 && page < p.num_pages;
      page = ok ? page : 0;
      return ((static_cast<int64_t>(page) * p.Hk + kvh) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
    };
    auto stage_load = [&](int kt) {
      const int kb = 64 * kt;
      if (krole) {
        bool ok;
        const int64_t row = row_of(kb + kkey, ok);
        const uint4* src = reinterpret_cast<const uint4*>(p.k_codes + row * D + 32 * kch);
        kc[0] = src[0];
        kc[1] = src[1];
        kse = p.k_scale[row * CH + kch];
      }
      if (vrole) {
        const int64_t row = row_of(kb + 8 * vkg, vok);
        const uint8_t* src = p.v_codes + row * D + 4 * vdq;
#pragma unroll
        for (int j = 0; j < 8; ++j) vc[j] = *reinterpret_cast<const uint32_t*>(src + j * D);
#pragma unroll
        for (int c = 0; c < 8 * CH / 16; ++c) {
          const uint4 w = reinterpret_cast<const uint4*>(p.v_scale + row * CH)[c];
          vse[4 * c] = w.x; vse[4 * c + 1] = w.y; vse[4 * c + 2] = w.z; vse[4 * c + 3] = w.w;
        }
      }
      {
        bool ok;
        const int64_t row = row_of(kb + lane, ok);
        ok = ok && kb + lane >= lo && kb + lane < hi;
        if constexpr (CH == 4) vw = *reinterpret_cast<const uint32_t*>(p.v_scale + row * CH);
        else vw = *reinterpret_cast<const uint16_t*>(p.v_scale + row * CH);
        vw = ok ? vw : 0;
        if constexpr (DT == kF16) {
          if constexpr (CH == 4) kw = *reinterpret_cast<const uint32_t*>(p.k_scale + row * CH);
          else kw = *reinterpret_cast<const uint16_t*>(p.k_scale + row * CH);
          kw = ok ? kw : 0;
        }
      }
    };
    auto stage_store = [&](int kt, uint8_t* buf) {
      const int kb = 64 * kt;
      const int t = wave_max_byte(vw);
      E = t > E ? t : E;
      if constexpr (DT == kF16) {
        Ek = wave_max_byte(kw);
        Ek = Ek > 64 ? Ek : 64;
      }
      if (krole) {
        const uint32_t w[8] = {kc[0].x, kc[0].y, kc[0].z, kc[0].w, kc[1].x, kc[1].y, kc[1].z, kc[1].w};
        uint32_t o[16];
        const float e = DT == kF16 ? rel_scale(kse, Ek) : __uint_as_float(kse << 23);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          o[2 * k] = DT == kF16 ? cvt_f16<false>(w[k], e) : cvt_bf16<false>(w[k], e);
          o[2 * k + 1] = DT == kF16 ? cvt_f16<true>(w[k], e) : cvt_bf16<true>(w[k], e);
        }
        uint4* dst = reinterpret_cast<uint4*>(buf + kkey * L::KP + 64 * kch);
#pragma unroll
        for (int k = 0; k < 4; ++k) dst[k] = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
      }
      if (vrole) {
        const bool edge = kb < lo || kb + 64 > hi;
        uint32_t o[8][2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t by;
          if constexpr (CH == 4) by = vse[j] >> (8 * (vdq / 8));
          else by = vse[j / 2] >> (16 * (j & 1) + 8 * (vdq / 8));
          by &= 0xffu;
          uint32_t w = vc[j];
          const int key = kb + 8 * vkg + j;
          if (!vok || (edge && (key < lo || key >= hi))) {  // never seen: nothing of it may reach the product
            w = 0;
            by = 1;
          }
          const float e = rel_scale(by, E);
          o[j][0] = cvt_f16<false>(w, e);
          o[j][1] = cvt_f16<true>(w, e);
        }
        // column 4 dq + c is V^T row c D/4 + dq, so that neighbouring lanes write neighbouring rows
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t sel = c & 1 ? 0x07060302u : 0x05040100u;
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = __builtin_amdgcn_perm(o[2 * j + 1][c / 2], o[2 * j][c / 2], sel);
          *reinterpret_cast<uint4*>(buf + L::KBYTES + (c * (D / 4) + vdq) * L::VP + 16 * vkg) =
              make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    };

    if (begin < end) {
      stage_load(begin);
      stage_store(begin, lds);
    }
    __syncthreads();
    for (int kt = begin; kt < end; ++kt) {
      const uint8_t* buf = lds + ((kt - begin) & 1) * L::BUF;
      const int kb = 64 * kt;
      const int Et = E, Ekt = Ek;
      if (kt + 1 < end) stage_load(kt + 1);
      if (kb < whi && kb + 64 > wlo) {
        v16f sc[2];
#pragma unroll
        for (int bl = 0; bl < 2; ++bl) {
          const uint8_t* kr = buf + (32 * bl + key_of(li)) * L::KP + 16 * g;
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[bl][r] = 0.0f;
#pragma unroll
          for (int k = 0; k < NKS; ++k) {
            const uint4 kop = *reinterpret_cast<const uint4*>(kr + 32 * k);
            if constexpr (DT == kBF16) sc[bl] = mfma32_bf16(kop, q[k], sc[bl]);
            else sc[bl] = mfma32_f16(kop, q[k], sc[bl]);
          }
        }
        // register r of block bl is key kb + 32 bl + 16 (r / 8) + 8 g + r % 8
        bool whole = kb >= wlo_all && kb + 64 <= whi_all;
        uint32_t pages = 0xfu;  // of the tile's four groups of 16 keys, those whose page is there
        {
          bool ok = true;
          if (lane < 4) {
            const int idx = (kb + 16 * lane) >> p.page_shift;
            const int page = idx < p.table_cols ? table[idx] : -1;
            ok = page >= 0 && page < p.num_pages;
          }
          pages = static_cast<uint32_t>(__ballot(ok)) & 0xfu;
          whole = whole && pages == 0xfu;
        }
        if (!whole) {
#pragma unroll
          for (int bl = 0; bl < 2; ++bl)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int key = kb + 32 * bl + 16 * (r >> 3) + 8 * g + (r & 7);
              if (key < lo_r || key >= hi_r || !((pages >> (2 * bl + (r >> 3))) & 1u)) sc[bl][r] = -INFINITY;
            }
        }
        const float c = DT == kF16 ? a.sml2 * ldexpf(1.0f, Ekt - 134) : a.sml2;
        float mx = -INFINITY;
#pragma unroll
        for (int bl = 0; bl < 2; ++bl)
#pragma unroll
          for (int r = 0; r < 16; r += 2) mx = fmaxf(mx, fmaxf(sc[bl][r], sc[bl][r + 1]));
        mx = max_x32(mx) * c;
        // p may grow to 2^8 past the maximum in use before that is moved (fp16 holds 65504)
        if (__any(mx > m + 8.0f) || Et != Eacc) {
          const float mn = fmaxf(m, mx);
          const float al = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
          const float ae = al * ldexpf(1.0f, Eacc - Et);
          m = mn;
          l *= al;
          Eacc = Et;
#pragma unroll
          for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[db][r] *= ae;
        }
        const float ms = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int bl = 0; bl < 2; ++bl)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int r = 8 * j + 2 * k;
              const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[bl][r], c, -ms));
              const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[bl][r + 1], c, -ms));
              l += p0 + p1;
              w[k] = pack_f16(p0, p1);
            }
            const uint4 pb = make_uint4(w[0], w[1], w[2], w[3]);
            const uint8_t* vr = buf + L::KBYTES + li * L::VP + 16 * g + 32 * (2 * bl + j);
#pragma unroll
            for (int db = 0; db < NDB; ++db)
              acc[db] = mfma32_f16(*reinterpret_cast<const uint4*>(vr + 32 * db * L::VP), pb, acc[db]);
          }
      }
      if (kt + 1 < end) stage_store(kt + 1, lds + ((kt + 1 - begin) & 1) * L::BUF);
      __syncthreads();
    }
    // V^T row x = c D/4 + dq holds column 4 dq + c.  Row 32 db + 8 (r / 4) + 4 g + r % 4 is lane (li, g)'s register r
    // of acc[db].
    l = add_x32(l);
    const float back = ldexpf(1.0f, Eacc - 134);
    if (rw + li < rows) {
      const int64_t tok = s.start + qi;
      const bool one = a.splits == 1;
      const float f = one ? (l > 0.0f ? back / l : 0.0f) : back;
      const int64_t at = split * R + tok * p.Hq + h;
      if (one && p.lse && g == 0) p.lse[tok * p.Hq + h] = row_lse(m, l);
      if (!one && g == 0) a.ml[at] = make_float2(m, l);
      if (one || l > 0.0f) {
        if constexpr (D == 128) {
          // c = db, dq = 8 (r / 4) + 4 g + r % 4: four consecutive columns from the four blocks
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const int col = 32 * r4 + 16 * g;
            float o[16];
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int db = 0; db < NDB; ++db) o[4 * k + db] = acc[db][4 * r4 + k] * f;
            if (one) {
              uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + tok * p.out_t + h * p.out_h + col);
              dst[0] = make_uint4(pack_dt<DT>(o[0], o[1]), pack_dt<DT>(o[2], o[3]), pack_dt<DT>(o[4], o[5]),
                                  pack_dt<DT>(o[6], o[7]));
              dst[1] = make_uint4(pack_dt<DT>(o[8], o[9]), pack_dt<DT>(o[10], o[11]), pack_dt<DT>(o[12], o[13]),
                                  pack_dt<DT>(o[14], o[15]));
            } else {
              float4* dst = reinterpret_cast<float4*>(a.acc + at * D + col);
#pragma unroll
              for (int k = 0; k < 4; ++k) dst[k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
            }
          }
        } else {
          // D = 64: row x = 16 c + dq; block db holds c = 2 db (r < 8) and 2 db + 1, dq = 8 ((r / 4) % 2) + 4 g + r % 4
#pragma unroll
          for (int half = 0; half < 2; ++half)
            {
              const int col = 32 * half + 16 * g;
              float o[16];
#pragma unroll
              for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[4 * k + c] = acc[c / 2][8 * (c & 1) + 4 * half + k] * f;
              if (one) {
                uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + tok * p.out_t + h * p.out_h + col);
                dst[0] = make_uint4(pack_dt<DT>(o[0], o[1]), pack_dt<DT>(o[2], o[3]), pack_dt<DT>(o[4], o[5]),
                                    pack_dt<DT>(o[6], o[7]));
                dst[1] = make_uint4(pack_dt<DT>(o[8], o[9]), pack_dt<DT>(o[10], o[11]), pack_dt<DT>(o[12], o[13]),
                                    pack_dt<DT>(o[14], o[15]));
              } else {
                float4* dst = reinterpret_cast<float4*>(a.acc + at * D + col);
#pragma unroll
                for (int k = 0; k < 4; ++k) dst[k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
              }
            }
        }
      }
    }
    __syncthreads();
  }
}

// ---- joining the parts of the keys ---------------------------------------------

// A wave per row: 2^(m_s - M) weights of the parts, summed in their order.
template <int DT, int D>
__global__ void __launch_bounds__(256) paged_combine_kernel(const Args a) {
  const lbfq_paged_params& p = a.p;
  const int64_t R = p.T * p.Hq;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= R) return;
  const int lane = threadIdx.x & 63;
  const int64_t tok = row / p.Hq;
  const int h = static_cast<int>(row - tok * p.Hq);
  uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + tok * p.out_t + h * p.out_h + lane * (D / 64);
  const bool mine = tok >= p.query_starts[0] && tok < p.query_starts[p.B];
  float M = -INFINITY, l = 0.0f, o[D / 64];
#pragma unroll
  for (int k = 0; k < D / 64; ++k) o[k] = 0.0f;
  if (mine) {
    for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.ml[s * R + row].x);
    for (int s = 0; s < a.splits; ++s) {
      const float2 x = a.ml[s * R + row];
      if (!(x.y > 0.0f)) continue;  // nothing in this part (its sums were not written)
      const float f = __builtin_amdgcn_exp2f(x.x - M);
      l = fmaf(x.y, f, l);
#pragma unroll
      for (int k = 0; k < D / 64; ++k) o[k] = fmaf(a.acc[(s * R + row) * D + lane * (D / 64) + k], f, o[k]);
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  if (mine || p.fill_rest) {
    if constexpr (D == 128) *reinterpret_cast<uint32_t*>(dst) = pack_dt<DT>(o[0] * inv, o[1] * inv);
    else *dst = static_cast<uint16_t>(pack_dt<DT>(o[0] * inv, 0.0f));
  }
  if (p.lse && lane == 0) p.lse[row] = row_lse(M, l);
}

// ---- host --------------------------------------------------------------------

struct Plan {
  bool decode;
  int tiles, splits;
};

constexpr int kDecodeRows = 16;

Plan plan(const lbfq_paged_params* p) {
  Plan x;
  const int64_t G = p->Hq / p->Hk;
  const int64_t most = p->max_query_len > 0 && p->max_query_len < p->T ? p->max_query_len : p->T;
  const int64_t rows = most * G;
  x.decode = rows <= kDecodeRows;
  const int64_t tile = x.decode ? 16 : 128;
  x.tiles = static_cast<int>((rows + tile - 1) / tile);
  const int64_t wgs = x.tiles * p->Hk * p->B;
  const int64_t keys = p->table_cols << p->page_shift;
  const int64_t want = x.decode ? 2048 : 512, least = x.decode ? 256 : 512;
  int64_t s = want / wgs;
  if (s > keys / least) s = keys / least;
  if (s > 64) s = 64;
  x.splits = s < 1 ? 1 : static_cast<int>(s);
  return x;
}

int64_t workspace(const lbfq_paged_params* p, const Plan& x) {
  if (x.splits == 1) return 0;
  const int64_t R = p->T * p->Hq;
  return x.splits * R * (static_cast<int64_t>(sizeof(float2)) + p->D * 4) + 16;
}

int check(const lbfq_paged_params* p) {
  const char* who = "lbfq_paged_attention";
  LBFQ_CHECK_ARG(p, "%s: null params", who);
  LBFQ_CHECK_ARG(p->D == 64 || p->D == 128, "%s: D must be 64 or 128", who);
  LBFQ_CHECK_ARG(p->dtype == kBF16 || p->dtype == kF16, "%s: queries are bf16 or fp16", who);
  LBFQ_CHECK_ARG(p->Hk > 0 && p->Hq > 0 && p->Hq % p->Hk == 0 && p->Hq < (1 << 16),
                 "%s: the query heads must be a multiple of the key heads", who);
  LBFQ_CHECK_ARG(p->T > 0 && p->B > 0 && p->T < (int64_t{1} << 30) && p->B < (int64_t{1} << 30),
                 "%s: bad number of tokens or sequences", who);
  LBFQ_CHECK_ARG(p->page_shift >= 4 && p->page_shift <= 10, "%s: pages hold 16 to 1024 tokens, a power of two", who);
  LBFQ_CHECK_ARG(p->num_pages > 0 && p->num_pages < (int64_t{1} << 31), "%s: bad number of pages", who);
  LBFQ_CHECK_ARG(p->table_cols > 0 && (p->table_cols << p->page_shift) <= (int64_t{1} << 30) &&
                     p->table_cols < (int64_t{1} << 30) && p->table_stride >= 0,
                 "%s: bad block table", who);
  LBFQ_CHECK_ARG(p->q && p->out && p->block_table && p->seq_lens && p->query_starts && p->k_codes && p->k_scale &&
                     p->v_codes && p->v_scale,
                 "%s: missing tensor", who);
  LBFQ_CHECK_ARG(((reinterpret_cast<uint64_t>(p->q) | reinterpret_cast<uint64_t>(p->out) |
                   reinterpret_cast<uint64_t>(p->k_codes) | reinterpret_cast<uint64_t>(p->v_codes) |
                   reinterpret_cast<uint64_t>(p->k_scale) | reinterpret_cast<uint64_t>(p->v_scale)) & 15) == 0 &&
                     ((p->q_t | p->q_h | p->out_t | p->out_h) & 7) == 0,
                 "%s: rows must be 16-byte aligned", who);
  LBFQ_CHECK_ARG(p->sm_scale > 0.0f && p->sm_scale < INFINITY, "%s: sm_scale must be positive and finite", who);
  LBFQ_CHECK_ARG(p->window >= 0 && p->window <= (int64_t{1} << 30), "%s: bad window", who);
  return 0;
}

}  // namespace

extern "C" int64_t lbfq_paged_attention_workspace_bytes(const lbfq_paged_params* p) {
  if (!p || p->Hk <= 0 || p->Hq <= 0 || p->T <= 0 || p->B <= 0 || p->table_cols <= 0) return 0;
  return workspace(p, plan(p));
}

extern "C" int lbfq_paged_attention(const lbfq_paged_params* p, lbfq_stream_t stream) {
  if (int rc = check(p)) return rc;
  const Plan x = plan(p);
  Args a{};
  a.p = *p;
  a.G = static_cast<int>(p->Hq / p->Hk);
  a.tiles = x.tiles;
  a.splits = x.splits;
  a.sml2 = p->sm_scale * kLog2e;
  const int64_t R = p->T * p->Hq;
  if (x.splits > 1) {
    LBFQ_CHECK_ARG(p->workspace && p->workspace_bytes >= workspace(p, x), "lbfq_paged_attention: workspace too small");
    LBFQ_CHECK_ARG((reinterpret_cast<uint64_t>(p->workspace) & 15) == 0, "lbfq_paged_attention: workspace alignment");
    a.acc = static_cast<float*>(p->workspace);
    a.ml = reinterpret_cast<float2*>(a.acc + x.splits * R * p->D);
  }
  LBFQ_CHECK_ARG(p->B < (int64_t{1} << 30) / (p->Hk * x.splits) / x.tiles, "lbfq_paged_attention: problem too large");
  a.main = p->B * p->Hk * x.tiles * x.splits;
  // rows that no sequence has: the combine kernel sees every row, otherwise some workgroups more
  const int64_t fill = (p->fill_rest || p->lse) && x.splits == 1 ? 8 : 0;
  const dim3 grid(static_cast<unsigned>(a.main + fill));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool bf = p->dtype == kBF16, d128 = p->D == 128;
  if (x.decode) {
    const dim3 block(256);
    if (bf && d128) hipLaunchKernelGGL((paged_decode_kernel<kBF16, 128>), grid, block, 0, st, a);
    else if (bf) hipLaunchKernelGGL((paged_decode_kernel<kBF16, 64>), grid, block, 0, st, a);
    else if (d128) hipLaunchKernelGGL((paged_decode_kernel<kF16, 128>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((paged_decode_kernel<kF16, 64>), grid, block, 0, st, a);
  } else {
    const dim3 block(256);
    if (bf && d128) hipLaunchKernelGGL((paged_chunk_kernel<kBF16, 128, 4>), grid, block, 0, st, a);
    else if (bf) hipLaunchKernelGGL((paged_chunk_kernel<kBF16, 64, 4>), grid, block, 0, st, a);
    else if (d128) hipLaunchKernelGGL((paged_chunk_kernel<kF16, 128, 4>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((paged_chunk_kernel<kF16, 64, 4>), grid, block, 0, st, a);
  }
  LBFQ_LAUNCH_CHECK("lbfq_paged_attention");
  if (x.splits > 1) {
    const dim3 gc(static_cast<unsigned>((R + 3) / 4)), block(256);
    if (bf && d128) hipLaunchKernelGGL((paged_combine_kernel<kBF16, 128>), gc, block, 0, st, a);
    else if (bf) hipLaunchKernelGGL((paged_combine_kernel<kBF16, 64>), gc, block, 0, st, a);
    else if (d128) hipLaunchKernelGGL((paged_combine_kernel<kF16, 128>), gc, block, 0, st, a);
    else hipLaunchKernelGGL((paged_combine_kernel<kF16, 64>), gc, block, 0, st, a);
    LBFQ_LAUNCH_CHECK("lbfq_paged_attention (combine)");
  }
  return 0;
}

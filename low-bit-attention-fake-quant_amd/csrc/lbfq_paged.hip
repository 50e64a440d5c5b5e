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
// Two kernels (for the cache in 8 bits; in 4 bits those of lbfq_paged4.hip and lbfq_paged4_chunk.hip).
//
// decode (up to 16 rows: one token of a sequence, 16x16x32 MFMA).  Bound by reading the cache, 2 D (1 + 1/32) bytes a key
// and head.  A wave takes 32 keys at a time straight into registers; a workgroup's four waves take turns, workgroups
// split the keys, and the parts are joined by their maxima (in LDS, then by the combine kernel).  Operands are bf16,
// which holds code * 2^e exactly (four significant bits); fp16 queries are two bf16 terms (eleven bits, exact); P is two
// bf16 terms (16 bits).  48 sequences of 8000 to 16000 keys, 32 / 8 heads of 128: 230 us, 5.3 TB/s of the 6.4 that a kernel
// that only reads reaches; the same loads without the arithmetic take 218.
//
// chunk (more rows, 32x32x16 MFMA).  A workgroup's four waves have 32 rows each; 64-key tiles are read once, converted to
// 16 bits and staged in LDS, one barrier a tile.  A wave and tile take 32 MFMAs of 32 cycles and about 240 VALU
// instructions, 32 of them exponentials, and the two share a SIMD's power and issue: so the loop runs the next tile's
// scores and this one's P V beside the softmax and the conversion, in an order fixed here.  V goes through fp16, times
// one power of two for the workgroup's part of the keys: every value that fits is exact, and a part whose scales lie too
// far apart for that takes a slower loop with V in bf16 and P in two bf16 terms.  So P can be fp16: 11 bits, where
// bf16's 8 would cost as much as the output's own rounding.  K is bf16 (exact) for bf16 queries, and for fp16 ones fp16
// under the same rule.  4680 tokens over 32760 keys, 12 heads of 128, all seen: 1.10 ms, 855 TFLOP/s, the matrix units
// busy 39% of the cycles at 2.1 GHz (a large library product: 1218 TFLOP/s).
#include "lbfq_paged_common.h"

using namespace lbfq;
using namespace lbfq::paged;

namespace {

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

// The page ids of the two halves of a tile (-1: none); the same in every lane.
__device__ __forceinline__ void load_pages(const lbfq_paged_params& p, const int32_t* table, int kb, int (&page)[2]) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int idx = (kb + 16 * t) >> p.page_shift;
    page[t] = idx < p.table_cols ? table[idx] : -1;
  }
}

template <int D>
__device__ __forceinline__ void load_tile(const lbfq_paged_params& p, const int (&pages)[2], int kvh, int kb, int n,
                                          int g, Tile<D>& x) {
  constexpr int NB = D / 16;
  int64_t row[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    x.ok[t] = pages[t] >= 0 && pages[t] < p.num_pages;
    const int page = x.ok[t] ? pages[t] : 0;
    row[t] = (static_cast<int64_t>(page * static_cast<int>(p.Hk) + kvh) << p.page_shift) +
             ((kb + 16 * t) & ((1 << p.page_shift) - 1));
    const uint8_t* kr = p.k_codes + row[t] * D + (n * D + 16 * g);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) x.k[t][c] = *reinterpret_cast<const uint4*>(kr + 64 * c);
    const uint8_t* ks = p.k_scale + row[t] * (D / 32) + n * (D / 32);
    if constexpr (D == 128) x.ks[t] = *reinterpret_cast<const uint32_t*>(ks);
    else x.ks[t] = *reinterpret_cast<const uint16_t*>(ks);
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint8_t* vr = p.v_codes + row[t] * D + (4 * g * D + NB * n);
    const uint8_t* vs = p.v_scale + row[t] * (D / 32) + 4 * g * (D / 32);
    if constexpr (D == 128) {
      const uint4 s = *reinterpret_cast<const uint4*>(vs);
      x.vs[t][0] = s.x; x.vs[t][1] = s.y; x.vs[t][2] = s.z; x.vs[t][3] = s.w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint2 v = *reinterpret_cast<const uint2*>(vr + i * D);
        x.v[t][i][0] = v.x; x.v[t][i][1] = v.y;
      }
    } else {
      const uint2 s = *reinterpret_cast<const uint2*>(vs);
      x.vs[t][0] = s.x; x.vs[t][1] = s.y;
#pragma unroll
      for (int i = 0; i < 4; ++i) x.v[t][i][0] = *reinterpret_cast<const uint32_t*>(vr + i * D);
    }
  }
}

template <int DT, int D>
__global__ void __launch_bounds__(256, 3) paged_decode_kernel(const Args a) {
  constexpr int NC = D / 64, NB = D / 16, NW = 4;
  const lbfq_paged_params& p = a.p;
  if (static_cast<int64_t>(blockIdx.x) >= a.main) {
    fill_rest<D>(p, blockIdx.x - a.main, gridDim.x - a.main);
    return;
  }
  __shared__ DecodeLds<D> join;
  // 32-bit indices: the divisions of 64-bit ones were most of this kernel's code and a fifth of a small call's time
  // The parts come last: those behind a short sequence's end then leave the XCDs (workgroups go to them in turn) and their
  // shader engines evenly loaded.
  const uint32_t Hk = static_cast<uint32_t>(p.Hk);
  const int split = static_cast<int>(blockIdx.x / a.combos);
  const uint32_t rest = blockIdx.x % a.combos;
  const int b = static_cast<int>(rest / Hk), kvh = static_cast<int>(rest % Hk);
  const Seq s = sequence(p, b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int32_t* table = p.block_table + b * p.table_stride;
  const int64_t R = p.T * p.Hq;
  const int G = a.G, rows = s.n * G;  // below 2^30: the host checks T * Hq
  for (int r0 = 0; r0 < rows; r0 += 16) {  // once, but for more new tokens than max_query_len
    // this lane's query; rows past the last repeat it and are not stored
    const int rr = r0 + n < rows ? r0 + n : rows - 1;
    const int qi = rr / G, h = kvh * G + (rr - qi * G);
    const int lo_r = s.lo(qi), hi_r = s.hi(qi);
    const int first = r0 / G;
    const int last = ((r0 + 16 < rows ? r0 + 16 : rows) - 1) / G;
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
            split_f16(w, q[c][u], q2[c][u]);
          }
        }
    }
    v4f acc[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[nb][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    int up = kUp;
    bool large = false;  // some block's unit is below the bytes

    const int kt0 = lo / 32, nt = hi > lo ? (hi + 31) / 32 - kt0 : 0;
    int per = (nt + a.splits - 1) / a.splits;
    per = per > a.least ? per : a.least;
    const int begin = kt0 + split * per;
    const int end = begin + per < kt0 + nt ? begin + per : kt0 + nt;
    int pages[2];
    load_pages(p, table, 32 * (begin + wave), pages);
    for (int kt = begin + wave; kt < end; kt += NW) {
      const int kb = 32 * kt;
      Tile<D> x;
      load_tile<D>(p, pages, kvh, kb, n, g, x);
      load_pages(p, table, 32 * (kt + NW), pages);
      // S^T: lane (n, g) has query n, keys 16 t + 4 g + i
      float sc[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        v4f d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float e = __uint_as_float(((x.ks[t] >> (16 * c + 8 * (g >> 1))) & 0xffu) << 23);
          const uint32_t kw[4] = {x.k[t][c].x, x.k[t][c].y, x.k[t][c].z, x.k[t][c].w};
          const uint4 k0 = make_uint4(cvt_bf16<8>(kw, 0, e), cvt_bf16<8>(kw, 1, e), cvt_bf16<8>(kw, 2, e), cvt_bf16<8>(kw, 3, e));
          const uint4 k1 = make_uint4(cvt_bf16<8>(kw, 4, e), cvt_bf16<8>(kw, 5, e), cvt_bf16<8>(kw, 6, e), cvt_bf16<8>(kw, 7, e));
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
      // this lane's block's scales of its eight keys
      int by[8], top = 0;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t w;
          if constexpr (D == 128) w = x.vs[t][i] >> (8 * (n >> 2));
          else w = x.vs[t][i / 2] >> (16 * (i & 1) + 8 * (n >> 3));
          by[4 * t + i] = static_cast<int>(w & 0xffu);
          top = by[4 * t + i] > top ? by[4 * t + i] : top;
        }
      if (__any(top + up > kTop)) {
        lower_unit<D>(top, up, acc);
        large = __any(up < 0);
      }
      if (large) {
#pragma unroll
        for (int j = 0; j < 8; ++j) by[j] = by[j] > -up ? by[j] : -up;
      }
      float mx = vmax(vmax(vmax(sc[0][0], sc[0][1]), vmax(sc[0][2], sc[0][3])),
                       vmax(vmax(sc[1][0], sc[1][1]), vmax(sc[1][2], sc[1][3])));
      mx = max_x32(max_x16(mx)) * a.sml2;
      if (__any(mx > m)) {
        const float mn = vmax(m, mx);
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
          const float e = __uint_as_float(static_cast<uint32_t>(by[4 * t + i] + up) << 23);
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            vv[4 * t + i][2 * c] = cvt_bf16<8>(x.v[t][i], 2 * c, e);
            vv[4 * t + i][2 * c + 1] = cvt_bf16<8>(x.v[t][i], 2 * c + 1, e);
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
    }
    join_waves<DT, D>(a, s, acc, m, l, up, join, r0, rows, split, kvh);
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

template <int DT, int D>
__global__ void __launch_bounds__(256, chunk_groups(DT, D)) paged_chunk_kernel(const Args a) {
  constexpr int NW = 4, QB = kChunkRows, NT = 64 * NW;
  static_assert(QB == 32 * NW, "32 rows a wave");
  constexpr int NKS = D / 16, NDB = D / 32, CH = D / 32;
  constexpr int KC = 64 * D / NT;  // K codes of a thread
  constexpr int KT = D / KC;       // threads of a key's row
  constexpr int VK = KC / 4;       // V keys of a thread, four columns each
  constexpr int WKEYS = 64 / NW;   // keys that a wave stages: of one page
  using L = Lds<D>;
  const lbfq_paged_params& p = a.p;
  if (static_cast<int64_t>(blockIdx.x) >= a.main) {
    fill_rest<D>(p, blockIdx.x - a.main, gridDim.x - a.main);
    return;
  }
  __shared__ __align__(16) uint8_t lds[2 * L::BUF];
  // Workgroups go to the eight XCDs in turn.  Pieces of up to eight neighbouring row tiles are dealt to them whole, so that
  // those that read the same keys share an L2; the pieces of all heads and parts (`combos`) with the last rows first,
  // which take longest under a causal mask, and turned by one XCD from round to round, so that none has all of a kind.
  // (No slots in vain: where seven of eight workgroups had nothing to do, the others shared a quarter of the chip: an
  // XCD's four shader engines take its workgroups in turn.  1024 keys, 512 heads of 128 rows: 203 us, dense 60.)
  const uint32_t ps = a.piece, round = blockIdx.x / (8 * ps), piece = round * 8 + (blockIdx.x + round) % 8;
  const int slot = a.slots - 1 - static_cast<int>(piece / a.combos * ps + blockIdx.x / 8 % ps);
  if (slot < 0) return;
  const uint32_t rest = piece % a.combos, splits = static_cast<uint32_t>(a.splits);
  const int split = static_cast<int>(rest % splits), kvh = static_cast<int>(rest / splits);
  const int G = a.G, Hk = static_cast<int>(p.Hk);
  const int b = sequence_at(p, G, slot), r0 = (slot - slot_of(p, G, b)) * QB;
  const Seq s = sequence(p, b);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 31, g = lane >> 5;
  const int32_t* table = p.block_table + b * p.table_stride;
  const int cols = static_cast<int>(p.table_cols), num_pages = static_cast<int>(p.num_pages);
  const int shift = p.page_shift, pmask = (1 << p.page_shift) - 1;
  const int64_t R = p.T * p.Hq;
  const int rows = s.n * G;  // below 2^30: the host checks T * Hq
  if (r0 < 0 || r0 >= rows) return;
  // Staging: wave w takes keys WKEYS w .. of a tile, which lie in one page.
  const int kkey = lane / KT, kq = lane % KT;           // K: key kkey of the wave's, columns KC kq ..
  const int vkg = lane / (D / 4), vdq = lane % (D / 4);  // V: keys VK vkg .. of the wave's, columns 4 vdq ..
  static_assert(64 / KT == WKEYS && 64 / (D / 4) * VK == WKEYS, "a wave's keys");
  const uint32_t koff = kkey * D + KC * kq, ksoff = kkey * CH + KC * kq / 32;
  const uint32_t voff = VK * vkg * D + 4 * vdq, vsoff = VK * vkg * CH;

  auto row_of = [&](int page, int key) -> int64_t {
    return (static_cast<int64_t>(page * Hk + kvh) << shift) + (key & pmask);
  };

  const int rw = r0 + wave * 32;
  const int rr = rw + li < rows ? rw + li : rows - 1;
  const int qi = rr / G, h = kvh * G + (rr - qi * G);
  const int lo_r = s.lo(qi), hi_r = s.hi(qi);
  const int first = r0 / G, last = ((r0 + QB < rows ? r0 + QB : rows) - 1) / G;
  const int lo = s.lo(first), hi = s.hi(last);  // keys that some row of the workgroup sees
  const int wf = __builtin_amdgcn_readfirstlane((rw < rows ? rw : rows - 1) / G);
  const int wl = __builtin_amdgcn_readfirstlane((rw + 31 < rows ? rw + 31 : rows - 1) / G);
  const int lo_all = s.lo(wl), hi_all = s.hi(wf);            // that every row of the wave sees

  const int kt0 = lo / 64, nt = hi > lo ? (hi + 63) / 64 - kt0 : 0;
  int per = (nt + a.splits - 1) / a.splits;
  per = per > a.least ? per : a.least;
  const int begin = kt0 + split * per;
  const int end = begin + per < kt0 + nt ? begin + per : kt0 + nt;

  v16f acc[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  Unit uv{134, false}, uk{134, false};
  uint32_t vtops = 0;  // V's unit: the byte that block b's scale vtops >> 8 b comes to is vtop
  int vtop = 134;
  if (begin < end) {
    uint4 q[NKS];
    {
      const uint16_t* qr = reinterpret_cast<const uint16_t*>(p.q) + (s.start + qi) * p.q_t + h * p.q_h + 8 * g;
#pragma unroll
      for (int k = 0; k < NKS; ++k) q[k] = *reinterpret_cast<const uint4*>(qr + 16 * k);
    }
    // Staging registers: codes and scales of a K tile and of a V tile.
    struct KRegs {
      uint32_t c[KC / 4], e;
    } kx, ky;
    uint32_t vc[VK], vse[VK * CH / 4];
    auto load_k = [&](KRegs& x, int kt, int page) {
      const int64_t row = row_of(page < 0 ? 0 : page, 64 * kt + WKEYS * wave);
      const uint8_t* ks = p.k_codes + row * D;
      const uint8_t* kss = p.k_scale + row * CH;
#pragma unroll
      for (int i = 0; i < KC / 16; ++i) {
        const uint4 w = *reinterpret_cast<const uint4*>(ks + koff + 16 * i);
        x.c[4 * i] = w.x; x.c[4 * i + 1] = w.y; x.c[4 * i + 2] = w.z; x.c[4 * i + 3] = w.w;
      }
      x.e = kss[ksoff];
    };
    auto load_v = [&](int kt, int page) {
      const int64_t row = row_of(page < 0 ? 0 : page, 64 * kt + WKEYS * wave);
      const uint8_t* vs = p.v_codes + row * D;
      const uint8_t* vss = p.v_scale + row * CH;
#pragma unroll
      for (int j = 0; j < VK; ++j) vc[j] = *reinterpret_cast<const uint32_t*>(vs + voff + j * D);
      if constexpr (D == 128) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 w = reinterpret_cast<const uint4*>(vss + vsoff)[i];
          vse[4 * i] = w.x; vse[4 * i + 1] = w.y; vse[4 * i + 2] = w.z; vse[4 * i + 3] = w.w;
        }
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(vss + vsoff);
        vse[0] = w.x; vse[1] = w.y;
      }
    };
    auto upto = [&](int kt) { return kt < end ? kt : end - 1; };  // steps past the end repeat it, unused
    // Page ids of the tiles from kt on: lane 4 i + w has that of tile kt + i's keys 16 w .., which wave w stages.  One load,
    // so one wait; looked up where they are needed, each id cost the time of a trip to memory (4680 tokens over 32760 keys,
    // 12 heads: 1.16 ms, so 1.10).
    auto group_of = [&](int kt) { return (64 * upto(kt + (lane >> 2 & 3)) + 16 * (lane & 3)) >> shift; };
    auto look = [&](int kt) {
      const int idx = group_of(kt);
      return table[idx < cols ? idx : cols - 1];
    };
    auto there = [&](int kt, int id) -> uint32_t {  // a bit per lane: the page is there
      return static_cast<uint32_t>(__ballot(group_of(kt) < cols && id >= 0 && id < num_pages));
    };
    auto page_in = [&](int id, uint32_t mask, int i) {  // of tile kt + i's keys of this wave, or -1; a scalar
      return mask >> (4 * i + wave) & 1u ? __builtin_amdgcn_readlane(id, 4 * i + wave) : -1;
    };
    // The first tiles are on their way while the scales are looked through.
    const int ids = look(begin);
    const uint32_t mask = there(begin, ids);
    const int page0 = page_in(ids, mask, 0), page1 = page_in(ids, mask, 1);
    load_k(kx, begin, page0);
    load_v(begin, page0);
    load_k(ky, upto(begin + 1), page1);
    // The span of the part's scales, over the keys that some row sees: four keys a thread and pass.
    {
      uint32_t sv = 0, sk = 0;
      const int k1 = 64 * end < hi ? 64 * end : hi;
      for (int key = 64 * begin + 4 * tid; key < k1; key += 4 * NT) {
        if (key + 4 <= lo) continue;
        const int idx = key >> shift;
        const int page = idx < cols ? table[idx] : -1;
        if (page < 0 || page >= num_pages) continue;
        const int64_t row = row_of(page, key);
        const bool whole = key >= lo && key + 4 <= k1;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          uint32_t x = reinterpret_cast<const uint32_t*>(p.v_scale + row * CH)[c];
          uint32_t y = DT == kF16 ? reinterpret_cast<const uint32_t*>(p.k_scale + row * CH)[c] : 0u;
          if (whole) {
            sv = span_add<4>(sv, x);
            if constexpr (DT == kF16) sk = span_add<4>(sk, y);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int ki = key + (4 * c + i) / CH;
              if (ki < lo || ki >= k1) continue;
              sv = span_add<1>(sv, x >> (8 * i));
              if constexpr (DT == kF16) sk = span_add<1>(sk, y >> (8 * i));
            }
          }
        }
      }
      uint32_t* red = reinterpret_cast<uint32_t*>(lds);
#pragma unroll
      for (int i = 1; i < 64; i <<= 1) {
        sv = span_join(sv, __shfl_xor(sv, i, 64));
        if constexpr (DT == kF16) sk = span_join(sk, __shfl_xor(sk, i, 64));
      }
      if (lane == 0) {
        red[wave] = sv;
        red[NW + wave] = sk;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        sv = span_join(sv, red[w]);
        sk = span_join(sk, red[NW + w]);
      }
      __syncthreads();
      auto unit = [&](uint32_t x) {
        x = __builtin_amdgcn_readfirstlane(x);
        Unit u;
        u.E = static_cast<int>(x & 0xffu);
        u.wide = u.E - (255 - static_cast<int>(x >> 16)) > span_of(8);
        if (x == 0) u.E = 134;
        return u;
      };
      uv = unit(sv);
      if constexpr (DT == kF16) {
        uk = unit(sk);
        if (uk.wide) uk.E = 134;
      }
      vtops = uv.wide ? block_tops<D, NT>(p, table, kvh, lo > 64 * begin ? lo : 64 * begin, k1, red) : uv.E * 0x01010101u;
      if (uv.wide) vtop = wide_top(64 * (end - begin));
    }
    const float c = DT == kF16 ? ldexpf(a.sml2, uk.E - 134) : a.sml2;
    const uint32_t kadd = static_cast<uint32_t>(134 - uk.E) << 23;
    // (wide: of this thread's block of columns)
    const int vup = uv.wide ? vtop - static_cast<int>(vtops >> 8 * (vdq / 8) & 0xffu) : 134 - uv.E;

    // Keys that no row sees, or that are not there: nothing of them may reach a product.
    auto clear_k = [&](KRegs& x, int kt, int page) {
      const int key0 = 64 * kt + WKEYS * wave;
      if (page >= 0 && key0 >= lo && key0 + WKEYS <= hi) return;
      if (page < 0 || key0 + kkey < lo || key0 + kkey >= hi) {
#pragma unroll
        for (int i = 0; i < KC / 4; ++i) x.c[i] = 0;
        x.e = static_cast<uint32_t>(uk.E);
      }
    };
    auto clear_v = [&](int kt, int page) {
      const int key0 = 64 * kt + WKEYS * wave;
      if (page >= 0 && key0 >= lo && key0 + WKEYS <= hi) return;
#pragma unroll
      for (int j = 0; j < VK; ++j)
        if (const int key = key0 + VK * vkg + j; page < 0 || key < lo || key >= hi) {
          vc[j] = 0;
          if constexpr (CH == 4) vse[j] = vtops;
          else vse[j / 2] = (vse[j / 2] & (j & 1 ? 0x0000ffffu : 0xffff0000u)) | (vtops & (j & 1 ? 0xffff0000u : 0xffffu));
        }
    };
    // Registers -> LDS, as fp16 in the part's unit or (WIDE, and K for bf16 queries) as bf16; in eight pieces each.
    struct Staged {
      uint32_t k[KC / 2], v[VK][2];
    };
    auto k_piece = [&](Staged& st, const KRegs& x, int k, uint8_t* buf, auto WIDE) {
      if (k >= KC / 4) return;  // (D = 64 has four)
      constexpr bool f16 = DT == kF16 && !WIDE;
      const float sc = __uint_as_float((x.e << 23) + (f16 ? kadd : 0u));
      st.k[2 * k] = f16 ? cvt_f16<8>(x.c + k, 0, sc) : cvt_bf16<8>(x.c + k, 0, sc);
      st.k[2 * k + 1] = f16 ? cvt_f16<8>(x.c + k, 1, sc) : cvt_bf16<8>(x.c + k, 1, sc);
      if (k & 1)
        *reinterpret_cast<uint4*>(buf + (WKEYS * wave + kkey) * L::KP + 2 * KC * kq + 8 * (k - 1)) =
            make_uint4(st.k[2 * k - 2], st.k[2 * k - 1], st.k[2 * k], st.k[2 * k + 1]);
    };
    auto v_piece = [&](Staged& st, int i, uint8_t* buf, auto WIDE) {
      if (i < 4) {  // a quarter of the keys, then a column in each piece
#pragma unroll
        for (int j = i * (VK / 4); j < (i + 1) * (VK / 4); ++j) {
          uint32_t by;
          if constexpr (CH == 4) by = __builtin_amdgcn_ubfe(vse[j], 8 * (vdq / 8), 8);
          else by = __builtin_amdgcn_ubfe(vse[j / 2], 16 * (j & 1) + 8 * (vdq / 8), 8);
          const int e = static_cast<int>(by) + vup;
          const float sc = __uint_as_float(static_cast<uint32_t>(WIDE && e < 0 ? 0 : e) << 23);
          st.v[j][0] = WIDE ? cvt_bf16<8>(vc + j, 0, sc) : cvt_f16<8>(vc + j, 0, sc);
          st.v[j][1] = WIDE ? cvt_bf16<8>(vc + j, 1, sc) : cvt_f16<8>(vc + j, 1, sc);
        }
      } else {
        // column 4 dq + c is V^T row c D/4 + dq, so that neighbouring lanes write neighbouring rows
        const int cc = i - 4;
        const uint32_t sel = cc & 1 ? 0x07060302u : 0x05040100u;
        uint32_t w[VK / 2];
#pragma unroll
        for (int j = 0; j < VK / 2; ++j) w[j] = __builtin_amdgcn_perm(st.v[2 * j + 1][cc / 2], st.v[2 * j][cc / 2], sel);
        uint8_t* dst = buf + L::KBYTES + (cc * (D / 4) + vdq) * L::VP + 2 * (WKEYS * wave + VK * vkg);
        if constexpr (VK == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
      }
    };
    auto store_k = [&](const KRegs& x, uint8_t* buf, auto WIDE) {
      Staged st;
#pragma unroll
      for (int i = 0; i < 8; ++i) k_piece(st, x, i, buf, WIDE);
    };
    auto store_v = [&](uint8_t* buf, auto WIDE) {
      Staged st;
#pragma unroll
      for (int i = 0; i < 8; ++i) v_piece(st, i, buf, WIDE);
    };
    // S^T of 32 keys: register r is key 32 bl + 16 (r / 8) + 8 g + r % 8 of the tile in buf
    auto scores = [&](const uint8_t* buf, int bl, v16f& sc, auto WIDE) {
      const uint8_t* kr = buf + (32 * bl + key_of_32(li)) * L::KP + 16 * g;
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = 0.0f;
#pragma unroll
      for (int k = 0; k < NKS; ++k) {
        const uint4 kop = *reinterpret_cast<const uint4*>(kr + 32 * k);
        if constexpr (DT == kF16 && WIDE) {  // bf16 keys, the query's eleven bits in two bf16 terms
          uint4 qh, ql;
          split_f16(q[k], qh, ql);
          sc = mfma32_bf16(kop, qh, sc);
          sc = mfma32_bf16(kop, ql, sc);
        } else if constexpr (DT == kBF16) {
          sc = mfma32_bf16(kop, q[k], sc);
        } else {
          sc = mfma32_f16(kop, q[k], sc);
        }
      }
    };
    // The tile's scores masked where a row does not see the key, the row's reference m brought up to date (and with it
    // the sums so far); returns what p is relative to.
    auto settle = [&](int kb, uint32_t here, v16f& s0, v16f& s1) -> float {
      if (!(kb >= lo_all && kb + 64 <= hi_all && here == 0xfu)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = kb + 16 * (r >> 3) + 8 * g + (r & 7);
          if (key < lo_r || key >= hi_r || !((here >> (r >> 3)) & 1u)) s0[r] = -INFINITY;
          if (key + 32 < lo_r || key + 32 >= hi_r || !((here >> (2 + (r >> 3))) & 1u)) s1[r] = -INFINITY;
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = vmax(mx, vmax(s0[r], s1[r]));
      mx = max_x32(mx) * c;
      // m is 7 below a maximum seen: p may grow to 2^15 before m is moved (fp16 holds 65504), and is a normal fp16 number,
      // with all its 11 bits, down to 2^-21 of the row's largest.
      if (__any(mx > m + 15.0f)) {
        const float mn = vmax(m, mx - 7.0f);
        const float al = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= al;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[db][r] *= al;
      }
      return m == -INFINITY ? 0.0f : m;
    };

    if (uv.wide || uk.wide) {
      // Rare (see Unit), and plain: one tile after the other.
      for (int kt = begin; kt < end; ++kt) {
        const int id = look(kt);
        const uint32_t here = there(kt, id);
        const int page = page_in(id, here, 0);
        load_k(kx, kt, page);
        load_v(kt, page);
        clear_k(kx, kt, page);
        clear_v(kt, page);
        if (uk.wide) store_k(kx, lds, std::true_type{});
        else store_k(kx, lds, std::false_type{});
        if (uv.wide) store_v(lds, std::true_type{});
        else store_v(lds, std::false_type{});
        __syncthreads();
        v16f sc[2];
#pragma unroll
        for (int bl = 0; bl < 2; ++bl) {
          if (uk.wide) scores(lds, bl, sc[bl], std::true_type{});
          else scores(lds, bl, sc[bl], std::false_type{});
        }
        const float ms = settle(64 * kt, here & 0xfu, sc[0], sc[1]);
#pragma unroll
        for (int bl = 0; bl < 2; ++bl)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint8_t* vr = lds + L::KBYTES + li * L::VP + 16 * g + 32 * (2 * bl + j);
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              x[k] = __builtin_amdgcn_exp2f(fmaf(sc[bl][8 * j + k], c, -ms));
              l += x[k];
            }
            uint32_t w[4], w2[4];
            if (uv.wide) {  // V is bf16 as it is: P in two bf16 terms (16 bits)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                w[k] = pack_bf16(x[2 * k], x[2 * k + 1]);
                w2[k] = pack_bf16(x[2 * k] - __uint_as_float(w[k] << 16),
                                  x[2 * k + 1] - __uint_as_float(w[k] & 0xffff0000u));
              }
#pragma unroll
              for (int db = 0; db < NDB; ++db) {
                const uint4 va = *reinterpret_cast<const uint4*>(vr + 32 * db * L::VP);
                acc[db] = mfma32_bf16(va, make_uint4(w[0], w[1], w[2], w[3]), acc[db]);
                acc[db] = mfma32_bf16(va, make_uint4(w2[0], w2[1], w2[2], w2[3]), acc[db]);
              }
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) w[k] = pack_f16(x[2 * k], x[2 * k + 1]);
#pragma unroll
              for (int db = 0; db < NDB; ++db)
                acc[db] = mfma32_f16(*reinterpret_cast<const uint4*>(vr + 32 * db * L::VP),
                                     make_uint4(w[0], w[1], w[2], w[3]), acc[db]);
            }
          }
        __syncthreads();
      }
    } else {
      constexpr std::false_type kNarrow{};
      uint8_t* const buf0 = lds;
      uint8_t* const buf1 = lds + L::BUF;
      // The pages and masks of the tiles on the way: of V's registers, of K's, of the next K; of the scores' tile and
      // the three after it.
      int pv = page1, pk = page_in(ids, mask, 2), pn = page_in(ids, mask, 3);
      clear_k(kx, begin, page0);
      clear_v(begin, page0);
      clear_k(ky, upto(begin + 1), page1);
      store_k(kx, buf0, kNarrow);
      store_v(buf0, kNarrow);
      store_k(ky, buf1, kNarrow);
      load_v(upto(begin + 1), pv);
      load_k(kx, upto(begin + 2), pk);
      uint32_t here0 = mask & 0xfu, here1 = mask >> 4 & 0xfu, here2 = mask >> 8 & 0xfu, here3 = mask >> 12 & 0xfu;
      __syncthreads();
      v16f sa, sb, sc_;
      scores(buf0, 0, sa, kNarrow);
      scores(buf0, 1, sb, kNarrow);
      __syncthreads();  // the first step puts another K tile there
      // Tile kt: its scores are in s0 and s1; the next tile's go to s2 and, when s0 is used up, s0 (three blocks for what
      // would be four).  In LDS: K of kt + 1 (nxt), V of kt (cur).  In the staging registers: K of kt + 2, V of kt + 1.
      auto step = [&](int kt, uint8_t* cur, uint8_t* nxt, v16f& s0, v16f& s1, v16f& s2) {
        // The step's products in order: of each half of the tile the next tile's scores (NKS products) and this one's
        // two quarters of P V (NDB each).  Their LDS operands are read kAhead products ahead, and each product is
        // followed by a piece of what the VALU has to do meanwhile: the softmax of the half beside the scores, the
        // conversion of the staged K (first half) or V tile (second) beside P V.  The order is fixed here; left to the
        // compiler, every read was next to its product.
        constexpr int HALF = NKS + 2 * NDB, kAhead = 5;
        const int id = look(kt + 4);  // back by the end of the step
        uint4 ring[kAhead];
        const uint8_t* const kr = nxt + key_of_32(li) * L::KP + 16 * g;
        const uint8_t* const vr = cur + L::KBYTES + li * L::VP + 16 * g;
        auto fetch = [&](int n) {
          if (n >= 2 * HALF) return;
          const int bl = n / HALF, i = n % HALF;
          const uint8_t* src = i < NKS ? kr + 32 * bl * L::KP + 32 * i
                                       : vr + 32 * ((i - NKS) % NDB) * L::VP + 32 * (2 * bl + (i - NKS) / NDB);
          ring[n % kAhead] = *reinterpret_cast<const uint4*>(src);
        };
#pragma unroll
        for (int n = 0; n < kAhead; ++n) fetch(n);
        const float ms = settle(64 * kt, here0, s0, s1);
        clear_k(kx, upto(kt + 2), pk);
        clear_v(upto(kt + 1), pv);
        Staged st;
#pragma unroll
        for (int bl = 0; bl < 2; ++bl) {
          uint32_t w[8];
          v16f& sc = bl == 0 ? s0 : s1;
          v16f& sn = bl == 0 ? s2 : s0;
#pragma unroll
          for (int r = 0; r < 16; ++r) sn[r] = 0.0f;
#pragma unroll
          for (int i = 0; i < HALF; ++i) {
            const int n = bl * HALF + i;
            const uint4 x = ring[n % kAhead];
            if (i < NKS) {
              sn = DT == kBF16 ? mfma32_bf16(x, q[i], sn) : mfma32_f16(x, q[i], sn);
              fetch(n + kAhead);
#pragma unroll
              for (int e = 0; e < 8 / NKS; ++e) {
                const int k = i * (8 / NKS) + e;
                const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[2 * k], c, -ms));
                const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[2 * k + 1], c, -ms));
                l += p0 + p1;
                asm volatile("" : "+v"(l));  // here: else all 32 are added up at the step's end, and wait in registers
                w[k] = pack_f16(p0, p1);
              }
            } else {
              const int j = (i - NKS) / NDB, db = (i - NKS) % NDB;
              acc[db] = mfma32_f16(x, make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]), acc[db]);
              fetch(n + kAhead);
#pragma unroll
              for (int e = 0; e < 4 / NDB; ++e) {
                const int k = (i - NKS) * (4 / NDB) + e;  // 0 .. 7
                if (bl == 0) k_piece(st, kx, k, cur, kNarrow);
                else v_piece(st, k, nxt, kNarrow);
              }
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        pv = pk;
        pk = pn;
        load_v(upto(kt + 2), pv);
        load_k(kx, upto(kt + 3), pk);
        const uint32_t mask = there(kt + 4, id);
        pn = page_in(id, mask, 0);
        here0 = here1;
        here1 = here2;
        here2 = here3;
        here3 = mask & 0xfu;
        __syncthreads();
      };
      // (two LDS buffers and three blocks of scores: the order comes round after six steps)
      for (int kt = begin; kt < end;) {
        step(kt, buf0, buf1, sa, sb, sc_);
        if (++kt >= end) break;
        step(kt, buf1, buf0, sc_, sa, sb);
        if (++kt >= end) break;
        step(kt, buf0, buf1, sb, sc_, sa);
        if (++kt >= end) break;
        step(kt, buf1, buf0, sa, sb, sc_);
        if (++kt >= end) break;
        step(kt, buf0, buf1, sc_, sa, sb);
        if (++kt >= end) break;
        step(kt, buf1, buf0, sb, sc_, sa);
        ++kt;
      }
    }
    l = add_x32(l);
  }
  if (rw + li < rows) {
    const int64_t tok = s.start + qi;
    const bool one = a.splits == 1;
    const float f = filled(l) ? 1.0f / l : 0.0f;
    const int64_t at = split * R + tok * p.Hq + h;
    if (one && p.lse && g == 0) p.lse[tok * p.Hq + h] = row_lse(m, l);
    if (!one && g == 0) a.ml[at] = make_float2(m, l);
    if (one || filled(l)) {
      // Register r of acc[db] is V^T row 32 db + 8 (r / 4) + 4 g + r % 4 = c D/4 + dq, column 4 dq + c: for piece i
      // the columns 32 i + 16 g + 4 k + c.  D = 128: c = db, r = 4 i + k; D = 64: c = 2 db + r / 8, r % 8 = 4 i + k.
#pragma unroll
      for (int i = 0; i < NDB; ++i) {
        const int col = 32 * i + 16 * g, e = static_cast<int>(vtops >> 8 * i & 0xffu) - vtop;
        float o[16];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int cc = 0; cc < 4; ++cc)
            o[4 * k + cc] = ldexpf((D == 128 ? acc[cc % NDB][4 * i + k] : acc[cc / 2][8 * (cc & 1) + 4 * (i & 1) + k]) * f, e);
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

// ---- joining the parts of the keys ---------------------------------------------

// The largest / the sum over a row's 16 or 64 lanes, in every one of them
template <int LPR>
__device__ __forceinline__ float lanes_max(float v) {
#define LBFQ_ROR(c) v = vmax(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), c, 0xf, 0xf, true)))
  LBFQ_ROR(0x128);  // row_ror:8, 4, 2, 1
  LBFQ_ROR(0x124);
  LBFQ_ROR(0x122);
  LBFQ_ROR(0x121);
#undef LBFQ_ROR
  return LPR == 64 ? max_x32(max_x16(v)) : v;
}
template <int LPR>
__device__ __forceinline__ float lanes_add(float v) {
#define LBFQ_ROR(c) v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), c, 0xf, 0xf, true))
  LBFQ_ROR(0x128);
  LBFQ_ROR(0x124);
  LBFQ_ROR(0x122);
  LBFQ_ROR(0x121);
#undef LBFQ_ROR
  return LPR == 64 ? add_x32(add_x16(v)) : v;
}

// LPR lanes a row, at least as many as parts: the parts' maxima and sums one to a lane, their outputs, each an average of
// its values, summed in the parts' order with weights l_s 2^(m_s - M) / l that add up to one.  At a few rows it is all
// latency: the first parts are on their way before the weights are known.  16 lanes for up to 16 parts of 4096 rows or
// more, which wide loads serve better than many waves (with 64 lanes -> 16, us of the whole call: 29000 rows of 64, 3 parts
// 62.7 -> 57.7; 16000 of 128, 2 parts 50.9 -> 48.4; but 1200 of 128, 5 parts 16.5 -> 16.8, and 32, 7 parts 9.8 -> 10.0), else 64.
template <int DT, int D, int LPR>
__global__ void __launch_bounds__(256) paged_combine_kernel(const Args a) {
  constexpr int U = LPR == 16 ? 8 : 16, DL = D / LPR, RPW = 64 / LPR;
  const lbfq_paged_params& p = a.p;
  const int lane = threadIdx.x & 63, sub = lane / LPR, li = lane % LPR;
  const uint32_t wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t Hq = static_cast<uint32_t>(p.Hq), R = static_cast<uint32_t>(p.T * p.Hq);  // below 2^30
  if (wave * RPW >= R) return;
  const bool there = wave * RPW + sub < R;  // rows past the last repeat it and are not stored
  const uint32_t row = there ? wave * RPW + sub : R - 1;
  const int tok = static_cast<int>(row / Hq);
  const int h = static_cast<int>(row - tok * Hq);
  float2 x = make_float2(-INFINITY, 0.0f);
  if (li < a.splits) x = a.ml[static_cast<int64_t>(li) * R + row];
  const float* src = a.acc + static_cast<int64_t>(row) * D + li * DL;
  float y[U][DL];
  auto load = [&](int s0) {
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (s0 + i < a.splits) {
        const float* from = src + static_cast<int64_t>(s0 + i) * R * D;
        if constexpr (DL % 4 == 0) {
#pragma unroll
          for (int k = 0; k < DL; k += 4) {
            const float4 v = *reinterpret_cast<const float4*>(from + k);
            y[i][k] = v.x; y[i][k + 1] = v.y; y[i][k + 2] = v.z; y[i][k + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int k = 0; k < DL; ++k) y[i][k] = from[k];
        }
      }
  };
  load(0);
  const bool mine = tok >= p.query_starts[0] && tok < p.query_starts[p.B];
  const bool some = mine && filled(x.y);  // else nothing in this part, and its outputs were not written
  const float M = lanes_max<LPR>(some ? x.x : -INFINITY);
  const float part = some ? x.y * __builtin_amdgcn_exp2f(x.x - M) : 0.0f;
  const float l = lanes_add<LPR>(part);
  const float f = filled(l) ? part / l : 0.0f;
  float o[DL];
#pragma unroll
  for (int k = 0; k < DL; ++k) o[k] = 0.0f;
  for (int s0 = 0; s0 < a.splits; s0 += U) {
    if (s0) load(s0);
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (s0 + i < a.splits) {
        float w;
        if constexpr (LPR == 64) w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), s0 + i));
        else w = __shfl(f, sub * LPR + s0 + i, 64);
#pragma unroll
        for (int k = 0; k < DL; ++k) o[k] = filled(w) ? fmaf(y[i][k], w, o[k]) : o[k];
      }
  }
  if (!there) return;
  if (mine || p.fill_rest) {
    uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + tok * p.out_t + h * p.out_h + li * DL;
    if constexpr (DL == 1) {
      *dst = static_cast<uint16_t>(pack_dt<DT>(o[0], 0.0f));
    } else {
      uint32_t w[DL / 2];
#pragma unroll
      for (int k = 0; k < DL / 2; ++k) w[k] = pack_dt<DT>(o[2 * k], o[2 * k + 1]);
      if constexpr (DL == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      else if constexpr (DL == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(dst) = w[0];
    }
  }
  if (p.lse && li == 0) p.lse[row] = row_lse(M, l);
}

// ---- host --------------------------------------------------------------------

struct Plan {
  bool decode;
  int splits, least;
  int64_t share;  // chunk in 4 bits: Args::share
  int64_t slots, groups, piece;  // chunk: row tiles of a head (slot_of), the pieces that they come in, row tiles of a piece
};

// Bytes of a row in each part: its average and its maximum and sum.  Parts are not made beyond a workspace of kMostBytes (a
// token buffer may be padded; those of calls that fill it take tens of MiB), one part needs none.  That also keeps the
// rows of a call in parts under the 2^26 waves that may join them.
int64_t part_bytes(const lbfq_paged_params* p) { return p->T * p->Hq * (static_cast<int64_t>(sizeof(float2)) + p->D * 4); }
constexpr int64_t kMostBytes = (int64_t{1} << 30) - 16;

// Parts of the keys, of 192 at least in decode (one token over 5003 keys, 8 key heads, parts of 128 / 192 / 256 / 512: 12.5 /
// 11.9 / 12.8 / 15.3 us) and 128 in chunks (100 tokens over 700 keys, 12 heads, 128 / 256 / 512: 16 / 20 / 23).  The lengths
// are on the device: the rule goes by the table's width, and a shorter sequence's parts are shorter, or fewer.
//
// decode: the 768 workgroups that run at a time at D = 128 (24 sequences of 2000 to 4000 keys, 8 key heads, 384 / 768 /
// 1536: 51 / 39 / 44 us; 3 of up to 40000, 384 / 768 / 1152: 57 / 41 / 46).
// decode in 4 bits: a workgroup alone on its CU takes 4.9 ns a key (its waves' own chain of instructions), and from about 192
// of them on they share the memory; joining parts costs 3.5 us.  So: as many parts of 300 keys or more as give 256
// workgroups, one for fewer than 1100 keys; and, to even out several sequences, parts of 4000 keys from 12000 on (us for 1 / 2 /
// 3 / 4 / 6 / 8 / 16 / 32 parts, * the rule's, 8 key heads of 128: one sequence of 700 keys 9.5* / 12.8 / 11.1 / 10.9 / 11.0 /
// 10.8; 5003 31 / 21 / 18 / 15 / 14 / 13 / 11.8* / 12.1; 40000 197 / 105 / 74 / 58 / 42 / 34 / 22 / 18.8*; 24 of 2000 to 4000
// 25.8* / 28.0 / 27.6 / 28.5 / 29.6; 48 of 8000 to 16000 152 / 134 / 127 / 121* / 124 / 127; 8 of 4000 to 8000, 40 heads 53.6*
// / 59.6 / 56.0 / 55.7 / 57.1 / 61.7; 12 of 1000 to 16000, 12 heads 79 / 54 / 50 / 46* / 47 / 44 / 50).  Evening out takes
// workgroups for at most six rounds of 512 places: where the sequences alone come to three rounds or more, it mostly costs (8
// key heads, 6016 to 12032 keys, 1 / 2 / 3 / 4 parts: 96 sequences 182 / 169 / 168* / 174; 128 226 / 225 / 229* / 230; 192 330 /
// 335* / 343 / 355; 256 420* / 429 / 447 / 457; 512 815* / 854 / 877 / 915; 512 of 750 to 12032 576* / 627 / 668 / 682).
// chunk, one sequence: the parts that take the least time by a count of tiles.  A part costs the time of 12 tiles besides
// its own (its start, and its sums written and read again), and an XCD has two or three workgroups a CU at a time.  Row
// tiles that see much the same keys go in whole rounds (us for 1 / 2 / 4 / 6 / 7 parts, * the rule's: 1560 tokens, 32760
// keys, 40 heads 1717 / 1407 / 1295 / 1287* / 1288; 700, 8000 keys, 12 heads 168 / 96 / 81 / 68* / 86).  A causal prompt's
// row tiles differ, the longest first, and fill the rounds up; a workgroup that is left alone on its CU takes 0.7 times as
// long (1 / 2 / 3 / 4 parts: 2500 tokens, 32 / 8 heads 81* / 109 / 126 / 139; 5000, 5 heads 112 / 76 / 64* / 75).
// chunk, several: lengths differ, and more and shorter parts even them out.  With w workgroups in a part, w s / (8 places)
// + c rounds of keys / (64 s) tiles + o each take the least time at s^2 = keys / w * places / 8 * c / o.  c / o = 1 / 15: over
// 25 batches of 2 to 16 sequences, up to 3000 new tokens and 20000 keys, the parts of 1 / 10, 12, 14, 15, 16 take 7.6, 5.2,
// 6.4, 4.4 and 3.9% longer than the best of them, but 1 / 16 gives the last call named here two parts (us for 1 / 2 / 3 / 4 / 5 /
// 6 / 8 parts, * the rule's: 16 sequences of up to 64 tokens and 2000 keys 51 / 48* / 54 / 56 / 61 / 65 / 77; 8 of 128 and 4000 90 /
// 71 / 57* / 72 / 69 / 67 / 76; 4 of 700 and 9001, 12 heads 192 / 142 / 117 / 127 / 120* / 115 / 123; 2 of 1024 and 16000 475 /
// 469 / 474 / 432* / 449 / 457 / 468; 2 of 300 and 5000 111 / 70 / 68 / 63* / 76 / 76 / 77; 4 of 509, fp16, window 4096 77 / 63 /
// 53* / 52 / 58 / 58 / 66).
//
// In 4 bits the last round is counted as what it takes where it does not fill the chip, 0.7 of a round up to half of it (us
// for 1 / 2 / 3 / 4 / 5 / 6 / 7 / 8 parts, * the rule's: 1560 tokens, 32760 keys, 40 heads 1513 / 1237 / 1155 /
// 1141 / 1110* / 1107 / 1106 / 1112; 700 tokens, 8000 keys, 12 heads 148 / 89 / 69 / 71 / 63 / 58* / 81; 5000, 5 heads, causal 100 / 73 /
// 62* / 68); and parts of several sequences that come out at a little over whole rounds are made fewer (2 of 300 and 5000 97 /
// 63 / 60 / 53* / 71 / 72; 8 of 128 and 4000 84 / 67* / 75 / 73; 4 of 700 and 9001, 12 heads 175 / 119 / 132 / 124 / 116* / 129).
int64_t rounds10(int64_t n, int64_t places) {
  const int64_t whole = n / places, rest = n % places;
  if (rest == 0) return 10 * whole;
  if (whole == 0) return 10;
  return 10 * whole + (2 * rest <= places ? 7 : 7 + (2 * rest - places) * 3 / places);
}

Plan plan(const lbfq_paged_params* p) {
  Plan x;
  x.share = 0;
  const int64_t G = p->Hq / p->Hk;
  const int64_t most = p->max_query_len > 0 && p->max_query_len < p->T ? p->max_query_len : p->T;
  x.decode = most * G <= kDecodeRows;
  const int64_t tiles = (p->T * G + kChunkRows - 1) / kChunkRows;
  x.slots = tiles + p->B - 1;
  x.groups = (x.slots + 7) / 8;
  x.piece = (x.slots + x.groups - 1) / x.groups;
  int64_t keys = p->table_cols << p->page_shift;  // that a row tile may see
  if (p->causal && p->window) keys = std::min(keys, p->window + std::min(most, kChunkRows / G + 1));
  const bool four = p->bits == 4;
  const int64_t least = !x.decode ? 128 : four ? 256 : 192;
  // (a lane each in the combine kernel)
  const int64_t limit = std::min({keys / least, int64_t{64}, kMostBytes / part_bytes(p)});
  const int64_t places = 32 * (four ? chunk4_groups(p->D) : chunk_groups(p->dtype, p->D));  // for workgroups on an XCD
  int64_t s = 1;
  if (x.decode && four) {
    if (keys >= 1100) s = std::min(256 / (p->B * p->Hk), keys / 300);
    if (p->B > 1 && keys >= 12000) s = std::max(s, std::min(keys / 4000, 6 * 512 / (p->B * p->Hk)));
  } else if (x.decode) {
    const int64_t wgs = p->B * p->Hk;
    s = (768 + wgs / 2) / wgs;
  } else if (p->B == 1) {
    const bool uneven = p->causal && !p->window && 2 * most > keys;
    const int64_t seeing = std::min(most, keys);  // (a padded buffer has more tokens than the table has keys)
    int64_t best = std::numeric_limits<int64_t>::max();
    for (int64_t n = 1; n <= limit; ++n) {
      const int64_t of_xcd = (x.groups * p->Hk * n + 7) / 8 * x.piece, longest = keys / n + 12 * 64;
      const int64_t cost = uneven ? std::max(of_xcd * ((keys - seeing / 2) / n + 12 * 64), 45 * longest)
                                  : (four ? rounds10(of_xcd, places) * places / 10 : (of_xcd + places - 1) / places * places) * longest;
      if (cost < best) best = cost, s = n;
    }
    // Two unequal parts (in 4 bits): row tiles that fill more than half of the chip, but not all of it, leave the last keys of
    // each to the places that are free, where they come one after the other (4680 tokens over 32760 keys, 12 heads, one part /
    // two equal / these: 861 / 885 / 838 us; 3800 tokens 787 / 777 / 693).  Joining them takes a tile's time for 550000 values.
    const int64_t wgs = x.slots * p->Hk, all = 8 * places, o = 12 * 64;
    if (four && !uneven && limit >= 2 && wgs < all && 2 * wgs > all) {
      const int64_t turns = (wgs + all - wgs - 1) / (all - wgs);
      const int64_t rest = (keys + o - turns * o) / (turns + 1);
      const int64_t join = 64 * (p->T * p->Hq * p->D / 550000 + 2);
      if (rest >= 128 && places * (keys - rest + o + join) < best) {
        s = 2;
        x.share = ((keys - rest) << 16) / keys;
      }
    }
  } else {
    const int64_t wgs = (tiles + p->B / 2) * p->Hk;
    while (120 * (s + 1) * (s + 1) * wgs <= places * keys && s < limit) ++s;
    if (const int64_t all = 8 * places, over = wgs * s % all; four && wgs * s > all && 3 * over < all)
      s = std::max<int64_t>((wgs * s - over) / wgs, 1);
  }
  x.splits = static_cast<int>(std::max<int64_t>(std::min(s, limit), 1));
  x.least = static_cast<int>(least / (x.decode && !four ? 32 : 64));
  return x;
}

// Workgroups that fill at most (a prompt of 2048 tokens in a buffer of 32048, 32 heads of 128, 128 / 256 / 512 / 1024: 119 / 101 /
// 93 / 85 us, without the buffer 57; one token of 48 sequences in one of 30000: 83 / 47 / 37 / 37).  What they have to fill
// is known on the device; without anything they end at once.
constexpr int64_t kMostFill = 512;

int64_t workspace(const lbfq_paged_params* p, const Plan& x) {
  return x.splits == 1 ? 0 : x.splits * part_bytes(p) + 16;
}

int check_sizes(const lbfq_paged_params* p) {
  const char* who = "lbfq_paged_attention";
  LBFQ_CHECK_ARG(p, "%s: null params", who);
  LBFQ_CHECK_ARG(p->bits == 0 || p->bits == 4 || p->bits == 8, "%s: codes have 4 or 8 bits", who);
  LBFQ_CHECK_ARG(p->D == 64 || p->D == 128, "%s: D must be 64 or 128", who);
  LBFQ_CHECK_ARG(p->dtype == kBF16 || p->dtype == kF16, "%s: queries are bf16 or fp16", who);
  LBFQ_CHECK_ARG(p->Hk > 0 && p->Hq > 0 && p->Hq % p->Hk == 0 && p->Hq < (1 << 16),
                 "%s: the query heads must be a multiple of the key heads", who);
  LBFQ_CHECK_ARG(p->T > 0 && p->B > 0 && p->T < (int64_t{1} << 30) && p->B < (int64_t{1} << 30),
                 "%s: bad number of tokens or sequences", who);
  LBFQ_CHECK_ARG(p->page_shift >= 4 && p->page_shift <= 10, "%s: pages hold 16 to 1024 tokens, a power of two", who);
  LBFQ_CHECK_ARG(p->T * p->Hq < (int64_t{1} << 30), "%s: problem too large", who);
  LBFQ_CHECK_ARG(p->num_pages > 0 && p->num_pages < (int64_t{1} << 31) / p->Hk, "%s: bad number of pages", who);
  LBFQ_CHECK_ARG(p->table_cols > 0 && p->table_cols <= (int64_t{1} << 30) >> p->page_shift && p->table_stride >= 0,
                 "%s: bad block table", who);
  LBFQ_CHECK_ARG(p->window >= 0 && p->window <= (int64_t{1} << 30), "%s: bad window", who);
  return 0;
}

int check(const lbfq_paged_params* p) {
  const char* who = "lbfq_paged_attention";
  if (int rc = check_sizes(p)) return rc;
  LBFQ_CHECK_ARG(p->q && p->out && p->block_table && p->seq_lens && p->query_starts && p->k_codes && p->k_scale &&
                     p->v_codes && p->v_scale,
                 "%s: missing tensor", who);
  LBFQ_CHECK_ARG(((reinterpret_cast<uint64_t>(p->q) | reinterpret_cast<uint64_t>(p->out) |
                   reinterpret_cast<uint64_t>(p->k_codes) | reinterpret_cast<uint64_t>(p->v_codes) |
                   reinterpret_cast<uint64_t>(p->k_scale) | reinterpret_cast<uint64_t>(p->v_scale)) & 15) == 0 &&
                     ((p->q_t | p->q_h | p->out_t | p->out_h) & 7) == 0,
                 "%s: rows must be 16-byte aligned", who);
  // (beyond, a scale of K times sm_scale could leave fp32's range)
  LBFQ_CHECK_ARG(p->sm_scale >= 0x1p-64f && p->sm_scale <= 0x1p15f, "%s: sm_scale must lie in 2^-64 .. 2^15", who);
  return 0;
}

}  // namespace

extern "C" int64_t lbfq_paged_attention_workspace_bytes(const lbfq_paged_params* p) {
  if (check_sizes(p)) return 0;
  return workspace(p, plan(p));
}

extern "C" int lbfq_paged_attention_parts(const lbfq_paged_params* p, int* share) {
  if (share) *share = 0;
  if (check_sizes(p)) return 0;
  const Plan x = plan(p);
  if (share) *share = static_cast<int>(x.share);
  return x.splits;
}

extern "C" int lbfq_paged_attention(const lbfq_paged_params* p, lbfq_stream_t stream) {
  if (int rc = check(p)) return rc;
  const Plan x = plan(p);
  Args a{};
  a.p = *p;
  a.G = static_cast<int>(p->Hq / p->Hk);
  a.slots = static_cast<int>(x.slots);
  a.splits = x.splits;
  a.least = x.least;
  a.sml2 = p->sm_scale * kLog2e;
  const int64_t R = p->T * p->Hq;
  if (x.splits > 1) {
    LBFQ_CHECK_ARG(p->workspace && p->workspace_bytes >= workspace(p, x), "lbfq_paged_attention: workspace too small");
    LBFQ_CHECK_ARG((reinterpret_cast<uint64_t>(p->workspace) & 15) == 0, "lbfq_paged_attention: workspace alignment");
    a.acc = static_cast<float*>(p->workspace);
    a.ml = reinterpret_cast<float2*>(a.acc + x.splits * R * p->D);
  }
  // (a launch has fewer than 2^32 threads)
  const int64_t combos = (x.decode ? p->B : x.splits) * p->Hk;
  a.main = x.decode ? combos * x.splits : (x.groups * combos + 7) / 8 * 8 * x.piece;
  LBFQ_CHECK_ARG(a.main < (1 << 24) - 8, "lbfq_paged_attention: problem too large");
  a.combos = static_cast<uint32_t>(combos);
  a.piece = static_cast<uint32_t>(x.piece);
  a.share = static_cast<uint32_t>(x.share);
  if (x.share) a.main = (x.slots * p->Hk + 7) / 8 * 8 * 2;
  // rows that no sequence has: the combine kernel sees every row, otherwise some workgroups more, one for 64 KiB that the
  // output holds
  const int64_t fill = (p->fill_rest || p->lse) && x.splits == 1
                           ? std::min({R * p->D / (1 << 15) + 1, kMostFill, (1 << 24) - 1 - a.main})
                           : 0;
  const dim3 grid(static_cast<unsigned>(a.main + fill));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool bf = p->dtype == kBF16, d128 = p->D == 128;
#define LBFQ_PA(KERNEL)                                                                              \
  do {                                                                                               \
    if (bf && d128) hipLaunchKernelGGL((KERNEL<kBF16, 128>), grid, dim3(256), 0, st, a);             \
    else if (bf) hipLaunchKernelGGL((KERNEL<kBF16, 64>), grid, dim3(256), 0, st, a);                 \
    else if (d128) hipLaunchKernelGGL((KERNEL<kF16, 128>), grid, dim3(256), 0, st, a);               \
    else hipLaunchKernelGGL((KERNEL<kF16, 64>), grid, dim3(256), 0, st, a);                          \
  } while (0)
  if (p->bits == 4) {
    if (x.decode) launch_decode4(a, grid.x, st);
    else launch_chunk4(a, grid.x, st);
  } else if (x.decode) {
    LBFQ_PA(paged_decode_kernel);
  } else {
    LBFQ_PA(paged_chunk_kernel);
  }
#undef LBFQ_PA
  LBFQ_LAUNCH_CHECK("lbfq_paged_attention");
  if (x.splits > 1) {
    const bool narrow = x.splits <= 16 && R >= 4096;
    const int64_t per = narrow ? 16 : 4;  // rows of a workgroup
    const dim3 gc(static_cast<unsigned>((R + per - 1) / per)), block(256);
#define LBFQ_PJ(DT, DD)                                                                               \
  do {                                                                                                \
    if (narrow) hipLaunchKernelGGL((paged_combine_kernel<DT, DD, 16>), gc, block, 0, st, a);          \
    else hipLaunchKernelGGL((paged_combine_kernel<DT, DD, 64>), gc, block, 0, st, a);                 \
  } while (0)
    if (bf && d128) LBFQ_PJ(kBF16, 128);
    else if (bf) LBFQ_PJ(kBF16, 64);
    else if (d128) LBFQ_PJ(kF16, 128);
    else LBFQ_PJ(kF16, 64);
#undef LBFQ_PJ
    LBFQ_LAUNCH_CHECK("lbfq_paged_attention (combine)");
  }
  return 0;
}

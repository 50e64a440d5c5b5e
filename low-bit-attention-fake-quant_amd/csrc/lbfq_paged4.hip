// Attention of single tokens over the paged cache in 4 bits: the decode kernel for E2M1 codes (the mathematics and the
// masks are lbfq_paged.hip's, which also joins the parts; more rows go to lbfq_paged4_chunk.hip).
//
// Reading the cache is half of what it is in 8 bits, so what the arithmetic costs comes to the fore.  Scores are formed
// from the codes as they lie in memory, by the block-scaled product (16x16x128, a lane's 16 bytes and its scale byte are
// one operand).  That takes 4- and 6-bit operands at twice the rate of 8-bit ones, and, other than with 8-bit operands
// (whose products span more powers of two than its sums keep: errors of 3e-6 of a score), it adds up theirs exactly to
// fp32's precision.  So a query goes in as four E2M3 terms with scales 2^-5 apart, relative to the largest of its 32
// columns: bf16's eight bits are exact down to 2^-11 of that, fp16's eleven to 2^-8, and what is left is below 2^-19 of
// it.  Four products of 16 cycles take the time of bf16's four, without converting K.  (Queries whose columns lie so far apart
// that this would be less than bf16 itself holds of them take four more: split_query.)
//
// V's scales change from key to key, along the sum, so V is converted to bf16 (exact).  P is two bf16 terms.
//
// A wave has two tiles of 64 keys in LDS besides the one in its registers, copied there without passing through registers,
// 16 bytes a lane: it never waits for a tile that it has only just asked for.  (The same kernel with a tile's loads into
// registers took 154 us where this one takes 118, with K's loads before and V's behind the arithmetic 196.)  48
// sequences of 8000 to 16000 keys, 32 / 8 heads of 128: 118 us, 5.3 TB/s; the same copies without softmax and P V 110, a
// kernel that only reads 6.1 TB/s; in pages of 64, of 32 120, of 16 128.  Heads of 64: 77 us, 4.0 TB/s (pages of 32 and 16: 87 and
// 84): 290 VALU instructions a tile of 64 keys, where heads of 128 have 350 for twice the bytes, and a chain of 3000 cycles for
// a wave alone.  Pages of 16 read 18% more than they need: scales of a head and page are 32 bytes.
#include <cstddef>

#include "lbfq_paged_common.h"

using namespace lbfq;
using namespace lbfq::paged;

namespace {

constexpr int kT = 4, kKeys = 16 * kT;  // a wave's tile: 64 keys, 16 at a time
constexpr int kBufs = 2;                // tiles of a wave in LDS: one on its way, one behind it

// A tile in LDS: rows of D / 2 bytes of codes as they lie in the cache, their 16-byte pieces exchanged (piece_of), and the
// rows' scales.
template <int D>
struct Ring {
  struct Tile {
    uint8_t k[kKeys * D / 2], v[kKeys * D / 2];
    uint8_t ks[256], vs[256];  // (D = 64 needs half)
  };
  Tile t[4][kBufs];
};

// Key of a row of S^T within its 16: row 4 g + i is key 4 i + g, so that the four lane groups' rows of V are neighbours, and
// V's reads, 64 lanes four bytes of all pieces of four rows, on distinct banks, as K's are.
__device__ __forceinline__ int key_of_16(int r) { return 4 * (r & 3) + (r >> 2); }

// Pages of 16 and of 32 tokens: a tile lies in four or two; of 64 and more: in one.  A tile's piece is what it has of a page.
__device__ __forceinline__ int pieces(const lbfq_paged_params& p) { return p.page_shift >= 6 ? 1 : 64 >> p.page_shift; }

// The page ids of a tile's pieces (-1: none).  Through the constant address space: a scalar load, which no wait for copies
// stands behind (the table does not change during the call).
typedef const int32_t __attribute__((address_space(4))) * Table;
struct Pages {
  int id[kT];
};
__device__ __forceinline__ void load_pages(const lbfq_paged_params& p, Table table, int kb, Pages& x) {
  const int first = kb >> p.page_shift, n = pieces(p), cols = static_cast<int>(p.table_cols);
  x.id[0] = first < cols ? table[first] : -1;
  if (n > 1) {
    x.id[1] = first + 1 < cols ? table[first + 1] : -1;
    if (n > 2) {
      x.id[2] = first + 2 < cols ? table[first + 2] : -1;
      x.id[3] = first + 3 < cols ? table[first + 3] : -1;
    }
  }
}

// Copies a tile into LDS, kCopies of them under way; bit t: the page of its 16 keys t is there (in the place of one that is
// not, page 0 is read).  A copy of 1 KiB is lane i's 16 bytes of row i / (D / 32), places exchanged; all copies of a piece
// have one base, and the lanes that a piece does not need for its last copy are off.
template <int D>
constexpr int kCopies = D == 128 ? 10 : 6;
template <int D>
__device__ __forceinline__ uint32_t fetch(const lbfq_paged_params& p, const Pages& pages, int kvh, int kb, int lane,
                                          uint32_t off, uint32_t lds) {
  using X = typename Ring<D>::Tile;
  constexpr int RB = D / 2, SB = D / 32;  // bytes of a row, and of its scales
  const int shift = p.page_shift;
  const uint32_t Hk = static_cast<uint32_t>(p.Hk), num = static_cast<uint32_t>(p.num_pages);
  auto row_of = [&](int id) {
    return static_cast<int64_t>((static_cast<uint32_t>(id) < num ? static_cast<uint32_t>(id) : 0u) * Hk + kvh) << shift;
  };
  if (shift >= 6) {
    const int64_t row = row_of(pages.id[0]) + (kb & ((1 << shift) - 1));
    copy_to(lds + offsetof(X, k));
    const uint8_t* k = p.k_codes + row * RB;
    copy16<0, true>(k, off);
    copy16<1024, true>(k, off);
    if constexpr (D == 128) copy16<2 * 1024, true>(k, off), copy16<3 * 1024, true>(k, off);
    copy_to(lds + offsetof(X, v));
    const uint8_t* v = p.v_codes + row * RB;
    copy16<0, true>(v, off);
    copy16<1024, true>(v, off);
    if constexpr (D == 128) copy16<2 * 1024, true>(v, off), copy16<3 * 1024, true>(v, off);
    const uint32_t so = D == 128 ? 4 * lane : 4 * (lane & 31);  // (D = 64: lanes 32 .. write what nobody reads)
    copy_to(lds + offsetof(X, ks));
    copy4<true>(p.k_scale + row * SB, so);
    copy_to(lds + offsetof(X, vs));
    copy4<true>(p.v_scale + row * SB, so);
    return static_cast<uint32_t>(pages.id[0]) < num ? 15u : 0u;
  }
  if (shift == 5) {
    const int64_t r0 = row_of(pages.id[0]), r1 = row_of(pages.id[1]);
    auto codes = [&](const uint8_t* base, uint32_t to) {
      copy_to(lds + to);
      const uint8_t* c = base + r0 * RB;
      copy16<0, true>(c, off);
      if constexpr (D == 128) copy16<1024, true>(c, off);
      copy_to(lds + to + 32 * RB);
      c = base + r1 * RB;
      copy16<0, true>(c, off);
      if constexpr (D == 128) copy16<1024, true>(c, off);
    };
    codes(p.k_codes, offsetof(X, k));
    codes(p.v_codes, offsetof(X, v));
    // (8 D / 32 lanes have the second piece's scales: their offset reaches over from the first's)
    const bool second = lane & (8 * SB);
    const uint8_t* const base[2] = {p.k_scale, p.v_scale};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      copy_to(lds + (i ? offsetof(X, vs) : offsetof(X, ks)));
      copy4v(base[i] + (second ? r1 : r0) * SB + 4 * (lane & (8 * SB - 1)));
    }
    return (static_cast<uint32_t>(pages.id[0]) < num ? 3u : 0u) | (static_cast<uint32_t>(pages.id[1]) < num ? 12u : 0u);
  }
  int64_t row[kT];
  uint32_t there = 0;
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    row[t] = row_of(pages.id[t]);
    there |= static_cast<uint32_t>(pages.id[t]) < num ? 1u << t : 0u;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint8_t* const base = i ? p.v_codes : p.k_codes;
    const uint32_t to = lds + (i ? offsetof(X, v) : offsetof(X, k));
    if constexpr (D == 128) {
#pragma unroll
      for (int t = 0; t < kT; ++t) {
        copy_to(to + 1024 * t);
        copy16<0, true>(base + row[t] * RB, off);
      }
    } else {  // a copy reaches over two pieces
#pragma unroll
      for (int t = 0; t < kT; t += 2) {
        // (two scalars: an array's place that goes by the lane lies in scratch memory, and each wait for that is one for all copies)
        const int64_t r0 = row[t], r1 = row[t + 1];
        copy_to(to + 512 * t);
        copy16v(base + (lane & 32 ? r1 : r0) * RB + (off & 511));
      }
    }
  }
  const int64_t a = lane & (4 * SB) ? row[1] : row[0], b = lane & (4 * SB) ? row[3] : row[2];
  const int64_t so = (lane & (8 * SB) ? b : a) * SB + 4 * (lane & (4 * SB - 1));
  copy_to(lds + offsetof(X, ks));
  copy4v(p.k_scale + so);
  copy_to(lds + offsetof(X, vs));
  copy4v(p.v_scale + so);
  return there;
}

// A query's columns in four E2M3 terms: D = 128 an operand each, D = 64 two terms to an operand (lanes g < 2 the first);
// byte i of e: the E8M0 scale of operand i.
template <int D>
struct Query {
  static constexpr int N = D / 32;
  u32x6 w[N];
  uint32_t e;
};

template <int DT, int D, bool REST = false>
__device__ __forceinline__ Query<D> query(const Columns& q, int g, bool* more = nullptr) {
  const Terms s = split_query<DT, REST>(q, more);
  Query<D> x;
  if constexpr (D == 128) {
#pragma unroll
    for (int t = 0; t < 4; ++t) x.w[t] = s.w[t];
    x.e = s.e;
  } else {  // (bytes 0 and 2, or 1 and 3)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 6; ++i) x.w[t][i] = g < 2 ? s.w[2 * t][i] : s.w[2 * t + 1][i];
    x.e = __builtin_amdgcn_perm(s.e, s.e, g < 2 ? 0x0c0c0200u : 0x0c0c0301u);
  }
  return x;
}

// K (E2M1, scale in byte T of ke) times operand I of the query (E2M3)
template <int T, int I>
__device__ __forceinline__ v4f product(const uint4& k, uint32_t ke, const u32x6& q, uint32_t qe, const v4f& c) {
  const i32x8 x = {static_cast<int>(k.x), static_cast<int>(k.y), static_cast<int>(k.z), static_cast<int>(k.w), 0, 0, 0, 0};
  const i32x8 y = {static_cast<int>(q[0]), static_cast<int>(q[1]), static_cast<int>(q[2]), static_cast<int>(q[3]),
                   static_cast<int>(q[4]), static_cast<int>(q[5]), 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 2, T, static_cast<int>(ke), I, static_cast<int>(qe));
}
template <int I, int D>
__device__ __forceinline__ void products(const uint4 (&k)[kT], uint32_t ke, const Query<D>& q, v4f (&sc)[kT]) {
  sc[0] = product<0, I>(k[0], ke, q.w[I], q.e, sc[0]);
  sc[1] = product<1, I>(k[1], ke, q.w[I], q.e, sc[1]);
  sc[2] = product<2, I>(k[2], ke, q.w[I], q.e, sc[2]);
  sc[3] = product<3, I>(k[3], ke, q.w[I], q.e, sc[3]);
  if constexpr (I + 1 < Query<D>::N) products<I + 1, D>(k, ke, q, sc);
}

// The same with the operands in LDS, one after the other
template <int I, int D>
__device__ __forceinline__ void products_of(const uint4 (&k)[kT], uint32_t ke, const uint32_t (*x)[64], int lane, v4f (&sc)[kT]) {
  u32x6 w;
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = x[6 * I + i][lane];
  const uint32_t e = x[6 * Query<D>::N][lane];
  sc[0] = product<0, I>(k[0], ke, w, e, sc[0]);
  sc[1] = product<1, I>(k[1], ke, w, e, sc[1]);
  sc[2] = product<2, I>(k[2], ke, w, e, sc[2]);
  sc[3] = product<3, I>(k[3], ke, w, e, sc[3]);
  asm volatile("" ::"v"(e) : "memory");
  if constexpr (I + 1 < Query<D>::N) products_of<I + 1, D>(k, ke, x, lane, sc);
}

template <int DT, int D>
__global__ void __launch_bounds__(256, decode4_groups(D)) paged_decode4_kernel(const Args a) {
  constexpr int NB = D / 16, NW = 4;
  const lbfq_paged_params& p = a.p;
  if (static_cast<int64_t>(blockIdx.x) >= a.main) {
    fill_rest<D>(p, blockIdx.x - a.main, gridDim.x - a.main);
    return;
  }
  __shared__ union {
    Ring<D> ring;
    DecodeLds<D> join;
  } lds;
  __shared__ uint32_t rest_lds[Query<D>::N * 6 + 1][64];  // each lane's four more terms, where a query takes them
  const uint32_t Hk = static_cast<uint32_t>(p.Hk);
  const int split = static_cast<int>(blockIdx.x / a.combos);
  const uint32_t rest = blockIdx.x % a.combos;
  const int b = static_cast<int>(rest / Hk), kvh = static_cast<int>(rest % Hk);
  const Seq s = sequence(p, b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const Table table = (Table)(reinterpret_cast<uintptr_t>(p.block_table + b * p.table_stride));
  const int G = a.G, rows = s.n * G;  // below 2^30: the host checks T * Hq
  for (int r0 = 0; r0 < rows; r0 += kDecodeRows) {  // once, but for more new tokens than max_query_len
    // this lane's query; rows past the last repeat it and are not stored
    const int rr = r0 + n < rows ? r0 + n : rows - 1;
    const int qi = rr / G, h = kvh * G + (rr - qi * G);
    const int lo_r = s.lo(qi), hi_r = s.hi(qi);
    const int first = r0 / G;
    const int last = ((r0 + kDecodeRows < rows ? r0 + kDecodeRows : rows) - 1) / G;
    const int lo = s.lo(first), hi = s.hi(last);          // keys that some row sees
    const int lo_all = s.lo(last), hi_all = s.hi(first);  // keys that every row sees
    const int kt0 = lo / kKeys, nt = hi > lo ? (hi + kKeys - 1) / kKeys - kt0 : 0;
    int per = (nt + a.splits - 1) / a.splits;
    per = per > a.least ? per : a.least;
    const int begin = kt0 + split * per;
    const int end = begin + per < kt0 + nt ? begin + per : kt0 + nt;
    v4f acc[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[nb][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    int up = kUp;
    bool large = false;  // some block's unit is below the bytes
    if (begin + wave < end) {
      Pages pages;
      load_pages(p, table, kKeys * (begin + wave), pages);
      Columns raw = load_columns(reinterpret_cast<const uint16_t*>(p.q) + (s.start + qi) * p.q_t + h * p.q_h +
                                 32 * (D == 128 ? g : g & 1));
      const int lr = lane / (D / 32);  // this lane's row and place of it in a copy
      const uint32_t off = D / 2 * lr + 16 * piece_of<D>(lr & 15, lane & (D / 32 - 1));
      const uint32_t ring = lds_addr(&lds.ring.t[wave][0]);
#pragma unroll
      for (int i = 0; i < 16; ++i) asm volatile("" : "+v"(raw.w[i]));  // (here: a wait for them later is one for the copies too)
      wait_for<0>();
      uint32_t there = fetch<D>(p, pages, kvh, kKeys * (begin + wave), lane, off, ring), next = 0;
      if (begin + wave + NW < end) {
        load_pages(p, table, kKeys * (begin + wave + NW), pages);
        next = fetch<D>(p, pages, kvh, kKeys * (begin + wave + NW), lane, off, ring + sizeof(typename Ring<D>::Tile));
      }
      load_pages(p, table, kKeys * (begin + wave + 2 * NW), pages);
      bool more;
      const Query<D> q = query<DT, D>(raw, g, &more);  // (while the tiles are on their way)
      more = __any(more);
      if (more) {  // (the same from all four waves)
        const Query<D> rest = query<DT, D, true>(raw, g);
#pragma unroll
        for (int i = 0; i < Query<D>::N; ++i)
#pragma unroll
          for (int k = 0; k < 6; ++k) rest_lds[6 * i + k][lane] = rest.w[i][k];
        rest_lds[6 * Query<D>::N][lane] = rest.e;
      }
      // This lane's places in a tile: its piece of K row key_of_16(n), and columns (D/16) n .. of V rows 4 i + g, of 16 keys
      using X = typename Ring<D>::Tile;
      const int kr = key_of_16(n), kpiece = D == 128 ? g : g & 1, vpiece = D == 128 ? n >> 2 : n >> 3;
      const int k_at = offsetof(X, k) + D / 2 * kr + 16 * piece_of<D>(kr, kpiece);
      const int ks_at = offsetof(X, ks) + D / 32 * kr + kpiece;
      const int vs_at = offsetof(X, vs) + D / 32 * g + vpiece;
      int v_at[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v_at[i] = offsetof(X, v) + D / 2 * (4 * i + g) + 16 * piece_of<D>(4 * i + g, vpiece) + D / 32 * (n & (D == 128 ? 3 : 7));
      int buf = 0;  // the tile's buffer, in bytes
      for (int kt = begin + wave; kt < end; kt += NW) {
        const int kb = kKeys * kt;
        if (kt + NW < end) wait_for<kCopies<D>>();
        else wait_for<0>();
        // The tile into registers, and the one after the next on its way into its place
        uint4 k[kT];
        uint32_t ks[kT], v[kT][4], vs[kT][4];
        const uint8_t* const x = reinterpret_cast<const uint8_t*>(&lds.ring.t[wave][0]) + buf;
#pragma unroll
        for (int t = 0; t < kT; ++t) {
          k[t] = *reinterpret_cast<const uint4*>(x + k_at + 8 * D * t);
          ks[t] = x[ks_at + D / 2 * t];
        }
#pragma unroll
        for (int t = 0; t < kT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            load_bytes<D / 32>(x + v_at[i] + 8 * D * t, &v[t][i]);
            vs[t][i] = x[vs_at + D / 2 * t + D / 8 * i];
          }
        const uint32_t here = there;
        there = next;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (kt + 2 * NW < end) {
          next = fetch<D>(p, pages, kvh, kKeys * (kt + 2 * NW), lane, off, ring + buf);
          load_pages(p, table, kKeys * (kt + 3 * NW), pages);
        }
        buf = buf ? 0 : sizeof(X);
        // S^T: lane (n, g) has query n, keys 16 t + 4 i + g
        const uint32_t ke = ks[0] | ks[1] << 8 | ks[2] << 16 | ks[3] << 24;
        v4f sc[kT];
#pragma unroll
        for (int t = 0; t < kT; ++t) sc[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        products<0, D>(k, ke, q, sc);
        if (more) {
          products_of<0, D>(k, ke, rest_lds, lane, sc);
        }
        if (!(kb >= lo_all && kb + kKeys <= hi_all && here == 15u)) {
#pragma unroll
          for (int t = 0; t < kT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = kb + 16 * t + 4 * i + g;
              if (!(here >> t & 1u) || key < lo_r || key >= hi_r) sc[t][i] = -INFINITY;
              // a scale that lies in the place of a key that no row sees may be anything; its codes are finite as they are
              if (!(here >> t & 1u) || key < lo || key >= hi) vs[t][i] = 127;
            }
        }
        int top = static_cast<int>(vs[0][0]);
#pragma unroll
        for (int t = 0; t < kT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = static_cast<int>(vs[t][i]) > top ? static_cast<int>(vs[t][i]) : top;
        if (__any(top + up > kTop)) {
          lower_unit<D>(top, up, acc);
          large = __any(up < 0);
        }
        if (large) {
#pragma unroll
          for (int t = 0; t < kT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) vs[t][i] = static_cast<int>(vs[t][i]) > -up ? vs[t][i] : static_cast<uint32_t>(-up);
        }
        float mx = vmax(vmax(sc[0][0], sc[0][1]), vmax(sc[0][2], sc[0][3]));
#pragma unroll
        for (int t = 1; t < kT; ++t) mx = vmax(vmax(mx, vmax(sc[t][0], sc[t][1])), vmax(sc[t][2], sc[t][3]));
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
#pragma unroll
        for (int u = 0; u < kT; u += 2) {
          uint32_t ph[4], pl[4];
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[u + t][i], a.sml2, -ms));
              const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[u + t][i + 1], a.sml2, -ms));
              l += p0 + p1;
              const uint32_t w = pack_bf16(p0, p1);
              ph[2 * t + i / 2] = w;
              pl[2 * t + i / 2] = pack_bf16(p0 - __uint_as_float(w << 16), p1 - __uint_as_float(w & 0xffff0000u));
            }
          const uint4 pb = make_uint4(ph[0], ph[1], ph[2], ph[3]), pc = make_uint4(pl[0], pl[1], pl[2], pl[3]);
          // V^T: for product nb lane (n, g) has row NB n + nb, its eight keys in P's order
          float e[8];
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) e[4 * t + i] = __uint_as_float((vs[u + t][i] + up) << 23);
#pragma unroll
          for (int c = 0; c < NB / 2; ++c) {  // two columns of a lane
            uint32_t vv[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) vv[j] = cvt_bf16<4>(&v[u + j / 4][j % 4], c, e[j]);
#pragma unroll
            for (int nb = 2 * c; nb < 2 * c + 2; ++nb) {
              const uint32_t sel = nb & 1 ? 0x07060302u : 0x05040100u;  // upper or lower halves of (second, first)
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) w[j] = __builtin_amdgcn_perm(vv[2 * j + 1], vv[2 * j], sel);
              const uint4 va = make_uint4(w[0], w[1], w[2], w[3]);
              acc[nb] = mfma16_bf16(va, pb, acc[nb]);
              acc[nb] = mfma16_bf16(va, pc, acc[nb]);
            }
          }
        }
        // (a product must not write over its own scale: it stays until here)
        asm volatile("" ::"v"(ke));
      }
    }
    __syncthreads();  // (the ring's place)
    join_waves<DT, D>(a, s, acc, m, l, up, lds.join, r0, rows, split, kvh);
    __syncthreads();  // the next rows use the same LDS
  }
}

}  // namespace

void lbfq::paged::launch_decode4(const Args& a, unsigned grid, hipStream_t st) {
  const bool bf = a.p.dtype == kBF16, d128 = a.p.D == 128;
  if (bf && d128) hipLaunchKernelGGL((paged_decode4_kernel<kBF16, 128>), dim3(grid), dim3(256), 0, st, a);
  else if (bf) hipLaunchKernelGGL((paged_decode4_kernel<kBF16, 64>), dim3(grid), dim3(256), 0, st, a);
  else if (d128) hipLaunchKernelGGL((paged_decode4_kernel<kF16, 128>), dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((paged_decode4_kernel<kF16, 64>), dim3(grid), dim3(256), 0, st, a);
}

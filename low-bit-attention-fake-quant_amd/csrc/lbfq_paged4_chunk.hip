// Attention of chunks of new tokens over the paged cache in 4 bits (the mathematics, the masks, the row tiles and their
// order are those of lbfq_paged.hip's chunk kernel, and so is the order of a step: the next tile's scores and this one's P V
// beside the softmax and the conversion of V).
//
// What is different is K.  It stays as it lies in memory: tiles are copied to LDS asynchronously, three of them there, and
// multiplied by the query's four E2M3 terms with the block-scaled product (32x32x64; see lbfq_paged4.hip): as many
// cycles as bf16's, but a quarter of the LDS reads, and no conversion.  (At 16 bits, a step's reads take as long as its
// products: 32 KiB for 16 + 16 of 32 cycles, four waves and two workgroups a CU.)  K's scales go into the product, so no
// span of them needs bf16.  (Queries that take eight terms, as parts whose V scales lie far apart, go through a plain loop.)
// P is one fp16 term, 11 bits, as in the 8-bit kernel: a second would be half as many products again.  V is converted as
// there, but staged as rows of keys, and turned by the reads that feed the products (with 16 permutations a step instead,
// heads of 64 took 2.5% longer, of 128 the same).
//
// 8192 tokens over 32768 keys, 8 heads of 128, all seen: 930 to 980 us, 1.12 to 1.18 PFLOP/s, where a large library product
// reaches 1.24 (with all codes zero 756: power).  4680 over 32760, 12 heads: 840 to 850 us, 1.11 to 1.12 PFLOP/s, the matrix
// units busy 56% of the cycles at 2.0 GHz (the 8-bit kernel 1040 to 1140).  200 VALU instructions a step besides 32 products
// of 32 cycles, 32 of them exponentials.  Heads of 64, twice the exponentials per product: 0.92.
#include "lbfq_paged_common.h"

using namespace lbfq;
using namespace lbfq::paged;

namespace {

template <int D>
struct Lds {
  // Pitch of a V row, one key's columns: 64 more than a multiple of 256 or of 128, so that the four rows that 32 lanes of a
  // transposing read take 64 bytes of are on distinct banks.
  static constexpr int VP = 2 * D + 64;
  // A tile's K: 16 keys of each wave that copies them, rows of D / 2 bytes, pieces exchanged (piece_of), and their scales
  // (what a copy of 64 lanes needs; D = 64 uses half of the codes' place, and the scales take 64 or 32 bytes)
  uint8_t k[3][4][1024], ks[3][4][256];
  uint8_t v[2][64 * VP];
};

// K (E2M1; scale in byte A of ke) times term B of the query
template <int A, int B>
__device__ __forceinline__ v16f product(const uint4& k, uint32_t ke, const Terms& q, const v16f& c) {
  const i32x8 x = {static_cast<int>(k.x), static_cast<int>(k.y), static_cast<int>(k.z), static_cast<int>(k.w), 0, 0, 0, 0};
  const u32x6& w = q.w[B];
  const i32x8 y = {static_cast<int>(w[0]), static_cast<int>(w[1]), static_cast<int>(w[2]), static_cast<int>(w[3]),
                   static_cast<int>(w[4]), static_cast<int>(w[5]), 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 2, A, static_cast<int>(ke), B, static_cast<int>(q.e));
}

// V^T as A operand of a product of 32 columns and 16 keys from rows of keys: a read that transposes 4 x 16 values between 16
// lanes gives each its column of four keys.  at: this lane's 8 bytes of the first four keys' rows.
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4* LdsRow;
template <int VP>
__device__ __forceinline__ uint4 v_operand(const uint8_t* at) {
  const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsRow)(at)));
  const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsRow)(at + 4 * VP)));
  return make_uint4(a.x, a.y, b.x, b.y);
}

template <int DT, int D>
__global__ void __launch_bounds__(256, chunk4_groups(D)) paged_chunk4_kernel(const Args a) {
  constexpr int NW = 4, QB = kChunkRows, NT = 64 * NW;
  static_assert(QB == 32 * NW, "32 rows a wave");
  constexpr int NC = D / 64, NKS = 4 * NC, NDB = D / 32, CH = D / 32, RB = D / 2;
  constexpr int VK = D / 32;      // V keys of a thread, eight columns each
  constexpr int WKEYS = 64 / NW;  // keys that a wave stages: of one page
  constexpr int kUnit = unit_of(4);
  using L = Lds<D>;
  const lbfq_paged_params& p = a.p;
  if (static_cast<int64_t>(blockIdx.x) >= a.main) {
    fill_rest<D>(p, blockIdx.x - a.main, gridDim.x - a.main);
    return;
  }
  __shared__ __align__(16) L lds;
  const int G = a.G, Hk = static_cast<int>(p.Hk);
  int split, kvh, slot, b = 0, r0;
  if (a.share) {
    // Two unequal parts of one sequence: all the longer ones first, each XCD a stretch of neighbouring row tiles.
    const uint32_t half = static_cast<uint32_t>(a.main) / 2, all = a.slots * static_cast<uint32_t>(Hk);
    split = blockIdx.x >= half;
    const uint32_t i = blockIdx.x - split * half, id = i % 8 * (half / 8) + i / 8;
    if (id >= all) return;
    kvh = static_cast<int>(id / a.slots);
    slot = static_cast<int>(id % a.slots);
    r0 = slot * QB;
  } else {
    // (the 8-bit kernel's order: neighbouring row tiles to one XCD, the last rows first)
    const uint32_t ps = a.piece, round = blockIdx.x / (8 * ps), piece = round * 8 + (blockIdx.x + round) % 8;
    slot = a.slots - 1 - static_cast<int>(piece / a.combos * ps + blockIdx.x / 8 % ps);
    if (slot < 0) return;
    const uint32_t rest = piece % a.combos, splits = static_cast<uint32_t>(a.splits);
    split = static_cast<int>(rest % splits);
    kvh = static_cast<int>(rest / splits);
    b = sequence_at(p, G, slot);
    r0 = (slot - slot_of(p, G, b)) * QB;
  }
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
  const int vkg = lane / (D / 8), vdq = lane % (D / 8);  // V: keys VK vkg .. of the wave's, columns 8 vdq ..
  static_assert(64 / (D / 8) * VK == WKEYS, "a wave's keys");
  const uint32_t voff = VK * vkg * RB + 4 * vdq, vsoff = VK * vkg * CH;
  const int lr = lane / CH & 15;  // K: row and piece of this lane's 16 bytes (D = 64: lanes 32 .. copy them again)
  const uint32_t koff = RB * lr + 16 * piece_of<D>(lr, lane % CH), ksoff = 4 * (lane & (4 * CH - 1));

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
  if (a.share) per = static_cast<int>((static_cast<int64_t>(nt) * a.share + 65535) >> 16);
  per = per > a.least ? per : a.least;
  const int begin = kt0 + split * per;  // (unequal parts: the second is the shorter one)
  const int end = begin + per < kt0 + nt ? begin + per : kt0 + nt;

  v16f acc[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  Unit uv{kUnit, false};
  uint32_t vtops = 0;  // V's unit: the byte that block b's scale vtops >> 8 b comes to is vtop
  int vtop = kUnit;
  if (begin < end) {
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
    // A tile's K into LDS (place b of three), its V into registers: of a page that is not there, page 0's
    auto copy_k = [&](int kt, int page, int b) {
      const int64_t row = row_of(page < 0 ? 0 : page, 64 * kt + WKEYS * wave);
      // (the same in every lane, which the compiler does not always see)
      const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(row >> 32));
      const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(row));
      const int64_t at = static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
      copy_to(lds_addr(lds.k[b][wave]));
      copy16<0, false>(p.k_codes + at * RB, koff);
      copy_to(lds_addr(lds.ks[b][wave]));
      copy4<false>(p.k_scale + at * CH, ksoff);
    };
    uint32_t vc[VK], vse[VK * CH / 4];
    auto load_v = [&](int kt, int page) {
      const int64_t row = row_of(page < 0 ? 0 : page, 64 * kt + WKEYS * wave);
      const uint8_t* vs = p.v_codes + row * RB;
#pragma unroll
      for (int j = 0; j < VK; ++j) load_bytes<4>(vs + voff + j * RB, vc + j);
      load_bytes<VK * CH>(p.v_scale + row * CH + vsoff, vse);
    };
    const int ids = look(begin);
    const uint32_t mask = there(begin, ids);
    const int page0 = page_in(ids, mask, 0), page1 = page_in(ids, mask, 1);
    int pv = page1, pk = page_in(ids, mask, 3);
    copy_k(begin, page0, 0);
    copy_k(upto(begin + 1), page1, 1);
    copy_k(upto(begin + 2), page_in(ids, mask, 2), 2);
    load_v(begin, page0);
    auto columns = [&](int row, int i) {  // this lane's 32 of step i
      const int query = row / G, head = kvh * G + (row - query * G);
      return reinterpret_cast<const uint16_t*>(p.q) + (s.start + query) * p.q_t + head * p.q_h + 64 * i + 32 * g;
    };
    Terms q[NC];
    bool more = false;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      bool x;
      q[i] = split_query<DT>(
          load_columns(reinterpret_cast<const uint16_t*>(p.q) + (s.start + qi) * p.q_t + h * p.q_h + 64 * i + 32 * g), &x);
      more |= x;
    }
    // The span of the part's V scales, over the keys that some row sees: four keys a thread and look, eight looks on their
    // way at a time (one after the other, each is two trips to memory: 32 looks were 5% of a long part).
    {
      constexpr int U = 8;
      uint32_t sv = 0;
      const int k1 = 64 * end < hi ? 64 * end : hi;
      for (int key0 = 64 * begin + 4 * tid; key0 < k1; key0 += 4 * NT * U) {
        int page[U];
        uint32_t x[U][CH];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int key = key0 + 4 * NT * u, idx = (key < k1 ? key : key0) >> shift;
          page[u] = table[idx < cols ? idx : cols - 1];
          if (idx >= cols || page[u] >= num_pages || key >= k1 || key + 4 <= lo) page[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) load_bytes<4 * CH>(p.v_scale + row_of(page[u] < 0 ? 0 : page[u], key0 + 4 * NT * u) * CH, x[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int key = key0 + 4 * NT * u;
          if (page[u] < 0) continue;
          if (key >= lo && key + 4 <= k1) {
#pragma unroll
            for (int c = 0; c < CH; ++c) sv = span_add<4>(sv, x[u][c]);
          } else {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (const int ki = key + (4 * c + i) / CH; ki >= lo && ki < k1) sv = span_add<1>(sv, x[u][c] >> (8 * i));
          }
        }
      }
      uint32_t* red = reinterpret_cast<uint32_t*>(lds.v[1]);
#pragma unroll
      for (int i = 1; i < 64; i <<= 1) sv = span_join(sv, __shfl_xor(sv, i, 64));
      more = __any(more);
      if (lane == 0) {
        red[wave] = sv;
        red[NW + wave] = more;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        sv = span_join(sv, red[w]);
        more |= red[NW + w] != 0;
      }
      __syncthreads();
      more = __builtin_amdgcn_readfirstlane(more);
      sv = __builtin_amdgcn_readfirstlane(sv);
      uv.E = static_cast<int>(sv & 0xffu);
      uv.wide = more || uv.E - (255 - static_cast<int>(sv >> 16)) > span_of(4);
      if (sv == 0) uv.E = kUnit;
      vtops = uv.wide ? block_tops<D, NT>(p, table, kvh, lo > 64 * begin ? lo : 64 * begin, k1, red) : uv.E * 0x01010101u;
      if (uv.wide) vtop = wide_top(64 * (end - begin));
    }
    const float c = a.sml2;
    // (wide: of this thread's block of columns)
    const int vup = uv.wide ? vtop - static_cast<int>(vtops >> 8 * (vdq / 4) & 0xffu) : kUnit - uv.E;

    // Keys that no row sees, or that are not there: their scales may be anything (their codes are finite as they are, and
    // what K has there ends in scores that are masked).
    auto clear_v = [&](int kt, int page) {
      const int key0 = 64 * kt + WKEYS * wave;
      if (page >= 0 && key0 >= lo && key0 + WKEYS <= hi) return;
#pragma unroll
      for (int j = 0; j < VK; ++j)
        if (const int key = key0 + VK * vkg + j; page < 0 || key < lo || key >= hi) {
          if constexpr (CH == 4) vse[j] = vtops;
          else vse[0] = (vse[0] & (j & 1 ? 0x0000ffffu : 0xffff0000u)) | (vtops & (j & 1 ? 0xffff0000u : 0xffffu));
        }
    };
    // V's key i of this thread's VK: registers -> LDS, as fp16 in the part's unit or (WIDE) as bf16
    auto put_v = [&](int i, uint8_t* buf, auto WIDE) {
      uint32_t by;
      if constexpr (CH == 4) by = __builtin_amdgcn_ubfe(vse[i], 8 * (vdq / 4), 8);
      else by = __builtin_amdgcn_ubfe(vse[0], 16 * i + 8 * (vdq / 4), 8);
      const int e = static_cast<int>(by) + vup;
      const float sc = __uint_as_float(static_cast<uint32_t>(WIDE && e < 0 ? 0 : e) << 23);
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = WIDE ? cvt_bf16<4>(vc + i, k, sc) : cvt_f16<4>(vc + i, k, sc);
      *reinterpret_cast<uint4*>(buf + (WKEYS * wave + VK * vkg + i) * L::VP + 16 * vdq) = make_uint4(w[0], w[1], w[2], w[3]);
    };
    auto store_v = [&](uint8_t* buf, auto WIDE) {
#pragma unroll
      for (int i = 0; i < VK; ++i) put_v(i, buf, WIDE);
    };
    // This lane's part in V's reads: keys 8 g + li % 16 / 4 (and four on), columns 16 (li / 16) + 4 (li % 4) ..
    const int vrow = (8 * g + (li & 15) / 4) * L::VP + 32 * (li >> 4) + 8 * (li & 3);
    // This lane's K row of a 32-key block, as A operand: its piece 2 i + g and the bytes 2 i + g of its scales (in bytes 2 i)
    const int kr = key_of_32(li), krow = RB * (kr & 15), ksrow = CH * (kr & 15);
    auto k_operand = [&](int b, int bl, int i) {
      return *reinterpret_cast<const uint4*>(lds.k[b][2 * bl + (kr >> 4)] + krow + 16 * piece_of<D>(kr & 15, (2 * i + g) & (CH - 1)));
    };
    auto k_scale = [&](int b, int bl) -> uint32_t {
      const uint8_t* at = lds.ks[b][2 * bl + (kr >> 4)] + ksrow;
      if constexpr (CH == 4) return *reinterpret_cast<const uint32_t*>(at) >> (8 * g);
      else return *reinterpret_cast<const uint16_t*>(at) >> (8 * g);
    };
    // Product n of a block's scores: step n / 4 of the columns, term n % 4
    auto score = [&](int n, const uint4& k, uint32_t ke, const v16f& sc, const Terms (&q)[NC]) -> v16f {
      switch (n) {  // (known once the loops are unrolled)
        case 0: return product<0, 0>(k, ke, q[0], sc);
        case 1: return product<0, 1>(k, ke, q[0], sc);
        case 2: return product<0, 2>(k, ke, q[0], sc);
        case 3: return product<0, 3>(k, ke, q[0], sc);
        case 4: return product<2, 0>(k, ke, q[NC - 1], sc);
        case 5: return product<2, 1>(k, ke, q[NC - 1], sc);
        case 6: return product<2, 2>(k, ke, q[NC - 1], sc);
        default: return product<2, 3>(k, ke, q[NC - 1], sc);
      }
    };
    // (a product must not write over its own scale: it stays until the block's scores are done)
    auto keep = [](uint32_t ke) { asm volatile("" ::"v"(ke)); };
    // S^T of 32 keys: register r is key 32 bl + 16 (r / 8) + 8 g + r % 8 of the tile in place b
    auto scores = [&](int b, int bl, v16f& sc, const Terms (&q)[NC], bool fresh = true) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = fresh ? 0.0f : sc[r];
      const uint32_t ke = k_scale(b, bl);
#pragma unroll
      for (int n = 0; n < NKS; ++n) sc = score(n, k_operand(b, bl, n / 4), ke, sc, q);
      keep(ke);
    };
    // The tile's scores masked where a row does not see the key, the row's reference m brought up to date (and with it
    // the sums so far); returns what p is relative to.
    auto settle = [&](int kb, uint32_t here, v16f& s0, v16f& s1) -> float {
      if (!(kb >= lo_all && kb + 64 <= hi_all && here == 0xfu)) {
        // seen: from lo_r on, fewer than `span` keys (of a page that is not there: none); one compare, and no branches
        const uint32_t at = static_cast<uint32_t>(kb + 8 * g - lo_r), span = hi_r > lo_r ? static_cast<uint32_t>(hi_r - lo_r) : 0u;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t n0 = here >> t & 1u ? span : 0u, n1 = here >> (t + 2) & 1u ? span : 0u;
#pragma unroll
          for (int i = 8 * t; i < 8 * t + 8; ++i) {
            s0[i] = at + (8 * t + i) < n0 ? s0[i] : -INFINITY;
            s1[i] = at + (8 * t + i + 32) < n1 ? s1[i] : -INFINITY;
          }
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

    if (uv.wide) {
      // Rare (see Unit, and split_query), and plain: one tile after the other.
      Terms rest[NC];
      if (more) {
        int row = rw + li < rows ? rw + li : rows - 1;
        asm volatile("" : "+v"(row));  // (the address formed again: it would wait in memory, there are no registers for it)
#pragma unroll
        for (int i = 0; i < NC; ++i) rest[i] = split_query<DT, true>(load_columns(columns(row, i)));
#pragma unroll
        for (int i = 0; i < NC; ++i) {  // (and these, in place of waiting meanwhile)
          bool x;
          q[i] = split_query<DT>(load_columns(columns(row, i)), &x);
        }
      }
      wait_for<0>();  // (the first tiles' copies)
      for (int kt = begin; kt < end; ++kt) {
        const int id = look(kt);
        const uint32_t here = there(kt, id);
        const int page = page_in(id, here, 0);
        copy_k(kt, page, 0);
        load_v(kt, page);
        clear_v(kt, page);
        store_v(lds.v[0], std::true_type{});
        wait_for<0>();
        __syncthreads();
        v16f sc[2];
#pragma unroll
        for (int bl = 0; bl < 2; ++bl) {
          scores(0, bl, sc[bl], q);
          if (more) scores(0, bl, sc[bl], rest, false);
        }
        const float ms = settle(64 * kt, here & 0xfu, sc[0], sc[1]);
#pragma unroll
        for (int bl = 0; bl < 2; ++bl)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint8_t* vr = lds.v[0] + vrow + 16 * (2 * bl + j) * L::VP;
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              x[k] = __builtin_amdgcn_exp2f(fmaf(sc[bl][8 * j + k], c, -ms));
              l += x[k];
            }
            uint32_t w[4], w2[4];  // V is bf16 as it is: P in two bf16 terms (16 bits)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              w[k] = pack_bf16(x[2 * k], x[2 * k + 1]);
              w2[k] = pack_bf16(x[2 * k] - __uint_as_float(w[k] << 16), x[2 * k + 1] - __uint_as_float(w[k] & 0xffff0000u));
            }
#pragma unroll
            for (int db = 0; db < NDB; ++db) {
              const uint4 va = v_operand<L::VP>(vr + 64 * db);
              acc[db] = mfma32_bf16(va, make_uint4(w[0], w[1], w[2], w[3]), acc[db]);
              acc[db] = mfma32_bf16(va, make_uint4(w2[0], w2[1], w2[2], w2[3]), acc[db]);
            }
          }
        __syncthreads();
      }
    } else {
      constexpr std::false_type kNarrow{};
      clear_v(begin, page0);
      store_v(lds.v[0], kNarrow);
      load_v(upto(begin + 1), pv);
      uint32_t here0 = mask & 0xfu, here1 = mask >> 4 & 0xfu, here2 = mask >> 8 & 0xfu, here3 = mask >> 12 & 0xfu;
      int pn = page_in(ids, mask, 2);
      wait_for<0>();
      __syncthreads();
      v16f sa, sb, sc_;
      scores(0, 0, sa, q);
      scores(0, 1, sb, q);
      __syncthreads();  // the first step puts another K tile there
      // Tile kt: its scores are in s0 and s1; the next tile's go to s2 and, when s0 is used up, s0 (three blocks for what
      // would be four).  In LDS: K of kt + 1 (place kn) and kt + 2, V of kt (cur); place kf is free.  In the staging
      // registers: V of kt + 1.
      auto step = [&](int kt, uint8_t* cur, uint8_t* nxt, int kn, int kf, v16f& s0, v16f& s1, v16f& s2) {
        // The step's products in order: of each half of the tile the next tile's scores (NKS products) and this one's
        // two quarters of P V (NDB each).  Their LDS operands are read kAhead products ahead, and each product is
        // followed by a piece of what the VALU has to do meanwhile: the softmax of the half beside the scores, the
        // conversion of the staged V tile beside P V.  The order is fixed here; left to the
        // compiler, every read was next to its product.  The further a wave is in its products, the higher its priority:
        // the SIMD's other wave then gives way, and does its waits, masks and maxima when this one does not multiply (4680
        // tokens over 32760 keys, 12 heads: 888 us without, 840; one level instead of two 865).
        constexpr int HALF = NKS + 2 * NDB, kAhead = 5;
        const int id = look(kt + 4);  // back by the end of the step
        uint4 ring[kAhead], kx[NC];
        uint32_t ke[2];
        const uint8_t* const vr = cur + vrow;
        auto fetch = [&](int n) {
          if (n >= 2 * HALF) return;
          const int bl = n / HALF, i = n % HALF;
          if (i < NKS) {
            if (i == 0) ke[bl] = k_scale(kn, bl);
            if (i % 4 == 0) kx[i / 4] = k_operand(kn, bl, i / 4);
          } else {
            ring[n % kAhead] = v_operand<L::VP>(vr + 16 * (2 * bl + (i - NKS) / NDB) * L::VP + 64 * ((i - NKS) % NDB));
          }
        };
#pragma unroll
        for (int n = 0; n < kAhead; ++n) fetch(n);
        const float ms = settle(64 * kt, here0, s0, s1);
        clear_v(upto(kt + 1), pv);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int bl = 0; bl < 2; ++bl) {
          uint32_t w[8];
          if (bl == 1) __builtin_amdgcn_s_setprio(2);
          v16f& sc = bl == 0 ? s0 : s1;
          v16f& sn = bl == 0 ? s2 : s0;
#pragma unroll
          for (int i = 0; i < HALF; ++i) {
            const int n = bl * HALF + i;
            if (i < NKS) {
              if (i == 0) {
#pragma unroll
                for (int r = 0; r < 16; ++r) sn[r] = 0.0f;
              }
              sn = score(i, kx[i / 4], ke[bl], sn, q);
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
              acc[db] = mfma32_f16(ring[n % kAhead], make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]), acc[db]);
              fetch(n + kAhead);
              if ((i - NKS) % 4 == 1) put_v(bl * (VK / 2) + (i - NKS) / 4, nxt, kNarrow);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          keep(ke[bl]);
          // (else the compiler moves these products to the next step, where their results are used: 871 us instead of 840;
          // heads of 64 have too few registers for them here, 48 us instead of 45 on 4 chunks of 509)
          if constexpr (D == 128) asm volatile("" ::"v"(sn));
        }
        __builtin_amdgcn_s_setprio(0);
        wait_for<0>();  // K of kt + 2, asked for a step ago
        // (id is looked at before the next copies: the compiler does not count those, and its wait for id would be for them too)
        const uint32_t mask = there(kt + 4, id);
        const int next_page = page_in(id, mask, 0);
        copy_k(upto(kt + 3), pk, kf);
        load_v(upto(kt + 2), pn);
        pv = pn;
        pn = pk;
        pk = next_page;
        here0 = here1;
        here1 = here2;
        here2 = here3;
        here3 = mask & 0xfu;
        __syncthreads();
      };
      // (two places for V, three for K and three blocks of scores: the order comes round after six steps)
      uint8_t* const v0 = lds.v[0];
      uint8_t* const v1 = lds.v[1];
      for (int kt = begin; kt < end;) {
        step(kt, v0, v1, 1, 0, sa, sb, sc_);
        if (++kt >= end) break;
        step(kt, v1, v0, 2, 1, sc_, sa, sb);
        if (++kt >= end) break;
        step(kt, v0, v1, 0, 2, sb, sc_, sa);
        if (++kt >= end) break;
        step(kt, v1, v0, 1, 0, sa, sb, sc_);
        if (++kt >= end) break;
        step(kt, v0, v1, 2, 1, sc_, sa, sb);
        if (++kt >= end) break;
        step(kt, v1, v0, 0, 2, sb, sc_, sa);
        ++kt;
      }
      wait_for<0>();  // (no copy may come after the workgroup's end)
    }
    l = add_x32(l);
  }
  if (rw + li < rows) {
    int row = rw + li;
    asm volatile("" : "+v"(row));  // (formed again, so that nothing waits for this in registers)
    const int query = row / G, head = kvh * G + (row - query * G);
    const int64_t tok = s.start + query;
    const bool one = a.splits == 1;
    const float f = filled(l) ? 1.0f / l : 0.0f;
    const int64_t at = split * R + tok * p.Hq + head;
    if (one && p.lse && g == 0) p.lse[tok * p.Hq + head] = row_lse(m, l);
    if (!one && g == 0) a.ml[at] = make_float2(m, l);
    if (one || filled(l)) {
      // Register r of acc[db] is column 32 db + 8 (r / 4) + 4 g + r % 4.
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const int e = static_cast<int>(vtops >> 8 * db & 0xffu) - vtop;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int col = 32 * db + 8 * k + 4 * g;
          float o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = ldexpf(acc[db][4 * k + i] * f, e);
          if (one)
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + tok * p.out_t + head * p.out_h + col) =
                make_uint2(pack_dt<DT>(o[0], o[1]), pack_dt<DT>(o[2], o[3]));
          else
            *reinterpret_cast<float4*>(a.acc + at * D + col) = make_float4(o[0], o[1], o[2], o[3]);
        }
      }
    }
  }
}

}  // namespace

void lbfq::paged::launch_chunk4(const Args& a, unsigned grid, hipStream_t st) {
  const bool bf = a.p.dtype == kBF16, d128 = a.p.D == 128;
  if (bf && d128) hipLaunchKernelGGL((paged_chunk4_kernel<kBF16, 128>), dim3(grid), dim3(256), 0, st, a);
  else if (bf) hipLaunchKernelGGL((paged_chunk4_kernel<kBF16, 64>), dim3(grid), dim3(256), 0, st, a);
  else if (d128) hipLaunchKernelGGL((paged_chunk4_kernel<kF16, 128>), dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((paged_chunk4_kernel<kF16, 64>), dim3(grid), dim3(256), 0, st, a);
}

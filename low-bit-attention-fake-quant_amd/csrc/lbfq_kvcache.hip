// The quantised paged K/V cache: rows written as they come, and read back.
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
// Both directions are bound by memory.  D/8 lanes hold a row, eight values each;
// a workgroup takes 64 consecutive tokens of one head of K or of V, so that the
// scales of its rows, four bytes each, fill whole lines from one workgroup, and a
// thread's rows (four at D = 128) are all on their way before the first is used.
// Writing 32760 tokens x 40 heads x 128 from bf16: 196 us, 5.2 TB/s of bytes read
// and written (a copy of 1 GiB reaches 5.1 to 5.5).  Reading 8 sequences of up to
// 16384 x 8 heads to bf16: 147 us, 4.7 TB/s (what only writes reaches 5.3).  A few
// tokens: 3.0 and 4.6 us, a launch's own time.
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
    float m = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(x[i][k]));
    m = fmaxf(m, __shfl_xor(m, 1, 64));
    m = fmaxf(m, __shfl_xor(m, 2, 64));
    const float sc = fminf(mx_scale_from_amax(fmaxf(m, kAmaxFloor)), 0x1p119f);
    const float inv = 1.0f / sc;  // exact: 2^-e
    float q[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = clamp448(x[i][k] * inv);
    if (slot[i] < 0 || slot[i] >= slots) continue;  // padding, or not in the cache
    const int64_t row = ((slot[i] >> p.page_shift) * H + h) * (int64_t{1} << p.page_shift) +
                        (slot[i] & ((int64_t{1} << p.page_shift) - 1));
    *reinterpret_cast<uint2*>(codes + row * D + 8 * lp) = make_uint2(cvt4_e4m3(q), cvt4_e4m3(q + 4));
    if ((lp & 3) == 0) scale[row * (D / 32) + lp / 4] = static_cast<uint8_t>(__float_as_uint(sc) >> 23);
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

int check_cache(const char* who, int64_t num_pages, int page_shift, int64_t H, int64_t D, const void* kc,
                const void* ks, const void* vc, const void* vs) {
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

}  // namespace

extern "C" int lbfq_kv_write(const lbfq_kv_write_params* p, lbfq_stream_t stream) {
  LBFQ_CHECK_ARG(p, "lbfq_kv_write: null params");
  if (int rc = check_cache("lbfq_kv_write", p->num_pages, p->page_shift, p->H, p->D, p->k_codes, p->k_scale,
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

extern "C" int lbfq_kv_read(const lbfq_kv_read_params* p, lbfq_stream_t stream) {
  LBFQ_CHECK_ARG(p, "lbfq_kv_read: null params");
  if (int rc = check_cache("lbfq_kv_read", p->num_pages, p->page_shift, p->H, p->D, p->k_codes, p->k_scale,
                           p->v_codes, p->v_scale))
    return rc;
  LBFQ_CHECK_ARG(p->dtype >= kF32 && p->dtype <= kBF16, "lbfq_kv_read: bad dtype %d", p->dtype);
  LBFQ_CHECK_ARG(p->B > 0 && p->max_len > 0 && p->max_len <= (int64_t{1} << 30), "lbfq_kv_read: bad number of tokens");
  LBFQ_CHECK_ARG((p->block_table || p->table_cols == 0) && p->seq_lens && p->k_out && p->v_out,
                 "lbfq_kv_read: missing tensor");
  LBFQ_CHECK_ARG(p->table_cols >= 0 && p->table_cols < (int64_t{1} << 40), "lbfq_kv_read: bad block table");
  const int64_t blocks = (p->max_len + kRows - 1) / kRows;
  LBFQ_CHECK_ARG(p->B < (int64_t{1} << 24) / (blocks * 2 * p->H), "lbfq_kv_read: problem too large");
  const dim3 grid(static_cast<unsigned>(p->B * blocks * 2 * p->H)), block(256);
  hipStream_t st = static_cast<hipStream_t>(stream);
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

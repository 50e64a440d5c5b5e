// The torch side of the cache operators (qk_norm.py, kv_cache.py): their checks of
// arguments, allocations and parameter structs, in front of the C entries.
//
// A call on a few tokens is bound by this part.  In Python with ctypes it took 14
// us for qk_norm_rope and 9.5 for write_kv_cache; here 5.6 and 3.9.  Kernels stay behind the C ABI (include/lbfq.h), in
// liblbfq_hip.so, which this module links to.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <initializer_list>
#include <limits>
#include <optional>
#include <string>
#include <utility>

#include "../../include/lbfq.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

// Set from Python: index -> the handle of torch's current stream there, and the package's error class.
// Never destroyed: a module's end may come after the interpreter's.
py::object* stream_of = nullptr;
py::object* library_error = nullptr;

std::string str(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + (s.size() == 1 ? ",)" : ")");
}
std::string str(const Tensor& t) { return str(t.sizes()); }

std::string name(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kDouble: return "torch.float64";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    case at::kByte: return "torch.uint8";
    case at::kFloat8_e4m3fn: return "torch.float8_e4m3fn";
    default: return std::string("torch.") + c10::toString(t);
  }
}

[[noreturn]] void bad_value(const std::string& m) { throw py::value_error(m); }
[[noreturn]] void bad_type(const std::string& m) { throw py::type_error(m); }

int dtype_code(at::ScalarType t) {
  if (t == at::kBFloat16) return LBFQ_BF16;
  if (t == at::kHalf) return LBFQ_F16;
  if (t == at::kFloat) return LBFQ_F32;
  bad_type("unsupported dtype " + name(t) + "; expected float32, float16 or bfloat16");
}

void check_rc(int rc, const char* what) {
  if (rc == 0) return;
  const char* m = lbfq_last_error();
  const std::string text = m && *m ? m : std::string(what) + " failed";
  if (rc == -1) bad_value(text);
  PyErr_SetString(library_error->ptr(), text.c_str());
  throw py::error_already_set();
}

void* stream(const Tensor& t) {
  return reinterpret_cast<void*>((*stream_of)(static_cast<int>(t.get_device())).cast<uintptr_t>());
}

// Launches go to the tensors' device, whichever is current.
struct On {
  c10::DeviceGuard guard;
  explicit On(const Tensor& t) : guard(t.device()) {}
};

// Last dimension contiguous and every row on a 16-byte boundary (any other strides go to the kernel)
bool rows_16b(const Tensor& t) {
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  const int64_t last = t.dim() - 1, step = 16 / static_cast<int64_t>(t.element_size());
  if (t.stride(last) != 1 && t.size(last) != 1) return false;
  for (int64_t i = 0; i < last; ++i)
    if (t.size(i) > 1 && t.stride(i) % step) return false;
  return true;
}
Tensor aligned(const Tensor& t) { return rows_16b(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// Stride of a dimension; of one of a single entry, whose stride may be anything, 0.
int64_t row_stride(const Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

bool on(const Tensor& t, int64_t index) { return t.is_cuda() && t.get_device() == index; }
std::string cuda(int64_t index) { return "cuda:" + std::to_string(index); }

void refuse_grad(const char* what) {
  bad_value(std::string(what) + " has no backward pass; detach its inputs or call it under torch.no_grad()");
}

// Forward mode: a dual tensor does not say requires_grad(), and an output without a tangent counts as one of zero.
// (torch.no_grad leaves this mode on.)
void refuse_tangent(const char* what, std::initializer_list<const Tensor*> inputs) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : inputs)
    if (t->defined() && t->_fw_grad(/*level=*/0).defined())
      bad_value(std::string(what) + " has no forward-mode derivative; call it on the primal parts of its inputs");
}

// Whether no two of the rows of t (n0, n1, d), contiguous, share memory.  With strides s0 <= s1: rows that lie j s1 and i s0
// from the first, i of the nearest two.  (One look where the rows of one dimension lie within a step of the other.)
bool rows_apart(const Tensor& t) {
  int64_t n0 = t.size(0), n1 = t.size(1), s0 = row_stride(t, 0), s1 = row_stride(t, 1);
  const int64_t d = t.size(2);
  if (n0 == 0 || n1 == 0) return true;
  if (n0 == 1) std::swap(n0, n1), std::swap(s0, s1);
  if (n0 == 1) return true;
  if (n1 == 1) return s0 >= d;
  if (s0 > s1) std::swap(n0, n1), std::swap(s0, s1);
  if (s0 < d) return false;
  for (int64_t j = 1; j < n1 && j * s1 < (n0 - 1) * s0 + d; ++j) {
    const int64_t i = j * s1 / s0;
    if ((i < n0 && j * s1 - i * s0 < d) || (i + 1 < n0 && (i + 1) * s0 - j * s1 < d)) return false;
  }
  return true;
}

// ---- Q/K norm and rotation -----------------------------------------------------

// q and k hold the (possibly copied) inputs: kept by the caller until the launch.
struct Norm {
  lbfq_qk_norm_params p{};
  Tensor q, k, qw, kw, cos, sin;
};

void weight(const OptTensor& w, const char* what, int64_t d, int64_t index, Tensor& held, const void*& ptr, int& dtype) {
  if (!w) return;
  if (w->dim() != 1 || w->size(0) != d)
    bad_value(std::string(what) + " must have shape (" + std::to_string(d) + ",); got " + str(*w));
  if (!on(*w, index)) bad_value(std::string(what) + " must live on " + cuda(index) + "; got " + w->device().str());
  dtype = dtype_code(w->scalar_type());
  held = w->contiguous();
  ptr = held.data_ptr();
}

void norm_params(Norm& n, const Tensor& q, const Tensor& k, const OptTensor& qw, const OptTensor& kw, const Tensor& cos,
                 const Tensor& sin, const OptTensor& positions, double eps, const std::string& pairs) {
  const int64_t dims = q.dim();
  if ((dims != 3 && dims != 4) || k.dim() != dims)
    bad_value("q and k must both be (B, S, H, D) or (T, H, D); got " + str(q) + " and " + str(k));
  if (!q.is_cuda() || !on(k, q.get_device()))
    bad_value("q and k must live on one CUDA device; got " + q.device().str() + " and " + k.device().str());
  const int64_t index = q.get_device();
  if (k.scalar_type() != q.scalar_type())
    bad_type("q and k must have one dtype; got " + name(q.scalar_type()) + " and " + name(k.scalar_type()));
  auto& p = n.p;
  p.dtype = dtype_code(q.scalar_type());
  const int64_t o = dims - 3;  // of the token dimension
  p.B = o ? q.size(0) : 1;
  p.S = q.size(o);
  p.Hq = q.size(o + 1);
  p.Hk = k.size(o + 1);
  p.D = q.size(o + 2);
  if (p.D != 64 && p.D != 128) bad_value("D must be 64 or 128; got " + std::to_string(p.D));
  if ((o && k.size(0) != p.B) || k.size(o) != p.S || k.size(o + 2) != p.D || p.Hq == 0 || p.Hk == 0)
    bad_value("q and k must agree in all but their heads; got " + str(q) + " and " + str(k));
  if (pairs != "adjacent" && pairs != "halves") bad_value("pairs must be 'adjacent' or 'halves'; got '" + pairs + "'");
  p.halves = pairs == "halves";
  if (!(eps >= 0.0 && eps <= std::numeric_limits<float>::max()))
    bad_value("eps must be finite and not negative; got " + std::to_string(eps));
  p.eps = static_cast<float>(eps);
  if (cos.dim() != 2 || sin.sizes() != cos.sizes())
    bad_value("cos and sin must be (P, R/2); got " + str(cos) + " and " + str(sin));
  if (cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat)
    bad_type("cos and sin must be float32; got " + name(cos.scalar_type()) + " and " + name(sin.scalar_type()));
  p.table_len = cos.size(0);
  const int64_t half = cos.size(1);
  if (half == 0 || half % 8 || 2 * half > p.D)
    bad_value("R must be a multiple of 16 up to D=" + std::to_string(p.D) + "; got " + std::to_string(2 * half));
  p.rot = static_cast<int>(2 * half);
  if (!on(cos, index) || !on(sin, index)) bad_value("cos and sin must live on " + cuda(index));
  if (!positions) {
    if (p.S > p.table_len)
      bad_value("the table has " + std::to_string(p.table_len) + " positions, q has " + std::to_string(p.S));
  } else {
    const Tensor& t = *positions;
    if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong)
      bad_type("positions must be int32 or int64; got " + name(t.scalar_type()));
    if (!on(t, index)) bad_value("positions must live on " + cuda(index) + "; got " + t.device().str());
    const bool one = t.dim() == 1 && t.size(0) == p.S, two = o && t.dim() == 2 && t.size(0) == p.B && t.size(1) == p.S;
    if (!one && !two)
      bad_value("positions must have shape (" + std::to_string(p.S) + ",)" +
                (o ? " or (" + std::to_string(p.B) + ", " + std::to_string(p.S) + ")" : "") + "; got " + str(t));
    p.positions = t.data_ptr();
    p.positions_i64 = t.scalar_type() == at::kLong;
    p.pos_s = t.stride(-1);
    p.pos_b = two ? t.stride(0) : 0;
  }
  weight(qw, "q_weight", p.D, index, n.qw, p.q_weight, p.q_weight_dtype);
  weight(kw, "k_weight", p.D, index, n.kw, p.k_weight, p.k_weight_dtype);
  auto table = [](const Tensor& t) {
    return t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t
                                                                                  : t.clone(at::MemoryFormat::Contiguous);
  };
  n.cos = table(cos);
  n.sin = table(sin);
  p.cos = n.cos.data_ptr<float>();
  p.sin = n.sin.data_ptr<float>();
  n.q = aligned(q);
  n.k = aligned(k);
  p.q = n.q.data_ptr();
  p.k = n.k.data_ptr();
  p.q_b = o ? row_stride(n.q, 0) : 0; p.q_s = row_stride(n.q, o); p.q_h = row_stride(n.q, o + 1);
  p.k_b = o ? row_stride(n.k, 0) : 0; p.k_s = row_stride(n.k, o); p.k_h = row_stride(n.k, o + 1);
}

std::tuple<Tensor, Tensor> norm_forward(const Tensor& q, const Tensor& k, const OptTensor& qw, const OptTensor& kw,
                                        const Tensor& cos, const Tensor& sin, const OptTensor& positions, double eps,
                                        const std::string& pairs) {
  Norm n;
  norm_params(n, q, k, qw, kw, cos, sin, positions, eps, pairs);
  Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
  if (q.numel()) {
    On dev(q);
    n.p.q_out = qo.data_ptr();
    n.p.k_out = ko.data_ptr();
    check_rc(lbfq_qk_norm_rope(&n.p, stream(q)), "lbfq_qk_norm_rope");
  }
  return {qo, ko};
}

// Of the outputs of norm_forward(the same arguments); want_qw / want_kw: the weights' gradients too
std::tuple<Tensor, Tensor, OptTensor, OptTensor> norm_backward(const Tensor& q, const Tensor& k, const OptTensor& qw,
                                                               const OptTensor& kw, const Tensor& cos, const Tensor& sin,
                                                               const OptTensor& positions, double eps,
                                                               const std::string& pairs, const Tensor& dyq_,
                                                               const Tensor& dyk_, bool want_qw, bool want_kw) {
  Norm n;
  norm_params(n, q, k, qw, kw, cos, sin, positions, eps, pairs);
  Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
  OptTensor dqw, dkw;
  const bool empty = q.numel() == 0;
  if (want_qw && qw) dqw = empty ? at::zeros(qw->sizes(), qw->options()) : at::empty(qw->sizes(), qw->options());
  if (want_kw && kw) dkw = empty ? at::zeros(kw->sizes(), kw->options()) : at::empty(kw->sizes(), kw->options());
  if (!empty) {
    if (dyq_.sizes() != q.sizes() || dyk_.sizes() != k.sizes() || dyq_.scalar_type() != q.scalar_type() ||
        dyk_.scalar_type() != k.scalar_type() || !on(dyq_, q.get_device()) || !on(dyk_, q.get_device()))
      bad_value("gradients must have the outputs' shapes, dtype and device");
    On dev(q);
    const Tensor dyq = aligned(dyq_), dyk = aligned(dyk_);
    const int64_t o = q.dim() - 3;
    lbfq_qk_norm_grads g{};
    g.dyq = dyq.data_ptr();
    g.dyk = dyk.data_ptr();
    g.dyq_b = o ? row_stride(dyq, 0) : 0; g.dyq_s = row_stride(dyq, o); g.dyq_h = row_stride(dyq, o + 1);
    g.dyk_b = o ? row_stride(dyk, 0) : 0; g.dyk_s = row_stride(dyk, o); g.dyk_h = row_stride(dyk, o + 1);
    g.dq = dq.data_ptr();
    g.dk = dk.data_ptr();
    Tensor partial;
    if (dqw || dkw) {
      partial = at::empty({lbfq_qk_norm_rope_bwd_rows(&n.p) * 2 * n.p.D}, q.options().dtype(at::kFloat));
      g.partial = partial.data_ptr<float>();
      g.dq_weight = dqw ? dqw->data_ptr() : nullptr;
      g.dk_weight = dkw ? dkw->data_ptr() : nullptr;
    }
    check_rc(lbfq_qk_norm_rope_bwd(&n.p, &g, stream(q)), "lbfq_qk_norm_rope_bwd");
  }
  return {dq, dk, dqw, dkw};
}

// The two as one differentiable operator.  (As a torch.autograd.Function in Python a training step on a few tokens took
// 100 us, as this 79; a node that only makes its four outputs takes 61.5.)
struct NormFunction : torch::autograd::Function<NormFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const OptTensor& qw,
                               const OptTensor& kw, const Tensor& cos, const Tensor& sin, const OptTensor& positions,
                               double eps, const std::string& pairs) {
    ctx->save_for_backward({q, k, qw.value_or(Tensor()), kw.value_or(Tensor()), cos, sin, positions.value_or(Tensor())});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["pairs"] = pairs;
    const auto [yq, yk] = norm_forward(q, k, qw, kw, cos, sin, positions, eps, pairs);
    return {yq, yk};
  }

  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const py::gil_scoped_acquire gil;  // (the engine's threads come without it; stream() and errors need it)
    const variable_list x = ctx->get_saved_variables();
    const auto given = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    const OptTensor qw = given(x[2]), kw = given(x[3]);
    // (an input that was not given has no edge)
    const bool want_qw = qw && ctx->needs_input_grad(2), want_kw = kw && ctx->needs_input_grad(qw ? 3 : 2);
    const bool again = at::GradMode::is_enabled();
    variable_list g;
    {
      const at::AutoGradMode off(false);
      auto [dq, dk, dqw, dkw] = norm_backward(x[0], x[1], qw, kw, x[4], x[5], given(x[6]), ctx->saved_data["eps"].toDouble(),
                                              ctx->saved_data["pairs"].toStringRef(), dy[0], dy[1], want_qw, want_kw);
      g = {dq, dk, dqw.value_or(Tensor()), dkw.value_or(Tensor())};
    }
    if (again) {  // create_graph: whoever differentiates these is told
      for (Tensor& t : g)
        if (t.defined()) t = t.detach().set_requires_grad(true);
      g = torch::autograd::DelayedError("qk_norm_rope has no second derivative", 4)(std::move(g));
    }
    g.resize(9);
    return g;
  }
};

std::tuple<Tensor, Tensor> norm(const Tensor& q, const Tensor& k, const OptTensor& qw, const OptTensor& kw, const Tensor& cos,
                                const Tensor& sin, const OptTensor& positions, double eps, const std::string& pairs) {
  const Tensor none;
  refuse_tangent("qk_norm_rope", {&q, &k, qw ? &*qw : &none, kw ? &*kw : &none, &cos, &sin});
  if (at::GradMode::is_enabled()) {
    if (cos.requires_grad() || sin.requires_grad())
      bad_value("qk_norm_rope has no gradient for cos and sin; detach them");
    if (q.requires_grad() || k.requires_grad() || (qw && qw->requires_grad()) || (kw && kw->requires_grad())) {
      const variable_list y = NormFunction::apply(q, k, qw, kw, cos, sin, positions, eps, pairs);
      return {y[0], y[1]};
    }
  }
  return norm_forward(q, k, qw, kw, cos, sin, positions, eps, pairs);
}

// A tensor was written in place: autograd is to know
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// First byte of a tensor and the one behind its last.
std::pair<int64_t, int64_t> extent(const Tensor& t) {
  const int64_t at = reinterpret_cast<int64_t>(t.data_ptr());
  int64_t n = 1;
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (t.size(i) == 0) return {at, at};
    n += (t.size(i) - 1) * t.stride(i);
  }
  return {at, at + n * static_cast<int64_t>(t.element_size())};
}

// Whether, for some |i| < n0 and |j| < n1, i s0 + j s1 lies in (lo, hi): rows that are so far apart
bool reached(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t lo, int64_t hi, bool both_ways) {
  if (n0 < n1) std::swap(n0, n1), std::swap(s0, s1);
  for (int64_t j = both_ways ? 1 - n1 : 0; j < n1; ++j) {
    const int64_t from = both_ways ? 1 - n0 : 0, a = lo - j * s1, b = hi - j * s1;
    if (s0 == 0) {
      if (a < 0 && b > 0) return true;
      continue;
    }
    int64_t i = a >= 0 ? a / s0 + 1 : 1 - (s0 - 1 - a) / s0;  // the least with i s0 > a
    if (i < from) i = from;
    if (i < n0 && i * s0 < b) return true;
  }
  return false;
}

// Whether a row of t (n0, n1, d) touches the bytes from x.first up to x.second.
bool rows_touch(const Tensor& t, std::pair<int64_t, int64_t> x) {
  const auto own = extent(t);
  if (x.first == x.second || own.first >= x.second || x.first >= own.second) return false;
  const int64_t e = static_cast<int64_t>(t.element_size());
  return reached(t.size(0), row_stride(t, 0) * e, t.size(1), row_stride(t, 1) * e, x.first - own.first - t.size(2) * e,
                 x.second - own.first, false);
}

// Whether out, whose rows are written while other rows of q are still to be read, may change those: it shares memory
// with q, but not row by row (each is read before it is written).
bool changes_queries(const Tensor& out, const Tensor& q) {
  if (!rows_touch(out, extent(q))) return false;
  for (int64_t i = 0; i < 2; ++i)
    if (row_stride(out, i) != row_stride(q, i)) return true;
  const int64_t e = static_cast<int64_t>(q.element_size()), row = q.size(2) * e;
  const int64_t apart = extent(out).first - extent(q).first;
  return apart != 0 && reached(q.size(0), row_stride(q, 0) * e, q.size(1), row_stride(q, 1) * e, apart - row, apart + row, true);
}

// ---- the cache ---------------------------------------------------------------------

struct Cache {
  const Tensor &kc, &ks, &vc, &vs;
  int64_t pages, heads, page, d, index;
  int shift;

  Cache(const Tensor& kc_, const Tensor& ks_, const Tensor& vc_, const Tensor& vs_) : kc(kc_), ks(ks_), vc(vc_), vs(vs_) {
    if (kc.dim() != 4) bad_value("cache codes must be (pages, H, page size, D); got " + str(kc));
    pages = kc.size(0); heads = kc.size(1); page = kc.size(2); d = kc.size(3);
    if (d != 64 && d != 128) bad_value("cache D must be 64 or 128; got " + std::to_string(d));
    if (page < 16 || page > 1024 || (page & (page - 1)))
      bad_value("cache page size must be a power of two from 16 to 1024; got " + std::to_string(page));
    const int64_t sshape[4] = {pages, heads, page, d / 32};
    const at::IntArrayRef want(sshape, 4);
    if (vc.sizes() != kc.sizes() || ks.sizes() != want || vs.sizes() != want)
      bad_value("cache tensors must be codes " + str(kc) + " and scales " + str(want) + "; got " + str(vc) + ", " + str(ks) +
                " and " + str(vs));
    if (kc.scalar_type() != at::kFloat8_e4m3fn || vc.scalar_type() != at::kFloat8_e4m3fn || ks.scalar_type() != at::kByte ||
        vs.scalar_type() != at::kByte)
      bad_type("cache codes must be float8_e4m3fn and scales uint8; got " + name(kc.scalar_type()) + ", " +
               name(vc.scalar_type()) + ", " + name(ks.scalar_type()) + " and " + name(vs.scalar_type()));
    if (!kc.is_cuda() || !on(ks, kc.get_device()) || !on(vc, kc.get_device()) || !on(vs, kc.get_device()))
      bad_value("cache tensors must live on one CUDA device");
    if (!kc.is_contiguous() || !ks.is_contiguous() || !vc.is_contiguous() || !vs.is_contiguous())
      bad_value("cache tensors must be contiguous");
    if (pages == 0 || heads == 0) bad_value("the cache is empty: " + str(kc));
    index = kc.get_device();
    shift = __builtin_ctzll(static_cast<unsigned long long>(page));
  }

  void refuse_derivatives(const char* what) const {
    if (at::GradMode::is_enabled() && (kc.requires_grad() || vc.requires_grad())) refuse_grad(what);
    refuse_tangent(what, {&kc, &vc});
  }

  template <class P>
  void set(P& p) const {
    p.k_codes = static_cast<uint8_t*>(kc.data_ptr());
    p.k_scale = static_cast<uint8_t*>(ks.data_ptr());
    p.v_codes = static_cast<uint8_t*>(vc.data_ptr());
    p.v_scale = static_cast<uint8_t*>(vs.data_ptr());
    p.num_pages = pages;
    p.page_shift = shift;
  }
};

Tensor index_tensor(const Tensor& t, const char* what, int64_t n, int64_t index, at::ScalarType type) {
  if (t.scalar_type() != type) bad_type(std::string(what) + " must be " + name(type) + "; got " + name(t.scalar_type()));
  if (t.dim() != 1 || t.size(0) != n)
    bad_value(std::string(what) + " must have shape (" + std::to_string(n) + ",); got " + str(t));
  if (!on(t, index)) bad_value(std::string(what) + " must live on " + cuda(index) + "; got " + t.device().str());
  return t.contiguous();
}

Tensor table_tensor(const Tensor& t, int64_t index) {
  if (t.dim() != 2 || t.scalar_type() != at::kInt)
    bad_type("block_table must be (B, pages) int32; got " + str(t) + " " + name(t.scalar_type()));
  if (!on(t, index)) bad_value("block_table must live on the cache's " + cuda(index) + "; got " + t.device().str());
  return t.stride(1) == 1 ? t : t.contiguous();
}

void kv_write(const Tensor& k_, const Tensor& v_, const Tensor& kc, const Tensor& ks, const Tensor& vc, const Tensor& vs,
           const Tensor& slots_) {
  const Cache c(kc, ks, vc, vs);
  if (k_.dim() != 3 || k_.size(1) != c.heads || k_.size(2) != c.d || v_.sizes() != k_.sizes())
    bad_value("k and v must be (T, " + std::to_string(c.heads) + ", " + std::to_string(c.d) + "); got " + str(k_) + " and " +
              str(v_));
  if (!on(k_, c.index) || !on(v_, c.index))
    bad_value("k and v must live on the cache's " + cuda(c.index) + "; got " + k_.device().str() + " and " +
              v_.device().str());
  if (v_.scalar_type() != k_.scalar_type())
    bad_type("k and v must have one dtype; got " + name(k_.scalar_type()) + " and " + name(v_.scalar_type()));
  lbfq_kv_write_params p{};
  p.dtype = dtype_code(k_.scalar_type());
  const Tensor slots = index_tensor(slots_, "slots", k_.size(0), c.index, at::kLong);
  if (at::GradMode::is_enabled() && (k_.requires_grad() || v_.requires_grad())) refuse_grad("write_kv_cache");
  c.refuse_derivatives("write_kv_cache");
  refuse_tangent("write_kv_cache", {&k_, &v_});
  if (k_.size(0) == 0) return;
  On dev(k_);
  const Tensor k = aligned(k_), v = aligned(v_);
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.T = k.size(0); p.H = c.heads; p.D = c.d;
  p.k_t = row_stride(k, 0); p.k_h = row_stride(k, 1);
  p.v_t = row_stride(v, 0); p.v_h = row_stride(v, 1);
  p.slots = slots.data_ptr<int64_t>();
  c.set(p);
  check_rc(lbfq_kv_write(&p, stream(k)), "lbfq_kv_write");
  for (const Tensor* t : {&kc, &ks, &vc, &vs}) written(*t);
}

std::tuple<Tensor, Tensor> kv_read(const Tensor& kc, const Tensor& ks, const Tensor& vc, const Tensor& vs,
                                const Tensor& block_table, const Tensor& seq_lens, int64_t max_len, at::ScalarType dtype) {
  const Cache c(kc, ks, vc, vs);
  const Tensor table = table_tensor(block_table, c.index);
  const int64_t b = table.size(0);
  const Tensor lens = index_tensor(seq_lens, "seq_lens", b, c.index, at::kInt);
  lbfq_kv_read_params p{};
  p.dtype = dtype_code(dtype);
  c.refuse_derivatives("read_kv_cache");
  if (max_len < 0) bad_value("max_len must not be negative; got " + std::to_string(max_len));
  Tensor k = at::empty({b, max_len, c.heads, c.d}, kc.options().dtype(dtype)), v = at::empty_like(k);
  if (b && max_len) {
    On dev(k);
    c.set(p);
    p.B = b; p.H = c.heads; p.D = c.d; p.max_len = max_len;
    p.block_table = table.data_ptr<int32_t>();
    p.table_stride = table.stride(0);
    p.table_cols = table.size(1);
    p.seq_lens = lens.data_ptr<int32_t>();
    p.k_out = k.data_ptr();
    p.v_out = v.data_ptr();
    check_rc(lbfq_kv_read(&p, stream(k)), "lbfq_kv_read");
  }
  return {k, v};
}

std::tuple<Tensor, OptTensor> attention(const Tensor& q_, const Tensor& kc, const Tensor& ks, const Tensor& vc,
                                        const Tensor& vs, const Tensor& block_table, const Tensor& seq_lens,
                                        const Tensor& query_starts, std::optional<int64_t> max_query_len,
                                        std::optional<double> sm_scale, bool causal, std::optional<int64_t> window,
                                        const OptTensor& out_, bool return_lse) {
  const Cache c(kc, ks, vc, vs);
  if (q_.dim() != 3 || q_.size(2) != c.d) bad_value("q must be (T, Hq, " + std::to_string(c.d) + "); got " + str(q_));
  if (!on(q_, c.index)) bad_value("q must live on the cache's " + cuda(c.index) + "; got " + q_.device().str());
  if (q_.scalar_type() != at::kBFloat16 && q_.scalar_type() != at::kHalf)
    bad_type("q must be bfloat16 or float16; got " + name(q_.scalar_type()));
  const int64_t t = q_.size(0), hq = q_.size(1);
  if (hq == 0 || hq % c.heads)
    bad_value("the query heads (" + std::to_string(hq) + ") must be a multiple of the cache's (" + std::to_string(c.heads) +
              ")");
  const Tensor table = table_tensor(block_table, c.index);
  const int64_t b = table.size(0);
  if (table.size(1) == 0) bad_value("block_table has no columns");
  const Tensor lens = index_tensor(seq_lens, "seq_lens", b, c.index, at::kInt);
  const Tensor starts = index_tensor(query_starts, "query_starts", b + 1, c.index, at::kInt);
  const double scale = sm_scale ? *sm_scale : 1.0 / std::sqrt(static_cast<double>(c.d));
  if (!(scale >= 0x1p-64 && scale <= 0x1p15))
    bad_value("sm_scale must lie in 2^-64 ... 2^15; got " + std::to_string(scale));
  if (window && *window <= 0) bad_value("window must be positive; got " + std::to_string(*window));
  if (max_query_len && *max_query_len < 0)
    bad_value("max_query_len must not be negative; got " + std::to_string(*max_query_len));
  if (at::GradMode::is_enabled() && q_.requires_grad()) refuse_grad("paged_attention");
  refuse_tangent("paged_attention", {&q_});
  c.refuse_derivatives("paged_attention");
  if (out_) {
    if (out_->sizes() != q_.sizes() || out_->scalar_type() != q_.scalar_type() || !on(*out_, c.index))
      bad_value("out must be " + str(q_) + " " + name(q_.scalar_type()) + " on " + cuda(c.index) + "; got " + str(*out_) +
                " " + name(out_->scalar_type()) + " on " + out_->device().str());
    if (!rows_16b(*out_) || !rows_apart(*out_))
      bad_value("out must have contiguous, distinct rows that start on 16-byte boundaries");
    if (at::GradMode::is_enabled() && out_->requires_grad()) refuse_grad("paged_attention");
    refuse_tangent("paged_attention", {&*out_});
  }
  On dev(q_);
  const Tensor out = out_ ? *out_ : at::empty(q_.sizes(), q_.options());
  OptTensor lse;
  if (return_lse) lse = at::empty({t, hq}, q_.options().dtype(at::kFloat));
  if (b == 0 || t == 0) {
    if (!out_) out.zero_();
    if (lse) lse->fill_(-std::numeric_limits<float>::infinity());
    return {out, lse};
  }
  if (out_) {
    for (const Tensor* x : {&c.kc, &c.ks, &c.vc, &c.vs, &table, &lens, &starts})
      if (rows_touch(out, extent(*x))) bad_value("out must not share memory with the cache, block_table, seq_lens or query_starts");
  }
  const Tensor q = out_ && changes_queries(out, q_) ? q_.clone(at::MemoryFormat::Contiguous) : aligned(q_);
  lbfq_paged_params p{};
  p.q = q.data_ptr();
  p.dtype = dtype_code(q.scalar_type());
  p.T = t; p.Hq = hq; p.Hk = c.heads; p.D = c.d; p.B = b;
  p.q_t = row_stride(q, 0); p.q_h = row_stride(q, 1);
  c.set(p);
  p.block_table = table.data_ptr<int32_t>();
  p.table_stride = table.stride(0);
  p.table_cols = table.size(1);
  p.seq_lens = lens.data_ptr<int32_t>();
  p.query_starts = starts.data_ptr<int32_t>();
  p.max_query_len = max_query_len ? *max_query_len : 0;
  p.sm_scale = static_cast<float>(scale);
  p.causal = causal;
  p.window = window ? std::min<int64_t>(*window, int64_t{1} << 30) : 0;
  p.out = out.data_ptr();
  p.out_t = row_stride(out, 0); p.out_h = row_stride(out, 1);
  p.lse = lse ? lse->data_ptr<float>() : nullptr;
  p.fill_rest = !out_;
  Tensor ws;  // of this call alone: torch's allocator keeps it until the launches are done
  if (const int64_t need = lbfq_paged_attention_workspace_bytes(&p)) {
    ws = at::empty({need}, q.options().dtype(at::kByte));
    p.workspace = ws.data_ptr();
    p.workspace_bytes = need;
  }
  check_rc(lbfq_paged_attention(&p, stream(q)), "lbfq_paged_attention");
  if (out_) written(out);
  return {out, lse};
}

}  // namespace

PYBIND11_MODULE(_lbfq_torch, m) {
  // (of pybind's own it would be a plain RuntimeError)
  py::register_local_exception_translator([](std::exception_ptr e) {
    try {
      if (e) std::rethrow_exception(e);
    } catch (const c10::OutOfMemoryError& x) {
      PyErr_SetString(py::module_::import("torch").attr("OutOfMemoryError").ptr(), x.what_without_backtrace());
    }
  });
  m.def("set_hooks", [](py::object stream, py::object error) {
    stream_of = new py::object(std::move(stream));
    library_error = new py::object(std::move(error));
  });
  m.def("qk_norm_rope", &norm);
  m.def("write_kv_cache", &kv_write);
  m.def("read_kv_cache", &kv_read);
  m.def("paged_attention", &attention);
}

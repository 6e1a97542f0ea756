// Further C++ torch operators over the C ABI (include/bcfft.h), in torch.ops.bcfft_native: the dense
// projections and top-logit distillation with their autograd nodes. What bcfft/dense.py and bcfft/distill.py
// do through ctypes and Python autograd Functions (170 us of host time for a forward and backward), in one
// dispatcher call and a C++ node each (27-95 us by operator and host). Same checks, errors and semantics as the Python path, which stays as
// the fallback when this library is not built. Host code only: the kernels are libbcfft.so's.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <cmath>
#include <cstdint>
#include <optional>
#include <string>
#include <tuple>

#include "bcfft.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return BCFFT_F32;
    case at::kHalf: return BCFFT_F16;
    case at::kBFloat16: return BCFFT_BF16;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t, "; BC engine supports float32/float16/bfloat16");
  }
  return BCFFT_NONE;
}
void check_status(int st, const char* what) {
  if (st == BCFFT_OK) return;
  std::string msg = std::string(what) + " failed: " + bcfft_status_string(st);
  if (st == BCFFT_ERR_HIP) msg += std::string(" (") + bcfft_last_hip_error() + ")";
  TORCH_CHECK(false, msg);
}
void require_device(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), what, ": the MI355X BC engine runs on ROCm device tensors only (got ", t.device(),
              "); move the module and inputs to the GPU. There is no CPU path in the product.");
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
const void* ptr(const OptTensor& t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool given(const OptTensor& t) { return t.has_value() && t->defined(); }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t.has_value() && wants_grad(*t); }
int64_t row_stride(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }
Tensor aligned16(const Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 ? t.clone(at::MemoryFormat::Contiguous) : t;
}
// FakeTensors, functionalised tensors and other subclasses have no memory to read here, and a trace would not hold
// the launches of a C++ autograd node: their shapes come from the Meta kernels, below autograd
bool traced(const Tensor& t) { return t.defined() && t.unsafeGetTensorImpl()->key_set().has(c10::DispatchKey::Python); }
bool traced(const OptTensor& t) { return t.has_value() && traced(*t); }
template <class... T>
void require_memory(const char* what, const T&... operands) {
  using c10::impl::TorchDispatchModeKey, c10::impl::TorchDispatchModeTLS;
  const bool mode = TorchDispatchModeTLS::any_modes_set() &&
                    (TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY) ||
                     TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE) ||
                     TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FUNCTIONAL));
  TORCH_CHECK(!(mode || (traced(operands) || ...)), what,
              ": records no gradient of a traced tensor (FakeTensor, torch.compile, make_fx, a subclass); run this call "
              "eagerly, e.g. under torch.compiler.disable");
}
// forward mode: below autograd a tangent would be dropped, and its absence read as a zero derivative
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }
template <class... T>
void refuse_forward_mode(const char* what, const T&... operands) {
  TORCH_CHECK(!(has_tangent(operands) || ...), what, ": no forward-mode derivatives (an operand is a dual tensor)");
}
// Where the backward itself is recorded (create_graph), a second differentiation raises instead of missing terms,
// whether or not the incoming gradient needs one: dx depends on w. What passes the incoming gradient on is left as it is.
variable_list first_order(variable_list out, const Tensor& upstream) {
  if (!at::GradMode::is_enabled()) return out;
  auto fail = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function whose backward is not differentiable", (int64_t)out.size());
  variable_list marked(out);
  for (Tensor& t : marked)
    if (t.defined()) t = t.detach().requires_grad_(true);
  marked = (*fail)(std::move(marked));
  for (size_t i = 0; i < out.size(); ++i)
    if (out[i].defined() && out[i].is_same(upstream)) marked[i] = out[i];
  return marked;
}

// ------------------------------------------------------------------ dense projections
constexpr int64_t MAX_FEATURES = 1 << 20, MAX_TOKENS = 1 << 23;

// (..., K) -> (N, K): adjacent elements, a 16-byte aligned start, rows on 16 bytes where K fills them
Tensor dense_rows(const Tensor& t) {
  const int64_t k = t.size(-1);
  Tensor x = t.dim() == 2 ? t : t.reshape({t.numel() / k, k});
  const int64_t e = x.element_size();
  const bool strided = x.size(0) > 1 && (x.stride(0) < k || x.stride(0) > MAX_FEATURES ||
                                         (x.stride(0) * e % 16 != 0 && k * e % 16 == 0));
  if (strided || (k > 1 && x.stride(1) != 1)) x = x.contiguous();
  return aligned16(x);
}
Tensor dense_weight(const Tensor& w) { return aligned16(w.contiguous()); }

void check_operand(const Tensor& x, const Tensor& t, const char* what, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), what, ": ", name, " is ", t.scalar_type(), " but x is ",
                   x.scalar_type(), "; all operands share one dtype");
  TORCH_CHECK_VALUE(t.device() == x.device(), what, ": ", name, " is on ", t.device(), " but x is on ", x.device(),
                    "; move it to x's device");
}
void check_weight(const Tensor& x, const Tensor& w, const Tensor& first, const char* what, const char* name) {
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) == x.size(-1) && w.sizes() == first.sizes(), what, ": ", name, " ",
                    w.sizes(), " must be (out_features, in_features = ", x.size(-1), ")");
}
void check_dense(const Tensor& x, const Tensor& w, int64_t act, const char* what) {
  const int64_t k = x.size(-1), m = w.size(0);
  TORCH_CHECK_VALUE(k >= 1 && k <= MAX_FEATURES && m >= 1 && m <= MAX_FEATURES, what, ": features (", k, ", ", m,
                    ") must lie in [1, ", MAX_FEATURES, "]");
  TORCH_CHECK_VALUE(x.numel() / k <= MAX_TOKENS, what, ": ", x.numel() / k, " rows, at most ", MAX_TOKENS);
  TORCH_CHECK_VALUE(act >= 0 && act <= BCFFT_ACT_GELU, what, ": activation code ", act);
}
void check_x(const Tensor& x, const char* what) {
  require_device(x, what);
  dtype_code(x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1, what, ": x must be (..., in_features), got a scalar");
}
std::vector<int64_t> with_last(at::IntArrayRef lead, int64_t last) {
  std::vector<int64_t> s(lead.begin(), lead.end());
  s.push_back(last);
  return s;
}
Tensor dense_workspace(int op, int64_t n, int64_t k, int64_t m, const Tensor& x, int64_t act, int64_t& bytes) {
  bytes = bcfft_dense_workspace_bytes(op, n, k, m, dtype_code(x.scalar_type()), (int)act);
  TORCH_CHECK_VALUE(bytes >= 0, "bcfft.dense: sizes (", n, ", ", k, ", ", m, ") are not served");
  return bytes ? at::empty({bytes}, x.options().dtype(at::kByte)) : Tensor();
}

constexpr const char* LINEAR = "bcfft.dense.linear";
std::tuple<Tensor, Tensor> linear_run(const Tensor& x, const Tensor& weight, const OptTensor& bias,
                                      const OptTensor& residual, int64_t act, bool keep) {
  check_x(x, LINEAR);
  check_weight(x, weight, weight, LINEAR, "weight");
  check_dense(x, weight, act, LINEAR);
  const int64_t m = weight.size(0);
  const std::vector<int64_t> shape = with_last(x.sizes().slice(0, x.dim() - 1), m);
  if (given(bias)) TORCH_CHECK_VALUE(bias->sizes() == at::IntArrayRef({m}), LINEAR, ": bias ", bias->sizes(), " must be [", m, "]");
  if (given(residual))
    TORCH_CHECK_VALUE(residual->sizes() == at::IntArrayRef(shape), LINEAR, ": residual ", residual->sizes(), " must be ", at::IntArrayRef(shape));
  check_operand(x, weight, LINEAR, "weight");
  if (given(bias)) check_operand(x, *bias, LINEAR, "bias");
  if (given(residual)) check_operand(x, *residual, LINEAR, "residual");
  const c10::DeviceGuard guard(x.device());
  Tensor y = at::empty(shape, x.options());
  const int64_t k = x.size(-1), n = x.numel() / k;
  Tensor z = keep ? at::empty({n, m}, x.options().dtype(at::kFloat)) : Tensor();
  if (n == 0) return {y, z};
  const Tensor xa = dense_rows(x), wa = dense_weight(weight);
  const Tensor ba = given(bias) ? bias->contiguous() : Tensor(), ra = given(residual) ? dense_rows(*residual) : Tensor();
  int64_t bytes;
  const Tensor ws = dense_workspace(BCFFT_DENSE_LINEAR, n, k, m, x, act, bytes);
  check_status(bcfft_dense_linear(xa.data_ptr(), dtype_code(x.scalar_type()), n, row_stride(xa), k, m, wa.data_ptr(),
                                  ptr(ba), ptr(ra), ra.defined() ? row_stride(ra) : 0, (int)act, y.data_ptr(),
                                  (float*)ptr(z), ptr(ws), bytes, stream_of(x)),
               "bcfft_dense_linear");
  return {y, z};
}

struct LinearFn : torch::autograd::Function<LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias,
                        const OptTensor& residual, int64_t act, bool keep) {
    auto [y, z] = linear_run(x, weight, bias, residual, act, keep);
    ctx->save_for_backward({x, weight, z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = given(bias);
    ctx->saved_data["residual"] = given(residual);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor& dy = grads[0];
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &z = saved[2];
    const int64_t act = ctx->saved_data["act"].toInt();
    const bool has_b = ctx->saved_data["bias"].toBool(), has_r = ctx->saved_data["residual"].toBool();
    const bool need_b = has_b && ctx->needs_input_grad(2), need_r = has_r && ctx->needs_input_grad(has_b ? 3 : 2);
    const int64_t k = x.size(-1), n = x.numel() / k, m = weight.size(0);
    Tensor dx, dw, db;
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(x.device());
      if (ctx->needs_input_grad(0)) dx = at::empty(x.sizes(), x.options());
      if (ctx->needs_input_grad(1)) dw = at::empty({m, k}, x.options());
      if (need_b) db = at::empty({m}, x.options());
      if (n == 0) {
        if (dw.defined()) dw.zero_();
        if (db.defined()) db.zero_();
      } else if (dx.defined() || dw.defined() || db.defined()) {
        const Tensor xa = dense_rows(x), wa = dense_weight(weight), da = dense_rows(dy);
        int64_t bytes;
        const Tensor ws = dense_workspace(BCFFT_DENSE_LINEAR_BACKWARD, n, k, m, x, act, bytes);
        check_status(bcfft_dense_linear_backward(xa.data_ptr(), dtype_code(x.scalar_type()), n, row_stride(xa), k, m,
                                                 wa.data_ptr(), da.data_ptr(), row_stride(da), (const float*)ptr(z),
                                                 (int)act, ptr(dx), ptr(dw), ptr(db), ptr(ws), bytes, stream_of(x)),
                     "bcfft_dense_linear_backward");
      }
    }
    return first_order({dx, dw, db, need_r ? dy : Tensor(), Tensor(), Tensor()}, dy);
  }
};

constexpr const char* GLU = "bcfft.dense.glu";
std::tuple<Tensor, Tensor> glu_run(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, int64_t act, bool keep) {
  check_x(x, GLU);
  check_weight(x, w_gate, w_gate, GLU, "w_gate");
  check_weight(x, w_up, w_gate, GLU, "w_up");
  check_dense(x, w_gate, act, GLU);
  check_operand(x, w_gate, GLU, "w_gate");
  check_operand(x, w_up, GLU, "w_up");
  const int64_t m = w_gate.size(0), k = x.size(-1), n = x.numel() / k;
  TORCH_CHECK_VALUE(2 * m <= MAX_FEATURES, GLU, ": out_features = ", m, ", at most ", MAX_FEATURES / 2);
  const c10::DeviceGuard guard(x.device());
  Tensor h = at::empty(with_last(x.sizes().slice(0, x.dim() - 1), m), x.options());
  Tensor gu = keep ? at::empty({2, n, m}, x.options().dtype(at::kFloat)) : Tensor();
  if (n == 0) return {h, gu};
  const Tensor xa = dense_rows(x), wg = dense_weight(w_gate), wu = dense_weight(w_up);
  int64_t bytes;
  const Tensor ws = dense_workspace(BCFFT_DENSE_GLU, n, k, m, x, act, bytes);
  check_status(bcfft_dense_glu(xa.data_ptr(), dtype_code(x.scalar_type()), n, row_stride(xa), k, m, wg.data_ptr(),
                               wu.data_ptr(), (int)act, h.data_ptr(), (float*)ptr(gu), ptr(ws), bytes, stream_of(x)),
               "bcfft_dense_glu");
  return {h, gu};
}

struct GluFn : torch::autograd::Function<GluFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_gate, const Tensor& w_up, int64_t act) {
    auto [h, gu] = glu_run(x, w_gate, w_up, act, true);
    ctx->save_for_backward({x, w_gate, w_up, gu});
    ctx->saved_data["act"] = act;
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor& dh = grads[0];
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w_gate = saved[1], &w_up = saved[2], &gu = saved[3];
    const int64_t act = ctx->saved_data["act"].toInt();
    const int64_t k = x.size(-1), n = x.numel() / k, m = w_gate.size(0);
    const bool need_g = ctx->needs_input_grad(1), need_u = ctx->needs_input_grad(2);
    Tensor dx, dw;
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(x.device());
      if (ctx->needs_input_grad(0)) dx = at::empty(x.sizes(), x.options());
      if (need_g || need_u) dw = at::empty({2, m, k}, x.options());
      if (n == 0) {
        if (dw.defined()) dw.zero_();
      } else {
        const Tensor xa = dense_rows(x), wg = dense_weight(w_gate), wu = dense_weight(w_up), da = dense_rows(dh);
        int64_t bytes;
        const Tensor ws = dense_workspace(BCFFT_DENSE_GLU_BACKWARD, n, k, m, x, act, bytes);
        check_status(bcfft_dense_glu_backward(xa.data_ptr(), dtype_code(x.scalar_type()), n, row_stride(xa), k, m,
                                              wg.data_ptr(), wu.data_ptr(), da.data_ptr(), row_stride(da),
                                              (const float*)gu.data_ptr(), (int)act, ptr(dx), ptr(dw), ptr(ws), bytes,
                                              stream_of(x)),
                     "bcfft_dense_glu_backward");
      }
    }
    return first_order({dx, need_g ? dw.select(0, 0) : Tensor(), need_u ? dw.select(0, 1) : Tensor(), Tensor()}, dh);
  }
};

// ------------------------------------------------------------------ distillation from top logits
constexpr int64_t MAX_ENTRIES = 1024, MAX_VOCAB = 1 << 18;
constexpr const char *TOPK = "bcfft.distill.topk_logits", *KL = "bcfft.distill.topk_kl", *KL_GRAD = "bcfft.distill.topk_kl_grad";

Tensor logit_rows(const Tensor& logits, const char* what) {
  require_device(logits, what);
  TORCH_CHECK_VALUE(logits.dim() >= 1, what, ": logits must be (..., vocabulary), got a scalar");
  dtype_code(logits.scalar_type());
  const int64_t v = logits.size(-1);
  TORCH_CHECK_VALUE(v > 0, what, ": empty vocabulary");
  Tensor x = logits.dim() == 2 ? logits : logits.reshape({logits.numel() / v, v});
  if ((v > 1 && x.stride(1) != 1) || (x.size(0) > 1 && x.stride(0) < v)) x = x.contiguous();
  return x;
}
void check_temperature(double t, const char* what) {
  TORCH_CHECK_VALUE(std::isfinite(t) && t >= 1e-6 && t <= 1e6, what, ": temperature must lie in [1e-6, 1e6], got ", t);
}

std::tuple<Tensor, Tensor, Tensor> topk_run(const Tensor& logits, int64_t k, double temperature) {
  const char* const what = TOPK;
  const Tensor x = logit_rows(logits, what);
  const int64_t n = x.size(0), v = x.size(1);
  TORCH_CHECK_VALUE(k >= 1 && k <= std::min(v, MAX_ENTRIES), what, ": k = ", k, " must lie in [1, min(vocabulary = ", v,
                    ", ", MAX_ENTRIES, ")]");
  check_temperature(temperature, what);
  const c10::DeviceGuard guard(x.device());
  const at::IntArrayRef lead = logits.sizes().slice(0, logits.dim() - 1);
  Tensor values = at::empty(with_last(lead, k), x.options()), indices = at::empty(with_last(lead, k), x.options().dtype(at::kInt));
  Tensor rest = at::empty(lead, x.options().dtype(at::kFloat));
  check_status(bcfft_topk_logits(ptr(x), dtype_code(x.scalar_type()), n, v, row_stride(x), (int)k, temperature, ptr(values),
                                 (int32_t*)ptr(indices), (float*)ptr(rest), stream_of(x)),
               "bcfft_topk_logits");
  return {values, indices, rest};
}

struct KlOperands {
  Tensor x, values, indices, rest, weight;
  int64_t n, v, k;
  double t;
};
KlOperands kl_operands(const Tensor& logits, const Tensor& values, const Tensor& indices, const OptTensor& rest,
                       const OptTensor& weight, double temperature, const char* what) {
  KlOperands o;
  o.x = logit_rows(logits, what);
  o.n = o.x.size(0);
  o.v = o.x.size(1);
  check_temperature(temperature, what);
  o.t = temperature;
  TORCH_CHECK_VALUE(o.v <= MAX_VOCAB, what, ": vocabulary of ", o.v, ", at most ", MAX_VOCAB);
  const at::IntArrayRef lead = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK_VALUE(values.sizes() == indices.sizes() && values.dim() >= 1 &&
                        values.sizes().slice(0, values.dim() - 1) == lead,
                    what, ": values ", values.sizes(), " and indices ", indices.sizes(), " must both be ", lead, " + (k,)");
  o.k = values.size(-1);
  TORCH_CHECK_VALUE(o.k >= 1 && o.k <= MAX_ENTRIES, what, ": k = ", o.k, " entries per row, must lie in [1, ", MAX_ENTRIES, "]");
  dtype_code(values.scalar_type());
  TORCH_CHECK_TYPE(indices.scalar_type() == at::kInt || indices.scalar_type() == at::kLong, what,
                   ": indices must be int32 or int64, got ", indices.scalar_type());
  auto constant = [&](const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.device() == logits.device(), what, ": ", name, " is on ", t.device(), " but logits is on ", logits.device());
    TORCH_CHECK_VALUE(!t.requires_grad(), what, ": ", name,
                      " requires grad, but the teacher's side and the weights are constants here: detach it");
  };
  auto per_row = [&](const OptTensor& t, const char* name) {
    if (!given(t)) return Tensor();
    TORCH_CHECK_VALUE(t->sizes() == lead && t->is_floating_point(), what, ": ", name, " must be floating point of shape ",
                      lead, ", got ", t->scalar_type(), " ", t->sizes());
    constant(*t, name);
    return t->reshape({o.n}).to(at::kFloat).contiguous();
  };
  o.rest = per_row(rest, "rest");
  o.weight = per_row(weight, "weight");
  constant(values, "values");
  constant(indices, "indices");
  o.values = values.reshape({o.n, o.k}).contiguous();
  o.indices = indices.reshape({o.n, o.k}).contiguous();
  return o;
}
std::tuple<Tensor, Tensor, Tensor> kl_run(const Tensor& logits, const KlOperands& o, bool stats, bool grad) {
  const c10::DeviceGuard guard(o.x.device());
  const at::IntArrayRef lead = logits.sizes().slice(0, logits.dim() - 1);
  Tensor loss = at::empty(lead, o.x.options().dtype(at::kFloat));
  Tensor st = stats ? at::empty({o.n, 4}, o.x.options().dtype(at::kFloat)) : Tensor();
  Tensor g = grad ? at::empty(logits.sizes(), o.x.options()) : Tensor();
  check_status(bcfft_distill_topk(ptr(o.x), dtype_code(o.x.scalar_type()), o.n, o.v, row_stride(o.x), ptr(o.values),
                                  dtype_code(o.values.scalar_type()), ptr(o.indices), (int)o.indices.element_size(), (int)o.k,
                                  (const float*)ptr(o.rest), (const float*)ptr(o.weight), o.t, (float*)ptr(loss),
                                  (float*)ptr(st), ptr(g), stream_of(o.x)),
               "bcfft_distill_topk");
  return {loss, st, g};
}

struct TopKKlFn : torch::autograd::Function<TopKKlFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& values, const Tensor& indices,
                        const OptTensor& rest, const OptTensor& weight, double temperature) {
    const KlOperands o = kl_operands(logits, values, indices, rest, weight, temperature, KL);
    auto [loss, stats, grad] = kl_run(logits, o, true, false);
    ctx->save_for_backward({logits, values, indices, given(rest) ? *rest : Tensor(), given(weight) ? *weight : Tensor(), stats});
    ctx->saved_data["temperature"] = temperature;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    Tensor g;
    {
      const at::NoGradGuard no_grad;
      const KlOperands o = kl_operands(s[0], s[1], s[2], s[3].defined() ? OptTensor(s[3]) : std::nullopt,
                                       s[4].defined() ? OptTensor(s[4]) : std::nullopt,
                                       ctx->saved_data["temperature"].toDouble(), KL);
      const c10::DeviceGuard guard(o.x.device());
      g = at::empty(s[0].sizes(), o.x.options());
      const Tensor up = grads[0].reshape({o.n}).to(at::kFloat).contiguous();
      check_status(bcfft_distill_topk_backward(ptr(o.x), dtype_code(o.x.scalar_type()), o.n, o.v, row_stride(o.x),
                                               ptr(o.values), dtype_code(o.values.scalar_type()), ptr(o.indices),
                                               (int)o.indices.element_size(), (int)o.k, (const float*)ptr(o.rest),
                                               (const float*)ptr(o.weight), o.t, (const float*)ptr(s[5]), (const float*)ptr(up),
                                               ptr(g), stream_of(o.x)),
                   "bcfft_distill_topk_backward");
    }
    return first_order({g, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, grads[0]);
  }
};

// ------------------------------------------------------------------ registered kernels
Tensor dense_linear_hip(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, int64_t act) {
  return std::get<0>(linear_run(x, weight, bias, residual, act, false));
}
Tensor dense_glu_hip(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, int64_t act) {
  return std::get<0>(glu_run(x, w_gate, w_up, act, false));
}
Tensor topk_kl_hip(const Tensor& logits, const Tensor& values, const Tensor& indices, const OptTensor& rest,
                   const OptTensor& weight, double temperature) {
  return std::get<0>(kl_run(logits, kl_operands(logits, values, indices, rest, weight, temperature, KL), false, false));
}
std::tuple<Tensor, Tensor> topk_kl_grad_hip(const Tensor& logits, const Tensor& values, const Tensor& indices,
                                            const OptTensor& rest, const OptTensor& weight, double temperature) {
  auto [loss, stats, grad] = kl_run(logits, kl_operands(logits, values, indices, rest, weight, temperature, KL_GRAD), false, true);
  return {loss, grad};
}

// Meta: shapes and dtypes
Tensor dense_linear_meta(const Tensor& x, const Tensor& weight, const OptTensor&, const OptTensor&, int64_t) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && weight.size(1) == x.size(-1), LINEAR, ": weight ", weight.sizes(),
                    " must be (out_features, in_features)");
  return at::empty(with_last(x.sizes().slice(0, x.dim() - 1), weight.size(0)), x.options());
}
Tensor dense_glu_meta(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, int64_t) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && w_gate.dim() == 2 && w_gate.size(1) == x.size(-1) && w_up.sizes() == w_gate.sizes(), GLU,
                    ": w_gate ", w_gate.sizes(), " and w_up ", w_up.sizes(), " must be (out_features, in_features)");
  return at::empty(with_last(x.sizes().slice(0, x.dim() - 1), w_gate.size(0)), x.options());
}
std::tuple<Tensor, Tensor, Tensor> topk_logits_meta(const Tensor& logits, int64_t k, double) {
  TORCH_CHECK_VALUE(logits.dim() >= 1 && k >= 1 && k <= logits.size(-1), "bcfft.distill.topk_logits: k = ", k);
  const at::IntArrayRef lead = logits.sizes().slice(0, logits.dim() - 1);
  return {at::empty(with_last(lead, k), logits.options()), at::empty(with_last(lead, k), logits.options().dtype(at::kInt)),
          at::empty(lead, logits.options().dtype(at::kFloat))};
}
Tensor topk_kl_meta(const Tensor& logits, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, double) {
  return at::empty(logits.sizes().slice(0, logits.dim() - 1), logits.options().dtype(at::kFloat));
}
std::tuple<Tensor, Tensor> topk_kl_grad_meta(const Tensor& logits, const Tensor&, const Tensor&, const OptTensor&,
                                             const OptTensor&, double) {
  return {at::empty(logits.sizes().slice(0, logits.dim() - 1), logits.options().dtype(at::kFloat)), at::empty(logits.sizes(), logits.options())};
}

// Autograd: a node where an operand needs a gradient, else straight to the device's kernel
template <class F>
auto below(const char* name, F) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<std::remove_pointer_t<F>>();
}
Tensor dense_linear_autograd(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, int64_t act) {
  refuse_forward_mode(LINEAR, x, weight, bias, residual);
  if (at::GradMode::is_enabled() && !x.is_meta()) {
    const bool inner = wants_grad(x) || wants_grad(weight) || wants_grad(bias);
    if (inner || wants_grad(residual)) {
      require_memory(LINEAR, x, weight, bias, residual);
      return LinearFn::apply(x, weight, bias, residual, act, inner && act != BCFFT_ACT_NONE);
    }
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = below("bcfft_native::dense_linear", &dense_linear_hip);
  return op.call(x, weight, bias, residual, act);
}
Tensor dense_glu_autograd(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, int64_t act) {
  refuse_forward_mode(GLU, x, w_gate, w_up);
  if (at::GradMode::is_enabled() && !x.is_meta() && (wants_grad(x) || wants_grad(w_gate) || wants_grad(w_up))) {
    require_memory(GLU, x, w_gate, w_up);
    return GluFn::apply(x, w_gate, w_up, act);
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = below("bcfft_native::dense_glu", &dense_glu_hip);
  return op.call(x, w_gate, w_up, act);
}
Tensor topk_kl_autograd(const Tensor& logits, const Tensor& values, const Tensor& indices, const OptTensor& rest,
                        const OptTensor& weight, double temperature) {
  refuse_forward_mode(KL, logits, values, rest, weight);
  if (at::GradMode::is_enabled() && !logits.is_meta() && wants_grad(logits)) {
    require_memory(KL, logits, values, indices, rest, weight);
    return TopKKlFn::apply(logits, values, indices, rest, weight, temperature);
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = below("bcfft_native::topk_kl", &topk_kl_hip);
  return op.call(logits, values, indices, rest, weight, temperature);
}
// no gradient flows through these two: the teacher is a constant, and the second returns its gradient
std::tuple<Tensor, Tensor, Tensor> topk_logits_autograd(const Tensor& logits, int64_t k, double temperature) {
  refuse_forward_mode(TOPK, logits);
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = below("bcfft_native::topk_logits", &topk_run);
  return op.call(logits, k, temperature);
}
std::tuple<Tensor, Tensor> topk_kl_grad_autograd(const Tensor& logits, const Tensor& values, const Tensor& indices,
                                                 const OptTensor& rest, const OptTensor& weight, double temperature) {
  refuse_forward_mode(KL_GRAD, logits, values, rest, weight);
  at::AutoDispatchBelowADInplaceOrView guard;
  static auto op = below("bcfft_native::topk_kl_grad", &topk_kl_grad_hip);
  return op.call(logits, values, indices, rest, weight, temperature);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(bcfft_native, m) {
  m.def("dense_linear(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int act) -> Tensor");
  m.def("dense_glu(Tensor x, Tensor w_gate, Tensor w_up, int act) -> Tensor");
  m.def("topk_logits(Tensor logits, int k, float temperature) -> (Tensor, Tensor, Tensor)");
  m.def("topk_kl(Tensor logits, Tensor values, Tensor indices, Tensor? rest, Tensor? weight, float temperature) -> Tensor");
  m.def("topk_kl_grad(Tensor logits, Tensor values, Tensor indices, Tensor? rest, Tensor? weight, float temperature) "
        "-> (Tensor, Tensor)");
}
// the CPU kernels are the device's: their first check names the missing CPU path
#define BCFFT_DEVICE_KERNELS(m)                 \
  m.impl("dense_linear", &dense_linear_hip);    \
  m.impl("dense_glu", &dense_glu_hip);          \
  m.impl("topk_logits", &topk_run);             \
  m.impl("topk_kl", &topk_kl_hip);              \
  m.impl("topk_kl_grad", &topk_kl_grad_hip);
TORCH_LIBRARY_IMPL(bcfft_native, CUDA, m) { BCFFT_DEVICE_KERNELS(m) }
TORCH_LIBRARY_IMPL(bcfft_native, CPU, m) { BCFFT_DEVICE_KERNELS(m) }
TORCH_LIBRARY_IMPL(bcfft_native, Meta, m) {
  m.impl("dense_linear", &dense_linear_meta);
  m.impl("dense_glu", &dense_glu_meta);
  m.impl("topk_logits", &topk_logits_meta);
  m.impl("topk_kl", &topk_kl_meta);
  m.impl("topk_kl_grad", &topk_kl_grad_meta);
}
TORCH_LIBRARY_IMPL(bcfft_native, Autograd, m) {
  m.impl("dense_linear", &dense_linear_autograd);
  m.impl("dense_glu", &dense_glu_autograd);
  m.impl("topk_logits", &topk_logits_autograd);
  m.impl("topk_kl", &topk_kl_autograd);
  m.impl("topk_kl_grad", &topk_kl_grad_autograd);
}

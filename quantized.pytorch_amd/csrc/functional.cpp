// The host side of qnn/functional.py as a CPython extension (qnn/_float.so): checks of arguments, rows,
// allocations and the autograd nodes of linear_act, layer_norm and topk_distill_loss, over the C entries
// of include/qnn.h (bound at run time to the library that qnn/_lib.py loaded).
//
// In C++ because the calls are short: a training step of a few microseconds of kernels took 130 to
// 150 us of Python on its two threads (the backward pass runs on autograd's own), and about 60 here, of
// which 48 are torch's for a node that does nothing.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <optional>

#include "../../include/qnn.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ------------------------------------------------------------------------------ the C entries
struct Api {
  decltype(&qnn_last_error) last_error;
  decltype(&qnn_linear_act_fwd_work) linear_act_fwd_work;
  decltype(&qnn_linear_act_fwd) linear_act_fwd;
  decltype(&qnn_linear_act_bwd_work) linear_act_bwd_work;
  decltype(&qnn_linear_act_bwd) linear_act_bwd;
  decltype(&qnn_layer_norm_fwd) layer_norm_fwd;
  decltype(&qnn_layer_norm_bwd_work) layer_norm_bwd_work;
  decltype(&qnn_layer_norm_bwd) layer_norm_bwd;
  decltype(&qnn_topk_distill_fwd_work) topk_distill_fwd_work;
  decltype(&qnn_topk_distill_fwd) topk_distill_fwd;
  decltype(&qnn_topk_distill_bwd) topk_distill_bwd;
} api;

void bind(const py::dict& address) {
#define QNN_BIND(name) \
  api.name = reinterpret_cast<decltype(api.name)>(py::cast<uintptr_t>(address[py::str("qnn_" #name)]))
  QNN_BIND(last_error);
  QNN_BIND(linear_act_fwd_work);
  QNN_BIND(linear_act_fwd);
  QNN_BIND(linear_act_bwd_work);
  QNN_BIND(linear_act_bwd);
  QNN_BIND(layer_norm_fwd);
  QNN_BIND(layer_norm_bwd_work);
  QNN_BIND(layer_norm_bwd);
  QNN_BIND(topk_distill_fwd_work);
  QNN_BIND(topk_distill_fwd);
  QNN_BIND(topk_distill_bwd);
#undef QNN_BIND
}

void ok(int status, const char* entry) {
  TORCH_CHECK(status == QNN_OK, entry, " failed (status ", status, "): ", api.last_error());
}

// ------------------------------------------------------------------------------ what all share
bool is_float(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf; }
int code_of(at::ScalarType t) { return t == at::kFloat ? QNN_F32 : t == at::kBFloat16 ? QNN_BF16 : QNN_F16; }

// The argument as a tensor.  What the kernels would lose without a word is refused: the tangent of a dual tensor
// (of a `constant` it is dropped as its gradient is), and the call itself under torch.jit.trace, which would
// record nothing but the empty output.
Tensor tensor_of(py::handle h, const char* op, const char* name, bool constant = false) {
  TORCH_CHECK_TYPE(THPVariable_Check(h.ptr()), "qnn: ", op, " expects a tensor for ", name, ", got ",
                   Py_TYPE(h.ptr())->tp_name);
  Tensor t = THPVariable_Unpack(h.ptr());
  TORCH_CHECK(constant || !t._fw_grad(/*level=*/0).defined(), "qnn: ", op, " has no forward-mode derivative (", name,
              " is a dual tensor with a tangent)");
  TORCH_CHECK(!torch::jit::tracer::isTracing(), "qnn: ", op, " cannot be recorded by torch.jit.trace");
  TORCH_CHECK(t.is_cuda(), "qnn: ", op, " runs on the MI355X path only (ROCm device tensor required for ", name,
              ", got ", t.device(), ")");
  return t;
}
OptTensor maybe_tensor_of(py::handle h, const char* op, const char* name) {
  if (h.is_none()) return std::nullopt;
  return tensor_of(h, op, name);
}
void same_device(const Tensor& t, const Tensor& first, const char* op, const char* name) {
  TORCH_CHECK(t.device() == first.device(), "qnn: ", op, " expects its tensors on one device, got ", name, " on ",
              t.device(), " and not ", first.device());
}

// t as a matrix of dense rows along its last dimension: itself, a view or a copy.  For the products rows
// also begin on 16-byte boundaries (or follow one another without a gap), strides within LONGEST.  A lazily negated
// view (of a conjugate's imaginary part) is copied: what lies in memory is not its value.
constexpr int64_t LONGEST = 1 << 21;  // of a row stride that the products take
struct Rows {
  Tensor t;
  int64_t ld = 0;
};
Rows rows_of(const Tensor& given, bool products = false) {
  const int64_t n = given.size(-1);
  Tensor t = given.dim() == 2 ? given : given.reshape({given.numel() / n, n});
  int64_t ld = t.size(0) <= 1 ? n : t.stride(0);
  const bool fits = !products || (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && ld <= LONGEST &&
                                  (ld * t.element_size() % 16 == 0 || ld == n));
  if ((t.stride(1) != 1 && n > 1) || ld < n || !fits || t.is_neg()) {
    t = t.clone(at::MemoryFormat::Contiguous);
    ld = n;
  }
  return {t, ld};
}
Tensor vector_of(const OptTensor& t) {
  if (!t) return Tensor();
  return t->is_contiguous() && !t->is_neg() ? *t : t->clone(at::MemoryFormat::Contiguous);
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor scratch(int64_t bytes, const Tensor& like) {
  return bytes ? at::empty({bytes}, like.options().dtype(at::kByte).requires_grad(false)) : Tensor();
}
qnn_stream_t stream_of(const Tensor& t) {
  return (qnn_stream_t)at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}
bool wants(const Tensor& t) { return t.requires_grad(); }
bool wants(const OptTensor& t) { return t && t->requires_grad(); }

// Gradients of gradients are not offered: under create_graph, gradients carry a node that says so where the gradient
// that came in is asked for one.  Where it is not they are constants, and a warning says what is missing of them if
// they depend (`depend`) on inputs that do require a gradient.
variable_list once(const variable_list& given, variable_list grads, const char* op, bool depend) {
  if (!at::GradMode::is_enabled()) return grads;
  bool any = false;
  for (const auto& g : given) any = any || (g.defined() && g.requires_grad());
  if (!any) {
    if (depend)
      TORCH_WARN("qnn: gradients of ", op, "'s gradients are not offered: those made here under create_graph are "
                 "constants, and what is computed from them sends nothing back to ", op, "'s inputs");
    return grads;
  }
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  return (*std::make_shared<torch::autograd::DelayedError>(
      std::string("qnn: gradients of ") + op + "'s gradients are not offered", grads.size()))(std::move(grads));
}

// ---------------------------------------------------------------------------------- linear_act
struct LinearOut {
  Tensor y, slope;
};
LinearOut linear_fwd(const Tensor& x, const Rows& x2, const Rows& w2, const Tensor& b, const Rows& r2, int act,
                     bool need_slope) {
  const int64_t m = x2.t.size(0), k = x2.t.size(1), n = w2.t.size(0);
  const int code = code_of(x.scalar_type());
  const c10::DeviceGuard guard(x.device());
  const auto opt = x.options().requires_grad(false);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = n;
  LinearOut o;
  o.y = at::empty(shape, opt);
  if (need_slope && act == QNN_ACT_RELU) o.slope = at::empty({m, (n + 7) / 8}, opt.dtype(at::kByte));
  if (need_slope && act == QNN_ACT_GELU)
    o.slope = at::empty({m, n}, opt.dtype(code == QNN_F32 ? at::kFloat : at::kShort));
  int64_t bytes = 0;
  ok(api.linear_act_fwd_work(m, n, k, code, &bytes), "qnn_linear_act_fwd_work");
  const Tensor work = scratch(bytes, x);
  ok(api.linear_act_fwd(ptr(x2.t), x2.ld, ptr(w2.t), w2.ld, ptr(b), ptr(r2.t), r2.ld, ptr(o.y), ptr(o.slope), m, n, k,
                        code, act, ptr(work), bytes, stream_of(x)),
     "qnn_linear_act_fwd");
  return o;
}

struct LinearAct : torch::autograd::Function<LinearAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& r,
                        int64_t act) {
    const Rows x2 = rows_of(x, true), w2 = rows_of(w, true), r2 = r ? rows_of(*r) : Rows{};
    LinearOut o = linear_fwd(x, x2, w2, vector_of(b), r2, (int)act, true);
    // the products take x for dw and w for dx
    ctx->save_for_backward({wants(w) ? x2.t : Tensor(), wants(x) ? w2.t : Tensor(), o.slope});
    ctx->saved_data["act"] = act;
    ctx->saved_data["has"] = (int64_t)((b ? 1 : 0) | (r ? 2 : 0));
    ctx->saved_data["x"] = x.sizes().vec();
    return o.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor& dy = grads[0];
    const int act = (int)ctx->saved_data["act"].toInt();
    const int64_t has = ctx->saved_data["has"].toInt();
    const std::vector<int64_t> shape = ctx->saved_data["x"].toIntVector();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool need_b = (has & 1) && ctx->needs_input_grad(2), need_r = (has & 2) && ctx->needs_input_grad(2 + (has & 1));
    const int64_t n = dy.size(-1), k = shape.back();
    variable_list out(5);
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(dy.device());
      const Rows dy2 = rows_of(dy, true);
      const int64_t m = dy2.t.size(0);
      const int code = code_of(dy.scalar_type());
      const auto opt = dy.options();
      const Rows x2 = need_w ? rows_of(saved[0], true) : Rows{Tensor(), k};
      const Rows w2 = need_x ? rows_of(saved[1], true) : Rows{Tensor(), k};
      Tensor dz;
      if (act != QNN_ACT_NONE) dz = at::empty(dy.sizes(), opt);
      if (need_x) out[0] = at::empty(shape, opt);
      if (need_w) out[1] = at::empty({n, k}, opt);
      if (need_b) out[2] = at::empty({n}, opt);
      if (act != QNN_ACT_NONE || need_x || need_w || need_b) {
        int64_t bytes = 0;
        ok(api.linear_act_bwd_work(m, n, k, code, &bytes), "qnn_linear_act_bwd_work");
        const Tensor work = scratch(bytes, dy);
        ok(api.linear_act_bwd(ptr(dy2.t), dy2.ld, ptr(saved[2]), ptr(x2.t), x2.ld, ptr(w2.t), w2.ld, ptr(dz),
                              ptr(out[0]), ptr(out[1]), ptr(out[2]), m, n, k, code, act, ptr(work), bytes,
                              stream_of(dy)),
           "qnn_linear_act_bwd");
      }
      if (need_r) out[3] = act != QNN_ACT_NONE ? dz : dy;
    }
    // without GELU the gradients are products of dy with the other operand
    return once(grads, std::move(out), "linear_act", act == QNN_ACT_GELU || (need_x && need_w));
  }
};

Tensor linear_act(py::handle hx, py::handle hw, py::handle hb, py::handle hr, int64_t act) {
  constexpr const char* op = "linear_act";
  const Tensor x = tensor_of(hx, op, "x"), w = tensor_of(hw, op, "weight");
  const OptTensor b = maybe_tensor_of(hb, op, "bias"), r = maybe_tensor_of(hr, op, "residual");
  const at::ScalarType t = x.scalar_type();
  TORCH_CHECK_TYPE(is_float(t), "qnn: linear_act expects x of float32, bfloat16 or float16, got ", t);
  const auto check = [&](const Tensor& v, const char* name) {
    TORCH_CHECK_TYPE(v.scalar_type() == t, "qnn: linear_act expects ", name, " of x's type ", t, ", got ", v.scalar_type());
    same_device(v, x, op, name);
  };
  check(w, "weight");
  if (b) check(*b, "bias");
  if (r) check(*r, "residual");
  TORCH_CHECK_VALUE(w.dim() == 2 && x.dim() >= 1 && x.size(-1) == w.size(1),
                    "qnn: linear_act needs x [..., in] and weight [out, in], got ", x.sizes(), " and ", w.sizes());
  const int64_t n = w.size(0), k = w.size(1);
  TORCH_CHECK_VALUE(n >= 1 && k >= 1 && n <= LONGEST && k <= LONGEST,
                    "qnn: linear_act needs 1 to 2^21 input and output features, got ", k, " and ", n);
  if (b) TORCH_CHECK_VALUE(b->dim() == 1 && b->size(0) == n, "qnn: linear_act needs bias [", n, "], got ", b->sizes());
  if (r)
    TORCH_CHECK_VALUE(r->dim() == x.dim() && r->size(-1) == n && r->sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1),
                      "qnn: linear_act needs a residual of the output's shape, got ", r->sizes(), " for x ", x.sizes(),
                      " and weight ", w.sizes());
  const py::gil_scoped_release release;
  if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b) || wants(r))) return LinearAct::apply(x, w, b, r, act);
  const at::NoGradGuard no_grad;
  return linear_fwd(x, rows_of(x, true), rows_of(w, true), vector_of(b), r ? rows_of(*r) : Rows{}, (int)act, false).y;
}

// ---------------------------------------------------------------------------------- layer_norm
Tensor norm_fwd(const Tensor& x, const Rows& x2, const Tensor& w, const Tensor& b, double eps, int wcode,
                const Tensor& stats) {
  const int64_t rows = x2.t.size(0), dim = x2.t.size(1);
  const c10::DeviceGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options().requires_grad(false));
  float* mean = stats.defined() ? stats.data_ptr<float>() : nullptr;
  ok(api.layer_norm_fwd(ptr(x2.t), x2.ld, ptr(w), ptr(b), ptr(y), mean, mean ? mean + rows : nullptr, rows, dim,
                        (float)eps, code_of(x.scalar_type()), wcode, stream_of(x)),
     "qnn_layer_norm_fwd");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, double eps,
                        int64_t wcode) {
    const Rows x2 = rows_of(x);
    const Tensor w2 = vector_of(w);
    const Tensor stats = at::empty({2, x2.t.size(0)}, x.options().dtype(at::kFloat).requires_grad(false));
    Tensor y = norm_fwd(x, x2, w2, vector_of(b), eps, (int)wcode, stats);
    ctx->save_for_backward({x2.t, w2, stats});
    ctx->saved_data["wcode"] = wcode;
    ctx->saved_data["has"] = (int64_t)((w ? 1 : 0) | (b ? 2 : 0));
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor& dy = grads[0];
    const int wcode = (int)ctx->saved_data["wcode"].toInt();
    const int64_t has = ctx->saved_data["has"].toInt();
    const bool need_x = ctx->needs_input_grad(0);
    const bool need_w = (has & 1) && ctx->needs_input_grad(1), need_b = (has & 2) && ctx->needs_input_grad(1 + (has & 1));
    variable_list out(5);
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(dy.device());
      const Rows dy2 = rows_of(dy), x2 = rows_of(saved[0]);
      const int64_t rows = x2.t.size(0), dim = x2.t.size(1);
      const int code = code_of(dy.scalar_type());
      const auto wopt = wcode == QNN_F32 ? dy.options().dtype(at::kFloat) : dy.options();
      if (need_x) out[0] = at::empty(dy.sizes(), dy.options());
      if (need_w) out[1] = at::empty({dim}, wopt);
      if (need_b) out[2] = at::empty({dim}, wopt);
      int64_t bytes = 0;
      if (need_w || need_b) ok(api.layer_norm_bwd_work(rows, dim, code, &bytes), "qnn_layer_norm_bwd_work");
      const Tensor work = scratch(bytes, dy);
      const float* mean = saved[2].data_ptr<float>();
      ok(api.layer_norm_bwd(ptr(dy2.t), dy2.ld, ptr(x2.t), x2.ld, ptr(saved[1]), mean, mean + rows, ptr(out[0]),
                            ptr(out[1]), ptr(out[2]), rows, dim, code, wcode, ptr(work), bytes, stream_of(dy)),
         "qnn_layer_norm_bwd");
    }
    return once(grads, std::move(out), "layer_norm", need_x);
  }
};

Tensor layer_norm(py::handle hx, py::handle hw, py::handle hb, double eps) {
  constexpr const char* op = "layer_norm";
  const Tensor x = tensor_of(hx, op, "x");
  const OptTensor w = maybe_tensor_of(hw, op, "weight"), b = maybe_tensor_of(hb, op, "bias");
  const at::ScalarType t = x.scalar_type();
  TORCH_CHECK_TYPE(is_float(t), "qnn: layer_norm expects x of float32, bfloat16 or float16, got ", t);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "qnn: layer_norm needs x [..., dim] with dim > 0, got ", x.sizes());
  TORCH_CHECK_VALUE(eps >= 0.0, "qnn: layer_norm needs eps >= 0, got ", eps);
  const int64_t dim = x.size(-1);
  int64_t wcode = code_of(t);
  const auto check = [&](const Tensor& v, const char* name) {
    TORCH_CHECK_TYPE(v.scalar_type() == t || v.scalar_type() == at::kFloat, "qnn: layer_norm expects ", name,
                     " of x's type ", t, " or float32, got ", v.scalar_type());
    same_device(v, x, op, name);
    TORCH_CHECK_VALUE(v.dim() == 1 && v.size(0) == dim, "qnn: layer_norm needs ", name, " [", dim, "], got ", v.sizes());
    wcode = code_of(v.scalar_type());
  };
  if (w) check(*w, "weight");
  if (b) check(*b, "bias");
  if (w && b)
    TORCH_CHECK_TYPE(w->scalar_type() == b->scalar_type(), "qnn: layer_norm needs weight and bias of one type, got ",
                     w->scalar_type(), " and ", b->scalar_type());
  const py::gil_scoped_release release;
  if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b))) return LayerNorm::apply(x, w, b, eps, wcode);
  const at::NoGradGuard no_grad;
  return norm_fwd(x, rows_of(x), vector_of(w), vector_of(b), eps, (int)wcode, Tensor());
}

// --------------------------------------------------------------------------- topk_distill_loss
enum { MEAN = 0, SUM = 1, NONE = 2 };  // reductions, as in qnn/functional.py

struct DistillOut {
  Tensor loss, stats;
};
DistillOut distill_fwd(const Tensor& s, const Rows& s2, const Rows& t2, const Rows& i2, double temp, int reduction) {
  const int64_t rows = s2.t.size(0), vocab = s2.t.size(1);
  const int code = code_of(s.scalar_type());
  const c10::DeviceGuard guard(s.device());
  const auto opt = s.options().dtype(at::kFloat).requires_grad(false);
  DistillOut o;
  o.stats = at::empty({4 * rows + 4}, opt);
  const Tensor row_loss = at::empty(s.sizes().slice(0, s.dim() - 1), opt);
  o.loss = reduction == NONE ? row_loss : at::empty({}, opt);
  int64_t bytes = 0;
  ok(api.topk_distill_fwd_work(rows, vocab, code, &bytes), "qnn_topk_distill_fwd_work");
  const Tensor work = scratch(bytes, s);
  ok(api.topk_distill_fwd(ptr(s2.t), s2.ld, ptr(t2.t), t2.ld, ptr(i2.t), i2.ld, rows, vocab, t2.t.size(1), (float)temp,
                          reduction == MEAN, code, code_of(t2.t.scalar_type()), (int)i2.t.element_size(),
                          row_loss.data_ptr<float>(), o.stats.data_ptr<float>(),
                          reduction == NONE ? nullptr : o.loss.data_ptr<float>(), ptr(work), bytes, stream_of(s)),
     "qnn_topk_distill_fwd");
  return o;
}

struct TopKDistill : torch::autograd::Function<TopKDistill> {
  static Tensor forward(AutogradContext* ctx, const Tensor& s, const Tensor& t, const Tensor& i, double temp,
                        int64_t reduction) {
    const Rows s2 = rows_of(s), t2 = rows_of(t), i2 = rows_of(i);
    DistillOut o = distill_fwd(s, s2, t2, i2, temp, (int)reduction);
    ctx->save_for_backward({s2.t, t2.t, i2.t, o.stats});
    ctx->saved_data["temp"] = temp;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["s"] = s.sizes().vec();
    return o.loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const double temp = ctx->saved_data["temp"].toDouble();
    const int reduction = (int)ctx->saved_data["reduction"].toInt();
    variable_list out(5);
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(saved[0].device());
      const Rows s2 = rows_of(saved[0]), t2 = rows_of(saved[1]), i2 = rows_of(saved[2]);
      const Tensor g = grads[0].contiguous().resolve_neg();
      out[0] = at::empty(ctx->saved_data["s"].toIntVector(), saved[0].options().requires_grad(false));
      ok(api.topk_distill_bwd(ptr(s2.t), s2.ld, ptr(t2.t), t2.ld, ptr(i2.t), i2.ld, saved[3].data_ptr<float>(),
                              g.data_ptr<float>(), reduction == NONE, ptr(out[0]), s2.t.size(0), s2.t.size(1),
                              t2.t.size(1), (float)temp, reduction == MEAN, code_of(s2.t.scalar_type()),
                              code_of(t2.t.scalar_type()), (int)i2.t.element_size(), stream_of(s2.t)),
         "qnn_topk_distill_bwd");
    }
    return once(grads, std::move(out), "topk_distill_loss", true);
  }
};

constexpr int64_t MAX_TOP = 1024;

Tensor topk_distill_loss(py::handle hs, py::handle ht, py::handle hi, double temp, int64_t reduction) {
  constexpr const char* op = "topk_distill_loss";
  const Tensor s = tensor_of(hs, op, "logits"), t = tensor_of(ht, op, "teacher_logits", true).detach(),
               i = tensor_of(hi, op, "teacher_index");
  TORCH_CHECK_TYPE(is_float(s.scalar_type()) && is_float(t.scalar_type()),
                   "qnn: topk_distill_loss expects logits and teacher_logits of float32, bfloat16 or float16, got ",
                   s.scalar_type(), " and ", t.scalar_type());
  TORCH_CHECK_TYPE(i.scalar_type() == at::kLong || i.scalar_type() == at::kInt,
                   "qnn: topk_distill_loss expects teacher_index of int64 or int32, got ", i.scalar_type());
  same_device(t, s, op, "teacher_logits");
  same_device(i, s, op, "teacher_index");
  TORCH_CHECK_VALUE(temp >= 0x1p-60 && temp <= 0x1p60,
                    "qnn: topk_distill_loss needs a positive, finite temperature (2^-60 to 2^60), got ", temp);
  TORCH_CHECK_VALUE(s.dim() >= 1 && s.size(-1) >= 1, "qnn: topk_distill_loss needs logits [..., vocab], got ", s.sizes());
  TORCH_CHECK_VALUE(t.sizes() == i.sizes() && t.dim() == s.dim() && t.sizes().slice(0, s.dim() - 1) == s.sizes().slice(0, s.dim() - 1),
                    "qnn: topk_distill_loss needs teacher_logits and teacher_index [..., top] beside logits ", s.sizes(),
                    ", got ", t.sizes(), " and ", i.sizes());
  TORCH_CHECK_VALUE(t.size(-1) >= 1 && t.size(-1) <= MAX_TOP, "qnn: topk_distill_loss takes 1 to ", MAX_TOP,
                    " entries a row, got ", t.size(-1));
  const py::gil_scoped_release release;
  if (at::GradMode::is_enabled() && wants(s)) return TopKDistill::apply(s, t, i, temp, reduction);
  const at::NoGradGuard no_grad;
  return distill_fwd(s, rows_of(s), rows_of(t), rows_of(i), temp, (int)reduction).loss;
}

}  // namespace

PYBIND11_MODULE(_float, m) {
  m.def("bind", &bind);
  m.def("linear_act", &linear_act);
  m.def("layer_norm", &layer_norm);
  m.def("topk_distill_loss", &topk_distill_loss);
}

// Python module _mixture_torch: the plain mixture-of-adapters operators of
// include/tensafe_he.h over torch tensors, with their autograd functions.
// provenloop_amd/mixture.py is its documentation and only caller.
//
// A call through ctypes and a Python autograd function costs more host time
// than the kernels of a small batch take on the GPU (one token's projection
// with its adapter: 24 us a call for 11 us of kernels), so the checks, the
// allocations and the graph's nodes are made here.
#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include "tensafe_he.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;
using Guard = c10::hip::OptionalHIPGuardMasqueradingAsCUDA;

#define NEED(ok, ...) TORCH_CHECK_VALUE(ok, __VA_ARGS__)

// A refusal of the library, as provenloop_amd/_lib.py raises it.
void check(int rc) {
  if (rc == 0) return;
  const std::string message = th_last_error();
  if (rc == TH_EINVAL) TORCH_CHECK_VALUE(false, message);
  pybind11::gil_scoped_acquire gil;  // also from autograd's threads
  pybind11::module_::import("provenloop_amd._lib").attr("check")(rc);
}

int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return TH_BF16;
    case at::kHalf: return TH_F16;
    case at::kFloat: return TH_F32;
    default: return 0;
  }
}
bool is_half(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }

void on_gpu(const char* name, const Tensor& first, std::initializer_list<Tensor> others = {}) {
  NEED(first.is_cuda(), name, ": tensors must be on the GPU (there is no CPU path)");
  for (const Tensor& t : others)
    NEED(!t.defined() || t.device() == first.device(), name, ": all tensors must be on one device");
}

// These functions are not torch's dispatched operators: a trace would hold their
// results as constants, and the results would have no tangents, which torch
// reads as zeros.
void not_traced(const char* name) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() && !Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY),
                              name, ": cannot be traced");
}
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const OptTensor& t) { return t && has_tangent(*t); }
template <class... Tensors>
void no_tangents(const char* name, const Tensors&... ts) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(ts) || ...), name, ": has no forward-mode derivative");
}

Tensor make(at::IntArrayRef size, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(size, type, like.device(), std::nullopt);
}
struct Work {
  Tensor t;
  void* p = nullptr;
  size_t bytes = 0;
};
Work work(size_t bytes, const Tensor& like) {
  Work w;
  if (bytes) {
    w.t = make({(int64_t)bytes}, at::kByte, like);
    w.p = w.t.data_ptr();
    w.bytes = bytes;
  }
  return w;
}
void* stream(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

// autograd's apply takes no undefined tensors
OptTensor optional(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

template <class P = void>
P* ptr(const Tensor& t) {
  return t.defined() ? (P*)t.data_ptr() : nullptr;
}

// t with unit column stride and rows that do not overlap (a copy only if it has none).
Tensor rows(const Tensor& t) {
  const int64_t d = t.dim(), width = t.size(d - 1);
  if (width > 1 && t.stride(d - 1) != 1) return t.contiguous();
  for (int64_t i = 0; i + 1 < d; ++i)
    if (t.size(i) > 1 && t.stride(i) < width) return t.contiguous();
  return t;
}
// Row stride; of a single row its length, which every row check takes.
int64_t ld(const Tensor& t) {
  const int64_t d = t.dim();
  return t.size(d - 2) > 1 ? t.stride(d - 2) : t.size(d - 1);
}

Tensor experts_of(const char* name, const Tensor& experts) {
  NEED(experts.scalar_type() == at::kInt, name, ": experts must be an int32 tensor");
  NEED(experts.dim() == 1 || experts.dim() == 2, name, ": experts must be [T] or [T, k]");
  return (experts.dim() == 1 ? experts.unsqueeze(1) : experts).contiguous();
}

// The gradients of a node are not differentiable themselves.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& t : grads)
    if (t.defined()) t.set_requires_grad(true);  // so that the error's node joins the graph
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "the mixture operators' gradients are not differentiable a second time", (int64_t)grads.size());
  return (*error)(std::move(grads));
}

// ---------------------------------------------------------------- grouping and gate
std::tuple<Tensor, Tensor, Tensor> group(const Tensor& given, int64_t n) {
  not_traced("group");
  const Tensor experts = experts_of("group", given);
  on_gpu("group", experts);
  NEED(n >= 1 && n <= 1 << 30, "group: the number of groups must be positive");
  Guard guard(experts.device());
  const int64_t t = experts.size(0), k = experts.size(1);
  size_t bytes;
  check(th_group_workspace(t, (uint32_t)n, (uint32_t)k, &bytes));  // refuses what is out of range
  Tensor order = make({t * k}, at::kInt, experts), offsets = make({n + 1}, at::kInt, experts);
  const Work w = work(bytes, experts);
  check(th_group(ptr<int32_t>(experts), t, (uint32_t)n, (uint32_t)k, ptr<int32_t>(order), ptr<int32_t>(offsets), w.p,
                 w.bytes, stream(experts)));
  return {experts, order, offsets};
}

int64_t mask_ld(const Tensor& mask) {
  return !mask.defined() || mask.dim() == 1 || mask.stride(0) == 0 ? 0 : ld(mask);
}

variable_list route_forward(const Tensor& logits, const Tensor& mask, int64_t k, bool normalize) {
  Guard guard(logits.device());
  const int64_t t = logits.size(0), e = logits.size(1);
  NEED(k >= 1 && k <= e, "route: choices must be in [1, number of experts]");
  size_t bytes;
  check(th_group_workspace(t, (uint32_t)e, (uint32_t)k, &bytes));
  Tensor weights = make({t, k}, at::kFloat, logits), experts = make({t, k}, at::kInt, logits);
  Tensor order = make({t * k}, at::kInt, logits), offsets = make({e + 1}, at::kInt, logits);
  const Work w = work(bytes, logits);
  check(th_route(type_of(logits), ptr(logits), ld(logits), t, (uint32_t)e, ptr<uint8_t>(mask), mask_ld(mask),
                 (uint32_t)k, normalize, ptr<float>(weights), ptr<int32_t>(experts), ptr<int32_t>(order),
                 ptr<int32_t>(offsets), w.p, w.bytes, stream(logits)));
  return {weights, experts, order, offsets};
}

struct Route : Function<Route> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& given_mask, int64_t k,
                               bool normalize) {
    const Tensor mask = given_mask ? *given_mask : Tensor();
    variable_list out = route_forward(logits, mask, k, normalize);
    ctx->save_for_backward({logits, mask, out[0], out[1]});
    ctx->saved_data["normalize"] = normalize;
    ctx->mark_non_differentiable({out[1], out[2], out[3]});
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &mask = saved[1];
    if (!grads[0].defined()) return variable_list(4);
    no_tangents("route's gradient", grads[0]);
    const Tensor dweights = grads[0].contiguous();
    Guard guard(logits.device());
    Tensor dlogits = make(logits.sizes(), logits.scalar_type(), logits);
    check(th_route_backward(type_of(logits), ptr(logits), ld(logits), logits.size(0), (uint32_t)logits.size(1),
                            ptr<uint8_t>(mask), mask_ld(mask), (uint32_t)saved[2].size(1),
                            ctx->saved_data["normalize"].toBool(), ptr<float>(saved[2]), ptr<int32_t>(saved[3]),
                            ptr<float>(dweights), ptr(dlogits), stream(logits)));
    return once({dlogits, Tensor(), Tensor(), Tensor()});
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> route(const Tensor& given, int64_t k, const OptTensor& given_mask,
                                                 bool normalize) {
  not_traced("route");
  no_tangents("route", given);
  NEED(type_of(given) != 0, "route: logits must be bf16, f16 or f32");
  NEED(given.dim() == 2, "route: logits must be [T, E]");
  Tensor mask = given_mask ? *given_mask : Tensor();
  on_gpu("route", given, {mask});
  const int64_t t = given.size(0), e = given.size(1);
  if (mask.defined()) {
    NEED(mask.scalar_type() == at::kBool, "route: mask must be bool");
    NEED((mask.dim() == 2 && mask.size(0) == t && mask.size(1) == e) || (mask.dim() == 1 && mask.size(0) == e),
         "route: mask must be [T, E] or [E]");
    if ((e > 1 && mask.stride(-1) != 1) ||
        (mask.dim() == 2 && t > 1 && mask.stride(0) > 0 && mask.stride(0) < e))
      mask = mask.contiguous();
  }
  const Tensor logits = rows(given);
  const variable_list out = logits.requires_grad() && at::GradMode::is_enabled()
                                ? Route::apply(logits, optional(mask), k, normalize)
                                : route_forward(logits, mask, k, normalize);
  return {out[0], out[1], out[2], out[3]};
}

// ---------------------------------------------------------------- grouped products
th_grouped grouped_args(const Tensor& x, const Tensor& w, int64_t t, int64_t k, const Tensor& order,
                        const Tensor& offsets) {
  th_grouped d{};
  d.dtype = type_of(x);
  d.x_per_slot = x.dim() == 3;
  d.tokens = t;
  d.choices = (uint32_t)k;
  d.experts = (uint32_t)w.size(0);
  d.d_in = (uint32_t)w.size(2);
  d.d_out = (uint32_t)w.size(1);
  d.x = ptr(x);
  d.w = ptr(w);
  d.ldx = ld(x);
  d.ldw = ld(w);
  d.ldwe = w.stride(0);
  d.order = ptr<int32_t>(order);
  d.offsets = ptr<int32_t>(offsets);
  return d;
}

Tensor grouped_forward(const Tensor& x, const Tensor& w, int64_t t, int64_t k, const Tensor& order,
                       const Tensor& offsets) {
  Guard guard(x.device());
  Tensor y = make({t, k, w.size(1)}, x.scalar_type(), x);
  const th_grouped d = grouped_args(x, w, t, k, order, offsets);
  check(th_grouped_matmul(&d, ptr(y), w.size(1), stream(x)));
  return y;
}

struct GroupedMatmul : Function<GroupedMatmul> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, int64_t t, int64_t k,
                        const Tensor& order, const Tensor& offsets) {
    ctx->save_for_backward({x, w, order, offsets});
    ctx->saved_data["t"] = t;
    ctx->saved_data["k"] = k;
    return grouped_forward(x, w, t, k, order, offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1];
    no_tangents("grouped_matmul's gradient", grads[0]);
    const Tensor dy = grads[0].contiguous();
    Guard guard(x.device());
    Tensor dx, dw;
    if (ctx->needs_input_grad(0)) dx = make(x.sizes(), x.scalar_type(), x);
    if (ctx->needs_input_grad(1)) dw = make(w.sizes(), w.scalar_type(), w);
    const th_grouped d = grouped_args(x, w, ctx->saved_data["t"].toInt(), ctx->saved_data["k"].toInt(), saved[2],
                                      saved[3]);
    size_t bytes;
    check(th_grouped_matmul_backward_workspace(&d, &bytes));
    const Work k = work(bytes, x);
    check(th_grouped_matmul_backward(&d, ptr(dy), w.size(1), ptr(dx), ptr(dw), k.p, k.bytes, stream(x)));
    return once({dx, dw, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor grouped_matmul(const Tensor& given_x, const Tensor& given_w, const Tensor& experts, const Tensor& order,
                      const Tensor& offsets, int64_t n_groups) {
  not_traced("grouped_matmul");
  no_tangents("grouped_matmul", given_x, given_w);
  NEED(is_half(given_x), "grouped_matmul: x must be bf16 or f16");
  NEED(given_w.scalar_type() == given_x.scalar_type(), "grouped_matmul: x and w must have one type");
  const int64_t t = experts.size(0), k = experts.size(1);
  NEED(given_w.dim() == 3 && given_w.size(0) == n_groups, "grouped_matmul: w must be [n_groups, d_out, d_in]");
  const int64_t d = given_w.size(2);
  NEED((given_x.dim() == 2 && given_x.size(0) == t && given_x.size(1) == d) ||
           (given_x.dim() == 3 && given_x.size(0) == t && given_x.size(1) == k && given_x.size(2) == d),
       "grouped_matmul: x must be [T, d_in] or [T, k, d_in]");
  on_gpu("grouped_matmul", given_x, {given_w, order, offsets});
  NEED(order.scalar_type() == at::kInt && order.is_contiguous() && order.numel() == t * k &&
           offsets.scalar_type() == at::kInt && offsets.is_contiguous() && offsets.numel() == n_groups + 1,
       "grouped_matmul: groups must be what group or route returns");
  const Tensor x = given_x.dim() == 3 ? given_x.contiguous() : rows(given_x), w = rows(given_w);
  if ((x.requires_grad() || w.requires_grad()) && at::GradMode::is_enabled())
    return GroupedMatmul::apply(x, w, t, k, order, offsets);
  return grouped_forward(x, w, t, k, order, offsets);
}

// ---------------------------------------------------------------- shared projection with adapters
struct Lora {
  Tensor x, weight, bias, a, b, experts, gate, scale, order, offsets;
  th_lora_linear_args args() const {
    th_lora_linear_args d{};
    d.dtype = type_of(x);
    d.choices = (uint32_t)experts.size(1);
    d.tokens = experts.size(0);
    d.d_in = (uint32_t)x.size(1);
    d.d_out = (uint32_t)weight.size(0);
    d.rank = (uint32_t)a.size(1);
    d.adapters = (uint32_t)a.size(0);
    d.x = ptr(x);
    d.weight = ptr(weight);
    d.bias = ptr(bias);
    d.a = ptr(a);
    d.b = ptr(b);
    d.ldx = ld(x);
    d.ldw = ld(weight);
    d.lda = ld(a);
    d.lda_adapter = a.stride(0);
    d.ldb = ld(b);
    d.ldb_adapter = b.stride(0);
    d.experts = ptr<int32_t>(experts);
    d.gate = ptr<float>(gate);
    d.scale = ptr<float>(scale);
    d.order = ptr<int32_t>(order);
    d.offsets = ptr<int32_t>(offsets);
    return d;
  }
};

Tensor lora_forward(const Lora& l, const Tensor& u) {
  Guard guard(l.x.device());
  const int64_t n = l.weight.size(0);
  Tensor y = make({l.x.size(0), n}, l.x.scalar_type(), l.x);
  const th_lora_linear_args d = l.args();
  size_t bytes;
  check(th_lora_linear_workspace(&d, u.defined(), &bytes));
  const Work w = work(bytes, l.x);
  check(th_lora_linear(&d, ptr(y), n, ptr<float>(u), w.p, w.bytes, stream(l.x)));
  return y;
}

struct LoraLinear : Function<LoraLinear> {
  // `l` holds all of them; its other tensors have no gradients
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& a, const Tensor& b, const OptTensor& gate,
                        Lora l) {
    l.x = x;
    l.a = a;
    l.b = b;
    l.gate = gate ? *gate : Tensor();
    if (!l.order.defined()) {  // the backward pass needs them again
      auto groups = group(l.experts, a.size(0));
      l.order = std::get<1>(groups);
      l.offsets = std::get<2>(groups);
    }
    // u rows: the rank rounded up to 4
    Tensor u = make({l.experts.numel(), (a.size(1) + 3) / 4 * 4}, at::kFloat, x);
    ctx->save_for_backward({x, a, b, l.gate, l.weight, l.bias, l.experts, l.scale, l.order, l.offsets, u});
    return lora_forward(l, u);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Lora l{s[0], s[4], s[5], s[1], s[2], s[6], s[3], s[7], s[8], s[9]};
    no_tangents("lora_linear's gradient", grads[0]);
    const Tensor dy = rows(grads[0]);
    Guard guard(l.x.device());
    Tensor out[4];
    for (int i = 0; i < 4; ++i)
      if (s[i].defined() && ctx->needs_input_grad(i)) out[i] = make(s[i].sizes(), s[i].scalar_type(), l.x);
    const th_lora_linear_args d = l.args();
    size_t bytes;
    check(th_lora_linear_backward_workspace(&d, &bytes));
    const Work w = work(bytes, l.x);
    check(th_lora_linear_backward(&d, ptr<float>(s[10]), ptr(dy), ld(dy), ptr(out[0]), ptr(out[1]), ptr(out[2]),
                                  ptr<float>(out[3]), w.p, w.bytes, stream(l.x)));
    variable_list result(5);
    for (int i = 0; i < 4; ++i) result[i] = out[i];
    return once(std::move(result));
  }
};

Tensor lora_linear(const Tensor& x, const Tensor& weight, const Tensor& a, const Tensor& b, const Tensor& given_experts,
                   const OptTensor& weights, const OptTensor& scale, const OptTensor& bias, const OptTensor& order,
                   const OptTensor& offsets) {
  not_traced("lora_linear");
  no_tangents("lora_linear", x, weight, a, b, weights, scale, bias);
  NEED(is_half(x), "lora_linear: x must be bf16 or f16");
  const at::ScalarType type = x.scalar_type();
  NEED(weight.scalar_type() == type, "lora_linear: weight must have x's type");
  NEED(a.scalar_type() == type, "lora_linear: lora_a must have x's type");
  NEED(b.scalar_type() == type, "lora_linear: lora_b must have x's type");
  NEED(!bias || bias->scalar_type() == type, "lora_linear: bias must have x's type");
  NEED(x.dim() == 2 && weight.dim() == 2 && weight.size(1) == x.size(1),
       "lora_linear: x must be [T, d_in] and weight [d_out, d_in]");
  NEED(a.dim() == 3 && a.size(2) == x.size(1), "lora_linear: lora_a must be [n, rank, d_in]");
  const int64_t n = a.size(0), d_out = weight.size(0);
  NEED(b.dim() == 3 && b.size(0) == n && b.size(1) == d_out && b.size(2) == a.size(1),
       "lora_linear: lora_b must be [n, d_out, rank]");
  const Tensor experts = experts_of("lora_linear", given_experts);
  NEED(experts.size(0) == x.size(0), "lora_linear: experts must have a row per token");
  NEED(!bias || (bias->dim() == 1 && bias->size(0) == d_out), "lora_linear: bias must be [d_out]");
  Lora l;
  if (weights) {
    l.gate = weights->dim() == 1 ? weights->unsqueeze(1) : *weights;
    NEED(l.gate.scalar_type() == at::kFloat && l.gate.sizes() == experts.sizes(),
         "lora_linear: weights must be float32 and shaped as experts");
    l.gate = l.gate.contiguous();
  }
  if (scale) {
    NEED(scale->scalar_type() == at::kFloat && scale->dim() == 1 && scale->size(0) == n,
         "lora_linear: scale must be float32 [n]");
    l.scale = scale->contiguous();
  }
  if (bias) l.bias = bias->contiguous();
  if (order) {
    NEED(offsets && order->scalar_type() == at::kInt && order->is_contiguous() && order->numel() == experts.numel() &&
             offsets->scalar_type() == at::kInt && offsets->is_contiguous() && offsets->numel() == n + 1,
         "lora_linear: groups must be what group or route returns for these experts");
    l.order = *order;
    l.offsets = *offsets;
  }
  on_gpu("lora_linear", x, {weight, a, b, experts, l.gate, l.scale, l.bias, l.order, l.offsets});
  l.x = rows(x);
  l.weight = rows(weight);
  l.a = rows(a);
  l.b = rows(b);
  l.experts = experts;
  if (at::GradMode::is_enabled()) {
    auto frozen = [](const Tensor& t) { return !t.defined() || !t.requires_grad(); };
    NEED(frozen(l.weight) && frozen(l.bias) && frozen(l.scale),
         "lora_linear: weight, bias and scale are frozen and have no gradient");
    if (!frozen(l.x) || !frozen(l.a) || !frozen(l.b) || !frozen(l.gate))
      return LoraLinear::apply(l.x, l.a, l.b, optional(l.gate), l);
  }
  return lora_forward(l, Tensor());
}

}  // namespace

PYBIND11_MODULE(_mixture_torch, m) {
  m.def("group", &group);
  m.def("route", &route);
  m.def("grouped_matmul", &grouped_matmul);
  m.def("lora_linear", &lora_linear);
}

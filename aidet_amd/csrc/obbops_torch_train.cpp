// The fused linear layer and the top-logit distillation loss as differentiable tensor operators: argument checks, memory,
// streams and the autograd nodes around obb_linear_* and obb_topk_distill_* (include/obbops.h).  In C++, because a step of a
// small head is bound by the host: a node in Python costs about 60 us a direction, these about 15.
#include <torch/extension.h>

#include <ATen/autocast_mode.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>

#include <tuple>
#include <unordered_set>
#include <vector>

#include "obbops.h"

namespace {

using c10::hip::HIPGuardMasqueradingAsCUDA;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<at::Tensor> MaybeTensor;

void *stream_of(const at::Tensor &t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
void check_rc(int rc, const char *what) { TORCH_CHECK(rc == OBB_OK, what, ": ", obb_last_error()); }

int code_of(at::ScalarType t) { return t == at::kFloat ? OBB_F32 : t == at::kBFloat16 ? OBB_BF16 : t == at::kHalf ? OBB_F16 : -1; }

int64_t leading(const at::Tensor &t) {
  int64_t n = 1;
  for (int64_t i = 0; i + 1 < t.dim(); i++) n *= t.size(i);
  return n;
}

// A tensor whose sign waits to be turned -- the imaginary part of a conjugate -- is turned: the kernels read memory.
at::Tensor turned(const at::Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }
MaybeTensor turned(const MaybeTensor &t) { return t && t->is_neg() ? MaybeTensor(t->resolve_neg()) : t; }

// (..., cols) as rows that the kernels read in place; copied only where the last dimension is not contiguous or rows overlap
struct Rows {
  at::Tensor t;
  int64_t ld;
  Rows(const at::Tensor &src, int64_t cols) {
    const int64_t m = leading(src);
    t = src.dim() == 2 ? src : src.reshape({m, cols});
    if ((cols > 1 && t.stride(1) != 1) || (m > 1 && t.stride(0) < cols)) t = t.contiguous();
    ld = std::max(t.stride(0), cols);
  }
};

at::Tensor workspace(size_t bytes, const at::Tensor &like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}
void *ptr(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// Forward mode has no rule here: a dual tensor is refused, not read as its primal alone (which would be a derivative of 0).
void check_no_tangent(const char *who, std::initializer_list<const at::Tensor *> tensors) {
  for (const at::Tensor *t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), who, " has no forward-mode derivative (an input is a dual tensor)");
}

// the gradients of a node that is differentiable once: they say so when somebody differentiates them
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list given;
  for (auto &g : grads)
    if (g.defined()) {
      g = g.detach();
      g.set_requires_grad(true);
      given.push_back(g);
    }
  if (given.empty()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that is differentiable once", (int64_t)given.size());
  variable_list out = (*error)(std::move(given));
  size_t i = 0;
  for (auto &g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

// A leaf's gradient is added up on the stream where its accumulator was made, and the accumulator lives as long as any graph
// of the leaf.  One of the default stream, which takes no part in a capture, would end a process that captures this pass: say so.
// All accumulators that this pass will reach from here are looked at, behind casts, views and other layers too.
void check_capture(void *stream) {
  hipStreamCaptureStatus status;
  if (hipStreamIsCapturing((hipStream_t)stream, &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
  const auto node = torch::autograd::get_current_node();
  const auto *exec = torch::autograd::get_current_graph_task_exec_info();
  if (!node) return;
  std::vector<torch::autograd::Node *> todo = {node.get()};
  std::unordered_set<torch::autograd::Node *> seen;
  while (!todo.empty()) {
    auto *at = todo.back();
    todo.pop_back();
    for (const auto &edge : at->next_edges()) {
      auto *next = edge.function.get();
      if (!next || !seen.insert(next).second) continue;
      if (exec && !exec->empty()) {
        const auto it = exec->find(next);
        if (it == exec->end() || !it->second.should_execute()) continue;
      }
      if (dynamic_cast<torch::autograd::AccumulateGrad *>(next)) {
        const auto s = next->stream();
        TORCH_CHECK(!s || s->id() != 0, "a backward pass is captured while a graph of the same leaves from the default stream is alive: free that graph's outputs before the capture");
      } else {
        todo.push_back(next);
      }
    }
  }
}

// ---- fused linear ------------------------------------------------------------------------------------------------------
void check_linear(const at::Tensor &x, const at::Tensor &w, const MaybeTensor &bias, const MaybeTensor &res, int64_t act) {
  TORCH_CHECK_VALUE(act >= OBB_ACT_NONE && act <= OBB_ACT_SILU, "unknown activation ", act);
  TORCH_CHECK_TYPE(code_of(x.scalar_type()) >= 0, "fused_linear takes float32, bfloat16 or float16, but got ", x.scalar_type());
  for (const at::Tensor *t : {&w, bias ? &*bias : &x, res ? &*res : &x})
    TORCH_CHECK_TYPE(t->scalar_type() == x.scalar_type(), "fused_linear takes tensors of one type: x is ", x.scalar_type(), ", another is ", t->scalar_type());
  TORCH_CHECK_VALUE(w.dim() == 2 && x.dim() >= 1 && x.size(-1) == w.size(1), "x must be (..., K) and weight (N, K): got ", x.sizes(), " and ", w.sizes());
  if (bias) TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == w.size(0), "bias must be (", w.size(0), ",), but got ", bias->sizes());
  if (res) {
    bool same = res->dim() == x.dim() && res->size(-1) == w.size(0);
    for (int64_t i = 0; same && i + 1 < x.dim(); i++) same = res->size(i) == x.size(i);
    TORCH_CHECK_VALUE(same, "residual must have the shape of the output, rows of x by ", w.size(0), ", but got ", res->sizes());
  }
  check_no_tangent("fused_linear", {&x, &w, bias ? &*bias : &x, res ? &*res : &x});
  for (const at::Tensor *t : {&x, &w, bias ? &*bias : &x, res ? &*res : &x}) {
    TORCH_CHECK_NOT_IMPLEMENTED(t->is_cuda(), "fused_linear runs on a HIP device only (a tensor is on ", t->device(), ")");
    TORCH_CHECK_VALUE(t->device() == x.device(), "x is on ", x.device(), ", another tensor on ", t->device());
  }
}

std::tuple<at::Tensor, at::Tensor> linear_forward(const at::Tensor &x, const at::Tensor &w, const MaybeTensor &bias, const MaybeTensor &res, int act, bool want_z) {
  const int64_t n = w.size(0), k = w.size(1), m = leading(x);
  HIPGuardMasqueradingAsCUDA guard(x.device());
  auto sizes = x.sizes().vec();
  sizes.back() = n;
  at::Tensor y = at::empty(sizes, x.options());
  at::Tensor z = want_z ? at::empty(sizes, x.options().dtype(at::kFloat)) : at::Tensor();
  if (y.numel() == 0) return {y, z};
  const Rows rx(x, k), rw(w, k);
  const at::Tensor b = bias ? bias->contiguous() : at::Tensor();
  at::Tensor r;
  int64_t ldr = 0;
  if (res) {
    r = res->dim() == 2 ? *res : res->reshape({m, n});
    if (m > 1 && r.stride(0) == 0 && (n == 1 || r.stride(1) == 1)) ldr = 0;      // one row for all
    else {
      const Rows rr(r, n);
      r = rr.t;
      ldr = rr.ld;
    }
  }
  const int code = code_of(x.scalar_type());
  const size_t bytes = obb_linear_workspace_bytes(m, n, k, code, OBB_LINEAR_FORWARD);
  const at::Tensor ws = workspace(bytes, x);
  check_rc(obb_linear_forward(ptr(rx.t), rx.ld, ptr(rw.t), rw.ld, ptr(b), ptr(r), ldr, m, n, k, code, act, ptr(y), (float *)ptr(z), ptr(ws), bytes, stream_of(x)),
           "obb_linear_forward");
  return {y, z};
}

struct FusedLinear : public torch::autograd::Function<FusedLinear> {
  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &w, const MaybeTensor &bias, const MaybeTensor &res, int64_t act) {
    at::AutoDispatchBelowADInplaceOrView below;
    // gelu and silu keep the pre-activation, in 32 bits: their slope is taken where the forward was; relu needs y only
    const bool smooth = act == OBB_ACT_GELU || act == OBB_ACT_SILU;
    at::Tensor y, z;
    std::tie(y, z) = linear_forward(x, w, bias, res, (int)act, smooth);
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = res.has_value();
    ctx->save_for_backward({x, w, smooth ? z : act == OBB_ACT_RELU ? y : at::Tensor()});
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const int64_t act = ctx->saved_data["act"].toInt();
    const bool bias = ctx->saved_data["bias"].toBool(), residual = ctx->saved_data["residual"].toBool();
    // (a node's inputs are counted without those that are not there)
    const int need = (ctx->needs_input_grad(0) ? 1 : 0) | (ctx->needs_input_grad(1) ? 2 : 0) | (bias && ctx->needs_input_grad(2) ? 4 : 0) |
                     (residual && ctx->needs_input_grad(bias ? 3 : 2) ? 8 : 0);
    const auto saved = ctx->get_saved_variables();
    variable_list out(5);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const at::Tensor x = saved[0], w = saved[1], kept = saved[2];
      const int64_t n = w.size(0), k = w.size(1), m = leading(x);
      HIPGuardMasqueradingAsCUDA guard(x.device());
      void *stream = stream_of(x);
      check_capture(stream);
      const int code = code_of(x.scalar_type());
      const at::Tensor dy = turned(grads[0]).contiguous();
      at::Tensor dz = dy;
      const bool want_dz = act != OBB_ACT_NONE && (need & 11);
      if (want_dz) dz = at::empty_like(dy);
      if (need & 4) out[2] = at::empty({n}, x.options());
      if (want_dz || (need & 4)) {
        const size_t bytes = need & 4 ? obb_linear_workspace_bytes(m, n, k, code, OBB_LINEAR_ACT_BACKWARD) : 0;
        const at::Tensor ws = workspace(bytes, x);
        check_rc(obb_linear_act_backward(ptr(dy), act == OBB_ACT_RELU ? ptr(kept) : nullptr, act > OBB_ACT_RELU ? (const float *)ptr(kept) : nullptr, m, n, code, (int)act,
                                         want_dz ? ptr(dz) : nullptr, ptr(out[2]), ptr(ws), bytes, stream),
                 "obb_linear_act_backward");
      }
      if (need & 1) {
        out[0] = at::empty(x.sizes(), x.options());
        const Rows rw(w, k);
        const size_t bytes = obb_linear_workspace_bytes(m, n, k, code, OBB_LINEAR_BACKWARD_INPUT);
        const at::Tensor ws = workspace(bytes, x);
        check_rc(obb_linear_backward_input(ptr(dz), ptr(rw.t), rw.ld, m, n, k, code, ptr(out[0]), ptr(ws), bytes, stream), "obb_linear_backward_input");
      }
      if (need & 2) {
        out[1] = at::empty({n, k}, x.options());
        const Rows rx(x, k);
        const size_t bytes = obb_linear_workspace_bytes(m, n, k, code, OBB_LINEAR_BACKWARD_WEIGHT);
        const at::Tensor ws = workspace(bytes, x);
        check_rc(obb_linear_backward_weight(ptr(dz), ptr(rx.t), rx.ld, m, n, k, code, ptr(out[1]), ptr(ws), bytes, stream), "obb_linear_backward_weight");
      }
      if (need & 8) out[3] = dz;
    }
    return once(std::move(out));
  }
};

at::Tensor linear(const at::Tensor &x, const at::Tensor &w, const MaybeTensor &bias, const MaybeTensor &res, int64_t act) {
  check_linear(x, w, bias, res, act);
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (bias && bias->requires_grad()) || (res && res->requires_grad())))
    return FusedLinear::apply(x, w, bias, res, act);
  return std::get<0>(linear_forward(x, w, bias, res, (int)act, false));
}

// under autocast the tensors are cast as those of torch's own linear layer are
at::Tensor cast(const at::Tensor &t, at::ScalarType type) { return code_of(t.scalar_type()) >= 0 ? t.to(type) : t; }

at::Tensor fused_linear(const at::Tensor &x_, const at::Tensor &w_, const MaybeTensor &bias_, const MaybeTensor &res_, int64_t act) {
  const at::Tensor x = turned(x_), w = turned(w_);
  const MaybeTensor bias = turned(bias_), res = turned(res_);
  if (x.is_cuda() && at::autocast::is_autocast_enabled(at::kCUDA)) {
    const auto type = at::autocast::get_autocast_dtype(at::kCUDA);
    c10::impl::ExcludeDispatchKeyGuard off(at::autocast::get_autocast_dispatch_key_from_device_type(at::kCUDA));
    const at::Tensor cx = cast(x, type), cw = cast(w, type);
    const MaybeTensor cb = bias ? MaybeTensor(cast(*bias, type)) : bias, cr = res ? MaybeTensor(cast(*res, type)) : res;
    return linear(cx, cw, cb, cr, act);
  }
  return linear(x, w, bias, res, act);
}

// ---- distillation ------------------------------------------------------------------------------------------------------
void check_distill(const at::Tensor &s, const at::Tensor &v, const at::Tensor &i, const MaybeTensor &weight) {
  TORCH_CHECK_TYPE(code_of(s.scalar_type()) >= 0 && code_of(v.scalar_type()) >= 0, "logits and teacher_values must be float32, bfloat16 or float16: got ", s.scalar_type(),
                   " and ", v.scalar_type());
  TORCH_CHECK_TYPE(i.scalar_type() == at::kLong || i.scalar_type() == at::kInt, "teacher_indices must be int64 or int32, but got ", i.scalar_type());
  bool same = s.dim() >= 1 && v.dim() == s.dim() && i.sizes() == v.sizes();
  for (int64_t d = 0; same && d + 1 < s.dim(); d++) same = v.size(d) == s.size(d);
  TORCH_CHECK_VALUE(same, "logits must be (..., C), teacher_values and teacher_indices (..., k): got ", s.sizes(), ", ", v.sizes(), " and ", i.sizes());
  TORCH_CHECK_VALUE(v.size(-1) <= OBB_DISTILL_MAX_K, "at most ", OBB_DISTILL_MAX_K, " teacher entries a row, but got ", v.size(-1));
  if (weight) {
    bool rows = weight->dim() == s.dim() - 1 && weight->is_floating_point();
    for (int64_t d = 0; rows && d < weight->dim(); d++) rows = weight->size(d) == s.size(d);
    TORCH_CHECK_VALUE(rows, "weight must be floating, one number a row of the logits: got ", weight->scalar_type(), " of ", weight->sizes());
    TORCH_CHECK_VALUE(!weight->requires_grad(), "weight is a constant: no gradient reaches it");
  }
  check_no_tangent("topk_distill_loss", {&s, weight ? &*weight : &s});
  for (const at::Tensor *t : {&s, &v, &i, weight ? &*weight : &s}) {
    TORCH_CHECK_NOT_IMPLEMENTED(t->is_cuda(), "topk_distill_loss runs on a HIP device only (a tensor is on ", t->device(), ")");
    TORCH_CHECK_VALUE(t->device() == s.device(), "logits are on ", s.device(), ", another tensor on ", t->device());
  }
}

// scale < 0: the rows' losses; else scale times their sum
struct TopkDistill : public torch::autograd::Function<TopkDistill> {
  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &logits, const at::Tensor &values, const at::Tensor &indices, const MaybeTensor &weight, double temperature,
                            double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t classes = logits.size(-1), rows = leading(logits), k = values.size(-1);
    HIPGuardMasqueradingAsCUDA guard(logits.device());
    const Rows s(logits, classes);
    const at::Tensor v = values.contiguous(), i = indices.contiguous();
    const at::Tensor w = weight ? weight->to(at::kFloat).contiguous() : at::Tensor();
    const auto f32 = logits.options().dtype(at::kFloat);
    const bool need = logits.requires_grad();
    at::Tensor row_loss = at::empty(logits.sizes().slice(0, logits.dim() - 1), f32);
    at::Tensor stats = need ? at::empty({rows, 2}, f32) : at::Tensor();
    at::Tensor total = scale < 0 ? at::Tensor() : at::empty({}, f32);
    const size_t bytes = obb_topk_distill_workspace_bytes(rows, classes);
    const at::Tensor ws = workspace(bytes, logits);
    check_rc(obb_topk_distill_forward(ptr(s.t), s.ld, rows, classes, code_of(logits.scalar_type()), ptr(v), ptr(i), (int)k, code_of(v.scalar_type()), (int)i.element_size(),
                                      (float)temperature, (const float *)ptr(w), (float *)ptr(row_loss), (float *)ptr(stats), scale < 0 ? 1.f : (float)scale, (float *)ptr(total),
                                      ptr(ws), bytes, stream_of(logits)),
             "obb_topk_distill_forward");
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["scale"] = scale;
    if (need) ctx->save_for_backward({logits, v, i, w, stats});
    return scale < 0 ? row_loss : total;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const double temperature = ctx->saved_data["temperature"].toDouble(), scale = ctx->saved_data["scale"].toDouble();
    const auto saved = ctx->get_saved_variables();
    variable_list out(6);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const at::Tensor logits = saved[0], v = saved[1], i = saved[2], w = saved[3], stats = saved[4];
      const int64_t classes = logits.size(-1), rows = leading(logits);
      HIPGuardMasqueradingAsCUDA guard(logits.device());
      check_capture(stream_of(logits));
      out[0] = at::empty(logits.sizes(), logits.options());
      if (out[0].numel() > 0) {
        const Rows s(logits, classes);
        const at::Tensor g = turned(grads[0]).to(at::kFloat).contiguous();
        check_rc(obb_topk_distill_backward(ptr(s.t), s.ld, rows, classes, code_of(logits.scalar_type()), ptr(v), ptr(i), (int)v.size(-1), code_of(v.scalar_type()),
                                           (int)i.element_size(), (float)temperature, (const float *)ptr(w), (const float *)ptr(stats), (const float *)ptr(g), scale < 0 ? 1 : 0,
                                           scale < 0 ? 1.f : (float)scale, ptr(out[0]), classes, stream_of(logits)),
                 "obb_topk_distill_backward");
      }
    }
    return once(std::move(out));
  }
};

at::Tensor topk_distill(const at::Tensor &logits, const at::Tensor &values, const at::Tensor &indices, double temperature, const MaybeTensor &weight, double scale) {
  check_distill(logits, values, indices, weight);
  // (the teacher's values are a constant: cut from whatever graph they come from)
  return TopkDistill::apply(turned(logits), turned(values.detach()), indices, turned(weight), temperature, scale);
}

}  // namespace

void bind_training_ops(py::module_ &m) {
  m.def("fused_linear", &fused_linear, "act(x @ weight.T + bias + residual)", py::arg("x"), py::arg("weight"), py::arg("bias") = py::none(), py::arg("residual") = py::none(),
        py::arg("act") = 0);
  m.def("topk_distill", &topk_distill, "distillation from a teacher's top logits: the rows' losses (scale < 0) or scale times their sum", py::arg("logits"),
        py::arg("teacher_values"), py::arg("teacher_indices"), py::arg("temperature") = 1.0, py::arg("weight") = py::none(), py::arg("scale") = -1.0);
}

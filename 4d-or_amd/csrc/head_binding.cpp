// head_binding.cpp — the torch side of the dense heads: argument checks, allocation and autograd nodes in C++ around the C entry
// points of pn2_hip.h (pointnet2_ops/head_ops.py is the public module).
//
// Why not ctypes like the other entry points: a training step of a scan-sized head is two kernels of 5 us, and its time is the host's.
// These nodes run on autograd's worker thread without the interpreter: forward and backward of the 72 x 256 -> 512 layer take 64 us
// (125 with nodes written in Python), 72 x 15 distillation 50 (100), one call without gradients 5 (11).  The entry points are those of
// the library that pointnet2_ops._ext has loaded: it hands their addresses over (bind), so there is one copy of the library and
// PN2_HIP_LIB stays in force.
#include <torch/extension.h>

#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <optional>
#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/pn2_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct {
  decltype(&pn2_linear_act_workspace_bytes) linear_bytes;
  decltype(&pn2_linear_act) linear;
  decltype(&pn2_linear_act_grad_workspace_bytes) linear_grad_bytes;
  decltype(&pn2_linear_act_grad) linear_grad;
  decltype(&pn2_label_logprobs_workspace_bytes) labels_bytes;
  decltype(&pn2_label_logprobs) labels;
  decltype(&pn2_label_logprobs_grad) labels_grad;
  decltype(&pn2_distill_topk_workspace_bytes) distill_bytes;
  decltype(&pn2_distill_topk) distill;
  decltype(&pn2_distill_topk_grad) distill_grad;
  decltype(&pn2_strerror) strerror;
  decltype(&pn2_last_hip_error) last_error;
  PyObject *timed;                                       // pointnet2_ops._ext._call: launches under the kernel timer
} lib;

// Look every entry point up by its name (address: pointnet2_ops._ext.address); called once, before anything else.
void bind(const py::function &address, py::object timed) {
  auto take = [&](auto &f, const char *name) { f = reinterpret_cast<std::decay_t<decltype(f)>>(address(name).cast<uintptr_t>()); };
  take(lib.linear_bytes, "pn2_linear_act_workspace_bytes");
  take(lib.linear, "pn2_linear_act");
  take(lib.linear_grad_bytes, "pn2_linear_act_grad_workspace_bytes");
  take(lib.linear_grad, "pn2_linear_act_grad");
  take(lib.labels_bytes, "pn2_label_logprobs_workspace_bytes");
  take(lib.labels, "pn2_label_logprobs");
  take(lib.labels_grad, "pn2_label_logprobs_grad");
  take(lib.distill_bytes, "pn2_distill_topk_workspace_bytes");
  take(lib.distill, "pn2_distill_topk");
  take(lib.distill_grad, "pn2_distill_topk_grad");
  take(lib.strerror, "pn2_strerror");
  take(lib.last_error, "pn2_last_hip_error");
  lib.timed = timed.release().ptr();                     // kept for the life of the process
}

// Enqueue f(stream) on the current stream of t's device.  `timed`: by way of the kernel timer, with the algorithm's bytes and
// operations (a call made while the timer runs is recorded, and so is its backward pass).
template <class F> void launch(const char *name, const Tensor &t, bool timed, double bytes, double flops, F f) {
  if (timed) {
    const py::gil_scoped_acquire gil;
    using namespace py::literals;
    py::reinterpret_borrow<py::object>(lib.timed)(name, t, "alg_bytes"_a = bytes, "alg_flops"_a = flops,
                                                  "fn"_a = py::cpp_function([&f](uintptr_t s) { return f((void *)s); }));
    return;
  }
  const c10::DeviceGuard guard(t.device());
  const int rc = f((void *)c10::hip::getCurrentHIPStream(t.device().index()).stream());
  TORCH_CHECK(rc == PN2_OK, name, " failed: ", lib.strerror(rc), " (rc=", rc, ", hipError=", lib.last_error(), ")");
}

Tensor workspace(size_t bytes, const Tensor &like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

int dtype_code(const Tensor &t, const char *name) {
  switch (t.scalar_type()) {
    case at::kFloat: return PN2_DT_F32;
    case at::kBFloat16: return PN2_DT_BF16;
    case at::kHalf: return PN2_DT_F16;
    default: TORCH_CHECK(false, name, " must be a float32, bfloat16 or float16 tensor");
  }
}
at::ScalarType slope_type(at::ScalarType t) { return t == at::kFloat ? at::kFloat : at::kShort; }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
template <class T> T *ptr_as(const Tensor &t) { return static_cast<T *>(ptr(t)); }

// (..., C) -> (rows, C) with a contiguous last axis; a copy only where the strides allow no view
Tensor matrix(const Tensor &t, const char *name) {
  TORCH_CHECK(t.dim() >= 1, name, " must be a tensor with at least one axis");
  const int64_t c = t.size(-1);
  TORCH_CHECK(c >= 1, name, " must have at least one column");
  const Tensor m = t.dim() == 2 ? t : t.reshape({t.numel() / c, c});
  return (c == 1 || m.stride(1) == 1 ? m : m.contiguous()).resolve_neg();
}
int64_t row_stride(const Tensor &m) { return m.size(0) > 1 ? m.stride(0) : m.size(1); }

// A launch goes around torch's dispatcher, so what the dispatcher would do beside it has to be refused here, or it would be left out
// without a word: the tangent of a forward-mode dual tensor, the node of a recorded graph (which would hold the outputs' allocation and
// no kernel), the code of a tensor subclass, the values of a tensor without memory of its own.
void check_plain(const char *op, std::initializer_list<std::pair<const Tensor *, const char *>> inputs) {
  bool recorded = torch::jit::tracer::isTracing();
  if (c10::impl::TorchDispatchModeTLS::any_modes_set()) {
    using c10::impl::TorchDispatchModeKey;
    for (const auto key : {TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL, TorchDispatchModeKey::FAKE})
      recorded |= c10::impl::TorchDispatchModeTLS::get_mode(key).has_value();
  }
  recorded |= c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
  TORCH_CHECK(!recorded, op, " cannot be recorded (torch.jit.trace, make_fx, export): its kernels run outside torch's dispatcher");
  const bool forward_mode = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (const auto &[t, name] : inputs) {
    if (!t->defined()) continue;
    TORCH_CHECK(!t->unsafeGetTensorImpl()->is_python_dispatch(), name, " must be a plain tensor, not a subclass with __torch_dispatch__");
    TORCH_CHECK(!forward_mode || !t->_fw_grad(0).defined(), op, " has no forward-mode derivative (", name, " is a dual tensor)");
    TORCH_CHECK(t->layout() == at::kStrided && t->has_storage() && (t->numel() == 0 || t->storage().data()), name,
                " must be a dense tensor with memory of its own");
  }
}

void check_device(const Tensor &lead, std::initializer_list<std::pair<const Tensor *, const char *>> others) {
  TORCH_CHECK(lead.is_cuda(), "CPU not supported");
  for (const auto &[t, name] : others) {
    if (!t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t->device() == lead.device(), name, " must be on ", lead.device());
  }
}

// A backward pass that is being captured must not go on to a node of a stream outside the capture: torch would make that stream wait
// for the captured one, which breaks the capture and can end the process.  It comes about where an eager graph of the same leaves is
// still alive, because the node that accumulates a leaf's gradient belongs to the stream of the leaf's first living graph.  Called on
// the node's own stream; looks at what lies behind the node (captures only).
void check_capture(const char *op) {
  auto capturing = [](hipStream_t s) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(s, &status) != hipSuccess) (void)hipGetLastError();
    return status != hipStreamCaptureStatusNone;
  };
  const auto here = c10::hip::getCurrentHIPStream();
  if (!capturing(here.stream())) return;
  using torch::autograd::Node;
  const auto first = torch::autograd::get_current_node();
  std::vector<Node *> todo;
  std::unordered_set<Node *> seen;
  if (first) todo.push_back(first.get());
  while (!todo.empty()) {
    Node *node = todo.back();
    todo.pop_back();
    for (const auto &edge : node->next_edges()) {
      Node *next = edge.function.get();
      if (!next || !seen.insert(next).second) continue;
      todo.push_back(next);
      const auto s = next->stream();
      if (!s || s->device_index() != here.device_index() || s->id() == here.id()) continue;
      // (the default stream is never captured; another one may have joined the capture)
      const bool joined = s->id() != 0 && capturing(c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED,
                                                                         c10::Stream(c10::Stream::UNSAFE, here.device(), s->id())).stream());
      TORCH_CHECK(joined, op, "'s backward pass is being captured while an eager graph of the same leaves is alive on another stream: "
                              "drop what holds that graph first, or give the captured pass leaves of its own (detach)");
    }
  }
}

// Each operator is differentiable once: where a graph of the backward pass is being built (create_graph), its results raise when
// they are differentiated.
variable_list once(variable_list out) {
  if (!at::GradMode::is_enabled()) return out;
  variable_list defined;
  for (const auto &t : out)
    if (t.defined()) defined.push_back(t.detach().set_requires_grad(true));
  if (defined.empty()) return out;
  const int n = (int)defined.size();
  defined = torch::autograd::DelayedError("trying to differentiate twice a function that can be differentiated once", n)
                .apply(std::move(defined));
  size_t next = 0;
  for (auto &t : out)
    if (t.defined()) t = defined[next++];
  return out;
}

// ------------------------------------------------------------------------------------------------------------ linear_act
struct LinearOut { Tensor y, slope; };
LinearOut run_linear(const Tensor &x, const Tensor &w, const Tensor &b, const Tensor &r, int64_t act, bool want_slope, bool timed) {
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  const int dt = dtype_code(x, "x");
  LinearOut o;
  o.y = at::empty({M, N}, x.options());
  if (want_slope && act) o.slope = at::empty({M, N}, x.options().dtype(slope_type(x.scalar_type())));
  if (M == 0) return o;
  const int64_t ldx = row_stride(x), ldw = row_stride(w);
  const size_t bytes = lib.linear_bytes(M, (int)N, (int)K, dt, x.data_ptr(), ldx, w.data_ptr(), ldw);
  const Tensor ws = workspace(bytes, x);
  const double es = x.element_size(), m = M, n = N, k = K;
  launch("pn2_linear_act", x, timed, es * (m * k + n * k + m * n * (1 + r.defined() + o.slope.defined())), 2 * m * n * k, [&](void *stream) {
    return lib.linear(M, (int)N, (int)K, dt, x.data_ptr(), ldx, w.data_ptr(), ldw, ptr(b), b.defined() ? dtype_code(b, "bias") : dt, (int)act,
                      ptr(r), r.defined() ? row_stride(r) : 0, o.y.data_ptr(), ptr(o.slope), ptr(ws), bytes, stream);
  });
  return o;
}

struct LinearAct : torch::autograd::Function<LinearAct> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const std::optional<Tensor> &bias,
                        const std::optional<Tensor> &residual, int64_t act, bool timed) {
    const Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
    const bool dx = x.requires_grad(), dw = w.requires_grad(), db = b.defined() && b.requires_grad();
    LinearOut o = run_linear(x, w, b, r, act, dx || dw || db, timed);
    ctx->save_for_backward({dw ? x : Tensor(), dx ? w : Tensor(), o.slope});
    ctx->saved_data["need"] = (int64_t)(dx | dw << 1 | db << 2 | (r.defined() && r.requires_grad()) << 3);
    ctx->saved_data["k"] = x.size(1);
    ctx->saved_data["timed"] = timed;
    ctx->saved_data["bias"] = (int64_t)(b.defined() ? b.scalar_type() : x.scalar_type());
    return o.y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    check_capture("linear_act");
    const int64_t need = ctx->saved_data["need"].toInt(), K = ctx->saved_data["k"].toInt();
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &slope = saved[2];
    Tensor dx, dw, db;
    if (need & 7) {
      check_plain("linear_act's gradient", {{&grads[0], "dy"}});
      const Tensor dy = matrix(grads[0], "dy");
      const int64_t M = dy.size(0), N = dy.size(1);
      const int dt = dtype_code(dy, "dy");
      const auto bias_type = (at::ScalarType)ctx->saved_data["bias"].toInt();
      auto make = [&](at::IntArrayRef shape, at::ScalarType t) {
        return M ? at::empty(shape, dy.options().dtype(t)) : at::zeros(shape, dy.options().dtype(t));
      };
      if (need & 1) dx = make({M, K}, dy.scalar_type());
      if (need & 2) dw = make({N, K}, dy.scalar_type());
      if (need & 4) db = make({N}, bias_type);
      if (M) {
        const int64_t ldy = row_stride(dy), ldx = x.defined() ? row_stride(x) : 0, ldw = w.defined() ? row_stride(w) : 0;
        const size_t bytes = lib.linear_grad_bytes(M, (int)N, (int)K, dt, dy.data_ptr(), ldy, slope.defined(), ptr(x), ldx, ptr(w), ldw,
                                                   (int)(need & 7));
        const Tensor ws = workspace(bytes, dy);
        const double es = dy.element_size(), m = M, n = N, k = K, products = dx.defined() + dw.defined();
        launch("pn2_linear_act_grad", dy, ctx->saved_data["timed"].toBool(), es * (m * n * (1 + slope.defined()) + (m * k + n * k) * products),
               2 * m * n * k * products, [&](void *stream) {
                 return lib.linear_grad(M, (int)N, (int)K, dt, dy.data_ptr(), ldy, ptr(slope), ptr(x), ldx, ptr(w), ldw, ptr(dx), ptr(dw),
                                        ptr(db), bias_type == at::kFloat ? PN2_DT_F32 : dt, ptr(ws), bytes, stream);
               });
      }
    }
    return once({dx, dw, db, need & 8 ? grads[0] : Tensor(), Tensor(), Tensor()});
  }
};

Tensor linear_act(const Tensor &x, const Tensor &weight, const std::optional<Tensor> &bias, int64_t act,
                  const std::optional<Tensor> &residual, bool timed) {
  const Tensor none;
  check_plain("linear_act", {{&x, "x"}, {&weight, "weight"}, {bias ? &*bias : &none, "bias"}, {residual ? &*residual : &none, "residual"}});
  const Tensor xm = matrix(x, "x");
  dtype_code(xm, "x");
  const int64_t K = xm.size(1);
  TORCH_CHECK(weight.dim() == 2 && weight.size(1) == K, "weight must have shape (N, ", K, ")");
  const int64_t N = weight.size(0);
  TORCH_CHECK(N >= 1, "weight must have at least one row");
  TORCH_CHECK(weight.scalar_type() == x.scalar_type(), "weight must have the type of x (", x.dtype(), ")");
  const Tensor wm = matrix(weight, "weight");
  Tensor b, r;
  if (bias) {
    b = bias->resolve_neg();
    TORCH_CHECK(b.dim() == 1 && b.size(0) == N && b.is_contiguous(), "bias must be a contiguous tensor of shape (", N, ",)");
    TORCH_CHECK(b.scalar_type() == x.scalar_type() || b.scalar_type() == at::kFloat, "bias must have the type of x (", x.dtype(),
                ") or float32");
  }
  auto shape = x.sizes().vec();
  shape.back() = N;
  if (residual) {
    TORCH_CHECK(residual->scalar_type() == x.scalar_type(), "residual must have the type of x (", x.dtype(), ")");
    bool fits = residual->dim() <= (int64_t)shape.size();
    for (int64_t n = 1; fits && n <= residual->dim(); ++n) fits = residual->size(-n) == shape[shape.size() - n] || residual->size(-n) == 1;
    TORCH_CHECK(fits, "residual must broadcast to ", at::IntArrayRef(shape));
    r = matrix(residual->expand(shape), "residual");
  }
  TORCH_CHECK(N <= (1 << 22) && K <= (1 << 22), "weight must have at most 4194304 rows and columns");
  check_device(xm, {{&wm, "weight"}, {&b, "bias"}, {&r, "residual"}});
  const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad()) ||
                                                   (residual && residual->requires_grad()));
  Tensor y = grad ? LinearAct::apply(xm, wm, bias ? std::make_optional(b) : std::nullopt, residual ? std::make_optional(r) : std::nullopt, act,
                                    timed)
                  : run_linear(xm, wm, b, r, act, false, timed).y;
  return x.dim() == 2 ? y : y.view(shape);
}

// ------------------------------------------------------------------------------------------------------- label_log_probs
struct Labels { Tensor log_prob, entropy, top_log_prob, top_index, stats; };
Labels run_labels(const Tensor &x, const Tensor &y, int64_t top, int64_t ignore, bool want_stats, bool timed) {
  const int64_t T = x.size(0), V = x.size(1);
  const auto f32 = x.options().dtype(at::kFloat);
  Labels o;
  o.log_prob = at::empty({T}, f32);
  o.entropy = at::empty({T}, f32);
  if (top) {
    o.top_log_prob = at::empty({T, top}, f32);
    o.top_index = at::empty({T, top}, x.options().dtype(at::kLong));
  }
  if (want_stats) o.stats = at::empty({T, 2}, f32);
  if (T == 0) return o;
  const int dt = dtype_code(x, "logits");
  const size_t bytes = lib.labels_bytes(T, (int)V, dt, (int)top);
  const Tensor ws = workspace(bytes, x);
  launch("pn2_label_logprobs", x, timed, (double)T * V * x.element_size() + T * (16.0 + 12.0 * top), 0, [&](void *stream) {
    return lib.labels(T, (int)V, row_stride(x), dt, x.data_ptr(), ptr_as<long long>(y), ignore, (int)top, ptr_as<float>(o.log_prob),
                      ptr_as<float>(o.entropy), ptr_as<float>(o.stats), ptr_as<float>(o.top_log_prob), ptr_as<long long>(o.top_index),
                      ptr(ws), bytes, stream);
  });
  return o;
}
Tensor grad_rows(const Tensor &g) {                    // the gradient of a row statistic, or undefined
  return g.defined() ? g.contiguous().resolve_neg() : g;
}

struct LabelLogProbs : torch::autograd::Function<LabelLogProbs> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &y, int64_t top, int64_t ignore, bool timed) {
    Labels o = run_labels(x, y, top, ignore, true, timed);
    ctx->saved_data["timed"] = timed;
    ctx->save_for_backward({x, y, o.stats, o.entropy});
    ctx->saved_data["ignore"] = ignore;
    ctx->set_materialize_grads(false);
    if (!top) return {o.log_prob, o.entropy};
    ctx->mark_non_differentiable({o.top_log_prob, o.top_index});
    return {o.log_prob, o.entropy, o.top_log_prob, o.top_index};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    check_capture("label_log_probs");
    check_plain("label_log_probs' gradient", {{&grads[0], "the gradient of log_prob"}, {&grads[1], "the gradient of entropy"}});
    const Tensor g = grad_rows(grads[0]), h = grad_rows(grads[1]);
    Tensor dx;
    if (g.defined() || h.defined()) {
      const auto saved = ctx->get_saved_variables();
      const Tensor &x = saved[0], &y = saved[1], &stats = saved[2], &entropy = saved[3];
      const int64_t T = x.size(0), V = x.size(1);
      dx = at::empty({T, V}, x.options());
      if (T)
        launch("pn2_label_logprobs_grad", x, ctx->saved_data["timed"].toBool(), 2.0 * T * V * x.element_size(), 0, [&](void *stream) {
          return lib.labels_grad(T, (int)V, row_stride(x), dtype_code(x, "logits"), x.data_ptr(), ptr_as<long long>(y),
                                 ctx->saved_data["ignore"].toInt(), ptr_as<float>(stats), ptr_as<float>(entropy), ptr_as<float>(g),
                                 ptr_as<float>(h), dx.data_ptr(), stream);
        });
    }
    return once({dx, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

std::tuple<Tensor, Tensor, std::optional<Tensor>, std::optional<Tensor>> label_log_probs(const Tensor &logits, const Tensor &labels,
                                                                                         int64_t top, int64_t ignore, bool timed) {
  check_plain("label_log_probs", {{&logits, "logits"}, {&labels, "labels"}});
  const Tensor x = matrix(logits, "logits");
  dtype_code(x, "logits");
  TORCH_CHECK(labels.scalar_type() == at::kLong, "labels must be a long tensor");
  const auto shape = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK(labels.sizes() == shape, "labels must be a tensor of shape ", shape);
  const int64_t V = x.size(1), most = V < 64 ? V : 64;
  TORCH_CHECK(V <= 0x7fffffff && x.size(0) <= 0x7fffffff, "logits must have fewer than 2^31 rows and columns");
  TORCH_CHECK(top >= 0 && top <= most, "top must lie in 0 .. min(columns, 64)");
  const Tensor y = labels.reshape({x.size(0)}).contiguous();
  check_device(x, {{&y, "labels"}});
  Tensor lp, ent, tlp, tix;
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    const variable_list o = LabelLogProbs::apply(x, y, top, ignore, timed);
    lp = o[0];
    ent = o[1];
    if (top) { tlp = o[2]; tix = o[3]; }
  } else {
    Labels o = run_labels(x, y, top, ignore, false, timed);
    lp = o.log_prob;
    ent = o.entropy;
    tlp = o.top_log_prob;
    tix = o.top_index;
  }
  if (logits.dim() != 2) {
    lp = lp.view(shape);
    ent = ent.view(shape);
    if (top) {
      auto wide = shape.vec();
      wide.push_back(top);
      tlp = tlp.view(wide);
      tix = tix.view(wide);
    }
  }
  if (!top) return {lp, ent, std::nullopt, std::nullopt};
  return {lp, ent, tlp, tix};
}

// --------------------------------------------------------------------------------------------------------- distill_top_k
std::pair<Tensor, Tensor> run_distill(const Tensor &x, const Tensor &index, const Tensor &values, double t, bool want_stats, bool timed) {
  const int64_t T = x.size(0), V = x.size(1);
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor loss = at::empty({T}, f32), stats;
  if (want_stats) stats = at::empty({T, 4}, f32);
  if (T == 0) return {loss, stats};
  const int dt = dtype_code(x, "logits");
  const size_t bytes = lib.distill_bytes(T, (int)V, dt);
  const Tensor ws = workspace(bytes, x);
  launch("pn2_distill_topk", x, timed, (double)T * V * x.element_size(), 0, [&](void *stream) {
    return lib.distill(T, (int)V, row_stride(x), dt, x.data_ptr(), (int)index.size(1), ptr_as<long long>(index),
                       dtype_code(values, "teacher_logits"), values.data_ptr(), (float)t, ptr_as<float>(loss), ptr_as<float>(stats),
                       ptr(ws), bytes, stream);
  });
  return {loss, stats};
}

struct DistillTopK : torch::autograd::Function<DistillTopK> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &index, const Tensor &values, double t, bool timed) {
    auto [loss, stats] = run_distill(x, index, values, t, true, timed);
    ctx->saved_data["timed"] = timed;
    ctx->save_for_backward({x, index, values, stats});
    ctx->saved_data["t"] = t;
    return loss;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    check_capture("distill_top_k");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &index = saved[1], &values = saved[2], &stats = saved[3];
    check_plain("distill_top_k's gradient", {{&grads[0], "the gradient of the loss"}});
    const Tensor g = grad_rows(grads[0]);
    const int64_t T = x.size(0), V = x.size(1);
    Tensor dx = at::empty({T, V}, x.options());
    if (T)
      launch("pn2_distill_topk_grad", x, ctx->saved_data["timed"].toBool(), 2.0 * T * V * x.element_size(), 0, [&](void *stream) {
        return lib.distill_grad(T, (int)V, row_stride(x), dtype_code(x, "logits"), x.data_ptr(), (int)index.size(1), ptr_as<long long>(index),
                                dtype_code(values, "teacher_logits"), values.data_ptr(), (float)ctx->saved_data["t"].toDouble(),
                                ptr_as<float>(stats), ptr_as<float>(g), dx.data_ptr(), stream);
      });
    return once({dx, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor distill_top_k(const Tensor &logits, const Tensor &teacher_index, const Tensor &teacher_logits, double temperature, bool timed) {
  check_plain("distill_top_k", {{&logits, "logits"}, {&teacher_index, "teacher_index"}, {&teacher_logits, "teacher_logits"}});
  const Tensor x = matrix(logits, "logits");
  dtype_code(x, "logits");
  TORCH_CHECK(teacher_index.scalar_type() == at::kLong, "teacher_index must be a long tensor");
  dtype_code(teacher_logits, "teacher_logits");
  const auto shape = logits.sizes().slice(0, logits.dim() - 1);
  for (const auto &[t, name] : {std::pair<const Tensor &, const char *>(teacher_index, "teacher_index"), {teacher_logits, "teacher_logits"}})
    TORCH_CHECK(t.dim() == logits.dim() && t.sizes().slice(0, t.dim() - 1) == shape, name, " must be a tensor of shape ", shape, " + (k,)");
  const int64_t k = teacher_index.size(-1);
  TORCH_CHECK(k >= 1 && k <= 0x7fffffff && teacher_logits.size(-1) == k, "teacher_index and teacher_logits must have shape ", shape,
              " + (k,), k >= 1");
  TORCH_CHECK(!teacher_logits.requires_grad(), "teacher_logits must not require a gradient (detach the teacher)");
  TORCH_CHECK(temperature > 0 && std::isfinite((float)temperature) && (float)temperature > 0, "temperature must be positive and finite");
  TORCH_CHECK(x.size(1) <= 0x7fffffff && x.size(0) <= 0x7fffffff, "logits must have fewer than 2^31 rows and columns");
  const Tensor index = teacher_index.reshape({x.size(0), k}).contiguous(), values = teacher_logits.reshape({x.size(0), k}).contiguous().resolve_neg();
  check_device(x, {{&index, "teacher_index"}, {&values, "teacher_logits"}});
  Tensor loss = at::GradMode::is_enabled() && logits.requires_grad() ? DistillTopK::apply(x, index, values, temperature, timed)
                                                                     : run_distill(x, index, values, temperature, false, timed).first;
  return logits.dim() == 2 ? loss : loss.view(shape);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  const py::call_guard<py::gil_scoped_release> free;
  m.def("linear_act", &linear_act, free);
  m.def("label_log_probs", &label_log_probs, free);
  m.def("distill_top_k", &distill_top_k, free);
}

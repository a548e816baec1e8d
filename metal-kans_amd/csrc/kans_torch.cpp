// residual_norm, linear_cross_entropy, embedding, dropout, causal_conv and selective_scan on torch tensors as autograd nodes around
// the library's entry points, and the optimizer's way through its parameters (host code, a Python module of its own).
//
// Small calls wait for the host, not for the GPU: torch runs a backward in a thread of its own, and each turn through the
// interpreter there starts with cold caches.  A forward and backward of 2047 x 1000 fp32 (36 us of kernels) took 165 us
// with both directions in Python, of which an empty Python autograd function takes 71; here 98.
//
// The library is bound by address (bind), so this module has no link to it and no HIP call of its own.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <cfloat>
#include <climits>
#include <cmath>
#include <limits>
#include <mutex>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "../../include/kans_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---- the library -----------------------------------------------------------------------------------
struct Library {
  decltype(&kans_last_error) last_error;
  decltype(&kans_stream_keep) stream_keep;
  decltype(&kans_residual_norm_forward) norm_forward;
  decltype(&kans_residual_norm_workspace) norm_workspace;
  decltype(&kans_residual_norm_backward) norm_backward;
  decltype(&kans_linear_xent_workspace) xent_workspace;
  decltype(&kans_linear_xent_forward) xent_forward;
  decltype(&kans_linear_xent_backward) xent_backward;
  decltype(&kans_adamw_step) adamw_step;
  decltype(&kans_embedding_forward) embedding_forward;
  decltype(&kans_embedding_workspace) embedding_workspace;
  decltype(&kans_embedding_backward) embedding_backward;
  decltype(&kans_dropout) dropout;
  decltype(&kans_causal_conv_forward) conv_forward;
  decltype(&kans_causal_conv_workspace) conv_workspace;
  decltype(&kans_causal_conv_backward) conv_backward;
  decltype(&kans_selective_scan_saved) scan_saved;
  decltype(&kans_selective_scan_workspace) scan_workspace;
  decltype(&kans_selective_scan_forward) scan_forward;
  decltype(&kans_selective_scan_backward) scan_backward;
} lib;
PyObject* kans_error;  // the package's exception for a negative code

struct Failure : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void check(long code, const char* what) {
  if (code < 0) throw Failure(std::string(what) + " failed with code " + std::to_string(code) + ": " + lib.last_error());
}

void bind(const py::dict& functions, py::object error) {
  auto get = [&](const char* name, auto& f) {
    f = reinterpret_cast<std::decay_t<decltype(f)>>(functions[name].cast<uintptr_t>());
  };
  get("kans_last_error", lib.last_error);
  get("kans_stream_keep", lib.stream_keep);
  get("kans_residual_norm_forward", lib.norm_forward);
  get("kans_residual_norm_workspace", lib.norm_workspace);
  get("kans_residual_norm_backward", lib.norm_backward);
  get("kans_linear_xent_workspace", lib.xent_workspace);
  get("kans_linear_xent_forward", lib.xent_forward);
  get("kans_linear_xent_backward", lib.xent_backward);
  get("kans_adamw_step", lib.adamw_step);
  get("kans_embedding_forward", lib.embedding_forward);
  get("kans_embedding_workspace", lib.embedding_workspace);
  get("kans_embedding_backward", lib.embedding_backward);
  get("kans_dropout", lib.dropout);
  get("kans_causal_conv_forward", lib.conv_forward);
  get("kans_causal_conv_workspace", lib.conv_workspace);
  get("kans_causal_conv_backward", lib.conv_backward);
  get("kans_selective_scan_saved", lib.scan_saved);
  get("kans_selective_scan_workspace", lib.scan_workspace);
  get("kans_selective_scan_forward", lib.scan_forward);
  get("kans_selective_scan_backward", lib.scan_backward);
  kans_error = error.release().ptr();
}

// ---- tensors ---------------------------------------------------------------------------------------
// The library's handle of torch's current stream.  Streams of torch's own live until the process ends, so the library may
// name them later; an external one (its id is its handle) it may not.
void* stream_of(const Tensor& t) {
  static std::mutex mutex;
  static std::unordered_set<void*> kept;
  const auto s = c10::hip::getCurrentHIPStream(t.get_device());
  void* h = s.stream();
  if (!h) return KANS_STREAM_LEGACY;  // (0 is the library's own stream)
  if ((uintptr_t)s.id() != (uintptr_t)h) {
    std::lock_guard<std::mutex> lock(mutex);
    if (!kept.count(h)) {
      check(lib.stream_keep(h), "kans_stream_keep");
      kept.insert(h);
    }
  }
  return h;
}

int type_of(at::ScalarType t) {
  return t == at::kFloat ? KANS_DT_F32 : t == at::kHalf ? KANS_DT_F16 : t == at::kBFloat16 ? KANS_DT_BF16 : -1;
}
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor contiguous(const std::optional<Tensor>& t) { return t ? t->contiguous() : Tensor(); }
Tensor bytes(const Tensor& like, long n) { return at::empty({n}, like.options().dtype(at::kByte)); }
bool wants_grad(std::initializer_list<const Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : inputs)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Results are written through pointers, which a tracer does not see: its graph would hold uninitialized memory.
void not_traced(const char* what) {
  const bool traced = torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
                      c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value();
  TORCH_CHECK(!traced, what, " cannot be traced: its kernels are not operators of torch's dispatcher");
}

// The nodes below differentiate backwards; a tangent would be lost without a word where no input requires grad.
void no_tangents(std::initializer_list<const Tensor*> inputs, const char* what) {
  for (const Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative");
}

// A backward under capture hands its gradients to the streams of the nodes before it.  Where one of these is the default
// stream -- an eager graph of the same leaf still lives and with it the node that collects the leaf's gradient -- the
// capture is torn and the process ends at its end: refused here, while there is a call to name.
bool capturing(c10::DeviceIndex device) {
  const auto current = c10::hip::getCurrentHIPStream(device);
  if (!current.stream()) return false;  // (the default stream is never under capture)
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(current.stream(), &status) == hipSuccess && status != hipStreamCaptureStatusNone;
}
void refuse_default_stream(torch::autograd::Node* node, const char* what) {
  const auto stream = node ? node->stream() : std::nullopt;
  TORCH_CHECK(!stream || stream->id() != 0, what,
              " under a graph capture: an autograd graph from outside of it, on the default stream, still holds an input; delete it first");
}

// In the forward: the nodes of the inputs as they are given.  (A copy in another layout has a node of its own.)
void capturable(std::initializer_list<const Tensor*> inputs, const char* what) {
  for (const Tensor* t : inputs) {
    if (!t->defined() || !t->requires_grad()) continue;
    if (!capturing(t->get_device())) return;
    refuse_default_stream((t->grad_fn() ? t->grad_fn() : torch::autograd::impl::try_get_grad_accumulator(*t)).get(), what);
  }
}

// In the backward, before it hands anything on: all nodes that its gradients reach.
void capturable_behind(const Tensor& grad, const char* what) {
  if (!capturing(grad.get_device())) return;
  const auto self = torch::autograd::get_current_node();
  std::vector<torch::autograd::Node*> next{self.get()};
  std::unordered_set<torch::autograd::Node*> seen;
  while (!next.empty()) {
    torch::autograd::Node* const node = next.back();
    next.pop_back();
    if (!node || !seen.insert(node).second) continue;
    if (node != self.get()) refuse_default_stream(node, what);
    for (uint32_t i = 0; i < node->num_outputs(); ++i)
      if (node->task_should_compute_output(i)) next.push_back(node->next_edge(i).function.get());
  }
}

// Gradients that cannot be differentiated again: an error to whoever tries, where the graph is kept for it.
variable_list once(variable_list grads, bool graph) {
  variable_list given;
  for (auto& g : grads)
    if (graph && g.defined()) given.push_back(g.detach().requires_grad_(true));
  if (given.empty()) return grads;
  const auto node = std::make_shared<torch::autograd::DelayedError>("metal_kans' torch operators have no second derivative",
                                                                   (int64_t)given.size());
  variable_list out = (*node)(std::move(given));
  size_t at = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[at++];
  return grads;
}

// ---- residual_norm ---------------------------------------------------------------------------------
struct Norm {
  Tensor x, block, gate, post, pre, dev;  // (undefined: not given)
  double scale;
  int64_t group;                          // rows that share a gate row
  int kind;
  double eps;
  at::ScalarType dt;                      // of the block

  long columns() const { return x.size(-1); }
  long rows() const { return x.numel() / columns(); }

  std::tuple<Tensor, Tensor, Tensor> forward(bool want_stats) const {
    Tensor y = block.defined() ? at::empty_like(x) : Tensor();
    Tensor h = at::empty(x.sizes(), x.options().dtype(dt));
    Tensor stats = want_stats ? at::empty({rows(), 2 + 2 * kind}, x.options().dtype(at::kFloat)) : Tensor();
    check(lib.norm_forward(type_of(x.scalar_type()), type_of(dt), kind, data(x), data(block), data(gate), group, data(post), data(pre),
                           (const float*)data(dev), scale, eps, data(y), data(h), (float*)data(stats), rows(), (int)columns(),
                           stream_of(x)),
          "kans_residual_norm_forward");
    return {y, h, stats};
  }

  // Gradients of the six inputs, undefined where need is false.
  variable_list backward(const Tensor& stats, Tensor dy, Tensor dh, const std::array<bool, 6>& need, at::IntArrayRef gate_shape) const {
    if (dy.defined()) dy = dy.contiguous();
    if (dh.defined()) dh = dh.contiguous();
    const Tensor* inputs[6] = {&x, &block, &gate, &post, &pre, &dev};
    variable_list d(6);
    // a gate that repeats in another way than by rows: its gradient is summed below, in fp32
    const bool wide = !gate_shape.empty() && need[2];
    for (int i = 0; i < 6; ++i)
      if (need[i] && inputs[i]->defined())
        d[i] = i == 2 && wide ? at::empty(x.sizes(), x.options().dtype(at::kFloat)) : at::empty_like(*inputs[i]);
    if (rows() == 0) {
      for (auto& g : d)
        if (g.defined()) g.zero_();
    } else {
      const long size = lib.norm_workspace(rows(), (int)columns(), gate.defined() ? group : 0);
      check(size, "kans_residual_norm_workspace");
      const Tensor ws = bytes(x, size);
      check(lib.norm_backward(type_of(x.scalar_type()), type_of(dt), kind, data(x), data(block), data(gate), group, data(post),
                              data(pre), (const float*)data(dev), scale, eps, (const float*)data(stats), data(dy), data(dh), data(d[0]),
                              data(d[1]), data(d[2]), wide, data(d[3]), data(d[4]), (float*)data(d[5]), rows(), (int)columns(),
                              data(ws), size, stream_of(x)),
            "kans_residual_norm_backward");
    }
    if (wide) d[2] = at::sum_to(d[2], gate_shape).to(dt);
    return d;
  }
};

struct NormFunction : torch::autograd::Function<NormFunction> {
  typedef std::optional<Tensor> Maybe;
  static variable_list forward(AutogradContext* ctx, Tensor x, Maybe block_, Maybe gate_, Maybe post_, Maybe pre_, Maybe dev_,
                               double scale, int64_t group, int64_t kind, double eps, int64_t dt) {
    auto given = [](Maybe& t) { return t ? *t : Tensor(); };
    Tensor block = given(block_), gate = given(gate_), post = given(post_), pre = given(pre_), dev = given(dev_);
    std::vector<int64_t> gate_shape;
    if (gate.defined() && group == 0) {  // repeats within a row or over leading dimensions
      gate_shape = gate.sizes().vec();
      gate = gate.expand(x.sizes()).contiguous();
      group = 1;
    }
    const Norm n{x, block, gate, post, pre, dev, scale, group, (int)kind, eps, (at::ScalarType)dt};
    auto [y, h, stats] = n.forward(true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, block, gate, post, pre, dev, stats});
    ctx->saved_data["numbers"] = std::vector<double>{scale, eps};
    std::vector<int64_t> rest{group, kind, dt};
    rest.insert(rest.end(), gate_shape.begin(), gate_shape.end());
    ctx->saved_data["rest"] = rest;
    if (y.defined()) return {y, h};
    return {h};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    const auto s = ctx->get_saved_variables();
    const auto numbers = ctx->saved_data["numbers"].toDoubleVector();
    const auto rest = ctx->saved_data["rest"].toIntVector();
    variable_list d(11);
    const Tensor dy = grads.size() == 2 ? grads[0] : Tensor(), dh = grads.back();
    if (!dy.defined() && !dh.defined()) return d;
    no_tangents({&dy, &dh}, "residual_norm's backward");
    capturable_behind(dy.defined() ? dy : dh, "residual_norm's backward");
    const Norm n{s[0], s[1], s[2], s[3], s[4], s[5], numbers[0], rest[0], (int)rest[1], numbers[1], (at::ScalarType)rest[2]};
    std::array<bool, 6> need;
    for (size_t i = 0, edge = 0; i < 6; ++i) need[i] = s[i].defined() && ctx->needs_input_grad(edge++);
    const variable_list six = once(n.backward(s[6], dy, dh, need, at::IntArrayRef(rest).slice(3)), graph);
    std::copy(six.begin(), six.end(), d.begin());
    return d;
  }
};

// The gate as rows that each serve `group` consecutive rows of x; group 0: it repeats in another way (over a
// leading dimension, or within a row).  None where it does not broadcast to x.
std::optional<int64_t> gate_group(const Tensor& gate, const Tensor& x) {
  const int64_t dims = x.dim(), pad = dims - gate.dim();
  if (pad < 0) return {};
  auto size = [&](int64_t i) { return i < pad ? 1 : gate.size(i - pad); };
  for (int64_t i = 0; i < dims; ++i)
    if (size(i) != 1 && size(i) != x.size(i)) return {};
  if (size(dims - 1) != x.size(dims - 1)) return 0;
  int64_t n = dims - 1, group = 1;
  while (n > 0 && size(n - 1) == 1) group *= x.size(--n);
  for (int64_t i = 0; i < n; ++i)
    if (size(i) != x.size(i)) return 0;
  return group;
}

// (y, h), y none without a block; none where the arguments do not fit together (the caller says why).
std::optional<std::tuple<std::optional<Tensor>, Tensor>> residual_norm(
    const Tensor& x, const std::optional<Tensor>& block, const std::optional<Tensor>& gate, const std::optional<Tensor>& dev,
    double scale, const std::optional<Tensor>& post, const std::optional<Tensor>& pre, int kind, double eps) {
  not_traced("residual_norm");
  if (x.dim() < 1 || x.size(-1) < 1 || kind < 0 || !(eps >= 0.0 && std::isfinite(eps))) return {};
  if (!block && (gate || post)) return {};
  const at::ScalarType dt = (block ? *block : pre ? *pre : x).scalar_type();
  auto fits = [&](const std::optional<Tensor>& t) { return !t || (t->scalar_type() == dt && t->is_cuda() && t->device() == x.device()); };
  auto vector = [&](const std::optional<Tensor>& t) { return fits(t) && (!t || (t->dim() == 1 && t->size(0) == x.size(-1))); };
  if (type_of(dt) < 0 || !x.is_cuda() || (x.scalar_type() != dt && x.scalar_type() != at::kFloat) || !fits(block) || !fits(gate) ||
      !vector(post) || !vector(pre) || (block && block->sizes() != x.sizes()))
    return {};
  if (dev && (dev->numel() != 1 || dev->scalar_type() != at::kFloat || dev->device() != x.device())) return {};
  TORCH_CHECK_VALUE(x.size(-1) <= INT_MAX, "x has more than 2^31 columns");
  int64_t group = std::max<int64_t>(x.numel() / x.size(-1), 1);
  Tensor g;
  if (gate) {
    g = gate->dim() ? *gate : gate->reshape({1});
    const auto of_gate = gate_group(g, x);
    if (!of_gate) return {};
    group = *of_gate;
    if (group) g = g.contiguous();
  }
  Norm n{x.contiguous(), contiguous(block), g, contiguous(post), contiguous(pre), Tensor(), scale, group, kind, eps, dt};
  if (dev && block) n.dev = *dev;  // (without a block the scale has no part in the result)
  no_tangents({&n.x, &n.block, &n.gate, &n.post, &n.pre, &n.dev}, "residual_norm");
  if (wants_grad({&n.x, &n.block, &n.gate, &n.post, &n.pre, &n.dev})) {
    auto maybe = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    const auto out = NormFunction::apply(n.x, maybe(n.block), maybe(n.gate), maybe(n.post), maybe(n.pre), maybe(n.dev), scale, group, (int64_t)kind, eps, (int64_t)dt);
    return {{block ? std::optional<Tensor>(out[0]) : std::nullopt, out.back()}};
  }
  if (group == 0) {
    n.gate = n.gate.expand(x.sizes()).contiguous();
    n.group = 1;
  }
  const auto [y, h, stats] = n.forward(false);
  return {{block ? std::optional<Tensor>(y) : std::nullopt, h}};
}

// ---- linear_cross_entropy --------------------------------------------------------------------------
struct Xent {
  Tensor h, w, target;
  int64_t ignore;
  int reduction;

  int type() const { return type_of(h.scalar_type()); }
  int n() const { return (int)h.size(0); }
  int d() const { return (int)h.size(1); }
  int v() const { return (int)w.size(0); }
  Tensor workspace(int backward) const {
    const long size = lib.xent_workspace(type(), n(), d(), v(), backward);
    check(size, "kans_linear_xent_workspace");
    return bytes(h, size);
  }

  std::tuple<Tensor, Tensor> forward() const {
    const auto f32 = h.options().dtype(at::kFloat);
    Tensor loss = reduction == 0 ? at::empty({n()}, f32) : at::empty({}, f32);
    Tensor state = at::empty({4 + 3L * n()}, h.options().dtype(at::kInt));
    if (n() == 0) {
      if (reduction != 0) loss.fill_(reduction == 1 ? std::numeric_limits<double>::quiet_NaN() : 0.0);
      return {loss, state};
    }
    const Tensor ws = workspace(0);
    check(lib.xent_forward(type(), data(h), data(w), (const int64_t*)data(target), n(), d(), v(), ignore, reduction,
                           (float*)data(loss), (int*)data(state), data(ws), ws.numel(), stream_of(h)),
          "kans_linear_xent_forward");
    return {loss, state};
  }

  variable_list backward(const Tensor& state, const Tensor& grad, bool need_h, bool need_w) const {
    Tensor dh = need_h ? at::empty_like(h) : Tensor(), dw = need_w ? at::empty_like(w) : Tensor();
    if (n() == 0) {
      if (dw.defined()) dw.zero_();
      return {dh, dw};
    }
    const Tensor ws = workspace(reduction == 0 ? 1 : 2), g = grad.contiguous();
    check(lib.xent_backward(type(), data(h), data(w), (const int64_t*)data(target), n(), d(), v(), ignore, reduction,
                            (const int*)data(state), (const float*)data(g), data(dh), data(dw), data(ws), ws.numel(), stream_of(h)),
          "kans_linear_xent_backward");
    return {dh, dw};
  }
};

struct XentFunction : torch::autograd::Function<XentFunction> {
  static variable_list forward(AutogradContext* ctx, Tensor h, Tensor w, Tensor target, int64_t ignore, int64_t reduction) {
    const auto [loss, state] = Xent{h, w, target, ignore, (int)reduction}.forward();
    ctx->save_for_backward({h, w, target, state});
    ctx->saved_data["rest"] = std::vector<int64_t>{ignore, reduction};
    return {loss};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    const auto s = ctx->get_saved_variables();
    const auto rest = ctx->saved_data["rest"].toIntVector();
    no_tangents({&grads[0]}, "linear_cross_entropy's backward");
    capturable_behind(grads[0], "linear_cross_entropy's backward");
    const Xent x{s[0], s[1], s[2], rest[0], (int)rest[1]};
    const variable_list d = once(x.backward(s[3], grads[0], ctx->needs_input_grad(0), ctx->needs_input_grad(1)), graph);
    return {d[0], d[1], Tensor(), Tensor(), Tensor()};
  }
};

// None where the arguments do not fit together (the caller says why).
std::optional<Tensor> linear_cross_entropy(const Tensor& hidden, const Tensor& weight, const Tensor& target, int64_t ignore,
                                           int reduction) {
  not_traced("linear_cross_entropy");
  if (reduction < 0 || hidden.dim() < 1 || weight.dim() != 2 || hidden.size(-1) != weight.size(1) || weight.size(0) == 0 ||
      weight.size(1) == 0 || target.sizes() != hidden.sizes().slice(0, hidden.dim() - 1))
    return {};
  if (type_of(hidden.scalar_type()) < 0 || weight.scalar_type() != hidden.scalar_type() || target.scalar_type() != at::kLong ||
      !hidden.is_cuda() || weight.device() != hidden.device() || target.device() != hidden.device())
    return {};
  // (sizes beyond an int are beyond the library's, which says so)
  TORCH_CHECK_VALUE(hidden.numel() / hidden.size(-1) <= INT_MAX && weight.size(0) <= INT_MAX && weight.size(1) <= INT_MAX,
                    "hidden and weight have more than 2^31 rows or columns");
  const Xent x{hidden.reshape({-1, hidden.size(-1)}).contiguous(), weight.contiguous(), target.reshape({-1}).contiguous(), ignore,
               reduction};
  no_tangents({&x.h, &x.w}, "linear_cross_entropy");
  const Tensor loss = wants_grad({&x.h, &x.w}) ? XentFunction::apply(x.h, x.w, x.target, ignore, (int64_t)reduction)[0]
                                               : std::get<0>(x.forward());
  return reduction == 0 ? loss.reshape(target.sizes()) : loss;
}

// ---- embedding -------------------------------------------------------------------------------------
struct EmbeddingFunction : torch::autograd::Function<EmbeddingFunction> {
  static Tensor call(const Tensor& tokens, const Tensor& w, double scale, int64_t ignore) {
    auto shape = tokens.sizes().vec();
    shape.push_back(w.size(1));
    Tensor out = at::empty(shape, w.options());
    if (tokens.numel() == 0) return out;
    check(lib.embedding_forward(type_of(w.scalar_type()), (const int64_t*)data(tokens), data(w), tokens.numel(), (int)w.size(1),
                                (int)w.size(0), ignore, scale, data(out), stream_of(w)),
          "kans_embedding_forward");
    return out;
  }

  static variable_list forward(AutogradContext* ctx, Tensor tokens, Tensor w, double scale, int64_t ignore) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({tokens});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["rest"] = std::vector<int64_t>{ignore, w.size(0), w.size(1)};
    return {call(tokens, w, scale, ignore)};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    if (!grads[0].defined()) return variable_list(4);
    no_tangents({&grads[0]}, "embedding's backward");
    capturable_behind(grads[0], "embedding's backward");
    const auto s = ctx->get_saved_variables();
    const auto rest = ctx->saved_data["rest"].toIntVector();
    const Tensor dout = grads[0].contiguous(), &tokens = s[0];
    const at::OptionalDeviceGuard device(dout.device());
    Tensor dw = at::empty({rest[1], rest[2]}, dout.options());
    const int type = type_of(dout.scalar_type()), D = (int)rest[2], V = (int)rest[1];
    const long size = lib.embedding_workspace(type, tokens.numel(), D, V);
    check(size, "kans_embedding_workspace");
    const Tensor ws = bytes(dout, size);
    check(lib.embedding_backward(type, (const int64_t*)data(tokens), data(dout), tokens.numel(), D, V, rest[0],
                                 ctx->saved_data["scale"].toDouble(), data(dw), data(ws), size, stream_of(dout)),
          "kans_embedding_backward");
    return {Tensor(), once({dw}, graph)[0], Tensor(), Tensor()};
  }
};

// None where the arguments do not fit together (the caller says why).
std::optional<Tensor> embedding(const Tensor& tokens, const Tensor& weight, double scale, int64_t ignore) {
  not_traced("embedding");
  if (weight.dim() != 2 || weight.size(0) == 0 || weight.size(1) == 0 || type_of(weight.scalar_type()) < 0 ||
      tokens.scalar_type() != at::kLong || !weight.is_cuda() || tokens.device() != weight.device() ||
      !(scale == 0.0 || (std::fabs(scale) >= FLT_MIN && std::fabs(scale) <= FLT_MAX)))
    return {};
  TORCH_CHECK_VALUE(weight.size(0) <= INT_MAX && weight.size(1) <= INT_MAX, "weight has more than 2^31 rows or columns");
  const Tensor t = tokens.contiguous(), w = weight.contiguous();
  no_tangents({&w}, "embedding");
  const at::OptionalDeviceGuard device(w.device());
  if (!wants_grad({&w})) return EmbeddingFunction::call(t, w, scale, ignore);
  capturable({&weight}, "embedding");
  return EmbeddingFunction::apply(t, w, scale, ignore)[0];
}

// ---- dropout ---------------------------------------------------------------------------------------
struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
  // The key is `dev`'s where that is given; used (where wanted) keeps it for the backward, since dev may hold another one by then.
  static Tensor call(const Tensor& x, double p, int64_t seed, const Tensor& dev, const Tensor& used, int64_t offset) {
    Tensor y = at::empty_like(x);
    if (x.numel() == 0) return y;
    check(lib.dropout(type_of(x.scalar_type()), data(x), data(y), x.numel(), p, seed, (const int64_t*)data(dev), (int64_t*)data(used),
                      offset, stream_of(x)),
          "kans_dropout");
    return y;
  }

  static variable_list forward(AutogradContext* ctx, Tensor x, double p, int64_t seed, std::optional<Tensor> dev, int64_t offset) {
    const Tensor used = dev ? at::empty({1}, dev->options()) : Tensor();
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({used});
    ctx->saved_data["p"] = p;
    ctx->saved_data["rest"] = std::vector<int64_t>{seed, offset};
    return {call(x, p, seed, dev ? *dev : Tensor(), used, offset)};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    if (!grads[0].defined()) return variable_list(5);
    no_tangents({&grads[0]}, "dropout's backward");
    capturable_behind(grads[0], "dropout's backward");
    const auto rest = ctx->saved_data["rest"].toIntVector();
    const Tensor dy = grads[0].contiguous();
    const at::OptionalDeviceGuard device(dy.device());
    const Tensor dx = call(dy, ctx->saved_data["p"].toDouble(), rest[0], ctx->get_saved_variables()[0], Tensor(), rest[1]);
    return {once({dx}, graph)[0], Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// None where the arguments do not fit together (the caller says why).
std::optional<Tensor> dropout(const Tensor& x, double p, int64_t seed, const std::optional<Tensor>& dev, int64_t offset) {
  not_traced("dropout");
  if (type_of(x.scalar_type()) < 0 || !x.is_cuda() || !(p >= 0.0 && p <= 1.0)) return {};
  if (dev && (dev->numel() != 1 || dev->scalar_type() != at::kLong || dev->device() != x.device())) return {};
  const Tensor in = x.contiguous();
  no_tangents({&in}, "dropout");
  const at::OptionalDeviceGuard device(in.device());
  if (!wants_grad({&in})) return DropoutFunction::call(in, p, seed, dev ? *dev : Tensor(), Tensor(), offset);
  capturable({&x}, "dropout");
  return DropoutFunction::apply(in, p, seed, dev, offset)[0];
}

// ---- causal_conv -----------------------------------------------------------------------------------
// A [B, L, C] tensor whose channels lie side by side, as it is where it can be read so.
Tensor with_channels(const Tensor& t) { return t.size(2) == 1 || t.stride(2) == 1 ? t : t.contiguous(); }
std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
Tensor given(const std::optional<Tensor>& t) { return t ? *t : Tensor(); }

// lengths and a state beside a [B, L, C] tensor
bool fits_lengths(const std::optional<Tensor>& lengths, const Tensor& x) {
  return !lengths || (lengths->dim() == 1 && lengths->size(0) == x.size(0) && lengths->scalar_type() == at::kLong &&
                      lengths->device() == x.device());
}
bool sizes_fit_int(const Tensor& x) { return x.size(0) <= INT_MAX && x.size(1) <= INT_MAX && x.size(2) <= INT_MAX; }

struct Conv {
  Tensor x, w, bias, lengths;  // (undefined: not given)
  bool silu;

  int B() const { return (int)x.size(0); }
  int L() const { return (int)x.size(1); }
  int D() const { return (int)x.size(2); }
  int W() const { return (int)w.size(1); }
  int type() const { return type_of(x.scalar_type()); }

  Tensor forward(const Tensor& state) const {
    Tensor y = at::empty(x.sizes(), x.options());
    check(lib.conv_forward(type(), data(x), stride(x, 0), stride(x, 1), data(w), data(bias), data(state), (const int64_t*)data(lengths),
                           silu, data(y), B(), L(), D(), W(), stream_of(x)),
          "kans_causal_conv_forward");
    return y;
  }

  variable_list backward(const Tensor& dy, const std::array<bool, 3>& need) const {
    Tensor dx = need[0] ? at::empty(x.sizes(), x.options()) : Tensor(), dw = need[1] ? at::empty_like(w) : Tensor(),
           dbias = need[2] ? at::empty_like(bias) : Tensor();
    const long size = lib.conv_workspace(type(), B(), L(), D(), W());
    check(size, "kans_causal_conv_workspace");
    const Tensor ws = need[1] || need[2] ? bytes(x, size) : Tensor();
    check(lib.conv_backward(type(), data(x), stride(x, 0), stride(x, 1), data(w), data(bias), (const int64_t*)data(lengths), silu, data(dy),
                            data(dx), data(dw), data(dbias), B(), L(), D(), W(), data(ws), size, stream_of(x)),
          "kans_causal_conv_backward");
    return {dx, dw, dbias};
  }
};

struct ConvFunction : torch::autograd::Function<ConvFunction> {
  typedef std::optional<Tensor> Maybe;
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor w, Maybe bias, Maybe lengths, bool silu) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, w, given(bias), given(lengths)});
    ctx->saved_data["silu"] = silu;
    return {Conv{x, w, given(bias), given(lengths), silu}.forward(Tensor())};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    variable_list d(5);
    if (!grads[0].defined()) return d;
    no_tangents({&grads[0]}, "causal_conv's backward");
    capturable_behind(grads[0], "causal_conv's backward");
    const auto s = ctx->get_saved_variables();
    const at::OptionalDeviceGuard device(s[0].device());
    const Conv c{s[0], s[1], s[2], s[3], ctx->saved_data["silu"].toBool()};
    std::array<bool, 3> need;
    for (size_t i = 0, edge = 0; i < 3; ++i) need[i] = s[i].defined() && ctx->needs_input_grad(edge++);
    const variable_list three = once(c.backward(grads[0].contiguous(), need), graph);
    std::copy(three.begin(), three.end(), d.begin());
    return d;
  }
};

// None where the arguments do not fit together (the caller says why).
std::optional<Tensor> causal_conv(const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias, int silu,
                                  const std::optional<Tensor>& state, const std::optional<Tensor>& lengths) {
  not_traced("causal_conv");
  const at::ScalarType dt = x.scalar_type();
  auto fits = [&](const Tensor& t) { return t.scalar_type() == dt && t.device() == x.device(); };
  if (silu < 0 || x.dim() != 3 || type_of(dt) < 0 || !x.is_cuda() || x.size(2) == 0 || w.dim() != 2 || w.size(0) != x.size(2) ||
      w.size(1) < 1 || w.size(1) > 8 || !fits(w) || !fits_lengths(lengths, x))
    return {};
  if (bias && (!fits(*bias) || bias->dim() != 1 || bias->size(0) != x.size(2))) return {};
  if (state && (!fits(*state) || !state->is_contiguous() || state->dim() != 3 || state->size(0) != x.size(0) ||
                state->size(1) != w.size(1) - 1 || state->size(2) != x.size(2)))
    return {};
  TORCH_CHECK_VALUE(sizes_fit_int(x), "x has a size of more than 2^31");
  const Conv c{with_channels(x), w.contiguous(), contiguous(bias), contiguous(lengths), silu != 0};
  no_tangents({&c.x, &c.w, &c.bias}, "causal_conv");
  const at::OptionalDeviceGuard device(x.device());
  if (wants_grad({&c.x, &c.w, &c.bias})) {
    TORCH_CHECK(!state, "causal_conv with a state has no gradients: call it under torch.no_grad()");
    const Tensor b = given(bias);
    capturable({&x, &w, &b}, "causal_conv");
    return ConvFunction::apply(c.x, c.w, maybe(c.bias), maybe(c.lengths), c.silu)[0];
  }
  TORCH_CHECK(!state || !(at::GradMode::is_enabled() && state->requires_grad()),
              "causal_conv with a state has no gradients: call it under torch.no_grad()");
  const Tensor y = c.forward(given(state));
  if (state && !state->is_inference()) state->unsafeGetTensorImpl()->bump_version();
  return y;
}

// ---- selective_scan --------------------------------------------------------------------------------
// (the scan's kernels take fewer than 2^23 elements between steps, and steps that are the same or apart)
Tensor with_steps(const Tensor& t) {
  const bool steps = t.size(1) <= 1 || t.stride(1) == 0 || (t.stride(1) >= t.size(2) && t.stride(1) < 1 << 23);
  return (t.size(2) == 1 || t.stride(2) == 1) && steps ? t : t.contiguous();
}

struct Scan {
  Tensor x, dt, A, B, C, skip, z, bias, lengths;  // (undefined: not given)
  bool softplus;

  int b() const { return (int)x.size(0); }
  int l() const { return (int)x.size(1); }
  int d() const { return (int)x.size(2); }
  int n() const { return (int)A.size(1); }
  int type() const { return type_of(x.scalar_type()); }
  // (of a single step or sequence there is none: it may be anything)
  static long stride(const Tensor& t, int i) { return t.defined() && t.size(i) > 1 ? t.stride(i) : 0; }
  Tensor workspace(int backward) const {
    const long size = lib.scan_workspace(b(), l(), d(), n(), backward);
    check(size, "kans_selective_scan_workspace");
    return bytes(x, size);
  }

  std::tuple<Tensor, Tensor> forward(const Tensor& state, bool save) const {
    Tensor out = at::empty(x.sizes(), x.options()), saved;
    if (save) {
      const long size = lib.scan_saved(b(), l(), d(), n());
      check(size, "kans_selective_scan_saved");
      saved = at::empty({size / 4}, x.options().dtype(at::kFloat));
    }
    const Tensor ws = workspace(0);
    check(lib.scan_forward(type(), data(x), stride(x, 0), stride(x, 1), data(dt), stride(dt, 0), stride(dt, 1), (const float*)data(A), data(B),
                           stride(B, 0), stride(B, 1), data(C), stride(C, 0), stride(C, 1), (const float*)data(skip), data(z), stride(z, 0),
                           stride(z, 1), (const float*)data(bias), softplus, (float*)data(state), (const int64_t*)data(lengths), data(out),
                           (float*)data(saved), b(), l(), d(), n(), data(ws), ws.numel(), stream_of(x)),
          "kans_selective_scan_forward");
    return {out, saved};
  }

  // Gradients of the eight inputs, undefined where need is false.
  variable_list backward(const Tensor& saved, const Tensor& dout, const std::array<bool, 8>& need) const {
    auto like = [&](const Tensor& t, bool on) { return on ? at::empty(t.sizes(), t.options()) : Tensor(); };
    // (the kernel writes dx, ddt and dz in any case)
    Tensor dx = like(x, true), ddt = like(dt, true), dA = like(A, need[2]), dB = like(B, need[3]), dC = like(C, need[4]),
           dskip = like(skip, need[5]), dz = like(z, z.defined()), dbias = like(bias, need[7]);
    const Tensor ws = workspace(1);
    check(lib.scan_backward(type(), data(x), stride(x, 0), stride(x, 1), data(dt), stride(dt, 0), stride(dt, 1), (const float*)data(A), data(B),
                            stride(B, 0), stride(B, 1), data(C), stride(C, 0), stride(C, 1), (const float*)data(skip), data(z), stride(z, 0),
                            stride(z, 1), (const float*)data(bias), softplus, (const int64_t*)data(lengths), (const float*)data(saved),
                            data(dout), data(dx), data(ddt), (float*)data(dA), data(dB), data(dC), (float*)data(dskip), data(dz),
                            (float*)data(dbias), b(), l(), d(), n(), data(ws), ws.numel(), stream_of(x)),
          "kans_selective_scan_backward");
    return {need[0] ? dx : Tensor(), need[1] ? ddt : Tensor(), dA, dB, dC, dskip, need[6] ? dz : Tensor(), dbias};
  }
};

struct ScanFunction : torch::autograd::Function<ScanFunction> {
  typedef std::optional<Tensor> Maybe;
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Maybe skip, Maybe z, Maybe bias,
                               Maybe lengths, bool softplus) {
    const Scan s{x, dt, A, B, C, given(skip), given(z), given(bias), given(lengths), softplus};
    auto [out, saved] = s.forward(Tensor(), true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, dt, A, B, C, s.skip, s.z, s.bias, s.lengths, saved});
    ctx->saved_data["softplus"] = softplus;
    return {out};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    variable_list d(10);
    if (!grads[0].defined()) return d;
    no_tangents({&grads[0]}, "selective_scan's backward");
    capturable_behind(grads[0], "selective_scan's backward");
    const auto s = ctx->get_saved_variables();
    const at::OptionalDeviceGuard device(s[0].device());
    const Scan scan{s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], ctx->saved_data["softplus"].toBool()};
    std::array<bool, 8> need;
    for (size_t i = 0, edge = 0; i < 8; ++i) need[i] = s[i].defined() && ctx->needs_input_grad(edge++);
    const variable_list eight = once(scan.backward(s[9], grads[0].contiguous(), need), graph);
    std::copy(eight.begin(), eight.end(), d.begin());
    return d;
  }
};

// None where the arguments do not fit together (the caller says why).
std::optional<Tensor> selective_scan(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                                     const std::optional<Tensor>& skip, const std::optional<Tensor>& z, const std::optional<Tensor>& bias,
                                     bool softplus, const std::optional<Tensor>& state, const std::optional<Tensor>& lengths) {
  not_traced("selective_scan");
  auto of_type = [&](const Tensor& t, at::ScalarType type) { return t.scalar_type() == type && t.device() == x.device(); };
  auto channel = [&](const std::optional<Tensor>& t) {
    return !t || (of_type(*t, at::kFloat) && t->dim() == 1 && t->size(0) == x.size(2));
  };
  if (x.dim() != 3 || type_of(x.scalar_type()) < 0 || !x.is_cuda() || x.size(2) == 0) return {};
  if (!of_type(A, at::kFloat) || A.dim() != 2 || A.size(0) != x.size(2) || A.size(1) < 1 || A.size(1) > 64) return {};
  auto wide = [&](const Tensor& t, int64_t channels) {
    return of_type(t, x.scalar_type()) && t.dim() == 3 && t.size(0) == x.size(0) && t.size(1) == x.size(1) && t.size(2) == channels;
  };
  if (!wide(dt, x.size(2)) || (z && !wide(*z, x.size(2))) || !wide(B, A.size(1)) || !wide(C, A.size(1)) || !channel(skip) ||
      !channel(bias) || !fits_lengths(lengths, x))
    return {};
  if (state && (!of_type(*state, at::kFloat) || !state->is_contiguous() || state->dim() != 3 || state->size(0) != x.size(0) ||
                state->size(1) != x.size(2) || state->size(2) != A.size(1)))
    return {};
  TORCH_CHECK_VALUE(sizes_fit_int(x), "x has a size of more than 2^31");
  const Scan s{with_steps(x), with_steps(dt), A.contiguous(), with_steps(B), with_steps(C), contiguous(skip),
         z ? with_steps(*z) : Tensor(), contiguous(bias), contiguous(lengths), softplus};
  no_tangents({&s.x, &s.dt, &s.A, &s.B, &s.C, &s.skip, &s.z, &s.bias}, "selective_scan");
  const at::OptionalDeviceGuard device(x.device());
  if (wants_grad({&s.x, &s.dt, &s.A, &s.B, &s.C, &s.skip, &s.z, &s.bias})) {
    TORCH_CHECK(!state, "selective_scan with a state has no gradients: call it under torch.no_grad()");
    const Tensor rest[] = {given(skip), given(z), given(bias)};
    capturable({&x, &dt, &A, &B, &C, &rest[0], &rest[1], &rest[2]}, "selective_scan");
    return ScanFunction::apply(s.x, s.dt, s.A, s.B, s.C, maybe(s.skip), maybe(s.z), maybe(s.bias), maybe(s.lengths), softplus)[0];
  }
  TORCH_CHECK(!state || !(at::GradMode::is_enabled() && state->requires_grad()),
              "selective_scan with a state has no gradients: call it under torch.no_grad()");
  const Tensor out = std::get<0>(s.forward(given(state), false));
  if (state && !state->is_inference()) state->unsafeGetTensorImpl()->bump_version();
  return out;
}

// ---- TorchAdamW ------------------------------------------------------------------------------------
// An arena's buffers (_Arena.flat), and what a parameter's state holds when it is the arena's own: views of them at the
// parameter's place, in its order of memory.
struct Arena {
  static constexpr int kKinds = 5;
  Tensor flat[kKinds];  // exp_avg, exp_avg_sq, their scales, master (undefined: none of these)

  explicit Arena(const py::dict& buffers) {
    for (int k = 0; k < kKinds; ++k)
      if (PyObject* t = PyDict_GetItemWithError(buffers.ptr(), name(k))) flat[k] = THPVariable_Unpack(t);
  }
  static PyObject* name(int k) {
    static PyObject* const names[kKinds] = {
        PyUnicode_InternFromString("exp_avg"), PyUnicode_InternFromString("exp_avg_sq"), PyUnicode_InternFromString("exp_avg_scale"),
        PyUnicode_InternFromString("exp_avg_sq_scale"), PyUnicode_InternFromString("master")};
    return names[k];
  }

  bool holds(PyObject* state, const Tensor& p, int64_t block) const {
    if (!state || !PyDict_Check(state)) return false;
    for (int k = 0; k < kKinds; ++k) {
      if (!flat[k].defined()) continue;
      PyObject* object = PyDict_GetItemWithError(state, name(k));
      if (!object || !THPVariable_Check(object)) return false;
      const Tensor& t = THPVariable_Unpack(object);
      const bool scale = k == 2 || k == 3;
      if (t.scalar_type() != flat[k].scalar_type() || t.storage().unsafeGetStorageImpl() != flat[k].storage().unsafeGetStorageImpl() ||
          t.storage_offset() != (scale ? block : block * 256))
        return false;
      if (scale) {
        if (t.dim() != 1 || t.size(0) != (p.numel() + 255) / 256 || !t.is_contiguous()) return false;
        continue;
      }
      if (t.sizes() != p.sizes()) return false;
      for (int64_t i = 0; i < p.dim(); ++i)
        if (p.size(i) != 1 && p.stride(i) != t.stride(i)) return false;
    }
    return true;
  }
};

// The state of parameter i, by start(i) where it is not there, or not the arena's own (a new tensor in its place, or the
// parameter in another order of memory).  A borrowed reference.
PyObject* state_of(const py::dict& state, PyObject* object, const Arena& arena, int64_t block, const py::object& start, size_t i) {
  const Tensor& p = THPVariable_Unpack(object);
  PyObject* s = PyDict_GetItemWithError(state.ptr(), object);
  if (!arena.holds(s, p, block)) {
    if (PyErr_Occurred()) throw py::error_already_set();
    start(i);
    s = PyDict_GetItemWithError(state.ptr(), object);
    if (!arena.holds(s, p, block)) {
      if (PyErr_Occurred()) throw py::error_already_set();
      throw py::value_error("a parameter's state is not the optimizer's own");
    }
  }
  return s;
}

// Puts every state that is there into the arena.
void adamw_hold(const py::dict& state, const py::list& params, const py::buffer& blocks, const py::dict& flat, const py::object& start) {
  const auto block_of = blocks.request();
  const Arena arena(flat);
  if (block_of.size != (py::ssize_t)params.size() || block_of.itemsize != 8) throw py::value_error("one block for each parameter");
  for (size_t i = 0; i < params.size(); ++i) {
    PyObject* object = PyList_GET_ITEM(params.ptr(), (Py_ssize_t)i);
    PyObject* s = PyDict_GetItemWithError(state.ptr(), object);
    if (!s && PyErr_Occurred()) throw py::error_already_set();
    if (s && PyObject_IsTrue(s) == 1) state_of(state, object, arena, ((const int64_t*)block_of.ptr)[i], start, i);
  }
}

// seen: int64 [2 n], each parameter's address and version behind its last step (version < 0: none).  Both are looked at before and
// noted behind the whole step, since views of one buffer share a version.
constexpr int64_t kStepped = -2;
int64_t version_of(const Tensor& p) { return p.is_inference() ? -1 : p._version(); }

py::buffer_info seen_of(const py::list& params, const py::buffer& seen) {
  py::buffer_info info = seen.request(/*writable=*/true);
  if (info.size != 2 * (py::ssize_t)params.size() || info.itemsize != 8) throw py::value_error("one address and version for each parameter");
  return info;
}

// Where a parameter with a gradient has changed since its last step: follow(i) brings its master in line.
void adamw_follow(const py::dict& state, const py::list& params, const py::buffer& blocks, const py::dict& flat, const py::object& start,
                  const py::buffer& seen, const py::object& follow) {
  const auto info = seen_of(params, seen), block_of = blocks.request();
  if (block_of.size != (py::ssize_t)params.size() || block_of.itemsize != 8) throw py::value_error("one block for each parameter");
  const Arena arena(flat);
  for (size_t i = 0; i < params.size(); ++i) {
    const int64_t* const was = (const int64_t*)info.ptr + 2 * i;
    PyObject* object = PyList_GET_ITEM(params.ptr(), (Py_ssize_t)i);
    const Tensor& p = THPVariable_Unpack(object);
    if (was[1] < 0 || (was[0] == (int64_t)(intptr_t)p.data_ptr() && was[1] == version_of(p)) || !p.grad().defined()) continue;
    PyObject* s = PyDict_GetItemWithError(state.ptr(), object);
    if (!s && PyErr_Occurred()) throw py::error_already_set();
    if (!s || PyObject_IsTrue(s) != 1) continue;
    state_of(state, object, arena, ((const int64_t*)block_of.ptr)[i], start, i);
    follow(i);
  }
}

void adamw_seen(const py::list& params, const py::buffer& seen) {
  const auto info = seen_of(params, seen);
  for (size_t i = 0; i < params.size(); ++i) {
    int64_t* const at = (int64_t*)info.ptr + 2 * i;
    if (at[1] != kStepped) continue;
    const Tensor& p = THPVariable_Unpack(PyList_GET_ITEM(params.ptr(), (Py_ssize_t)i));
    at[0] = (int64_t)(intptr_t)p.data_ptr();
    at[1] = version_of(p);
  }
}

// One step of the parameters of an arena that have gradients.  state: the optimizer's, by parameter; start(i) puts parameter i's into the arena.
// seen: marks those that a step has written for adamw_seen.
// numel, blocks: int64 per parameter; flat: the arena's buffers.  A step of 9 small tensors takes 17 us, of 48 with 8-bit
// states and their values 27; with this loop in Python 23 and 66.
void adamw_step(const py::dict& state, const py::list& params, const py::buffer& numel, const py::buffer& blocks, const py::dict& flat,
                int type, int bits, const py::object& start, double lr, double beta1, double beta2, double eps, double decay,
                const std::optional<py::buffer>& seen) {
  not_traced("TorchAdamW.step");
  const auto n_of = numel.request(), block_of = blocks.request();
  const size_t n = params.size();
  if ((size_t)n_of.size != n || (size_t)block_of.size != n || n_of.itemsize != 8 || block_of.itemsize != 8)
    throw py::value_error("one size and block for each parameter");
  std::optional<py::buffer_info> marks;
  if (seen) marks = seen_of(params, *seen);
  const Arena arena(flat);
  const Tensor &m = arena.flat[0], &v = arena.flat[1], &ms = arena.flat[2], &vs = arena.flat[3], &master = arena.flat[4];
  static PyObject* const step_name = PyUnicode_InternFromString("step");
  struct One {
    Tensor p, grad;
    PyObject* state;
    int64_t* seen;
  };
  std::vector<One> ones;
  std::vector<void*> at;
  std::vector<const void*> grads;
  std::vector<long> sizes, places, steps;
  ones.reserve(n), at.reserve(n), grads.reserve(n), sizes.reserve(n), places.reserve(n), steps.reserve(n);
  for (size_t i = 0; i < n; ++i) {
    PyObject* object = PyList_GET_ITEM(params.ptr(), (Py_ssize_t)i);
    const Tensor& p = THPVariable_Unpack(object);
    Tensor g = p.grad();
    if (!g.defined()) continue;
    if (g.layout() != at::kStrided || type_of(g.scalar_type()) != type || g.device() != m.device())
      throw py::type_error("gradients must be dense tensors of their parameter's dtype and device");
    if (type_of(p.scalar_type()) != type || p.device() != m.device() || p.numel() != ((const int64_t*)n_of.ptr)[i])
      throw py::value_error("a parameter's dtype, device or size changed under its optimizer");
    // (the kernel writes numel consecutive places)
    if (p.numel() > 1 && !p.is_non_overlapping_and_dense())
      throw py::value_error("parameters must be dense (no gaps or overlaps in memory)");
    if (g.sizes() != p.sizes()) throw py::value_error("a gradient has another shape than its parameter");
    if (g.strides() != p.strides()) {  // (elements are paired by their place in memory)
      at::NoGradGuard no_grad;
      g = at::empty_like(p).copy_(g);
    }
    PyObject* s = state_of(state, object, arena, ((const int64_t*)block_of.ptr)[i], start, i);
    PyObject* step = PyDict_GetItemWithError(s, step_name);
    const long count = step ? PyLong_AsLong(step) : -1;
    if (PyErr_Occurred()) throw py::error_already_set();
    if (!step) throw py::value_error("a parameter's state has no step");
    ones.push_back({p, g, s, marks ? (int64_t*)marks->ptr + 2 * i : nullptr});
    at.push_back(p.data_ptr());
    grads.push_back(g.data_ptr());
    sizes.push_back(p.numel());
    places.push_back(((const int64_t*)block_of.ptr)[i]);
    steps.push_back(count + 1);
  }
  if (ones.empty()) return;
  check(lib.adamw_step(type, bits, (int)ones.size(), at.data(), grads.data(), sizes.data(), places.data(), steps.data(), data(m),
                       data(v), (float*)data(ms), (float*)data(vs), (float*)data(master), lr, beta1, beta2, eps, decay, stream_of(m)),
        "kans_adamw_step");
  for (size_t i = 0; i < ones.size(); ++i) {
    const py::int_ step(steps[i]);
    if (PyDict_SetItem(ones[i].state, step_name, step.ptr()) < 0) throw py::error_already_set();
    ones[i].p.unsafeGetTensorImpl()->bump_version();
    if (ones[i].seen) ones[i].seen[1] = kStepped;
  }
}

}  // namespace

PYBIND11_MODULE(_kans_torch, m) {
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Failure& e) {
      PyErr_SetString(kans_error ? kans_error : PyExc_RuntimeError, e.what());
    }
  });
  m.def("bind", &bind);
  m.def("residual_norm", &residual_norm, py::call_guard<py::gil_scoped_release>());
  m.def("adamw_step", &adamw_step, py::arg("state"), py::arg("params"), py::arg("numel"), py::arg("blocks"), py::arg("flat"),
        py::arg("type"), py::arg("bits"), py::arg("start"), py::arg("lr"), py::arg("beta1"), py::arg("beta2"), py::arg("eps"),
        py::arg("decay"), py::arg("seen") = py::none());
  m.def("adamw_hold", &adamw_hold);
  m.def("adamw_follow", &adamw_follow);
  m.def("adamw_seen", &adamw_seen);
  m.def("linear_cross_entropy", &linear_cross_entropy, py::call_guard<py::gil_scoped_release>());
  m.def("embedding", &embedding, py::call_guard<py::gil_scoped_release>());
  m.def("dropout", &dropout, py::call_guard<py::gil_scoped_release>());
  m.def("causal_conv", &causal_conv, py::call_guard<py::gil_scoped_release>());
  m.def("selective_scan", &selective_scan, py::call_guard<py::gil_scoped_release>());
}

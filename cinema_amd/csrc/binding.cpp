// Python entry points of the plain MLP operators: argument checks, output allocation and the autograd nodes of linear_act and
// layer_norm, and the gradient norm over lists of tensors, on top of the C ABI of libcinema_hip.so (include/cinema_hip.h).
// Native because these calls are small: a node in Python spent 150 us of host time on a layer norm's forward and backward
// pass whose kernels take 12 us (64 x 256), most of it between the interpreter and the autograd engine's own thread.
#include <torch/extension.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <ATen/autocast_mode.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <dlfcn.h>
#include <algorithm>
#include <array>
#include <limits>
#include "../../include/cinema_hip.h"

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

namespace {

struct Api {
  decltype(&cinema_last_error) last_error;
  decltype(&cinema_linear_work_bytes) linear_work_bytes;
  decltype(&cinema_linear_forward) linear_forward;
  decltype(&cinema_linear_backward) linear_backward;
  decltype(&cinema_layer_norm_work_bytes) layer_norm_work_bytes;
  decltype(&cinema_layer_norm_forward) layer_norm_forward;
  decltype(&cinema_layer_norm_backward) layer_norm_backward;
  decltype(&cinema_grad_norm_work_bytes) grad_norm_work_bytes;
  decltype(&cinema_grad_norm) grad_norm;
  decltype(&cinema_grad_norm_f64) grad_norm_f64;
  decltype(&cinema_grad_clip) grad_clip;
} api = {};
PyObject *error_class = nullptr;      // cinema_amd._lib.CinemaHipError

// `path`: the library that _lib.load() has opened already
void bind(const std::string &path, py::object error) {
  void *h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(h != nullptr, "cannot open ", path, ": ", dlerror());
  auto get = [&](auto &slot, const char *name) {
    slot = reinterpret_cast<std::remove_reference_t<decltype(slot)>>(dlsym(h, name));
    TORCH_CHECK(slot != nullptr, path, " has no ", name);
  };
  get(api.last_error, "cinema_last_error");
  get(api.linear_work_bytes, "cinema_linear_work_bytes");
  get(api.linear_forward, "cinema_linear_forward");
  get(api.linear_backward, "cinema_linear_backward");
  get(api.layer_norm_work_bytes, "cinema_layer_norm_work_bytes");
  get(api.layer_norm_forward, "cinema_layer_norm_forward");
  get(api.layer_norm_backward, "cinema_layer_norm_backward");
  get(api.grad_norm_work_bytes, "cinema_grad_norm_work_bytes");
  get(api.grad_norm, "cinema_grad_norm");
  get(api.grad_norm_f64, "cinema_grad_norm_f64");
  get(api.grad_clip, "cinema_grad_clip");
  Py_XDECREF(error_class);
  error_class = error.release().ptr();
}

[[noreturn]] void raise(const std::string &text) {
  py::gil_scoped_acquire gil;           // the engine's threads come without it
  PyErr_SetString(error_class != nullptr ? error_class : PyExc_RuntimeError, text.c_str());
  throw py::error_already_set();
}
void check(int rc, const char *what) {
  if (rc != 0) raise(std::string(what) + " failed (code " + std::to_string(rc) + "): " + api.last_error());
}

int dtype_of(at::ScalarType t) {
  return t == at::kFloat ? CINEMA_DT_F32 : t == at::kBFloat16 ? CINEMA_DT_BF16 : t == at::kHalf ? CINEMA_DT_F16 : -1;
}
void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
const void *data(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *out(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
Tensor workspace(int64_t bytes, const char *what, const Tensor &like) {
  if (bytes < 0) check(-1, what);
  return bytes == 0 ? Tensor() : at::empty({bytes}, like.options().dtype(at::kByte));
}
bool wants_grad(const Tensor &t) { return t.defined() && t.requires_grad(); }

// rows of `k` values as the kernels read them: contiguous, or a matrix whose rows are at least a row apart; a copy otherwise
struct Rows { Tensor t; int64_t ld; };
Rows rows_of(const Tensor &t, int64_t k) {
  if (t.is_contiguous()) return {t, k};
  if (t.dim() == 2 && (k == 1 || t.stride(1) == 1) && t.stride(0) >= k) return {t, t.size(0) > 1 ? t.stride(0) : k};
  return {t.contiguous(), k};
}
// what a node keeps: the variable itself (so that a later write to it is noticed), or the copy that was made of it
SavedVariable saved(const Tensor &variable, const Rows &r) { return SavedVariable(r.t.is_same(variable) ? variable : r.t, false); }

// A saved tensor as it came back.  Hooks on saved tensors (offloading, checkpointing) give back the values, not the layout, and a
// leaf's .data may have been exchanged: what the kernels rely on is checked here, and strides are taken from the result.
Tensor unpacked(const SavedVariable &saved, const char *what, const char *name, at::IntArrayRef sizes, at::ScalarType type, const Tensor &grad) {
  Tensor t = saved.unpack();
  if (!t.defined()) return t;
  if (t.is_neg()) t = t.resolve_neg();
  TORCH_CHECK(t.layout() == at::kStrided && t.sizes() == sizes && t.scalar_type() == type && t.device() == grad.device(), "cinema_amd ", what,
              ": ", name, " was saved as ", sizes, " of ", type, " on ", grad.device(), " and came back as ", t.sizes(), " of ", t.scalar_type(),
              " on ", t.device());
  return t;
}
Tensor dense(const Tensor &t) { return t.defined() ? t.contiguous() : t; }

void check_rows(const char *what, const Tensor &x) {
  TORCH_CHECK_TYPE(dtype_of(x.scalar_type()) >= 0, what, ": rows are fp32, bf16 or fp16, got ", x.scalar_type());
}
void check_companion(const char *what, const char *name, const Tensor &t, const Tensor &x, bool may_be_f32) {
  if (!t.defined()) return;
  TORCH_CHECK_VALUE(t.device() == x.device(), what, ": ", name, " is on ", t.device(), ", the rows are on ", x.device());
  TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type() || (may_be_f32 && t.scalar_type() == at::kFloat), what, ": ", name, " has type ",
                   t.scalar_type(), ", the rows ", x.scalar_type(), may_be_f32 ? " (it may be fp32)" : "");
}
// lazily negated views become plain tensors; forward-mode tangents would be dropped in silence
void check_plain(const char *what, Tensor &t) {
  if (!t.defined()) return;
  if (t.is_neg()) t = t.resolve_neg();
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "cinema_amd ", what, ": no forward-mode derivative");
}
// A tracer records the allocation of the result and not the launch that fills it: the recorded program would return whatever the
// memory holds.  (torch.compile does not look into these calls; it breaks its graph around them and runs them as they are.)
void check_not_traced(const char *what) {
  using c10::impl::TorchDispatchModeTLS;
  using c10::impl::TorchDispatchModeKey;
  const bool traced = torch::jit::tracer::isTracing() || TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY) ||
                      TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE) || TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FUNCTIONAL);
  TORCH_CHECK_NOT_IMPLEMENTED(!traced, "cinema_amd ", what, ": cannot be traced (torch.jit.trace, make_fx, fake tensors)");
}
void check_gpu(const char *what, const Tensor &x) {
  TORCH_CHECK(x.is_cuda(), "cinema_amd ", what, " runs HIP kernels: the input must live on the GPU");
}
void first_order_only(const char *what) {
  // under create_graph=True the results would silently carry no graph
  TORCH_CHECK(!at::GradMode::is_enabled(), "cinema_amd ", what, ": the gradients have no second derivative (create_graph=True)");
}

// A leaf's accumulator node runs on the stream it was made on and lives as long as an eager graph that uses the leaf.  One of
// the default stream cannot take part in a capture: the captured backward pass would end the process from the engine's thread.
// Asked of the caller's own tensors: a cast (autocast's) hides its leaf behind a node.
template <typename Inputs>
void check_capture(const char *what, const Inputs &inputs) {
  if (!at::GradMode::is_enabled() || std::none_of(inputs.begin(), inputs.end(), [](const Tensor *t) { return wants_grad(*t); })) return;
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  for (const Tensor *t : inputs) {
    if (!wants_grad(*t) || t->grad_fn()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto stream = node ? node->stream() : std::nullopt;
    TORCH_CHECK(!stream || stream->id() != 0, "cinema_amd ", what, ": captured with gradients while an eager graph of the default stream ",
                "uses the same leaves; release its results first, or capture under torch.no_grad()");
  }
}

// for callers that cast their leaves themselves
void check_capture_of(const std::string &what, const std::vector<Tensor> &tensors) {
  std::vector<const Tensor *> on_gpu;
  for (const Tensor &t : tensors)
    if (t.is_cuda()) on_gpu.push_back(&t);
  check_capture(what.c_str(), on_gpu);
}

// ---- linear_act ------------------------------------------------------------------------------------------------------------
struct LinearActBackward : public Node {
  SavedVariable x, w, z;
  int64_t m, k, n;
  int act;
  std::vector<int64_t> x_shape;
  at::ScalarType bias_type, z_type;
  std::mutex mutex;

  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex);
    variable_list got(4);
    if (!grads[0].defined()) return got;
    first_order_only("linear_act");
    const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1), need_b = task_should_compute_output(2);
    if (task_should_compute_output(3)) got[3] = grads[0];
    if (!need_x && !need_w && !need_b) return got;
    const c10::DeviceGuard guard(grads[0].device());
    const Tensor g = grads[0].resolve_neg().contiguous();
    const auto o = g.options();
    if (need_x) got[0] = m ? at::empty(x_shape, o) : at::zeros(x_shape, o);
    if (need_w) got[1] = m ? at::empty({n, k}, o) : at::zeros({n, k}, o);
    if (need_b) got[2] = m ? at::empty({n}, o.dtype(bias_type)) : at::zeros({n}, o.dtype(bias_type));
    if (m == 0) return got;
    const auto t = g.scalar_type();
    const Tensor xs = unpacked(x, "linear_act", "x", x_shape, t, g), ws = dense(unpacked(w, "linear_act", "weight", {n, k}, t, g)),
                 zs = dense(unpacked(z, "linear_act", "the pre-activation", {m, n}, z_type, g));
    const int dt = dtype_of(t);
    const Rows xr = need_w ? rows_of(xs, k) : Rows{Tensor(), k};
    const void *xp = data(xr.t), *wp = need_x ? data(ws) : nullptr;
    const Tensor work = workspace(api.linear_work_bytes(xp, xr.ld, wp, m, k, n, act, dt, 1), "cinema_linear_work_bytes", g);
    check(api.linear_backward(data(g), data(zs), zs.defined() && z_type == at::kFloat, xp, xr.ld, wp, m, k, n, act, dt,
                              bias_type == at::kFloat, out(got[0]), out(got[1]), out(got[2]), out(work), stream_of(g)),
          "cinema_linear_backward");
    return got;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex);
    x.reset_data();
    w.reset_data();
    z.reset_data();
  }
  std::string name() const override { return "LinearActBackward"; }
};

const char *const ACTIVATIONS[] = {"none", "relu", "gelu", "gelu_tanh", "silu"};      // CINEMA_ACT_*

Tensor linear_act(Tensor x, Tensor w, const MaybeTensor &bias, const MaybeTensor &residual, const std::string &activation) {
  const char *what = "linear_act";
  check_not_traced(what);
  int act = -1;
  for (int i = 0; i < 5; ++i)
    if (activation == ACTIVATIONS[i]) act = i;
  TORCH_CHECK_VALUE(act >= 0, what, ": unknown activation '", activation, "', choose from none, relu, gelu, gelu_tanh, silu");
  Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
  if (x.is_cuda()) check_capture(what, std::array{&x, &w, &b, &r});
  if (x.is_cuda() && at::autocast::is_autocast_enabled(at::kCUDA)) {
    const auto t = at::autocast::get_autocast_dtype(at::kCUDA);
    x = x.to(t);
    w = w.to(t);
    if (r.defined()) r = r.to(t);
    if (b.defined() && b.scalar_type() != at::kFloat) b = b.to(t);
  }
  for (Tensor *t : {&x, &w, &b, &r}) check_plain(what, *t);
  check_rows(what, x);
  check_companion(what, "weight", w, x, false);
  check_companion(what, "bias", b, x, true);
  check_companion(what, "residual", r, x, false);
  TORCH_CHECK_VALUE(w.dim() == 2 && w.numel() > 0 && x.dim() >= 1 && x.size(-1) == w.size(1), what, ": rows ", x.sizes(), " do not fit a weight ",
                    w.sizes());
  const int64_t n = w.size(0), k = w.size(1), m = x.numel() / k;
  std::vector<int64_t> y_shape = x.sizes().vec();
  y_shape.back() = n;
  TORCH_CHECK_VALUE(!b.defined() || (b.dim() == 1 && b.size(0) == n), what, ": bias ", b.sizes(), " for ", n, " outputs");
  TORCH_CHECK_VALUE(!r.defined() || r.sizes() == at::IntArrayRef(y_shape), what, ": residual ", r.sizes(), " for an output of ",
                    at::IntArrayRef(y_shape));
  check_gpu(what, x);
  const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || wants_grad(b) || wants_grad(r));
  const bool inner = grad && (x.requires_grad() || w.requires_grad() || wants_grad(b));      // something besides the residual
  Tensor y, z, wc, bc;
  Rows xr, rr;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    y = at::empty(y_shape, x.options());
    // 16-bit rows keep fp16 pre-activations; where few of them make a gradient their rounding would show, and fp32 costs nothing
    if (inner && act != CINEMA_ACT_NONE)
      z = at::empty({m, n}, x.options().dtype(x.scalar_type() == at::kFloat || m * n <= 1 << 18 || n * k <= 2048 || m * k <= 256
                                                               ? at::kFloat : at::kHalf));
    xr = rows_of(x, k);
    wc = w.contiguous();
    if (b.defined()) bc = b.contiguous();
    if (r.defined()) rr = rows_of(r, n);
    if (m > 0) {
      const int dt = dtype_of(x.scalar_type());
      const Tensor work = workspace(api.linear_work_bytes(data(xr.t), xr.ld, data(wc), m, k, n, act, dt, 0), "cinema_linear_work_bytes", x);
      check(api.linear_forward(data(xr.t), xr.ld, data(wc), data(bc), bc.defined() && bc.scalar_type() == at::kFloat, data(rr.t), rr.ld, m, k, n,
                               act, dt, out(z), z.defined() && z.scalar_type() == at::kFloat, out(y), out(work), stream_of(x)),
            "cinema_linear_forward");
    }
  }
  if (grad) {
    auto node = std::shared_ptr<LinearActBackward>(new LinearActBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, b, r));
    if (w.requires_grad()) node->x = saved(x, xr);
    if (x.requires_grad()) node->w = SavedVariable(wc.is_same(w) ? w : wc, false);
    node->z = SavedVariable(z, false);
    node->m = m;
    node->k = k;
    node->n = n;
    node->act = act;
    node->x_shape = x.sizes().vec();
    node->bias_type = b.defined() ? b.scalar_type() : x.scalar_type();
    node->z_type = z.defined() ? z.scalar_type() : at::kFloat;
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---- layer_norm ------------------------------------------------------------------------------------------------------------
struct LayerNormBackward : public Node {
  SavedVariable x, w, stats;
  int64_t m, d;
  std::vector<int64_t> x_shape;
  at::ScalarType w_type;
  std::mutex mutex;

  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex);
    variable_list got(3);
    if (!grads[0].defined()) return got;
    first_order_only("layer_norm");
    const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1), need_b = task_should_compute_output(2);
    const c10::DeviceGuard guard(grads[0].device());
    const Tensor g = grads[0].resolve_neg().contiguous();
    const auto o = g.options();
    if (need_x) got[0] = m ? at::empty(x_shape, o) : at::zeros(x_shape, o);
    if (need_w) got[1] = m ? at::empty({d}, o.dtype(w_type)) : at::zeros({d}, o.dtype(w_type));
    if (need_b) got[2] = m ? at::empty({d}, o.dtype(w_type)) : at::zeros({d}, o.dtype(w_type));
    if (m == 0 || !(need_x || need_w || need_b)) return got;
    const Rows xr = rows_of(unpacked(x, "layer_norm", "x", x_shape, g.scalar_type(), g), d);
    const Tensor ws = dense(unpacked(w, "layer_norm", "weight", {d}, w_type, g)),
                 st = dense(unpacked(stats, "layer_norm", "the statistics", {2, m}, at::kFloat, g));
    const int dt = dtype_of(g.scalar_type());
    Tensor work;
    if (need_w || need_b) work = workspace(api.layer_norm_work_bytes(m, d, dt), "cinema_layer_norm_work_bytes", g);
    const float *mean = st.const_data_ptr<float>();
    check(api.layer_norm_backward(data(g), data(xr.t), xr.ld, data(ws), w_type == at::kFloat, mean, mean + m, m, d, dt, out(got[0]), out(got[1]),
                                  out(got[2]), out(work), stream_of(g)),
          "cinema_layer_norm_backward");
    return got;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex);
    x.reset_data();
    w.reset_data();
    stats.reset_data();
  }
  std::string name() const override { return "LayerNormBackward"; }
};

Tensor layer_norm(Tensor x, const MaybeTensor &weight, const MaybeTensor &bias, double eps) {
  const char *what = "layer_norm";
  check_not_traced(what);
  Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  if (x.is_cuda()) check_capture(what, std::array{&x, &w, &b});
  if (x.is_cuda() && at::autocast::is_autocast_enabled(at::kCUDA)) {
    x = x.to(at::kFloat);
    if (w.defined()) w = w.to(at::kFloat);
    if (b.defined()) b = b.to(at::kFloat);
  }
  for (Tensor *t : {&x, &w, &b}) check_plain(what, *t);
  check_rows(what, x);
  check_companion(what, "weight", w, x, true);
  check_companion(what, "bias", b, x, true);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, what, ": rows ", x.sizes(), " have no values");
  const int64_t d = x.size(-1), m = x.numel() / d;
  TORCH_CHECK_VALUE(!w.defined() || (w.dim() == 1 && w.size(0) == d), what, ": weight ", w.sizes(), " for rows of ", d);
  TORCH_CHECK_VALUE(!b.defined() || (b.dim() == 1 && b.size(0) == d), what, ": bias ", b.sizes(), " for rows of ", d);
  TORCH_CHECK_TYPE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), what, ": weight is ", w.scalar_type(), ", bias ",
                   b.scalar_type());
  TORCH_CHECK_VALUE(eps >= 0, what, ": eps = ", eps);
  check_gpu(what, x);
  const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(w) || wants_grad(b));
  const at::ScalarType w_type = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type();
  Tensor y, stats, wc, bc;
  Rows xr;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    y = at::empty(x.sizes(), x.options());
    if (grad) stats = at::empty({2, m}, x.options().dtype(at::kFloat));
    xr = rows_of(x, d);
    if (w.defined()) wc = w.contiguous();
    if (b.defined()) bc = b.contiguous();
    if (m > 0) {
      float *mean = grad ? stats.mutable_data_ptr<float>() : nullptr;
      check(api.layer_norm_forward(data(xr.t), xr.ld, data(wc), data(bc), w_type == at::kFloat, m, d, (float)eps, dtype_of(x.scalar_type()),
                                   out(y), mean, grad ? mean + m : nullptr, stream_of(x)),
            "cinema_layer_norm_forward");
    }
  }
  if (grad) {
    auto node = std::shared_ptr<LayerNormBackward>(new LayerNormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
    node->x = saved(x, xr);
    node->w = SavedVariable(!w.defined() || wc.is_same(w) ? w : wc, false);
    node->stats = SavedVariable(stats, false);
    node->m = m;
    node->d = d;
    node->x_shape = x.sizes().vec();
    node->w_type = w_type;
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---- gradient norm ---------------------------------------------------------------------------------------------------------
typedef std::pair<uintptr_t, uintptr_t> Span;     // bytes [first, second)

Span extent(const Tensor &t) {
  int64_t last = 0;
  for (int64_t k = 0; k < t.dim(); ++k) last += (t.size(k) - 1) * t.stride(k);
  const uintptr_t p = (uintptr_t)t.const_data_ptr();
  return {p, p + (last + 1) * t.element_size()};
}

// the memory of `t` as runs of neighbouring values
void append_runs(const Tensor &t, std::vector<Span> &runs) {
  std::vector<std::pair<int64_t, int64_t>> dims;      // stride, size
  for (int64_t k = 0; k < t.dim(); ++k)
    if (t.size(k) > 1) dims.emplace_back(t.stride(k), t.size(k));
  std::sort(dims.begin(), dims.end());
  int64_t run = 1;
  size_t d = 0;
  for (; d < dims.size() && dims[d].first == run; ++d) run *= dims[d].second;
  const int64_t count = t.numel() / run;
  TORCH_CHECK_VALUE((int64_t)runs.size() + count <= 1 << 24, "clip_grad_norm_: gradients are interleaved too finely to tell whether they overlap");
  const uintptr_t p = (uintptr_t)t.const_data_ptr(), es = t.element_size();
  for (int64_t n = 0; n < count; ++n) {
    int64_t at = 0, left = n;
    for (size_t k = d; k < dims.size(); ++k) {
      at += left % dims[k].second * dims[k].first;
      left /= dims[k].second;
    }
    runs.emplace_back(p + at * es, p + (at + run) * es);
  }
}

// Gradients are scaled side by side, so none may share memory with another.  Where the extents of two meet (columns of one
// table, say), their runs are compared.
void check_apart(const std::vector<Tensor> &grads) {
  std::vector<std::pair<Span, size_t>> all;
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].numel() > 0) all.emplace_back(extent(grads[i]), i);
  std::sort(all.begin(), all.end());
  std::vector<bool> meets(all.size(), false);
  for (size_t i = 1, far = 0; i < all.size(); ++i) {      // far: the one before i that reaches furthest
    if (all[i].first.first < all[far].first.second) meets[i] = meets[far] = true;
    if (all[i].first.second > all[far].first.second) far = i;
  }
  std::vector<Span> runs;
  for (size_t i = 0; i < all.size(); ++i)
    if (meets[i]) append_runs(grads[all[i].second], runs);
  std::sort(runs.begin(), runs.end());
  for (size_t i = 1; i < runs.size(); ++i)
    TORCH_CHECK_VALUE(runs[i].first >= runs[i - 1].second, "clip_grad_norm_: a gradient is listed twice or overlaps another");
}

// the norm of all gradients before clipping; max_norm given: clips them in place.  `wide`: gets the norm in 64 bits too
Tensor take_norm(const std::vector<Tensor> &grads, double norm_type, std::optional<double> max_norm, Tensor *wide) {
  check_not_traced("gradient norm");
  const double inf = std::numeric_limits<double>::infinity();
  TORCH_CHECK_VALUE(norm_type == 1. || norm_type == 2. || norm_type == inf, "norm_type is 1, 2 or inf, got ", norm_type);
  TORCH_CHECK_VALUE(!max_norm || *max_norm >= 0, "max_norm = ", max_norm.value_or(0));
  const int kind = norm_type == inf ? 0 : (int)norm_type;
  if (grads.empty()) return at::zeros({}, at::kFloat);
  std::vector<cinema_grad_tensor> table(grads.size());
  std::vector<Tensor> copies(grads.size());
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor &g = grads[i];
    TORCH_CHECK_TYPE(g.layout() == at::kStrided, "gradient norm: sparse gradients are not supported");
    TORCH_CHECK_VALUE(!g.is_neg(), "gradient norm: lazily negated gradients are not supported");
    const int dt = dtype_of(g.scalar_type());
    TORCH_CHECK_TYPE(dt >= 0, "gradient norm: gradients are fp32, bf16 or fp16, got ", g.scalar_type());
    TORCH_CHECK_VALUE(g.device() == grads[0].device(),
                      "gradient norm: the gradients are on several devices; combine the norms of each (grad_norm) instead");
    if (!g.is_contiguous()) {
      for (int64_t k = 0; max_norm && k < g.dim(); ++k)
        TORCH_CHECK_VALUE(g.stride(k) != 0 || g.size(k) <= 1, "clip_grad_norm_: an expanded gradient cannot be scaled in place");
      at::AutoDispatchBelowADInplaceOrView below;
      copies[i] = g.contiguous();
    }
    const Tensor &c = copies[i].defined() ? copies[i] : g;
    table[i] = {const_cast<void *>(c.const_data_ptr()), c.numel(), dt, 0};
  }
  if (max_norm) check_apart(grads);
  if (!grads[0].is_cuda()) raise("gradient norm runs HIP kernels: the gradients must live on the GPU");
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(grads[0].device());
  const Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
  const int n = (int)grads.size();
  const Tensor work = workspace(api.grad_norm_work_bytes(n), "cinema_grad_norm_work_bytes", norm);
  void *st = stream_of(norm);
  if (wide != nullptr) {
    *wide = at::empty({}, norm.options().dtype(at::kDouble));
    check(api.grad_norm_f64(table.data(), n, kind, out(work), norm.mutable_data_ptr<float>(), wide->mutable_data_ptr<double>(), st),
          "cinema_grad_norm_f64");
    return norm;
  }
  if (!max_norm) {
    check(api.grad_norm(table.data(), n, kind, out(work), norm.mutable_data_ptr<float>(), st), "cinema_grad_norm");
    return norm;
  }
  check(api.grad_clip(table.data(), n, kind, (float)*max_norm, out(work), norm.mutable_data_ptr<float>(), st), "cinema_grad_clip");
  for (size_t i = 0; i < grads.size(); ++i) {
    if (copies[i].defined()) const_cast<Tensor &>(grads[i]).copy_(copies[i]);
    if (!grads[i].is_inference()) grads[i].unsafeGetTensorImpl()->bump_version();     // written behind autograd's back, copy_ below it too
  }
  return norm;
}
Tensor grad_norm(const std::vector<Tensor> &grads, double norm_type, std::optional<double> max_norm) {
  return take_norm(grads, norm_type, max_norm, nullptr);
}
// the norm as fp32, and in 64 bits
std::pair<Tensor, Tensor> grad_norm_wide(const std::vector<Tensor> &grads, double norm_type) {
  Tensor wide;
  const Tensor norm = take_norm(grads, norm_type, std::nullopt, &wide);
  return {norm, wide.defined() ? wide : norm.to(at::kDouble)};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("linear_act", &linear_act);
  m.def("layer_norm", &layer_norm);
  m.def("check_capture", &check_capture_of);
  m.def("grad_norm", &grad_norm);
  m.def("grad_norm_wide", &grad_norm_wide);
}

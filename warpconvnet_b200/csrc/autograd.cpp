// Nodes of autograd's graph for RMS norm, dropout and linear layers: what their gradient needs is kept here, and the engine calls the C
// entry points without Python.  A training step of small layers waits for the host: an autograd function in Python takes some 50 us both
// ways before it does anything, most of it for the interpreter's lock in the engine's thread (both ways, us, that way and this: linear
// 2 000 x 96 -> 20 fp16 123, 96; dropout 2 001 x 64 fp32 81, 64; RMS norm 240 000 x 96 bf16 127, 100).
// A node runs the gradient of tensors that lie as the kernels read them; all else (rows that have to be copied, a graph of the gradient)
// goes to the operator's function in Python, which gives the same.
//
// The calls themselves are made here too where nothing has to be copied, cast or refused (us of the host for one row: RMS norm 9, here 5;
// linear 12, here 6, of 8-bit operands 15 and 6; the three above both ways then take 73, 52 and
// 78).  Arguments that the functions here do not take get no result, and Python goes on with them.
//
// A way of calling and no more: where this extension is not built, autograd functions in Python make the same calls.
#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/grad_mode.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <dlfcn.h>

#include <atomic>
#include <cstring>
#include <limits>
#include <locale>

#include "../../include/wcn_b200.h"

#ifndef WCN_BUILT_WITH   // torch.__version__
#error "compile with csrc/build.py"
#endif
#define WCN_BUILT_WITH_MARK "built with torch " WCN_BUILT_WITH   // (which build.py looks for in the file)

namespace py = pybind11;
using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

struct Functions {   // of the loaded library
  decltype(&wcn_status_string) status_string = nullptr;
  decltype(&wcn_training_launches) launches = nullptr;
  decltype(&wcn_linear_workspace_bytes) linear_bytes = nullptr;
  decltype(&wcn_linear_backward) linear = nullptr;
  decltype(&wcn_linear) linear_forward = nullptr;
  decltype(&wcn_linear_8bit) linear_8bit = nullptr;
  decltype(&wcn_rms_norm) norm_forward = nullptr;
  decltype(&wcn_rms_norm_workspace_bytes) norm_bytes = nullptr;
  decltype(&wcn_rms_norm_backward) norm = nullptr;
  decltype(&wcn_dropout) dropout = nullptr;
} native;
// The operators' functions in Python, kept for good: a node may outlive the interpreter's lock.
py::object *linear_in_python, *norm_in_python, *dropout_in_python;
struct Launched {   // kernels since they were last asked for
  std::atomic<int64_t> linear{0}, norm{0}, dropout{0}, linear_forward{0}, norm_forward{0}, linear_8bit{0};
} launched;

void check(int status, const char* what) {
  TORCH_CHECK(!status, "libwcn_b200 ", what, " failed: ", native.status_string(status), " (", status, ")");
}
void* at_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool in_rows(const Tensor& t) { return !t.defined() || t.is_contiguous(); }
bool on_lines(const Tensor& t, int64_t whole) { return t.is_contiguous() && t.size(1) % whole == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
py::object given(const Tensor& t) { return t.defined() ? py::cast(t) : py::none(); }
variable_list taken(const py::tuple& got) {
  variable_list out(got.size());
  for (size_t i = 0; i < got.size(); ++i)
    if (!got[i].is_none()) out[i] = got[i].cast<Tensor>();
  return out;
}
// Runs `call`, which asks Python: an exception there is the engine's, as one of C++ that holds no Python object.
template <typename F> variable_list ask(F call) {
  py::gil_scoped_acquire lock;
  try {
    return taken(call());
  } catch (py::error_already_set& e) {
    python_error raised;
    e.restore();
    raised.persist();
    throw std::move(raised);
  }
}

struct LinearNode : Node {
  SavedVariable x, weight, bias, seed, x_rows, w_rows;
  int64_t act = 0, least = 0, number = 0, code = 0;
  void* status = nullptr;
  std::string name() const override { return "LinearBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&x, &weight, &bias, &seed, &x_rows, &w_rows}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::unique_lock<std::mutex> lock(mutex_);
    Tensor dy = grads[0];
    if (!dy.defined()) return variable_list(4);
    const Tensor xt = x.unpack(), wt = weight.unpack(), bt = bias.unpack(), st = seed.unpack(), xr = x_rows.unpack(), wr = w_rows.unpack();
    lock.unlock();
    bool need[4];
    for (int i = 0; i < 4; ++i) need[i] = task_should_compute_output(i);
    const int64_t whole = code == WCN_F32 ? 1 : 8;
    if (c10::GradMode::is_enabled() || xr.defined() || wr.defined() || !dy.is_contiguous() || !on_lines(xt, whole) || !on_lines(wt, whole) || !in_rows(bt))
      return ask([&] {
        return (*linear_in_python)(given(xt), given(wt), given(bt), given(st), given(xr), given(wr), act, least, number, code,
                                   py::make_tuple(need[0], need[1], need[2], need[3]), given(dy));
      });
    variable_list out(4);
    if (need[3]) out[3] = dy;
    if (!need[0] && !need[1] && !need[2]) return out;
    c10::DeviceGuard device(xt.device());
    const int64_t n = xt.size(0), k = xt.size(1), m = wt.size(0);
    if (need[0]) out[0] = at::empty({n, k}, xt.options().requires_grad(false));
    if (need[1]) out[1] = at::empty({m, k}, wt.options().requires_grad(false));
    if (need[2]) out[2] = at::empty({m}, wt.options().requires_grad(false));
    const bool aligned = m % whole == 0 && reinterpret_cast<uintptr_t>(dy.data_ptr()) % (2 * whole) == 0;   // (fp32: always)
    int64_t size = 0;
    check(native.linear_bytes(n, k, m, code, need[0] + 2 * need[1] + 4 * need[2], act, least, aligned, &size), "wcn_linear_workspace_bytes");
    Tensor ws;
    if (size) ws = at::empty({size}, xt.options().dtype(at::kByte).requires_grad(false));
    check(native.linear(xt.data_ptr(), k, n, k, wt.data_ptr(), k, m, code, at_of(bt), act, dy.data_ptr(), m, least, number,
                        static_cast<const int64_t*>(at_of(st)), at_of(out[0]), at_of(out[1]), at_of(out[2]), at_of(ws), size,
                        static_cast<int32_t*>(status), stream_of(xt)),
          "wcn_linear_backward");
    launched.linear += native.launches();
    return out;
  }
};

struct NormNode : Node {
  SavedVariable x, residual, weight, h, rstd;
  bool sum = false;   // h = x + residual is a result
  double eps = 0;
  int64_t code = 0;
  std::string name() const override { return "RMSNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&x, &residual, &weight, &h, &rstd}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::unique_lock<std::mutex> lock(mutex_);
    Tensor dy = grads[0], dh = sum ? grads[1] : Tensor();
    if (!dy.defined() && !dh.defined()) return variable_list(3);
    const Tensor xt = x.unpack(), rt = residual.unpack(), wt = weight.unpack(), ht = sum ? h.unpack(shared_from_this()) : Tensor(), st = rstd.unpack();
    lock.unlock();
    const bool need[3] = {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2)};
    const Tensor rows = sum ? ht : xt;
    if (c10::GradMode::is_enabled() || !dy.defined() || !rows.size(0) || !dy.is_contiguous() || !in_rows(dh) || !rows.is_contiguous() ||
        (wt.defined() && (wt.scalar_type() != at::kFloat || !wt.is_contiguous())))
      return ask([&] {
        return (*norm_in_python)(given(xt), given(rt), given(wt), given(ht), given(st), eps, py::make_tuple(need[0], need[1], need[2]), given(dy), given(dh));
      });
    variable_list out(3);
    c10::DeviceGuard device(rows.device());
    const int64_t n = rows.size(0), c = rows.size(1);
    Tensor dx, ws;
    int64_t size = 0;
    if (need[0] || need[1]) dx = at::empty({n, c}, rows.options().requires_grad(false));
    if (need[2]) {
      out[2] = at::empty({c}, wt.options().requires_grad(false));
      check(native.norm_bytes(n, c, &size), "wcn_rms_norm_workspace_bytes");
      ws = at::empty({size}, rows.options().dtype(at::kByte).requires_grad(false));
    }
    check(native.norm(rows.data_ptr(), c, dy.data_ptr(), c, at_of(dh), c, n, c, code, static_cast<const float*>(at_of(wt)),
                      static_cast<const float*>(st.data_ptr()), at_of(dx), static_cast<float*>(at_of(out[2])), at_of(ws), size, stream_of(rows)),
          "wcn_rms_norm_backward");
    launched.norm += native.launches();
    if (need[0]) out[0] = dx;
    if (need[1]) out[1] = dx;
    return out;
  }
};

struct DropoutNode : Node {
  SavedVariable seed;
  int64_t least = 0, number = 0, code = 0;
  std::string name() const override { return "DropoutBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    seed.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::unique_lock<std::mutex> lock(mutex_);
    Tensor dy = grads[0];
    if (!dy.defined()) return variable_list(2);
    const Tensor st = seed.unpack();
    lock.unlock();
    const bool need[2] = {task_should_compute_output(0), task_should_compute_output(1)};
    if (c10::GradMode::is_enabled() || !dy.is_contiguous() || !dy.numel())
      return ask([&] { return (*dropout_in_python)(given(st), least, number, py::make_tuple(need[0], need[1]), given(dy)); });
    variable_list out(2);
    if (need[1]) out[1] = dy;
    if (!need[0]) return out;
    c10::DeviceGuard device(dy.device());
    out[0] = at::empty(dy.sizes(), dy.options().requires_grad(false));
    check(native.dropout(dy.data_ptr(), dy.size(1), nullptr, dy.size(1), dy.size(0), dy.size(1), code, least, number, static_cast<const int64_t*>(at_of(st)),
                         out[0].data_ptr(), stream_of(dy)),
          "wcn_dropout");
    launched.dropout += 1;
    return out;
  }
};

SavedVariable kept(const std::optional<Tensor>& t) { return SavedVariable(t.value_or(Tensor()), false); }

Tensor linear(Tensor y, Tensor x, Tensor weight, std::optional<Tensor> bias, std::optional<Tensor> residual, std::optional<Tensor> seed,
              std::optional<Tensor> x_rows, std::optional<Tensor> w_rows, int64_t act, int64_t least, int64_t number, int64_t code, int64_t status) {
  auto node = std::shared_ptr<LinearNode>(new LinearNode(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x, weight, bias.value_or(Tensor()), residual.value_or(Tensor())));
  node->x = kept(x), node->weight = kept(weight), node->bias = kept(bias), node->seed = kept(seed);
  node->x_rows = kept(x_rows), node->w_rows = kept(w_rows);
  node->act = act, node->least = least, node->number = number, node->code = code, node->status = reinterpret_cast<void*>(status);
  torch::autograd::set_history(y, node);
  return y;
}

void norm(Tensor y, std::optional<Tensor> h, Tensor x, std::optional<Tensor> residual, std::optional<Tensor> weight, Tensor rstd, double eps, int64_t code) {
  auto node = std::shared_ptr<NormNode>(new NormNode(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x, residual.value_or(Tensor()), weight.value_or(Tensor())));
  node->sum = h.has_value(), node->eps = eps, node->code = code;
  torch::autograd::set_history(y, node);
  if (h) {
    torch::autograd::set_history(*h, node);
    node->h = SavedVariable(*h, true);
  }
  node->x = kept(x), node->residual = kept(residual), node->weight = kept(weight), node->rstd = kept(rstd);
}

void dropout(Tensor y, Tensor x, std::optional<Tensor> residual, std::optional<Tensor> seed, int64_t least, int64_t number, int64_t code) {
  auto node = std::shared_ptr<DropoutNode>(new DropoutNode(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x, residual.value_or(Tensor())));
  node->seed = kept(seed);
  node->least = least, node->number = number, node->code = code;
  torch::autograd::set_history(y, node);
}

// ------------------------------------------------------------------ calls

constexpr int MOST_DEVICES = 64;
void* status_words[MOST_DEVICES];   // null: Python has not made it yet

// A device's tensor as it is in memory: no subclass that answers for itself, no wrapper of a function transform.
bool plain(const Tensor& t, const at::Device& device, at::ScalarType type) {
  return t.device() == device && t.scalar_type() == type && t.layout() == at::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch() && t.is_contiguous();
}
// Whether x, [n, c], is taken: on the current device, of a type whose code is set.
bool rows_taken(const Tensor& x, int64_t most_rows, int64_t most_columns, int& code) {
  if (!x.is_cuda() || x.dim() != 2 || x.size(0) < 1 || x.size(0) > most_rows || x.size(1) < 1 || x.size(1) > most_columns) return false;
  switch (x.scalar_type()) {
    case at::kFloat: code = WCN_F32; break;
    case at::kHalf: code = WCN_F16; break;
    case at::kBFloat16: code = WCN_BF16; break;
    default: return false;
  }
  return plain(x, x.device(), x.scalar_type()) && x.device().index() < MOST_DEVICES && x.device().index() == c10::cuda::current_device();
}
bool same_rows(const std::optional<Tensor>& t, const Tensor& x, int64_t n, int64_t c) {
  return !t || (t->dim() == 2 && t->size(0) == n && t->size(1) == c && plain(*t, x.device(), x.scalar_type()));
}
bool wants(const Tensor& t) { return t.requires_grad(); }
bool wants(const std::optional<Tensor>& t) { return t && t->requires_grad(); }
Tensor rows_like(const Tensor& x, int64_t n, int64_t c) { return at::empty({n, c}, x.options().requires_grad(false)); }

std::optional<Tensor> run_linear(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias, const std::optional<Tensor>& residual, int64_t act,
                                 int64_t least, int64_t number, int64_t most_rows, int64_t most_inputs, int64_t most_outputs) {
  int code = 0;
  if (!rows_taken(x, most_rows, most_inputs, code) || at::autocast::is_autocast_enabled(at::kCUDA)) return std::nullopt;
  const int64_t n = x.size(0), k = x.size(1), whole = code == WCN_F32 ? 1 : 8;
  if (weight.dim() != 2 || weight.size(1) != k || weight.size(0) < 1 || weight.size(0) > most_outputs || !plain(weight, x.device(), x.scalar_type()))
    return std::nullopt;
  const int64_t m = weight.size(0);
  void* const status = status_words[x.device().index()];
  if (!status || !on_lines(x, whole) || !on_lines(weight, whole) || !same_rows(residual, x, n, m) ||
      (bias && (bias->dim() != 1 || bias->size(0) != m || !plain(*bias, x.device(), x.scalar_type()))))
    return std::nullopt;
  Tensor y = rows_like(x, n, m), ws;
  int64_t size = 0;
  if (code == WCN_F32) check(native.linear_bytes(n, k, m, code, 0, act, least, 0, &size), "wcn_linear_workspace_bytes");
  if (size) ws = at::empty({size}, x.options().dtype(at::kByte).requires_grad(false));
  check(native.linear_forward(x.data_ptr(), k, n, k, weight.data_ptr(), k, m, code, bias ? bias->data_ptr() : nullptr, act,
                              residual ? residual->data_ptr() : nullptr, m, least, number, nullptr, y.data_ptr(), at_of(ws), size,
                              static_cast<int32_t*>(status), stream_of(x)),
        "wcn_linear");
  launched.linear_forward += native.launches();
  if (c10::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias) || wants(residual)))
    return linear(y, x, weight, bias, residual, std::nullopt, std::nullopt, std::nullopt, act, least, number, code, reinterpret_cast<int64_t>(status));
  return y;
}

// eight: codes and scales in the norm's place, and no graph.
py::object run_norm(const Tensor& x, const std::optional<Tensor>& weight, double eps, const std::optional<Tensor>& residual, bool eight, double least_eps,
                    int64_t most_rows, int64_t most_channels) {
  int code = 0;
  if (!rows_taken(x, most_rows, most_channels, code) || !(eps >= least_eps) || eps > std::numeric_limits<float>::max()) return py::none();
  const int64_t n = x.size(0), c = x.size(1);
  if (!same_rows(residual, x, n, c) || (weight && (weight->dim() != 1 || weight->size(0) != c || !plain(*weight, x.device(), at::kFloat)))) return py::none();
  const bool graph = c10::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(residual));
  if (eight && graph) return py::none();   // (refused there)
  Tensor y, rstd, scale;
  std::optional<Tensor> h;
  {
    py::gil_scoped_release others;
    y = eight ? at::empty({n, c}, x.options().dtype(at::kFloat8_e4m3fn).requires_grad(false)) : rows_like(x, n, c);
    if (eight) scale = at::empty({n}, x.options().dtype(at::kFloat).requires_grad(false));
    if (residual) h = rows_like(x, n, c);
    if (graph) rstd = at::empty({n}, x.options().dtype(at::kFloat).requires_grad(false));
    const float number = static_cast<float>(eps);
    int32_t bits;
    std::memcpy(&bits, &number, 4);
    check(native.norm_forward(x.data_ptr(), c, residual ? residual->data_ptr() : nullptr, c, n, c, code,
                              weight ? static_cast<const float*>(weight->data_ptr()) : nullptr, bits, h ? h->data_ptr() : nullptr, eight ? nullptr : y.data_ptr(),
                              static_cast<float*>(at_of(rstd)), eight ? y.data_ptr() : nullptr, static_cast<float*>(at_of(scale)), stream_of(x)),
          "wcn_rms_norm");
    launched.norm_forward += 1;
  }
  if (eight) return h ? py::make_tuple(y, scale, *h) : py::make_tuple(y, scale);
  if (graph) norm(y, h, x, residual, weight, rstd, eps, code);
  return h ? py::object(py::make_tuple(y, *h)) : py::cast(y);
}

std::optional<Tensor> run_linear_8bit(const Tensor& x, const Tensor& x_scale, const Tensor& weight, const Tensor& weight_scale, const std::optional<Tensor>& bias,
                                      int64_t act, const std::optional<Tensor>& residual, int64_t code, int64_t most_rows, int64_t most_inputs,
                                      int64_t most_outputs) {
  if (!x.is_cuda() || x.dim() != 2 || weight.dim() != 2 || x.device().index() >= MOST_DEVICES || x.device().index() != c10::cuda::current_device())
    return std::nullopt;
  const int64_t n = x.size(0), k = x.size(1), m = weight.size(0);
  const at::Device device = x.device();
  const at::ScalarType type = code == WCN_F16 ? at::kHalf : at::kBFloat16;
  void* const status = status_words[device.index()];
  if (!status || n < 1 || n > most_rows || k < 1 || k > most_inputs || m < 1 || m > most_outputs || weight.size(1) != k ||
      !plain(x, device, at::kFloat8_e4m3fn) || !plain(weight, device, at::kFloat8_e4m3fn) || !on_lines(x, 16) || !on_lines(weight, 16))
    return std::nullopt;
  if (x_scale.dim() != 1 || x_scale.size(0) != n || !plain(x_scale, device, at::kFloat) || weight_scale.dim() != 1 || weight_scale.size(0) != m ||
      !plain(weight_scale, device, at::kFloat) || (bias && (bias->dim() != 1 || bias->size(0) != m || !plain(*bias, device, type))) ||
      (residual && (residual->dim() != 2 || residual->size(0) != n || residual->size(1) != m || !plain(*residual, device, type))))
    return std::nullopt;
  if (c10::GradMode::is_enabled() && (wants(x) || wants(x_scale) || wants(weight) || wants(weight_scale) || wants(bias) || wants(residual)))
    return std::nullopt;   // (refused there)
  Tensor y = at::empty({n, m}, x.options().dtype(type).requires_grad(false));
  check(native.linear_8bit(x.data_ptr(), k, static_cast<const float*>(x_scale.data_ptr()), n, k, weight.data_ptr(), k,
                           static_cast<const float*>(weight_scale.data_ptr()), m, code, bias ? bias->data_ptr() : nullptr, act,
                           residual ? residual->data_ptr() : nullptr, residual ? m : 0, y.data_ptr(), static_cast<int32_t*>(status), stream_of(x)),
        "wcn_linear_8bit");
  launched.linear_8bit += native.launches();
  return y;
}

std::optional<Tensor> run_dropout(const Tensor& x, const std::optional<Tensor>& residual, int64_t least, int64_t number, int64_t most_rows,
                                  int64_t most_columns) {
  int code = 0;
  if (!rows_taken(x, most_rows, most_columns, code) || !same_rows(residual, x, x.size(0), x.size(1))) return std::nullopt;
  const int64_t n = x.size(0), c = x.size(1);
  Tensor y = rows_like(x, n, c);
  check(native.dropout(x.data_ptr(), c, residual ? residual->data_ptr() : nullptr, c, n, c, code, least, number, nullptr, y.data_ptr(), stream_of(x)),
        "wcn_dropout");
  launched.dropout += 1;
  if (c10::GradMode::is_enabled() && (wants(x) || wants(residual))) dropout(y, x, residual, std::nullopt, least, number, code);
  return y;
}

// Whether this file has a C++ library of its own in it.  Two of them in a process share some of their objects and not others: a number in
// the text of an error then ends the process.
bool own_library() {
  Dl_info here, there;
  const std::locale& (*const classic)() = &std::locale::classic;
  return dladdr(reinterpret_cast<const void*>(&own_library), &here) && dladdr(reinterpret_cast<const void*>(classic), &there) && here.dli_fbase == there.dli_fbase;
}

template <typename F> void take(F& function, const py::dict& addresses, const char* name) {
  function = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

}  // namespace

PYBIND11_MODULE(_autograd, m) {
  // Nodes and saved variables are laid out as the torch has them that this file was compiled with: no other one may run it.
  const std::string version = py::str(py::module_::import("torch").attr("__version__"));
  if (version != WCN_BUILT_WITH) throw py::import_error("_autograd.so was " WCN_BUILT_WITH_MARK ", not " + version);
  if (own_library()) throw py::import_error("_autograd.so is linked with a C++ library of its own");
  m.def("bind", [](const py::dict& a, py::object l, py::object n, py::object d) {
    take(native.status_string, a, "wcn_status_string");
    take(native.launches, a, "wcn_training_launches");
    take(native.linear_bytes, a, "wcn_linear_workspace_bytes");
    take(native.linear, a, "wcn_linear_backward");
    take(native.linear_forward, a, "wcn_linear");
    take(native.linear_8bit, a, "wcn_linear_8bit");
    take(native.norm_forward, a, "wcn_rms_norm");
    take(native.norm_bytes, a, "wcn_rms_norm_workspace_bytes");
    take(native.norm, a, "wcn_rms_norm_backward");
    take(native.dropout, a, "wcn_dropout");
    linear_in_python = new py::object(l), norm_in_python = new py::object(n), dropout_in_python = new py::object(d);
  });
  m.def("launches", [] { return py::make_tuple(launched.linear.exchange(0), launched.norm.exchange(0), launched.dropout.exchange(0),
                                                    launched.linear_forward.exchange(0), launched.norm_forward.exchange(0), launched.linear_8bit.exchange(0)); });
  m.def("linear", &linear);
  m.def("norm", &norm);
  m.def("dropout", &dropout);
  m.def("status", [](int64_t device, uintptr_t word) {
    if (device >= 0 && device < MOST_DEVICES) status_words[device] = reinterpret_cast<void*>(word);
  });
  // A launch waits where a stream's queue is full, as long as the GPU takes (for another thread's launch, it may be): Python's other threads go on.
  m.def("run_linear", &run_linear, py::call_guard<py::gil_scoped_release>());
  m.def("run_linear_8bit", &run_linear_8bit, py::call_guard<py::gil_scoped_release>());
  m.def("run_norm", &run_norm);   // (itself, as its results are Python's)
  m.def("run_dropout", &run_dropout, py::call_guard<py::gil_scoped_release>());
}

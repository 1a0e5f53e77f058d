// The host side of the operators of a training step beside its products and
// attention cores, as a Python module: the autograd node of the norms over rows,
// calls of rotary positions, and the lists of tensors of the gradient norm and of an AdamW
// step.  Calls of small inputs are bound by the host, and lists of some hundred
// tensors by what each costs, so what a call does once its options are checked
// is done here.  Allocations are torch's; the arithmetic is the library's,
// reached by the addresses that bind() is given.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cstring>
#include <optional>

#include "../../include/terra_swin.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

decltype(&terra_swin_layer_norm) norm_entry = nullptr;
decltype(&terra_swin_layer_norm_bwd) norm_backward_entry = nullptr;
decltype(&terra_swin_rotary) rotary_entry = nullptr;
decltype(&terra_swin_gradient_norm_workspace) gradient_norm_workspace_entry = nullptr;
decltype(&terra_swin_gradient_norm) gradient_norm_entry = nullptr;
decltype(&terra_swin_adamw) adamw_entry = nullptr;
decltype(&terra_last_error) last_error = nullptr;

void check(int status, const char* what) {
  TORCH_CHECK(status != TERRA_ERR_LAUNCH, what, ": ", last_error());
  TORCH_CHECK_VALUE(status == TERRA_OK, what, ": ", last_error());
}

const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// The current stream of the tensor's device.
void* current_stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// Counts a tensor that a kernel writes as changed (a graph that saved its values refuses them then).
void changed(const Tensor& t) {
  if (!t.is_inference()) torch::autograd::impl::bump_version(t);  // an inference tensor is in no graph
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return TERRA_DTYPE_F32;
    case at::kHalf: return TERRA_DTYPE_F16;
    case at::kBFloat16: return TERRA_DTYPE_BF16;
    default: return -1;
  }
}

at::ScalarType scalar_type(int code) {
  return code == TERRA_DTYPE_F32 ? at::kFloat : code == TERRA_DTYPE_F16 ? at::kHalf : at::kBFloat16;
}

template <typename D>
void fill(D* desc, const std::string& bytes) {
  TORCH_CHECK(bytes.size() == sizeof(D), "descriptor of ", bytes.size(), " bytes, expected ", sizeof(D));
  std::memcpy(desc, bytes.data(), sizeof(D));
}

// ---- norms over rows -------------------------------------------------------------

// What the checked arguments of a call say about it, but the tensors.
struct NormCall {
  terra_swin_layer_norm_desc desc;
  int64_t workspace;  // of the backward, fp32 values
};

std::shared_ptr<NormCall> make_norm_call(const std::string& desc, int64_t workspace) {
  auto c = std::make_shared<NormCall>();
  fill(&c->desc, desc);
  c->workspace = workspace;
  return c;
}

// A parameter as the kernels take it: packed, of the call's dtype.
Tensor parameter(const Tensor& t, const NormCall& c) {
  return t.defined() ? t.to(scalar_type(c.desc.param_dtype)).contiguous() : t;
}

void norm_forward(const NormCall& c, const Tensor& x, const Tensor& y, const Tensor& weight, const Tensor& bias,
                  const Tensor& statistics) {
  const Tensor w = parameter(weight, c), b = parameter(bias, c);
  if (c.desc.rows > 0)
    check(norm_entry(x.const_data_ptr(), y.data_ptr(), &c.desc, ptr(w), ptr(b),
                     statistics.defined() ? static_cast<float*>(statistics.data_ptr()) : nullptr, current_stream(x)),
          "terra_swin_layer_norm");
}

Tensor new_statistics(const NormCall& c, const Tensor& x) {
  return at::empty({c.desc.rows, 2}, x.options().dtype(at::kFloat));
}

Tensor new_output(const NormCall& c, const Tensor& x) {
  return at::empty(x.sizes(), x.options().dtype(scalar_type(c.desc.y_dtype)));
}

struct NormGradients {
  Tensor dx, dweight, dbias;
};

// dy packed, of y's dtype; x with the strides of the call.
NormGradients norm_gradients(const NormCall& c, const Tensor& dy, const Tensor& x, const Tensor& weight, const Tensor& bias,
                             const Tensor& statistics, bool need_x, bool need_w, bool need_b) {
  const c10::DeviceGuard guard(x.device());
  const Tensor w = parameter(weight, c);
  NormGradients g;
  Tensor work;
  if (need_x) g.dx = at::empty(x.sizes(), x.options());
  const auto params = x.options().dtype(scalar_type(c.desc.param_dtype));
  if (need_w) g.dweight = at::empty({c.desc.channels}, params);
  if (need_b) g.dbias = at::empty({c.desc.channels}, params);
  if (need_w || need_b) work = at::empty({c.workspace}, x.options().dtype(at::kFloat));
  if (need_x || need_w || need_b)
    check(norm_backward_entry(dy.const_data_ptr(), x.const_data_ptr(), static_cast<const float*>(statistics.const_data_ptr()),
                              need_x ? g.dx.data_ptr() : nullptr, &c.desc, ptr(w), need_w ? g.dweight.data_ptr() : nullptr,
                              need_b ? g.dbias.data_ptr() : nullptr,
                              work.defined() ? static_cast<float*>(work.data_ptr()) : nullptr, current_stream(x)),
          "terra_swin_layer_norm_bwd");
  if (need_w) g.dweight = g.dweight.to(weight.scalar_type());
  if (need_b) g.dbias = g.dbias.to(bias.scalar_type());
  return g;
}

// The same in torch's operations, in fp32 where the types are shorter, for a
// backward pass that is to be differentiated itself.
variable_list norm_gradients_in_operations(const NormCall& c, const Tensor& dy, const Tensor& x, const Tensor& weight,
                                           const Tensor& bias) {
  const Tensor xf = x.to(at::kFloat), d = dy.to(at::kFloat);
  const Tensor centred = c.desc.norm == TERRA_NORM_LAYER ? xf - xf.mean(-1, true) : xf;
  const Tensor r = (centred * centred).mean(-1, true).add(static_cast<double>(c.desc.eps)).rsqrt(), xh = centred * r;
  const Tensor g = weight.defined() ? d * weight.to(at::kFloat) : d;
  Tensor dx = g - xh * (g * xh).mean(-1, true);
  if (c.desc.norm == TERRA_NORM_LAYER) dx = dx - g.mean(-1, true);
  auto over_rows = [](const Tensor& t, const Tensor& like) { return t.reshape({-1, t.size(-1)}).sum(0).to(like.scalar_type()); };
  return {(dx * r).to(x.scalar_type()), weight.defined() ? over_rows(d * xh, weight) : Tensor(),
          bias.defined() ? over_rows(d, bias) : Tensor()};
}

struct LayerNormBackward : public torch::autograd::Node {
  std::shared_ptr<NormCall> call;
  SavedVariable x, weight, bias, statistics;
  std::vector<int64_t> x_strides;
  bool has_weight = false, has_bias = false;

  std::string name() const override { return "LayerNormBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    weight.reset_data();
    bias.reset_data();
    statistics.reset_data();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const Tensor dy = grads[0];
    if (!dy.defined()) return variable_list(3);
    Tensor xv = x.unpack(), wv, bv;
    if (has_weight) wv = weight.unpack();
    if (has_bias) bv = bias.unpack();
    if (at::GradMode::is_enabled()) return norm_gradients_in_operations(*call, dy, xv, wv, bv);  // create_graph
    NormCall c = *call;
    if (xv.strides() != at::IntArrayRef(x_strides)) {  // tensors saved by a hook may come back with others
      xv = xv.contiguous();
      c.desc.inner = 1;
      c.desc.inner_stride = c.desc.outer_stride = c.desc.channels;
    }
    const auto g = norm_gradients(c, dy.to(scalar_type(c.desc.y_dtype)).contiguous(), xv, wv, bv, statistics.unpack(),
                                  task_should_compute_output(0), has_weight && task_should_compute_output(1),
                                  has_bias && task_should_compute_output(2));
    return {g.dx, g.dweight, g.dbias};
  }
};

Tensor layer_norm(const std::shared_ptr<NormCall>& call, const Tensor& x, const std::optional<Tensor>& weight,
                  const std::optional<Tensor>& bias) {
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  bool grad = x.requires_grad(), tangent = x._fw_grad(0).defined();
  for (const Tensor& t : {w, b})
    if (t.defined()) {
      grad = grad || t.requires_grad();
      tangent = tangent || t._fw_grad(0).defined();
    }
  TORCH_CHECK_NOT_IMPLEMENTED(!tangent, "layer_norm has no forward-mode derivative");
  grad = grad && at::GradMode::is_enabled();
  Tensor y, statistics;
  {
    const at::AutoGradMode off(false);
    const c10::DeviceGuard guard(x.device());
    y = new_output(*call, x);
    if (grad) statistics = new_statistics(*call, x);
    norm_forward(*call, x, y, w, b, statistics);
  }
  if (!grad) return y;
  std::shared_ptr<LayerNormBackward> node(new LayerNormBackward(), torch::autograd::deleteNode);
  node->set_next_edges({torch::autograd::impl::gradient_edge(x),
                        w.defined() ? torch::autograd::impl::gradient_edge(w) : torch::autograd::Edge(),
                        b.defined() ? torch::autograd::impl::gradient_edge(b) : torch::autograd::Edge()});
  node->call = call;
  node->x = SavedVariable(x, false);
  node->x_strides = x.strides().vec();
  node->has_weight = w.defined();
  node->has_bias = b.defined();
  if (w.defined()) node->weight = SavedVariable(w, false);
  if (b.defined()) node->bias = SavedVariable(b, false);
  node->statistics = SavedVariable(statistics, false);
  torch::autograd::set_history(y, node);
  return y;
}

// Without autograd: y, or with `keep` (y, statistics).
pybind11::object layer_norm_forward(const std::shared_ptr<NormCall>& call, const Tensor& x, const std::optional<Tensor>& weight,
                                    const std::optional<Tensor>& bias, bool keep, const std::optional<Tensor>& out) {
  Tensor y, statistics;
  {
    const pybind11::gil_scoped_release no_gil;
    const at::AutoGradMode off(false);
    const c10::DeviceGuard guard(x.device());
    if (out.has_value()) {
      TORCH_CHECK_VALUE(out->sizes() == x.sizes() && out->scalar_type() == scalar_type(call->desc.y_dtype) &&
                            out->is_contiguous() && out->device() == x.device(),
                        "out must be a contiguous ", scalar_type(call->desc.y_dtype), " tensor of shape ", x.sizes(), " on ", x.device());
      y = *out;
      changed(y);
    } else {
      y = new_output(*call, x);
    }
    if (keep) statistics = new_statistics(*call, x);
    norm_forward(*call, x, y, weight.value_or(Tensor()), bias.value_or(Tensor()), statistics);
  }
  if (!keep) return pybind11::cast(y);
  return pybind11::make_tuple(y, statistics);
}

pybind11::tuple layer_norm_backward(const std::shared_ptr<NormCall>& call, const Tensor& dy, const Tensor& x,
                                    const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                                    const Tensor& statistics, bool need_x, bool need_w, bool need_b) {
  NormGradients g;
  {
    const pybind11::gil_scoped_release no_gil;
    const at::AutoGradMode off(false);
    TORCH_CHECK_VALUE(dy.device() == x.device() && statistics.device() == x.device(), "tensors on different devices: ",
                      x.device(), ", ", dy.device(), " and ", statistics.device());
    TORCH_CHECK_VALUE(dy.sizes() == x.sizes() && dy.scalar_type() == scalar_type(call->desc.y_dtype) && dy.is_contiguous(),
                      "dy must be a contiguous ", scalar_type(call->desc.y_dtype), " tensor of shape ", x.sizes());
    TORCH_CHECK_VALUE(statistics.scalar_type() == at::kFloat && statistics.is_contiguous() && statistics.dim() == 2 &&
                          statistics.size(0) == call->desc.rows && statistics.size(1) == 2,
                      "statistics must be those of the forward: a contiguous float32 [", call->desc.rows, ", 2] tensor");
    g = norm_gradients(*call, dy, x, weight.value_or(Tensor()), bias.value_or(Tensor()), statistics, need_x,
                       need_w && weight.has_value(), need_b && bias.has_value());
  }
  auto maybe = [](const Tensor& t) -> pybind11::object { return t.defined() ? pybind11::cast(t) : pybind11::none(); };
  return pybind11::make_tuple(maybe(g.dx), maybe(g.dweight), maybe(g.dbias));
}

// ---- rotary positions ------------------------------------------------------------

struct RotaryCall {
  terra_swin_rotary_desc desc;  // with y packed, and x's strides for y's in place
};

std::shared_ptr<RotaryCall> make_rotary_call(const std::string& desc) {
  auto c = std::make_shared<RotaryCall>();
  fill(&c->desc, desc);
  return c;
}

Tensor rotary(const std::shared_ptr<RotaryCall>& call, const Tensor& x, const Tensor& positions, const Tensor& turns,
              const std::optional<Tensor>& out) {
  const at::AutoGradMode off(false);
  const c10::DeviceGuard guard(x.device());
  Tensor y;
  if (out.has_value()) {
    y = *out;  // checked with the options
    changed(y);
  } else {
    y = at::empty(x.sizes(), x.options());
  }
  if (call->desc.tokens > 0)
    check(rotary_entry(x.const_data_ptr(), y.data_ptr(), positions.const_data_ptr(),
                       static_cast<const double*>(turns.const_data_ptr()), &call->desc, current_stream(x)), "terra_swin_rotary");
  return y;
}

// The gradient's call: the turn back, from a packed gradient into a packed one.
std::shared_ptr<RotaryCall> backward_call(const RotaryCall& c) {
  auto b = std::make_shared<RotaryCall>(c);
  auto& d = b->desc;
  d.inverse = !d.inverse;
  d.x_head_stride = d.y_head_stride = d.head_dim;
  d.x_inner_stride = d.y_inner_stride = static_cast<int64_t>(d.heads) * d.head_dim;
  d.x_outer_stride = d.y_outer_stride = d.inner * d.x_inner_stride;
  return b;
}

Tensor rotary_with_gradient(const std::shared_ptr<RotaryCall>& call, const Tensor& x, const Tensor& positions, const Tensor& turns);

// A linear map: its gradient is turned back, and may be differentiated again.
struct RotaryBackward : public torch::autograd::Node {
  std::shared_ptr<RotaryCall> call;  // of the gradient
  SavedVariable positions, turns;

  std::string name() const override { return "RotaryBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    positions.reset_data();
    turns.reset_data();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(1);
    return {rotary_with_gradient(call, grads[0].contiguous(), positions.unpack(), turns.unpack())};
  }
};

Tensor rotary_with_gradient(const std::shared_ptr<RotaryCall>& call, const Tensor& x, const Tensor& positions, const Tensor& turns) {
  Tensor y = rotary(call, x, positions, turns, std::nullopt);
  if (!x.requires_grad() || !at::GradMode::is_enabled()) return y;
  std::shared_ptr<RotaryBackward> node(new RotaryBackward(), torch::autograd::deleteNode);
  node->set_next_edges({torch::autograd::impl::gradient_edge(x)});
  node->call = backward_call(*call);
  node->positions = SavedVariable(positions, false);
  node->turns = SavedVariable(turns, false);
  torch::autograd::set_history(y, node);
  return y;
}

// ---- lists of tensors --------------------------------------------------------------

void check_member(const Tensor& t, const char* what, size_t i, const c10::Device& device) {
  TORCH_CHECK(t.device().is_cuda(), "terra_amd kernels run on ROCm devices only (", what, " ", i, " is on '", t.device(),
              "'); there is no CPU fallback");
  TORCH_CHECK_VALUE(t.device() == device, "tensors on different devices: ", device, " and ", t.device(), " (", what, " ", i, ")");
  TORCH_CHECK_TYPE(t.layout() == at::kStrided, what, " ", i, " is not dense (", t.layout(), ")");
  TORCH_CHECK_TYPE(dtype_code(t.scalar_type()) >= 0, "dtype ", t.scalar_type(), " of ", what, " ", i,
                   " not supported here (supported: float32, bfloat16, float16)");
}

// The norm, the clip factor and whether the norm is infinite or NaN, as one fp32 tensor of three.
Tensor gradient_norm(const std::vector<Tensor>& grads, double max_norm) {
  TORCH_CHECK_VALUE(!grads.empty(), "gradient_norm needs one gradient at least");
  const pybind11::gil_scoped_release no_gil;
  const at::AutoGradMode off(false);
  const c10::Device device = grads[0].device();
  std::vector<terra_swin_tensor> list;
  std::vector<Tensor> copies;  // of what does not lie side by side
  list.reserve(grads.size());
  for (size_t i = 0; i < grads.size(); ++i) {
    check_member(grads[i], "gradient", i, device);
    Tensor g = grads[i];
    if (!g.is_contiguous() && !g.is_non_overlapping_and_dense()) copies.push_back(g = g.contiguous());
    list.push_back({g.const_data_ptr(), g.numel(), dtype_code(g.scalar_type())});
  }
  const c10::DeviceGuard guard(device);
  const int count = static_cast<int>(list.size()), n = gradient_norm_workspace_entry(list.data(), count);
  check(n < 0 ? n : TERRA_OK, "terra_swin_gradient_norm_workspace");
  const auto options = grads[0].options();
  Tensor work = at::empty({n}, options.dtype(at::kDouble)), result = at::empty({3}, options.dtype(at::kFloat));
  check(gradient_norm_entry(list.data(), count, max_norm, static_cast<float*>(result.data_ptr()),
                            static_cast<double*>(work.data_ptr()), current_stream(result)), "terra_swin_gradient_norm");
  return result;
}

// The address of an option that may be a number in device memory.
const void* scalar_ptr(const std::optional<Tensor>& t, at::ScalarType type, const c10::Device& device, const char* name) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK_VALUE(t->scalar_type() == type && t->numel() == 1 && t->device() == device, name, " must be one ", type,
                    " value on ", device, " (got ", t->scalar_type(), ", ", t->numel(), " values on ", t->device(), ")");
  return t->const_data_ptr();
}

struct AdamOptions {
  double lr, beta1, beta2, eps, weight_decay;
  int64_t step;
  std::optional<Tensor> step_tensor, lr_tensor, grad_factor, found_inf, seed;
  uint32_t stream;
  bool maximize;
};

// places: the tensors' numbers in the random numbers' counter, as many as there are tensors, or none: their places in the list.
void adamw_step(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& firsts,
                const std::vector<Tensor>& seconds, const std::vector<std::optional<Tensor>>& scales,
                const std::vector<uint32_t>& places, const AdamOptions& o) {
  const pybind11::gil_scoped_release no_gil;
  const at::AutoGradMode off(false);
  if (params.empty()) return;
  const size_t n = params.size();
  TORCH_CHECK_VALUE(grads.size() == n && firsts.size() == n, "as many gradients and moments as parameters (got ", n, ", ",
                    grads.size(), " and ", firsts.size(), ")");
  TORCH_CHECK_VALUE(places.empty() || places.size() == n, "as many places as parameters (got ", n, " and ", places.size(), ")");
  const c10::Device device = params[0].device();
  std::vector<terra_swin_adamw_tensor> list;
  list.reserve(n);
  std::vector<Tensor> copies;  // of gradients of other strides
  bool scaled_any = false;
  for (size_t i = 0; i < n; ++i) {
    const Tensor &p = params[i], &m = firsts[i], &v = seconds[i];
    Tensor g = grads[i];
    check_member(p, "parameter", i, device);
    check_member(g, "gradient", i, device);
    TORCH_CHECK_VALUE(g.sizes() == p.sizes(), "gradient ", i, " of shape ", g.sizes(), " for a parameter of ", p.sizes());
    TORCH_CHECK_VALUE(p.is_contiguous() || p.is_non_overlapping_and_dense(), "parameter ", i,
                      " does not lie side by side in memory (strides ", p.strides(), ")");
    if (g.strides() != p.strides()) {
      Tensor same = at::empty_strided(p.sizes(), p.strides(), g.options());
      copies.push_back(g = same.copy_(g));
    }
    const bool scaled = scales[i].has_value();
    scaled_any = scaled_any || scaled;
    const at::ScalarType held = scaled ? at::kFloat8_e4m3fn : at::kFloat;
    for (const Tensor* t : {&m, &v})
      TORCH_CHECK_VALUE(t->device() == device && t->scalar_type() == held && t->sizes() == p.sizes() && t->strides() == p.strides(),
                        "the moments of parameter ", i, " must be ", held, " tensors of its shape and strides on ", device);
    if (scaled) {
      const Tensor& s = *scales[i];
      TORCH_CHECK_VALUE(s.device() == device && s.scalar_type() == at::kFloat && s.is_contiguous() && s.dim() == 2 &&
                            s.size(0) == 2 && s.size(1) == (p.numel() + 255) / 256,
                        "the scales of parameter ", i, " must be a contiguous float32 [2, ", (p.numel() + 255) / 256, "] tensor on ", device);
    }
    list.push_back({const_cast<void*>(p.const_data_ptr()), g.const_data_ptr(), const_cast<void*>(m.const_data_ptr()),
                    const_cast<void*>(v.const_data_ptr()),
                    scaled ? static_cast<float*>(const_cast<void*>(scales[i]->const_data_ptr())) : nullptr, p.numel(),
                    places.empty() ? static_cast<uint32_t>(i) : places[i], dtype_code(p.scalar_type()), dtype_code(g.scalar_type())});
  }
  TORCH_CHECK_VALUE(!scaled_any || o.seed.has_value(), "moments in 8 bits need a seed (see dropout_seed)");
  const c10::DeviceGuard guard(device);
  terra_swin_adamw_desc d = {};
  d.lr = o.lr, d.beta1 = o.beta1, d.beta2 = o.beta2, d.eps = o.eps, d.weight_decay = o.weight_decay;
  d.step = o.step;
  d.step_ptr = scalar_ptr(o.step_tensor, at::kLong, device, "step");
  d.lr_ptr = static_cast<const float*>(scalar_ptr(o.lr_tensor, at::kFloat, device, "lr"));
  d.grad_factor = static_cast<const float*>(scalar_ptr(o.grad_factor, at::kFloat, device, "grad_factor"));
  d.found_inf = static_cast<const float*>(scalar_ptr(o.found_inf, at::kFloat, device, "found_inf"));
  d.seed = scalar_ptr(o.seed, at::kLong, device, "seed");
  d.stream_id = o.stream;
  d.maximize = o.maximize;
  check(adamw_entry(list.data(), static_cast<int>(n), &d, current_stream(params[0])), "terra_swin_adamw");
  for (size_t i = 0; i < n; ++i) {
    changed(params[i]);
    changed(firsts[i]);
    changed(seconds[i]);
    if (scales[i].has_value()) changed(*scales[i]);
  }
}

template <typename F>
void entry(F& f, uintptr_t address) {
  f = reinterpret_cast<F>(address);
}

void bind(uintptr_t norm, uintptr_t norm_backward, uintptr_t rotate, uintptr_t gradient_norm_workspace,
          uintptr_t gradient_norm, uintptr_t adamw, uintptr_t error) {
  entry(norm_entry, norm);
  entry(norm_backward_entry, norm_backward);
  entry(rotary_entry, rotate);
  entry(gradient_norm_workspace_entry, gradient_norm_workspace);
  entry(gradient_norm_entry, gradient_norm);
  entry(adamw_entry, adamw);
  entry(last_error, error);
}

}  // namespace

PYBIND11_MODULE(_training, m) {
  pybind11::class_<NormCall, std::shared_ptr<NormCall>>(m, "NormCall").def(pybind11::init(&make_norm_call));
  pybind11::class_<RotaryCall, std::shared_ptr<RotaryCall>>(m, "RotaryCall").def(pybind11::init(&make_rotary_call));
  m.def("bind", &bind);
  m.def("layer_norm_forward", &layer_norm_forward);
  m.def("layer_norm_backward", &layer_norm_backward);
  const auto no_gil = pybind11::call_guard<pybind11::gil_scoped_release>();  // a launch may wait for room in the queue
  m.def("rotary", &rotary, no_gil);
  // What saves tensors may call hooks in Python: their exceptions pass as they are.
  m.def("layer_norm", torch::wrap_pybind_function_no_gil(&layer_norm));
  m.def("rotary_with_gradient", torch::wrap_pybind_function_no_gil(&rotary_with_gradient));
  m.def("gradient_norm", &gradient_norm);
  m.def("adamw_step", [](const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& firsts,
                         const std::vector<Tensor>& seconds, const std::vector<std::optional<Tensor>>& scales,
                         const std::vector<uint32_t>& places, double lr,
                         double beta1, double beta2, double eps, double weight_decay, int64_t step,
                         const std::optional<Tensor>& step_tensor, const std::optional<Tensor>& lr_tensor,
                         const std::optional<Tensor>& grad_factor, const std::optional<Tensor>& found_inf,
                         const std::optional<Tensor>& seed, uint32_t stream, bool maximize) {
    adamw_step(params, grads, firsts, seconds, scales, places,
               {lr, beta1, beta2, eps, weight_decay, step, step_tensor, lr_tensor, grad_factor, found_inf, seed, stream, maximize});
  });
}

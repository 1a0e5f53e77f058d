// The host side of the regularised operators, as a Python module beside the
// library: what a call of dropout and of GELU with dropout does once its
// arguments are checked, and the autograd node of the end of a half-block.
// Calls of small inputs are bound by the host: a dropout of 3136 x 96 took 7.9 us
// from Python, 4.3 so (x * 2: 4.7); and the backward of a node written in Python runs in the
// autograd engine's thread, which has to wait for the interpreter: a training
// step of 3136 x 96 fp32 took 76 us with the engine in the caller's thread and up
// to 160 with its own, 50 and 101 with this one (x * 2 and its gradient: 18 and
// 41).  Allocations are torch's; the arithmetic is the library's, reached by the
// addresses that bind() is given.
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
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

decltype(&terra_swin_residual_norm) forward_entry = nullptr;
decltype(&terra_swin_residual_norm_bwd) backward_entry = nullptr;
decltype(&terra_swin_dropout) dropout_entry = nullptr;
decltype(&terra_swin_gelu_dropout) gelu_entry = nullptr;
decltype(&terra_swin_gelu_dropout_bwd) gelu_backward_entry = nullptr;
decltype(&terra_last_error) last_error = nullptr;

void check(int status, const char* what) {
  TORCH_CHECK(status != TERRA_ERR_LAUNCH, what, ": ", last_error());
  TORCH_CHECK_VALUE(status == TERRA_OK, what, ": ", last_error());
}

// The parameters of a call, in the order of the entry points.
enum Param { kPostWeight, kPostBias, kGate, kNextWeight, kNextBias, kParams };

const float* f32(const Tensor& t) { return t.defined() ? static_cast<const float*>(t.const_data_ptr()) : nullptr; }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

// What the checked arguments of a call say about it, but the tensors.
struct Call {
  terra_swin_residual_norm_desc desc;
  bool covered;       // the backward writes all of dh
  int64_t workspace;  // of the backward, fp32 values
};

std::shared_ptr<Call> make_call(const std::string& desc, bool covered, int64_t workspace) {
  auto c = std::make_shared<Call>();
  TORCH_CHECK(desc.size() == sizeof(c->desc), "descriptor of ", desc.size(), " bytes, expected ", sizeof(c->desc));
  std::memcpy(&c->desc, desc.data(), sizeof(c->desc));
  c->covered = covered;
  c->workspace = workspace;
  return c;
}

// The current stream of the tensor's device.
void* current_stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

Tensor packed_like(const Tensor& t) { return t.is_contiguous() ? at::empty_like(t) : at::empty(t.sizes(), t.options()); }

Tensor packed_f32(const Tensor& t) {
  if (!t.defined() || (t.scalar_type() == at::kFloat && t.is_contiguous())) return t;
  return t.to(at::kFloat).contiguous();
}

// ---- dropout, GELU with dropout -----------------------------------------------

// What the checked arguments of a call say about it, but the tensors.
struct Rows {
  int dtype;
  int64_t rows, columns, stride;
  double p;
  uint32_t stream;
  int64_t workspace;  // of the backward's column sums, fp32 values
};

std::shared_ptr<Rows> make_rows(int dtype, int64_t rows, int64_t columns, int64_t stride, double p, uint32_t stream,
                                int64_t workspace) {
  return std::make_shared<Rows>(Rows{dtype, rows, columns, stride, p, stream, workspace});
}

const void* seed_ptr(const std::optional<Tensor>& seed, const Tensor& x, double p) {
  if (!seed.has_value()) {
    TORCH_CHECK_VALUE(p == 0.0, "dropout with p > 0 needs a seed (see dropout_seed)");
    return nullptr;
  }
  TORCH_CHECK_VALUE(seed->scalar_type() == at::kLong && seed->numel() == 1 && seed->device() == x.device(),
                    "seed must be one int64 value on ", x.device());
  return seed->const_data_ptr();
}

// `out`, checked and counted as written (a graph that saved its values refuses
// them then), or a new packed tensor like `like`.
Tensor output(const std::optional<Tensor>& out, const Tensor& like) {
  if (!out.has_value()) return packed_like(like);
  TORCH_CHECK_VALUE(out->sizes() == like.sizes() && out->scalar_type() == like.scalar_type() && out->is_contiguous() &&
                        out->device() == like.device(),
                    "out must be a contiguous ", like.scalar_type(), " tensor of shape ", like.sizes(), " on ", like.device());
  if (!out->is_inference()) torch::autograd::impl::bump_version(*out);  // an inference tensor is in no graph
  return *out;
}

Tensor dropout(const std::shared_ptr<Rows>& c, const Tensor& x, const std::optional<Tensor>& seed,
               const std::optional<Tensor>& out) {
  const pybind11::gil_scoped_release no_gil;  // a launch may wait for room in the queue
  const at::AutoGradMode off(false);
  const void* s = seed_ptr(seed, x, c->p);
  const c10::DeviceGuard guard(x.device());
  Tensor y = output(out, x);
  if (c->rows > 0)
    check(dropout_entry(x.const_data_ptr(), y.data_ptr(), c->dtype, c->rows, c->columns, c->stride, c->p, s, c->stream,
                        current_stream(x)), "terra_swin_dropout");
  return y;
}

Tensor gelu_dropout(const std::shared_ptr<Rows>& c, const Tensor& h, const std::optional<Tensor>& seed,
                    const std::optional<Tensor>& out) {
  const pybind11::gil_scoped_release no_gil;
  const at::AutoGradMode off(false);
  const void* s = seed_ptr(seed, h, c->p);
  const c10::DeviceGuard guard(h.device());
  Tensor a = output(out, h);
  if (c->rows > 0)
    check(gelu_entry(h.const_data_ptr(), a.data_ptr(), c->dtype, c->rows, c->columns, c->p, s, c->stream, current_stream(h)),
          "terra_swin_gelu_dropout");
  return a;
}

// dh, or with `column_sums` (dh, its sums over the rows).
pybind11::object gelu_dropout_backward(const std::shared_ptr<Rows>& c, const Tensor& dout, const Tensor& h,
                                       const std::optional<Tensor>& seed, bool column_sums, const std::optional<Tensor>& out) {
  Tensor dh, sums, work;
  {
    const pybind11::gil_scoped_release no_gil;
    const at::AutoGradMode off(false);
    TORCH_CHECK_VALUE(dout.device() == h.device(), "tensors on different devices: ", h.device(), " and ", dout.device());
    TORCH_CHECK_VALUE(dout.sizes() == h.sizes() && dout.scalar_type() == h.scalar_type() && dout.is_contiguous(),
                      "dout must be a contiguous ", h.scalar_type(), " tensor of shape ", h.sizes(), " like h");
    const void* s = seed_ptr(seed, h, c->p);
    const c10::DeviceGuard guard(h.device());
    dh = output(out, h);
    if (column_sums) {
      const auto f32_there = h.options().dtype(at::kFloat);
      sums = c->rows > 0 ? at::empty({c->columns}, f32_there) : at::zeros({c->columns}, f32_there);
      work = at::empty({c->workspace}, f32_there);
    }
    if (c->rows > 0)
      check(gelu_backward_entry(dout.const_data_ptr(), h.const_data_ptr(), dh.data_ptr(), c->dtype, c->rows, c->columns, c->p,
                                s, c->stream, column_sums ? static_cast<float*>(sums.data_ptr()) : nullptr,
                                column_sums ? static_cast<float*>(work.data_ptr()) : nullptr, current_stream(h)),
            "terra_swin_gelu_dropout_bwd");
  }
  if (!column_sums) return pybind11::cast(dh);
  return pybind11::make_tuple(dh, sums);
}

// ---- the end of a half-block ---------------------------------------------------

constexpr const char* kOnce = "residual_norm cannot be differentiated twice: its gradient has no gradient";

struct ResidualNormBackward : public torch::autograd::Node {
  std::shared_ptr<Call> call;
  SavedVariable h, x, seed, params[kParams];
  std::vector<int64_t> h_strides, x_strides;
  bool seeded = false, has[kParams] = {};
  PyObject* link = nullptr;  // a ResidualLink that takes x's gradient, or null

  ~ResidualNormBackward() override {
    if (link != nullptr && Py_IsInitialized()) {
      pybind11::gil_scoped_acquire gil;
      Py_DECREF(link);
    }
  }

  std::string name() const override { return "ResidualNormBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    h.reset_data();
    x.reset_data();
    seed.reset_data();
    for (auto& p : params) p.reset_data();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const Tensor dy = grads[0], dz = grads.size() > 1 ? grads[1] : Tensor();
    variable_list out;
    {
      at::AutoGradMode off(false);
      out = gradients(dy, dz);
    }
    if (!at::GradMode::is_enabled()) return out;
    // Asked for with create_graph: gradients that refuse to be differentiated, tied
    // to all they depend on, since a pass to one of those would leave them out otherwise.
    torch::autograd::edge_list sources = next_edges();
    for (const Tensor& t : {dy, dz})
      if (t.defined()) sources.push_back(torch::autograd::impl::gradient_edge(t));
    const std::shared_ptr<torch::autograd::Node> refuse(new torch::autograd::Error(kOnce, std::move(sources)),
                                                        torch::autograd::deleteNode);
    for (auto& t : out)
      if (t.defined()) torch::autograd::set_history(t, refuse);
    return out;
  }

  variable_list gradients(Tensor dy, Tensor dz) {
    Tensor hv = h.unpack(), xv = x.unpack(), ps[kParams], own[kParams];
    for (int i = 0; i < kParams; ++i)
      if (has[i]) {
        own[i] = params[i].unpack();
        ps[i] = packed_f32(own[i]);
      }
    const Tensor sv = seeded ? seed.unpack() : Tensor();
    terra_swin_residual_norm_desc d = call->desc;
    if (hv.strides() != at::IntArrayRef(h_strides)) {  // tensors saved by a hook may come back with others
      hv = hv.contiguous();
      d.h_stride = d.channels;
    }
    if (xv.strides() != at::IntArrayRef(x_strides)) {
      xv = xv.contiguous();
      d.x_stride = d.channels;
    }
    if (dy.defined()) dy = dy.contiguous();
    if (dz.defined()) dz = dz.contiguous();
    const c10::DeviceGuard guard(hv.device());
    Tensor dh = call->covered ? packed_like(hv) : at::zeros(hv.sizes(), hv.options());
    Tensor dx = packed_like(xv), dps[kParams], work;
    float* dp[kParams] = {};
    for (int i = 0, edge = 2; i < kParams; ++i) {
      if (!has[i]) continue;
      if (task_should_compute_output(edge++)) {
        dps[i] = at::empty_like(ps[i]);
        dp[i] = static_cast<float*>(dps[i].data_ptr());
        if (!work.defined()) work = at::empty({call->workspace}, ps[i].options());
      }
    }
    check(backward_entry(hv.const_data_ptr(), xv.const_data_ptr(), ptr(dy), ptr(dz), dh.data_ptr(), dx.data_ptr(), &d,
                         f32(ps[kPostWeight]), f32(ps[kPostBias]), f32(ps[kGate]), f32(ps[kNextWeight]), ptr(sv),
                         dp[kPostWeight], dp[kPostBias], dp[kGate], dp[kNextWeight], dp[kNextBias],
                         work.defined() ? static_cast<float*>(work.data_ptr()) : nullptr, current_stream(hv)),
          "terra_swin_residual_norm_bwd");
    if (link != nullptr) {
      pybind11::gil_scoped_acquire gil;
      pybind11::handle(link).attr("grad") = dx;
      dx = Tensor();
    }
    variable_list out = {dh, dx};
    for (int i = 0; i < kParams; ++i)
      if (has[i]) out.push_back(dps[i].defined() ? dps[i].to(own[i].scalar_type()) : Tensor());
    return out;
  }
};

// y, or with a next norm (y, z); `link` None or the ResidualLink of x.
pybind11::object residual_norm(const std::shared_ptr<Call>& call, const Tensor& h, const Tensor& x,
                               const std::optional<Tensor>& post_weight, const std::optional<Tensor>& post_bias,
                               const std::optional<Tensor>& gate, const std::optional<Tensor>& next_weight,
                               const std::optional<Tensor>& next_bias, const std::optional<Tensor>& seed,
                               const pybind11::object& link) {
  const std::optional<Tensor>* given[kParams] = {&post_weight, &post_bias, &gate, &next_weight, &next_bias};
  Tensor ps[kParams], y, z;
  {
    const pybind11::gil_scoped_release no_gil;
    const at::AutoGradMode off(false);
    const c10::DeviceGuard guard(h.device());
    for (int i = 0; i < kParams; ++i)
      if (given[i]->has_value()) ps[i] = packed_f32(**given[i]);
    y = packed_like(x);
    if (call->desc.next_norm != TERRA_NORM_NONE) z = at::empty(x.sizes(), h.options());
    if (call->desc.rows > 0)
      check(forward_entry(h.const_data_ptr(), x.const_data_ptr(), y.data_ptr(), z.defined() ? z.data_ptr() : nullptr,
                          &call->desc, f32(ps[kPostWeight]), f32(ps[kPostBias]), f32(ps[kGate]), f32(ps[kNextWeight]),
                          f32(ps[kNextBias]), seed.has_value() ? seed->const_data_ptr() : nullptr, current_stream(h)),
            "terra_swin_residual_norm");
  }
  bool grad = h.requires_grad() || x.requires_grad(), tangent = h._fw_grad(0).defined() || x._fw_grad(0).defined();
  for (const auto* p : given)
    if (p->has_value()) {
      grad = grad || (*p)->requires_grad();
      tangent = tangent || (*p)->_fw_grad(0).defined();
    }
  TORCH_CHECK_NOT_IMPLEMENTED(!tangent, "residual_norm has no forward-mode derivative");
  if (grad && at::GradMode::is_enabled()) {
    std::shared_ptr<ResidualNormBackward> node(new ResidualNormBackward(), torch::autograd::deleteNode);
    torch::autograd::edge_list edges = {torch::autograd::impl::gradient_edge(h), torch::autograd::impl::gradient_edge(x)};
    for (int i = 0; i < kParams; ++i)
      if (given[i]->has_value()) {
        edges.push_back(torch::autograd::impl::gradient_edge(**given[i]));
        node->has[i] = true;
        node->params[i] = SavedVariable(**given[i], false);
      }
    node->set_next_edges(std::move(edges));
    node->call = call;
    node->h = SavedVariable(h, false);
    node->x = SavedVariable(x, false);
    node->h_strides = h.strides().vec();
    node->x_strides = x.strides().vec();
    if (seed.has_value()) {
      node->seeded = true;
      node->seed = SavedVariable(*seed, false);
    }
    if (!link.is_none()) node->link = pybind11::object(link).release().ptr();
    torch::autograd::set_history(y, node);
    if (z.defined()) torch::autograd::set_history(z, node);
  }
  if (!z.defined()) return pybind11::cast(y);
  return pybind11::make_tuple(y, z);
}

template <typename F>
void entry(F& f, uintptr_t address) {
  f = reinterpret_cast<F>(address);
}

void bind(uintptr_t forward, uintptr_t backward, uintptr_t drop, uintptr_t gelu, uintptr_t gelu_backward, uintptr_t error) {
  entry(forward_entry, forward);
  entry(backward_entry, backward);
  entry(dropout_entry, drop);
  entry(gelu_entry, gelu);
  entry(gelu_backward_entry, gelu_backward);
  entry(last_error, error);
}

}  // namespace

PYBIND11_MODULE(_regularize, m) {
  pybind11::class_<Call, std::shared_ptr<Call>>(m, "Call").def(pybind11::init(&make_call));
  pybind11::class_<Rows, std::shared_ptr<Rows>>(m, "Rows").def(pybind11::init(&make_rows));
  m.def("bind", &bind);
  m.def("dropout", &dropout);
  m.def("gelu_dropout", &gelu_dropout);
  m.def("gelu_dropout_backward", &gelu_dropout_backward);
  m.def("residual_norm", &residual_norm);
}

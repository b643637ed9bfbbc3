// Torch side of the layers with dropout and gradients (ops.dropout, ops.linear_act, ops.groupnorm_act): argument checks,
// allocation and autograd nodes around the C ABI of libsdmi.  Native, because such a layer's kernels are often shorter than
// the Python that launches them: torch runs backward passes in a thread of its own, where an autograd.Function's Python
// starts on cold caches and takes the interpreter lock back and forth (dropout of 9217x333 with a residual, forward and
// backward, 12 us of kernels: 88 us a pass through Python, 50 through here, of which torch's own engine is most; a forward
// call of groupnorm_act on 2x8x8x1280, 5.7 us: 14.2 and 9.0).  The library is bound at run time by address, so that both
// sides of the package use one copy of it.  A call's kernels are launched without the interpreter lock.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/sdmi.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> OptTensor;

// ---- the library -----------------------------------------------------------------------------------
struct Api {
  decltype(&sdmi_last_error) last_error = nullptr;
  decltype(&sdmi_dropout) dropout = nullptr;
  decltype(&sdmi_linear_act_workspace_bytes) linear_ws = nullptr;
  decltype(&sdmi_linear_act) linear = nullptr;
  decltype(&sdmi_linear_act_backward_workspace_bytes) linear_bwd_ws = nullptr;
  decltype(&sdmi_linear_act_backward) linear_bwd = nullptr;
  decltype(&sdmi_groupnorm_act_workspace_bytes) groupnorm_ws = nullptr;
  decltype(&sdmi_groupnorm_act) groupnorm = nullptr;
  decltype(&sdmi_groupnorm_act_backward) groupnorm_bwd = nullptr;
} api;

void bind(const py::dict& addresses) {
  Api a;
  auto take = [&](const char* name, auto& fn) {
    fn = reinterpret_cast<std::decay_t<decltype(fn)>>(addresses[name].cast<uintptr_t>());
  };
  take("sdmi_last_error", a.last_error);
  take("sdmi_dropout", a.dropout);
  take("sdmi_linear_act_workspace_bytes", a.linear_ws);
  take("sdmi_linear_act", a.linear);
  take("sdmi_linear_act_backward_workspace_bytes", a.linear_bwd_ws);
  take("sdmi_linear_act_backward", a.linear_bwd);
  take("sdmi_groupnorm_act_workspace_bytes", a.groupnorm_ws);
  take("sdmi_groupnorm_act", a.groupnorm);
  take("sdmi_groupnorm_act_backward", a.groupnorm_bwd);
  api = a;
}

void done(int code, const char* name) {
  if (code != 0)
    throw std::runtime_error(std::string("libsdmi ") + name + " failed (" + std::to_string(code) + "): " + api.last_error());
}
// the tensors' device for the length of a call, and its current stream
struct Here {
  c10::DeviceGuard guard;
  void* stream;
  explicit Here(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.get_device()).stream()) {}
};

// ---- checks ------------------------------------------------------------------------------------------
std::string dtype_name(at::ScalarType t) { return c10::getDtypeNames(t).first; }

int dtype_code(const Tensor& x) {
  TORCH_CHECK_VALUE(x.is_cuda(), "x is on ", x.device(), ": there is no CPU path");
  switch (x.scalar_type()) {
    case at::kFloat: return SDMI_DTYPE_F32;
    case at::kHalf: return SDMI_DTYPE_F16;
    case at::kBFloat16: return SDMI_DTYPE_BF16;
    default: TORCH_CHECK_VALUE(false, "x is ", dtype_name(x.scalar_type()), ", expected float32, float16 or bfloat16");
  }
  return -1;
}
void check_like(const char* what, const Tensor& t, const Tensor& x, at::ScalarType dtype) {
  TORCH_CHECK_VALUE(t.device() == x.device(), what, " is on ", t.device(), ", expected ", x.device());
  TORCH_CHECK_VALUE(t.scalar_type() == dtype, what, " is ", dtype_name(t.scalar_type()), ", expected ", dtype_name(dtype));
}
// What records torch's operators (torch.jit.trace, make_fx, export) would record the allocation of a result and not the launch
// that fills it, and give back whatever is in that memory when it runs.
void check_not_traced() {
  using c10::impl::TorchDispatchModeTLS;
  const bool traced = torch::jit::tracer::isTracing() ||
                      TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value() ||
                      c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
  TORCH_CHECK_NOT_IMPLEMENTED(!traced, "the layers with dropout cannot be traced: their launches are no operators of torch");
}
// A wrapper subclass (DTensor, a fake tensor) has no memory of its own: its address is null, and an optional one would count as
// missing.
void check_memory(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t.unsafeGetTensorImpl()->is_python_dispatch(),
                              "the layers with dropout need tensors each with memory of its own, no subclasses that hand their operators to Python");
}
void check_memory(const OptTensor& t) { if (t) check_memory(*t); }
// forward-mode tangents would be lost without a word
template <typename... T> void check_no_tangent(const T&... t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(torch::autograd::isFwGradDefined(t) || ...),
                              "the layers with dropout have no forward-mode derivatives");
}
void check_shape(const char* what, const Tensor& t, at::IntArrayRef shape) {
  TORCH_CHECK_VALUE(t.sizes() == shape, what, " has shape ", t.sizes(), ", expected ", shape);
}
void check_columns(int64_t n) {
  TORCH_CHECK_VALUE(n <= (int64_t)1 << 30, "rows of ", n, " columns are too long: at most 2^30");
}

// a tensor whose memory holds its values: not a view that torch negates lazily (the imaginary part of a conjugate), nor zeros
// that it keeps without memory
Tensor in_memory(const Tensor& t) {
  if (C10_UNLIKELY(t.is_neg())) return t.resolve_neg();
  if (C10_UNLIKELY(t._is_zerotensor())) return t.clone();
  return t;
}

struct Drop {
  double p = 0.0;
  int64_t seed = 0, offset = 0;
  Tensor seed_t;                  // defined: the seed is read there when the kernel runs
};
const int64_t* address(const Tensor& seed_t) { return seed_t.defined() ? seed_t.const_data_ptr<int64_t>() : nullptr; }

Drop drop_state(double p, py::handle seed, int64_t offset, const Tensor& x) {
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "dropout probability ", p, " is not in [0, 1]");
  TORCH_CHECK_VALUE(offset >= 0 && offset <= 0xFFFFFFFFll, "dropout offset ", offset, " does not fit 32 bits");
  Drop d;
  if (p == 0.0) return d;
  TORCH_CHECK_VALUE(!seed.is_none(), "dropout needs a seed");
  d.p = p;
  d.offset = offset;
  if (THPVariable_Check(seed.ptr())) {
    d.seed_t = THPVariable_Unpack(seed.ptr());
    check_memory(d.seed_t);
    check_like("seed", d.seed_t, x, at::kLong);
    TORCH_CHECK_VALUE(d.seed_t.numel() == 1, "seed holds ", d.seed_t.numel(), " numbers, expected one");
    d.seed_t = in_memory(d.seed_t);
    return d;
  }
  const py::object i = py::reinterpret_steal<py::object>(PyNumber_Index(seed.ptr()));
  if (!i) throw py::error_already_set();
  int over = 0;
  d.seed = PyLong_AsLongLongAndOverflow(i.ptr(), &over);
  if (over > 0) {
    d.seed = (int64_t)PyLong_AsUnsignedLongLong(i.ptr());
    if (PyErr_Occurred()) { PyErr_Clear(); over = -1; }
  }
  TORCH_CHECK_VALUE(over >= 0, "seed does not fit 64 bits");
  return d;
}
int act_code(const std::optional<std::string>& act) {
  if (!act) return 0;
  if (*act == "silu") return 1;
  if (*act == "gelu") return 2;
  if (*act == "quick_gelu") return 3;
  TORCH_CHECK_VALUE(false, "unknown activation '", *act, "': None, 'silu', 'gelu' or 'quick_gelu'");
  return -1;
}

// a tensor as (rows, cols) with unit column stride: a view where the strides allow it
struct Rows { Tensor t; int64_t ld = 0, rows = 0; };
Rows rows_of(const Tensor& given, int64_t cols) {
  const Tensor t = in_memory(given);
  Rows r{t, cols, cols ? t.numel() / cols : 0};
  if (t.is_contiguous()) return r;
  r.t = t.reshape({r.rows, cols});
  if (cols > 1 && r.t.stride(1) != 1) r.t = r.t.contiguous();
  r.ld = r.rows > 1 ? r.t.stride(0) : cols;
  return r;
}
const void* in(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor workspace(int64_t bytes, const Tensor& like) {
  return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}
at::DimVector with_last(const Tensor& t, int64_t last) {
  at::DimVector s(t.sizes().begin(), t.sizes().end());
  s.back() = last;
  return s;
}
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

// Results of a backward pass carry no graph: where one is wanted of them, using it raises.
void first_derivatives_only(variable_list& grads, size_t computed) {
  if (!at::GradMode::is_enabled()) return;
  for (size_t i = 0; i < computed; ++i)
    if (grads[i].defined()) {
      auto error = std::make_shared<torch::autograd::DelayedError>("the layers with dropout have first derivatives only", 1);
      Tensor t = grads[i].detach();
      t.set_requires_grad(true);
      grads[i] = (*error)(variable_list{t})[0];
    }
}
template <typename N> std::shared_ptr<N> node() { return std::shared_ptr<N>(new N(), torch::autograd::deleteNode); }
SavedVariable saved(const Tensor& t) { return SavedVariable(t, false); }

// ---- dropout -------------------------------------------------------------------------------------------
Tensor run_dropout(const Tensor& x, const Tensor& resid, const Drop& d, int dt) {
  at::NoGradGuard no_grad;
  const int64_t cols = x.dim() ? x.size(-1) : 1;
  const Tensor y = at::empty(x.sizes(), x.options());
  const Rows rx = rows_of(x, cols), rr = resid.defined() ? rows_of(resid, cols) : Rows();
  const Here here(x);
  done(api.dropout(in(rx.t), rx.ld, in(rr.t), rr.ld, out(y), rx.rows, (int)cols, d.p, d.seed, address(d.seed_t), d.offset, dt,
                   here.stream), "dropout");
  return y;
}

struct DropoutNode : Node {
  std::string name() const override { return "DropoutBackward"; }
  Drop d;
  int dt = 0;
  SavedVariable seed;
  bool seeded = false;
  variable_list apply(variable_list&& grads) override {
    variable_list g(2);
    const Tensor dy = grads[0];
    if (!dy.defined()) return g;
    if (task_should_compute_output(0)) {
      Drop now = d;
      if (seeded) now.seed_t = seed.unpack();
      g[0] = run_dropout(dy, Tensor(), now, dt);
    }
    if (task_should_compute_output(1)) g[1] = dy;
    first_derivatives_only(g, 1);
    return g;
  }
  void release_variables() override { seed.reset_data(); }
};

Tensor dropout(const Tensor& x, double p, py::handle seed, int64_t offset, const OptTensor& resid_) {
  check_not_traced();
  check_memory(x); check_memory(resid_);
  const Drop d = drop_state(p, seed, offset, x);
  const py::gil_scoped_release no_gil;
  check_columns(x.dim() ? x.size(-1) : 1);
  const int dt = dtype_code(x);
  const Tensor resid = resid_ ? *resid_ : Tensor();
  check_no_tangent(x, resid);
  if (resid.defined()) {
    check_like("resid", resid, x, x.scalar_type());
    check_shape("resid", resid, x.sizes());
  }
  const Tensor y = run_dropout(x, resid, d, dt);
  if (at::GradMode::is_enabled() && (wants(x) || wants(resid))) {
    auto n = node<DropoutNode>();
    n->d = d;
    n->d.seed_t = Tensor();
    n->dt = dt;
    n->seeded = d.seed_t.defined();
    if (n->seeded) n->seed = saved(d.seed_t);
    n->set_next_edges(torch::autograd::collect_next_edges(x, resid));
    torch::autograd::set_history(y, n);
  }
  return y;
}

// ---- linear ----------------------------------------------------------------------------------------------
struct LinearNode : Node {
  std::string name() const override { return "LinearActBackward"; }
  Drop d;
  int dt = 0, act = 0, k = 0, n = 0;
  at::DimVector xshape;
  SavedVariable x, w, preact, seed;
  bool seeded = false;
  variable_list apply(variable_list&& grads) override {
    variable_list g(4);
    const Tensor dy = grads[0];
    if (!dy.defined()) return g;
    const int want = (task_should_compute_output(0) ? 1 : 0) | (task_should_compute_output(1) ? 2 : 0) |
                     (task_should_compute_output(2) ? 4 : 0);
    if (want) {
      at::NoGradGuard no_grad;
      const Rows rd = rows_of(dy, n);
      Rows rx, rw;
      if (want & 1) {
        rw = rows_of(w.unpack(), k);
        g[0] = at::empty(xshape, dy.options());
      }
      if (want & 2) {
        rx = rows_of(x.unpack(), k);
        g[1] = at::empty({n, k}, dy.options());
      }
      if (want & 4) g[2] = at::empty({n}, dy.options().dtype(at::kFloat));
      const Tensor z = act ? preact.unpack() : Tensor(), seed_t = seeded ? seed.unpack() : Tensor();
      const Tensor ws = workspace(api.linear_bwd_ws(rd.rows, k, n, act, d.p, want, dt), dy);
      const Here here(dy);
      done(api.linear_bwd(in(rd.t), rd.ld, (const float*)in(z), in(rx.t), rx.ld, in(rw.t), rw.ld, out(g[0]), out(g[1]),
                          (float*)out(g[2]), rd.rows, k, n, act, d.p, d.seed, address(seed_t), d.offset, out(ws), dt,
                          here.stream), "linear_act_backward");
    }
    if (task_should_compute_output(3)) g[3] = dy;
    first_derivatives_only(g, 3);
    return g;
  }
  void release_variables() override {
    x.reset_data(); w.reset_data(); preact.reset_data(); seed.reset_data();
  }
};

Tensor linear_act(const Tensor& x, const Tensor& w, const OptTensor& bias_, const std::optional<std::string>& act_,
                  const OptTensor& resid_, double p, py::handle seed, int64_t offset) {
  check_not_traced();
  check_memory(x); check_memory(w); check_memory(bias_); check_memory(resid_);
  const Drop d = drop_state(p, seed, offset, x);
  const py::gil_scoped_release no_gil;
  const int act = act_code(act_);
  TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1) && w.numel() > 0, "x ", x.sizes(), " and w ",
                    w.sizes(), " do not fit (..., K) and (N, K)");
  const int64_t n = w.size(0), k = w.size(1);
  check_columns(std::max(n, k));
  const int dt = dtype_code(x);
  check_like("w", w, x, x.scalar_type());
  Tensor bias = bias_ ? *bias_ : Tensor();
  const Tensor resid = resid_ ? *resid_ : Tensor();
  check_no_tangent(x, w, bias, resid);
  const at::DimVector shape = with_last(x, n);
  if (bias.defined()) {
    check_like("bias", bias, x, at::kFloat);
    check_shape("bias", bias, {n});
    bias = in_memory(bias).contiguous();
  }
  if (resid.defined()) {
    check_like("resid", resid, x, x.scalar_type());
    check_shape("resid", resid, shape);
  }
  const bool grad = at::GradMode::is_enabled(), gx = grad && wants(x), gw = grad && wants(w), gb = grad && wants(bias);
  const Tensor y = at::empty(shape, x.options());
  Tensor preact;
  {
    at::NoGradGuard no_grad;
    const Rows rx = rows_of(x, k), rw = rows_of(w, k), rr = resid.defined() ? rows_of(resid, n) : Rows();
    if (act && (gx || gw || gb)) preact = at::empty({rx.rows, n}, x.options().dtype(at::kFloat));
    const Tensor ws = workspace(api.linear_ws(rx.rows, (int)k, (int)n, dt), x);
    const Here here(x);
    done(api.linear(in(rx.t), rx.ld, in(rw.t), rw.ld, (const float*)in(bias), in(rr.t), rr.ld, out(y), (float*)out(preact),
                    rx.rows, (int)k, (int)n, act, d.p, d.seed, address(d.seed_t), d.offset, out(ws), dt, here.stream),
         "linear_act");
  }
  if (gx || gw || gb || (grad && wants(resid))) {
    auto nd = node<LinearNode>();
    nd->d = d;
    nd->d.seed_t = Tensor();
    nd->dt = dt; nd->act = act; nd->k = (int)k; nd->n = (int)n;
    nd->xshape = at::DimVector(x.sizes().begin(), x.sizes().end());
    if (gw) nd->x = saved(x);
    if (gx) nd->w = saved(w);
    if (preact.defined()) nd->preact = saved(preact);
    nd->seeded = d.seed_t.defined();
    if (nd->seeded) nd->seed = saved(d.seed_t);
    nd->set_next_edges(torch::autograd::collect_next_edges(x, w, bias, resid));
    torch::autograd::set_history(y, nd);
  }
  return y;
}

// ---- group norm --------------------------------------------------------------------------------------------
struct GroupNormNode : Node {
  std::string name() const override { return "GroupNormActBackward"; }
  Drop d;
  int dt = 0, act = 0, groups = 0, b = 0, c0 = 0, c1 = 0;
  int64_t hw = 0;
  SavedVariable x, x1, gamma, beta, stats, seed;
  bool seeded = false;
  variable_list apply(variable_list&& grads) override {
    variable_list g(4);
    if (!grads[0].defined()) return g;
    {
      at::NoGradGuard no_grad;
      const Tensor dy = in_memory(grads[0]).contiguous(), tx = x.unpack(), tx1 = c1 ? x1.unpack() : Tensor(), tg = gamma.unpack(),
                   tb = beta.unpack(), ts = stats.unpack(), seed_t = seeded ? seed.unpack() : Tensor();
      const bool need_x = task_should_compute_output(0), need_x1 = task_should_compute_output(1);
      Tensor dx, dx1;
      if (need_x || need_x1) {
        dx = at::empty(tx.sizes(), tx.options());
        if (c1) dx1 = at::empty(tx1.sizes(), tx1.options());
      }
      if (task_should_compute_output(2)) g[2] = at::empty(tg.sizes(), tg.options());
      if (task_should_compute_output(3)) g[3] = at::empty(tb.sizes(), tb.options());
      const Tensor ws = workspace(api.groupnorm_ws(b, hw, c0, c1, groups, dt, 1), tx);
      const Here here(tx);
      done(api.groupnorm_bwd(in(dy), in(tx), c0, in(tx1), c1, b, hw, groups, (const float*)in(tg), (const float*)in(tb),
                             (const float*)in(ts), act, d.p, d.seed, address(seed_t), d.offset, out(dx), out(dx1),
                             (float*)out(g[2]), (float*)out(g[3]), out(ws), dt, here.stream), "groupnorm_act_backward");
      if (need_x) g[0] = dx;
      if (need_x1) g[1] = dx1;
    }
    first_derivatives_only(g, 4);
    return g;
  }
  void release_variables() override {
    x.reset_data(); x1.reset_data(); gamma.reset_data(); beta.reset_data(); stats.reset_data(); seed.reset_data();
  }
};

Tensor groupnorm_act(const Tensor& x_, const Tensor& gamma_, const Tensor& beta_, double eps,
                     const std::optional<std::string>& act_, const OptTensor& x1_, int64_t groups, double p, py::handle seed,
                     int64_t offset) {
  check_not_traced();
  check_memory(x_); check_memory(gamma_); check_memory(beta_); check_memory(x1_);
  const Drop d = drop_state(p, seed, offset, x_);
  const py::gil_scoped_release no_gil;
  const int act = act_code(act_), dt = dtype_code(x_);
  check_no_tangent(x_, gamma_, beta_);
  TORCH_CHECK_VALUE(x_.dim() >= 2, "x ", x_.sizes(), " has no batch and channel dimension");
  const int64_t b = x_.size(0), c0 = x_.size(-1);
  int64_t c1 = 0, hw = 1;
  if (x1_) {
    check_like("x1", *x1_, x_, x_.scalar_type());
    check_no_tangent(*x1_);
    c1 = x1_->dim() ? x1_->size(-1) : 0;
    check_shape("x1", *x1_, with_last(x_, c1));
  }
  const int64_t c = c0 + c1;
  TORCH_CHECK_VALUE(c0 > 0 && groups >= 1 && c % groups == 0, c, " channels do not split into ", groups, " groups");
  TORCH_CHECK_VALUE(c <= 8192 && b <= 65535, "batch ", b, " of ", c, " channels: at most 65535 and 8192 are supported");
  check_like("gamma", gamma_, x_, at::kFloat);
  check_shape("gamma", gamma_, {c});
  check_like("beta", beta_, x_, at::kFloat);
  check_shape("beta", beta_, {c});
  for (int64_t i = 1; i + 1 < x_.dim(); ++i) hw *= x_.size(i);
  const Tensor x = in_memory(x_).contiguous(), x1 = c1 ? in_memory(*x1_).contiguous() : Tensor(),
               gamma = in_memory(gamma_).contiguous(), beta = in_memory(beta_).contiguous();
  const Tensor y = at::empty(with_last(x, c), x.options()), stats = at::empty({b, groups, 2}, gamma.options());
  {
    at::NoGradGuard no_grad;
    const Tensor ws = workspace(api.groupnorm_ws((int)b, hw, (int)c0, (int)c1, (int)groups, dt, 0), x);
    const Here here(x);
    done(api.groupnorm(in(x), (int)c0, in(x1), (int)c1, (int)b, hw, (int)groups, (float)eps, (const float*)in(gamma),
                       (const float*)in(beta), act, d.p, d.seed, address(d.seed_t), d.offset, out(y), (float*)out(stats),
                       out(ws), dt, here.stream), "groupnorm_act");
  }
  if (at::GradMode::is_enabled() && (wants(x) || wants(x1) || wants(gamma) || wants(beta))) {
    auto nd = node<GroupNormNode>();
    nd->d = d;
    nd->d.seed_t = Tensor();
    nd->dt = dt; nd->act = act; nd->groups = (int)groups; nd->b = (int)b; nd->c0 = (int)c0; nd->c1 = (int)c1; nd->hw = hw;
    nd->x = saved(x);
    if (c1) nd->x1 = saved(x1);
    nd->gamma = saved(gamma); nd->beta = saved(beta); nd->stats = saved(stats);
    nd->seeded = d.seed_t.defined();
    if (nd->seeded) nd->seed = saved(d.seed_t);
    nd->set_next_edges(torch::autograd::collect_next_edges(x, x1, gamma, beta));
    torch::autograd::set_history(y, nd);
  }
  return y;
}

}  // namespace

PYBIND11_MODULE(sdmi_layers, m) {
  m.def("bind", &bind);
  m.def("dropout", torch::wrap_pybind_function(&dropout));
  m.def("linear_act", torch::wrap_pybind_function(&linear_act));
  m.def("groupnorm_act", torch::wrap_pybind_function(&groupnorm_act));
}

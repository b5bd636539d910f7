// libdtf_torch.so: the entry points that work on torch tensors directly (checks, allocation, launch, autograd), without the Python and
// ctypes steps of ops/hip_ops.py.  A small call is bound by the host, not by the GPU: a norm's forward pass through ctypes took 13.6 us
// where its kernel takes 2.4, and a Python backward function costs two hand-overs of the interpreter lock on top (143 us for a forward
// and backward pass of 100 x 1024 fp32 whose kernels take 11).  What does not fit a kernel is refused here, as ValueError.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>

#include "adamw.h"
#include "linear_w4.h"
#include "rms_norm.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
struct NativeError : std::runtime_error {  // native.NativeError on the Python side
  using std::runtime_error::runtime_error;
};
void check(int rc, const char* what) {
  if (rc != 0) throw NativeError(c10::str(what, " failed with code ", rc, rc == -22 ? " (shape/alignment precondition violated)" : ""));
}
// A node that raises in a backward pass towards any of the operands.  (Its edges lead to them: one that hung from a leaf of its own would not
// be visited by a gradient with respect to them alone.)
template <typename... Operands> std::shared_ptr<torch::autograd::Node> refusal(const char* message, const Operands&... operands) {
  return std::make_shared<torch::autograd::Error>(message, torch::autograd::collect_next_edges(operands...));
}
// Forward mode: what has no rule for tangents refuses them
template <typename... Operands> void no_tangents(const char* what, const Operands&... operands) {
  const bool any = (torch::autograd::isFwGradDefined(operands) || ...);
  TORCH_CHECK_NOT_IMPLEMENTED(!any, what, " has no forward-mode derivative");
}
template <typename F> auto without_grad(F f) {
  const at::NoGradGuard no_grad;
  return f();
}
bool is_rows(const Tensor& t) {
  return t.is_cuda() && t.layout() == at::kStrided && (t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16) && t.dim() >= 1;
}
// A side operand: fp32, contiguous, of n elements on like's device
void check_f32(const Tensor& t, const char* name, int64_t n, const Tensor& like) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.scalar_type() == at::kFloat && t.is_contiguous() && !t.is_neg() && t.numel() == n && t.device() == like.device(), name,
                    " must be a contiguous CUDA tensor of ", n, " float32 values on ", like.device(), " (got ", t.scalar_type(), " ", t.sizes(),
                    " on ", t.device(), ")");
}

// ------------------------------------------------------------------------------------------------ RMS norm
struct Rows {  // rows of the last dimension: any stride between rows, none inside one (else a copy)
  Tensor keep;
  const void* p = nullptr;
  long ld = 0;
  Rows(const Tensor& t, const Tensor* like, const char* name) {
    TORCH_CHECK_VALUE(is_rows(t), name, " must be a CUDA tensor of float32 or bfloat16 rows (got ", t.scalar_type(), " ", t.sizes(), " on ",
                      t.device(), ")");
    TORCH_CHECK_VALUE(!like || (t.scalar_type() == like->scalar_type() && t.sizes() == like->sizes() && t.device() == like->device()), name, " (",
                      t.scalar_type(), " ", t.sizes(), " on ", t.device(), ") must have the type, shape and device of the other rows");
    if (t.numel() == 0) return;
    keep = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
    if (keep.is_neg() || (keep.size(1) > 1 && keep.stride(1) != 1)) keep = keep.resolve_neg().contiguous();  // (the imaginary part of a conjugate: negated lazily)
    p = keep.const_data_ptr();
    ld = keep.stride(0);
  }
};
void check_weight(const Tensor& w, const Tensor& x, double eps) {
  TORCH_CHECK_VALUE(w.is_cuda() && w.scalar_type() == at::kFloat && w.is_contiguous() && !w.is_neg() && w.dim() == 1 && w.device() == x.device() && w.size(0) >= 1 &&
                        x.size(-1) == w.size(0),
                    "weight must be contiguous float32 of the rows' length on their device (got ", w.scalar_type(), " ", w.sizes(), " on ",
                    w.device(), " for rows ", x.sizes(), " on ", x.device(), ")");
  TORCH_CHECK_VALUE(w.size(0) <= INT_MAX / 2, "rows of ", w.size(0), " elements");
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative (got ", eps, ")");
}

// y, rstd or the rows' scales, h (x itself without a residual)
std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& w, const OptTensor& residual, double eps, bool eight) {
  const Rows rx(x, nullptr, "x");
  check_weight(w, x, eps);
  RmsNormArgs a{};
  Tensor h = x;
  std::optional<Rows> rr;
  if (residual) rr.emplace(*residual, &x, "residual");
  const c10::DeviceGuard guard(x.device());
  if (rr) h = at::empty(x.sizes(), x.options());
  const Tensor y = at::empty(x.sizes(), eight ? x.options().dtype(at::kFloat8_e4m3fn) : x.options());
  const Tensor side = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  if (x.numel()) {
    if (rr) {
      a.res = rr->p;
      a.ld_res = rr->ld;
      a.h = h.mutable_data_ptr();
    }
    a.x = rx.p;
    a.ld_x = rx.ld;
    a.w = w.const_data_ptr<float>();
    a.y = y.mutable_data_ptr();
    (eight ? a.q_scale : a.rstd) = side.mutable_data_ptr<float>();
    a.dim = (int)w.size(0);
    a.rows = x.numel() / a.dim;
    a.bf16 = x.scalar_type() == at::kBFloat16;
    a.eps = (float)eps;
    check(dtf_rms_norm_fwd(&a, stream_of(x)), "rms_norm_fwd");
  }
  return {y, side, h};
}
// The results record no backward pass: one through them raises where `operands` require a gradient (h without a residual is x, whose gradient is
// its own)
template <typename... Operands>
void refuse_backward(const std::tuple<Tensor, Tensor, Tensor>& out, const OptTensor& residual, const char* message, const Operands&... operands) {
  if (!torch::autograd::compute_requires_grad(operands...)) return;
  const auto fn = refusal(message, operands...);
  torch::autograd::set_history(std::get<0>(out), fn);
  torch::autograd::set_history(std::get<1>(out), fn);
  if (residual) torch::autograd::set_history(std::get<2>(out), fn);
}
std::tuple<Tensor, Tensor, Tensor> rms_norm_forward(const Tensor& x, const Tensor& w, const OptTensor& residual, double eps) {
  no_tangents("rms_norm_forward", OptTensor(x), residual);
  const auto out = without_grad([&] { return norm_forward(x, w, residual, eps, false); });
  // (not the weight: a layer's parameter is passed as it is by those who call rms_norm_backward themselves)
  refuse_backward(out, residual, "rms_norm_forward has no backward pass of its own: autograd.rms_norm has", x, residual);
  const auto& [y, rstd, h] = out;
  return {y, h, rstd};
}
std::tuple<Tensor, Tensor, Tensor> rms_norm_e4m3(const Tensor& x, const Tensor& w, const OptTensor& residual, double eps) {
  no_tangents("rms_norm_e4m3", OptTensor(x), OptTensor(w), residual);
  const auto out = without_grad([&] { return norm_forward(x, w, residual, eps, true); });
  refuse_backward(out, residual, "rms_norm_e4m3 is for inference: it has no backward pass", x, w, residual);
  return out;
}

std::tuple<Tensor, OptTensor> rms_norm_backward(const Tensor& dy, const Tensor& x, const Tensor& rstd, const Tensor& w, const OptTensor& residual,
                                                const OptTensor& dh, bool need_dw) {
  const at::NoGradGuard no_grad;
  const Rows rx(x, nullptr, "x");
  check_weight(w, x, 0.0);
  const Rows rd(dy, &x, "dy");
  check_f32(rstd, "rstd", x.numel() / w.size(0), x);
  std::optional<Rows> rr, rg;
  if (residual) rr.emplace(*residual, &x, "residual");
  if (dh) rg.emplace(*dh, &x, "dh");
  const c10::DeviceGuard guard(x.device());
  const Tensor dx = at::empty(x.sizes(), x.options());
  OptTensor dw;
  if (x.numel() == 0) {
    if (need_dw) dw = at::zeros(w.sizes(), w.options());
    return {dx, dw};
  }
  RmsNormArgs a{};
  a.dim = (int)w.size(0);
  a.rows = x.numel() / a.dim;
  a.blocks = dtf_rms_norm_bwd_blocks(a.rows, a.dim);
  Tensor part;
  if (need_dw) {
    dw = at::empty(w.sizes(), w.options());
    a.dw = dw->mutable_data_ptr<float>();
    if (a.blocks) {
      part = at::empty({a.blocks, a.dim}, w.options());
      a.part = part.mutable_data_ptr<float>();
    }
  }
  if (rr) {
    a.res = rr->p;
    a.ld_res = rr->ld;
  }
  if (rg) {
    a.dh = rg->p;
    a.ld_dh = rg->ld;
  }
  a.x = rx.p;
  a.ld_x = rx.ld;
  a.dy = rd.p;
  a.ld_dy = rd.ld;
  a.w = w.const_data_ptr<float>();
  a.y = dx.mutable_data_ptr();
  a.rstd = const_cast<float*>(rstd.const_data_ptr<float>());  // (only read)
  a.bf16 = x.scalar_type() == at::kBFloat16;
  check(dtf_rms_norm_bwd(&a, stream_of(x)), "rms_norm_bwd");
  return {dx, dw};
}

struct RMSNormFunction : torch::autograd::Function<RMSNormFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& residual,
                                                double eps) {
    auto [y, rstd, h] = norm_forward(x, w, residual, eps, false);
    ctx->save_for_backward({x, rstd, w, residual ? *residual : Tensor()});
    ctx->set_materialize_grads(false);
    return residual ? torch::autograd::variable_list{y, h} : torch::autograd::variable_list{y};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[2], dy = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor();
    const OptTensor residual = saved[3].defined() ? OptTensor(saved[3]) : std::nullopt;
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_r = residual && ctx->needs_input_grad(2);
    Tensor dx, dw;
    if (dy.defined()) {
      auto [a, b] = rms_norm_backward(dy, x, saved[1], w, residual, dh.defined() ? OptTensor(dh) : std::nullopt, need_w);
      dx = a;
      if (b) dw = *b;
    } else {  // only h went into the loss
      dx = dh;
      if (need_w) dw = at::zeros(w.sizes(), w.options());
    }
    torch::autograd::variable_list out{need_x ? dx : Tensor(), dw, need_r ? dx : Tensor(), Tensor()};
    // Under create_graph: the kernels record nothing, so that a second derivative through them would be silently wrong.  dx and dw depend on
    // x, the residual and dy (dx on w and dh too, but it is asked for only where x or the residual requires a gradient).  h's own
    // gradient is dh itself, whose graph goes on.
    if (dy.defined() && at::GradMode::is_enabled() && (dy.requires_grad() || x.requires_grad() || (residual && residual->requires_grad()))) {
      auto refuse = refusal("rms_norm is differentiable once", dy, dh, x, w, residual);
      for (auto& t : out)
        if (t.defined()) torch::autograd::set_history(t = t.detach(), refuse);
    }
    return out;
  }
};
py::object rms_norm(const Tensor& x, const Tensor& w, const OptTensor& residual, double eps) {
  auto out = RMSNormFunction::apply(x, w, residual, eps);
  if (out.size() == 1) return py::cast(out[0]);
  return py::make_tuple(out[0], out[1]);
}

// ------------------------------------------------------------------------------------------------ products with 4-bit weights
constexpr int64_t W4_MAX_ROWS = 65535 * 5;
Tensor w4_product(const Tensor& x, const Tensor& wq, const Tensor& scales, int64_t N, const OptTensor& bias, bool relu, const OptTensor& x_scale,
                  bool out_bf16) {
  const at::NoGradGuard no_grad;
  TORCH_CHECK_VALUE(wq.scalar_type() == at::kByte && wq.dim() == 4 && wq.size(2) == 64 && wq.size(3) == 16 && wq.is_contiguous() && wq.numel() > 0 &&
                        scales.scalar_type() == at::kBFloat16 && scales.dim() == 3 && scales.is_contiguous() && scales.size(0) == wq.size(0) &&
                        scales.size(2) == 16 && scales.device() == wq.device() &&
                        (scales.size(1) == wq.size(1) || scales.size(1) == 2 * wq.size(1) || scales.size(1) == 4 * wq.size(1)),
                    "not a pair from quantize_w4: ", wq.scalar_type(), " ", wq.sizes(), ", ", scales.scalar_type(), " ", scales.sizes());
  const auto type = x.scalar_type();
  TORCH_CHECK_VALUE(x.is_cuda() && x.layout() == at::kStrided && (type == at::kFloat || type == at::kBFloat16 || type == at::kFloat8_e4m3fn) &&
                        x.dim() >= 1 && x.device() == wq.device(),
                    "x must be a CUDA tensor of float32, bfloat16 or float8_e4m3fn on the weights' device (got ", type, " on ", x.device(), ")");
  const int64_t K = x.size(-1);
  TORCH_CHECK_VALUE(K >= 1 && (K + 127) / 128 == wq.size(1) && N >= 1 && (N + 15) / 16 == wq.size(0), "x ", x.sizes(), " and ", N,
                    " outputs do not fit weights of ", wq.size(1), " x ", wq.size(0), " tiles of 128 x 16");
  TORCH_CHECK_VALUE(K < INT_MAX - 128 && N < INT_MAX - 16, "weights of ", K, " x ", N);
  TORCH_CHECK_VALUE(x_scale || type != at::kFloat8_e4m3fn, "e4m3 rows need their x_scale");
  const int64_t M = x.numel() / K;
  if (bias) check_f32(*bias, "bias", N, x);
  if (x_scale) check_f32(*x_scale, "x_scale", M, x);
  TORCH_CHECK_VALUE(M <= W4_MAX_ROWS, "at most ", W4_MAX_ROWS, " rows (got ", M, ")");
  const c10::DeviceGuard guard(x.device());
  auto shape = x.sizes().vec();
  shape.back() = N;
  const Tensor y = at::empty(shape, x.options().dtype(out_bf16 ? at::kBFloat16 : at::kFloat));
  if (M == 0) return y;
  Tensor rows = x.dim() == 2 ? x : x.reshape({-1, K});
  if (rows.is_neg() || (K > 1 && rows.stride(1) != 1)) rows = rows.resolve_neg().contiguous();
  LinearW4Args a{};
  a.x = rows.const_data_ptr();
  a.wq = wq.const_data_ptr();
  a.scales = static_cast<const uint16_t*>(scales.const_data_ptr());
  a.bias = bias ? bias->const_data_ptr<float>() : nullptr;
  a.x_scale = x_scale ? x_scale->const_data_ptr<float>() : nullptr;
  a.y = y.mutable_data_ptr();
  a.M = M;
  a.ldx = rows.stride(0);
  a.N = (int)N;
  a.K = (int)K;
  a.group = (int)(wq.size(1) * 128 / scales.size(1));
  a.xtype = type == at::kFloat ? X_F32 : type == at::kBFloat16 ? X_BF16 : X_E4M3;
  a.relu = relu;
  a.out_bf16 = out_bf16;
  check(dtf_linear_w4(&a, stream_of(x)), "linear_w4");
  return y;
}
Tensor linear_w4(const Tensor& x, const Tensor& wq, const Tensor& scales, int64_t N, const OptTensor& bias, bool relu, const OptTensor& x_scale,
                 bool out_bf16) {
  no_tangents("linear_w4", OptTensor(x), bias, x_scale);
  const Tensor y = w4_product(x, wq, scales, N, bias, relu, x_scale, out_bf16);
  if (torch::autograd::compute_requires_grad(x, scales, bias, x_scale))
    torch::autograd::set_history(y, refusal("linear_w4 is for inference: it has no backward pass", x, scales, bias, x_scale));
  return y;
}

// ------------------------------------------------------------------------------------------------ AdamW
// The parameters of one group (optim/adamw.py keeps the arenas and tables whose addresses are in `launch`).
struct AdamWGroup {
  std::vector<Tensor> params;
  std::vector<int64_t> sizes;
  std::vector<at::ScalarType> types;
  AdamWLaunch a{};
  std::vector<Tensor> grads;  // between gather and launch
  std::vector<uint64_t> pp, gg;
  std::vector<uint8_t> kind;

  AdamWGroup(std::vector<Tensor> p, const std::map<std::string, uint64_t>& at, int nchunks, int bits, uint32_t seed) : params(std::move(p)) {
    for (const auto& t : params) {
      sizes.push_back(t.numel());
      types.push_back(t.scalar_type());
    }
    const auto get = [&](const char* k) {
      const auto i = at.find(k);
      return i == at.end() ? uint64_t(0) : i->second;
    };
    a.shape = reinterpret_cast<const int64_t*>(get("shape"));
    a.chunks = reinterpret_cast<const void*>(get("chunks"));
    a.step = reinterpret_cast<int*>(get("step"));
    a.m = reinterpret_cast<void*>(get("m"));
    a.v = reinterpret_cast<void*>(get(bits == 8 ? "r" : "v"));
    a.m_scale = reinterpret_cast<float*>(get("m_scale"));
    a.r_scale = reinterpret_cast<float*>(get("r_scale"));
    a.ntensors = (int)params.size();
    a.nchunks = nchunks;
    a.bits = bits;
    a.seed = seed;
  }

  // The parameters' gradients, or the given ones; whatever does not fit the group is refused before anything is changed.  Whether
  // there is one at all.
  bool gather(const std::optional<std::vector<OptTensor>>& given) {
    const size_t n = params.size();
    TORCH_CHECK_VALUE(!given || given->size() == n, given ? given->size() : 0, " gradients for ", n, " parameters");
    std::vector<Tensor> found(n);
    std::vector<uint64_t> p(n), g(n);
    std::vector<uint8_t> k(n);
    const auto device = params[0].device();
    bool any = false;
    for (size_t i = 0; i < n; ++i) {
      const Tensor& t = params[i];
      TORCH_CHECK_VALUE(t.scalar_type() == types[i] && t.numel() == sizes[i] && t.device() == device && t.is_contiguous() && !t.is_neg(),
                        "a parameter's type, size, device or layout has changed since it was given to AdamW");
      Tensor d = given ? (*given)[i].value_or(Tensor()) : t.grad();
      if (!d.defined()) continue;
      TORCH_CHECK_VALUE(d.layout() == at::kStrided && (d.scalar_type() == at::kFloat || d.scalar_type() == at::kBFloat16),
                        "gradients are dense float32 or bfloat16 tensors (got ", d.scalar_type(), ", ", d.layout(), ")");
      TORCH_CHECK_VALUE(d.device() == device && d.sizes() == t.sizes(), "a gradient of shape ", d.sizes(), " on ", d.device(),
                        " for a parameter of shape ", t.sizes(), " on ", device);
      if (sizes[i] == 0) continue;
      found[i] = d.resolve_neg().contiguous();
      p[i] = reinterpret_cast<uint64_t>(t.data_ptr());
      g[i] = reinterpret_cast<uint64_t>(found[i].const_data_ptr());
      k[i] = (types[i] == at::kBFloat16 ? 1 : 0) | (d.scalar_type() == at::kBFloat16 ? 2 : 0);
      any = true;
    }
    grads.swap(found);
    pp.swap(p);
    gg.swap(g);
    kind.swap(k);
    return any;
  }

  void launch(double lr, double beta1, double beta2, double eps, double weight_decay, double grad_scale) {
    TORCH_CHECK(grads.size() == params.size(), "no gradients were gathered");
    a.lr = lr;
    a.beta1 = beta1;
    a.beta2 = beta2;
    a.b1 = (float)beta1;
    a.ob1 = (float)(1.0 - beta1);
    a.b2 = (float)beta2;
    a.ob2 = (float)(1.0 - beta2);
    a.eps = (float)eps;
    a.decay = (float)(1.0 - lr * weight_decay);
    a.grad_scale = (float)grad_scale;
    const c10::DeviceGuard guard(params[0].device());
    // (a step's own, like its graph's: steps over different parameters of a group may run at once, on two streams or from two captured graphs)
    const Tensor live = at::empty({(int64_t)params.size() * dtf_sizeof_adamw_live()}, params[0].options().dtype(at::kByte));
    a.live = live.mutable_data_ptr();
    const int rc = dtf_adamw(&a, pp.data(), gg.data(), kind.data(), stream_of(params[0]));
    for (size_t i = 0; i < grads.size(); ++i)
      if (grads[i].defined() && !params[i].is_inference()) params[i].unsafeGetTensorImpl()->bump_version();  // (a backward pass that saved the old values is refused)
    grads.clear();
    check(rc, "adamw");
  }
};

}  // namespace

PYBIND11_MODULE(libdtf_torch, m) {
  static const py::object error = py::module_::import("distributed_tensorflow_amd.native").attr("NativeError");
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const NativeError& e) {
      PyErr_SetString(error.ptr(), e.what());
    }
  });
  m.def("rms_norm_forward", &rms_norm_forward);
  m.def("rms_norm_e4m3", &rms_norm_e4m3);
  m.def("rms_norm_backward", &rms_norm_backward);
  m.def("rms_norm", &rms_norm);
  m.def("linear_w4", &linear_w4);
  py::class_<AdamWGroup>(m, "AdamWGroup")
      .def(py::init<std::vector<Tensor>, const std::map<std::string, uint64_t>&, int, int, uint32_t>())
      .def("gather", &AdamWGroup::gather)
      .def("launch", &AdamWGroup::launch);
}

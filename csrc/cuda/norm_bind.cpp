// Torch bindings of the norm kernels (norm.h).
#include "layer_bind.h"

#include <array>
#include <vector>

#include "norm.h"

namespace {
using namespace ngl::bind;
namespace norm = ngl::norm;

int64_t check_rows(const torch::Tensor& x, const OptTensor& w, const OptTensor& residual, double eps) {
  const auto t = x.scalar_type();
  TORCH_CHECK(t == torch::kFloat32 || is_half(t), "x must be float32, bfloat16 or float16; got ", t);
  TORCH_CHECK(x.dim() >= 1, "x needs at least one dimension");
  const int64_t width = x.size(-1);
  TORCH_CHECK(width > 0 && width <= norm::kMaxWidth, "rows must have 1 to ", text(norm::kMaxWidth), " elements; got ", text(width));
  if (w.has_value()) {
    TORCH_CHECK(w->dim() == 1 && w->size(0) == width, "weight must be [", text(width), "]; got ", text(w->sizes()));
    TORCH_CHECK(w->scalar_type() == t || w->scalar_type() == torch::kFloat32, "weight must be ", t,
                " or float32; got ", w->scalar_type());
  }
  if (residual.has_value()) {
    TORCH_CHECK(residual->sizes() == x.sizes(), "residual must have the shape of x, ", text(x.sizes()), "; got ",
                text(residual->sizes()));
    TORCH_CHECK(residual->scalar_type() == t || residual->scalar_type() == torch::kFloat32, "residual must be ", t,
                " or float32; got ", residual->scalar_type());
  }
  TORCH_CHECK(eps >= 0, "eps must not be negative; got ", std::to_string(eps));
  return width;
}

struct Out {
  torch::Tensor y, scale, stream;  // scale only in 8 bits, stream only with a residual
};
Out run_forward(const torch::Tensor& x, const OptTensor& weight, double eps, const OptTensor& residual, bool fp8,
                c10::optional<at::ScalarType> out_dtype) {
  const int64_t width = check_rows(x, weight, residual, eps), rows = x.numel() / width;
  const auto y_t = fp8 ? at::kFloat8_e4m3fn : out_dtype.has_value() ? *out_dtype : x.scalar_type();
  TORCH_CHECK(fp8 || y_t == x.scalar_type() || (x.scalar_type() == torch::kFloat32 && is_half(y_t)),
              "out_dtype must be ", x.scalar_type(), x.scalar_type() == torch::kFloat32 ? ", bfloat16 or float16" : "",
              "; got ", y_t);
  TORCH_CHECK(weight.has_value() || (fp8 && !residual.has_value()), "weight is needed");
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (there is no CPU path)");
  if (weight.has_value()) need_cuda(*weight, x, "weight");
  if (residual.has_value()) need_cuda(*residual, x, "residual");
  const c10::cuda::CUDAGuard guard(x.device());
  auto y = new_cuda(x.sizes(), y_t, x);
  torch::Tensor scale, stream;
  if (fp8) scale = new_cuda(x.sizes().slice(0, x.dim() - 1), torch::kFloat32, x);
  if (residual.has_value()) stream = new_cuda(x.sizes(), residual->scalar_type(), x);
  if (rows == 0) return {y, scale, stream};
  const Rows xr = rows_of(x, rows, width);
  Rows rr{xr.t, 0};
  norm::Forward f;
  std::memset(&f, 0, sizeof(f));
  f.rows = rows, f.width = width;
  f.x_type = f.stream_type = f.w_type = type_of(x.scalar_type());
  f.x = xr.p(), f.ldx = xr.ld;
  if (residual.has_value()) {
    rr = rows_of(*residual, rows, width);
    f.residual = rr.p(), f.ldr = rr.ld;
    f.stream_type = type_of(residual->scalar_type());
    f.stream = stream.data_ptr();
  }
  torch::Tensor w;
  if (weight.has_value()) {
    w = weight->contiguous();
    f.w = w.data_ptr();
    f.w_type = type_of(w.scalar_type());
  }
  f.y = y.data_ptr();
  f.y_type = type_of(y_t);
  f.scale = fp8 ? scale.data_ptr<float>() : nullptr;
  f.eps = (float)eps;
  ck(norm::forward(f, sm_count(x.get_device()), at::cuda::getCurrentCUDAStream()), "rms_norm");
  return {y, scale, stream};
}

// dx, dresidual (dx again where the types agree; undefined without residual), dweight.
std::array<torch::Tensor, 3> gradients(const torch::Tensor& dy, const torch::Tensor& ds, const torch::Tensor& s,
                                       const torch::Tensor& weight, double eps, at::ScalarType x_type,
                                       bool has_residual, bool need_w) {
  const int64_t width = s.size(-1), rows = s.numel() / width;
  TORCH_CHECK(s.is_cuda(), "the stream must be a CUDA tensor (there is no CPU path)");
  const c10::cuda::CUDAGuard guard(s.device());
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  const bool split = has_residual && s.scalar_type() != x_type;
  auto dx = new_cuda(s.sizes(), x_type, s);
  torch::Tensor dres, dw;
  if (split) dres = new_cuda(s.sizes(), s.scalar_type(), s);
  if (need_w) dw = new_cuda({width}, weight.scalar_type(), s);
  if (rows == 0) {
    if (need_w) dw.zero_();
    return {dx, has_residual ? (split ? dres : dx) : torch::Tensor(), dw};
  }
  const torch::Tensor dyt = dy.defined() ? dy.to(x_type) : torch::zeros(s.sizes(), s.options().dtype(x_type));
  TORCH_CHECK(dyt.sizes() == s.sizes(), "gradient must have the output's shape");
  const Rows yr = rows_of(dyt, rows, width), sr = rows_of(s, rows, width);
  Rows er{sr.t, 0};
  norm::Backward b;
  std::memset(&b, 0, sizeof(b));
  b.rows = rows, b.width = width;
  b.x_type = type_of(x_type), b.stream_type = type_of(s.scalar_type());
  b.dy = yr.p(), b.lddy = yr.ld;
  b.s = sr.p(), b.lds = sr.ld;
  if (ds.defined()) {
    er = rows_of(ds.to(s.scalar_type()), rows, width);
    b.ds = er.p(), b.ldds = er.ld;
  }
  const auto w = weight.contiguous();
  b.w = w.data_ptr();
  b.w_type = type_of(w.scalar_type());
  b.dx = dx.data_ptr();
  b.dres = split ? dres.data_ptr() : nullptr;
  b.eps = (float)eps;
  const int sms = sm_count(s.get_device());
  b.parts = norm::backward_parts(rows, width, sms);
  torch::Tensor part;
  if (need_w) {
    part = new_cuda({b.parts, width}, torch::kFloat32, s);
    b.partial = part.data_ptr<float>();
    b.dw = dw.data_ptr();
  }
  ck(norm::backward(b, st), "rms_norm backward");
  return {dx, has_residual ? (split ? dres : dx) : torch::Tensor(), dw};
}

namespace ag = torch::autograd;

class NormFn : public ag::Function<NormFn> {
 public:
  static ag::variable_list forward(ag::AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& weight,
                                   const OptTensor& residual, double eps, c10::optional<at::ScalarType> out_dtype) {
    Out o = run_forward(x, weight, eps, residual, false, out_dtype);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({residual.has_value() ? o.stream : x, weight});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["type"] = (int64_t)x.scalar_type();
    ctx->saved_data["residual"] = residual.has_value();
    return residual.has_value() ? ag::variable_list{o.y, o.stream} : ag::variable_list{o.y};
  }
  static ag::variable_list backward(ag::AutogradContext* ctx, ag::variable_list grads) {
    const bool has_r = ctx->saved_data["residual"].toBool();
    const torch::Tensor ds = has_r ? grads[1] : torch::Tensor();
    const torch::Tensor none;
    seen_by_all("the gradient of rms_norm", grads[0], ds);
    if (!grads[0].defined() && !ds.defined()) return {none, none, none, none, none};
    const auto saved = ctx->get_saved_variables();
    const bool nr = has_r && ctx->needs_input_grad(2);
    auto g = gradients(grads[0], ds, saved[0], saved[1], ctx->saved_data["eps"].toDouble(),
                       (at::ScalarType)ctx->saved_data["type"].toInt(), has_r, ctx->needs_input_grad(1));
    return once({ctx->needs_input_grad(0) ? g[0] : none, g[2], nr ? g[1] : none, none, none}, "rms_norm");
  }
};

// (y,) or (y, stream).
std::vector<torch::Tensor> rms_norm(const torch::Tensor& x, const torch::Tensor& weight, double eps,
                                    const OptTensor& residual,
                                    c10::optional<at::ScalarType> out_dtype) {
  seen_by_all("rms_norm", x, weight, residual);
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(residual)))
    return NormFn::apply(x, weight, residual, eps, out_dtype);
  Out o = run_forward(x, weight, eps, residual, false, out_dtype);
  if (residual.has_value()) return {o.y, o.stream};
  return {o.y};
}
std::vector<torch::Tensor> rms_norm_fp8(const torch::Tensor& x, const OptTensor& weight, double eps,
                                        const OptTensor& residual) {
  seen_by_all("rms_norm_fp8", x, weight, residual);
  const at::NoGradGuard no_grad;
  Out o = run_forward(x, weight, eps, residual, true, c10::nullopt);
  if (residual.has_value()) return {o.y, o.scale, o.stream};
  return {o.y, o.scale};
}

// (x, weight, eps, residual, out_dtype)
PyObject* py_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 5, "rms_norm");
  return wrap_all(rms_norm(tensor_arg(a[0], "x"), tensor_arg(a[1], "weight"), float_arg(a[2]),
                           opt_tensor_arg(a[3], "residual"), opt_dtype_arg(a[4], "out_dtype")));
  END_HANDLE_TH_ERRORS
}
// (x, weight or None, eps, residual)
PyObject* py_rms_norm_fp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 4, "rms_norm_fp8");
  return wrap_all(rms_norm_fp8(tensor_arg(a[0], "x"), opt_tensor_arg(a[1], "weight"), float_arg(a[2]),
                               opt_tensor_arg(a[3], "residual")));
  END_HANDLE_TH_ERRORS
}
PyMethodDef kMethods[] = {
    {"rms_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&py_rms_norm)), METH_FASTCALL, nullptr},
    {"rms_norm_fp8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&py_rms_norm_fp8)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

void register_norm(pybind11::module& m) {
  if (PyModule_AddFunctions(m.ptr(), kMethods) != 0) throw pybind11::error_already_set();
}

// Torch bindings of the norm kernels (norm.h).
#include "layer_bind.h"

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

// y (or codes), scale (undefined unless fp8), stream (undefined without residual).
std::vector<torch::Tensor> rms_norm_forward(torch::Tensor x, OptTensor weight, double eps, OptTensor residual,
                                            bool fp8) {
  const int64_t width = check_rows(x, weight, residual, eps), rows = x.numel() / width;
  TORCH_CHECK(weight.has_value() || (fp8 && !residual.has_value()), "weight is needed");
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (there is no CPU path)");
  if (weight.has_value()) need_cuda(*weight, x, "weight");
  if (residual.has_value()) need_cuda(*residual, x, "residual");
  const c10::cuda::CUDAGuard guard(x.device());
  auto y = torch::empty(x.sizes(), x.options().dtype(fp8 ? at::kFloat8_e4m3fn : x.scalar_type()));
  torch::Tensor scale, stream;
  if (fp8) scale = torch::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(torch::kFloat32));
  if (residual.has_value()) stream = torch::empty(x.sizes(), residual->options());
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
  f.scale = fp8 ? scale.data_ptr<float>() : nullptr;
  f.eps = (float)eps;
  ck(norm::forward(f, sm_count(x.get_device()), at::cuda::getCurrentCUDAStream()), "rms_norm");
  return {y, scale, stream};
}

// dx, dresidual (dx again where the types agree; undefined without residual), dweight.
std::vector<torch::Tensor> rms_norm_backward(OptTensor dy, OptTensor ds, torch::Tensor s, torch::Tensor weight,
                                             double eps, at::ScalarType x_type, bool has_residual, bool need_w) {
  const int64_t width = s.size(-1), rows = s.numel() / width;
  TORCH_CHECK(s.is_cuda(), "the stream must be a CUDA tensor (there is no CPU path)");
  const c10::cuda::CUDAGuard guard(s.device());
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  const bool split = has_residual && s.scalar_type() != x_type;
  auto dx = torch::empty(s.sizes(), s.options().dtype(x_type));
  torch::Tensor dres, dw;
  if (split) dres = torch::empty(s.sizes(), s.options());
  if (need_w) dw = torch::empty({width}, weight.options());
  if (rows == 0) {
    if (need_w) dw.zero_();
    return {dx, has_residual ? (split ? dres : dx) : torch::Tensor(), dw};
  }
  const torch::Tensor dyt = dy.has_value() ? dy->to(x_type) : torch::zeros(s.sizes(), s.options().dtype(x_type));
  TORCH_CHECK(dyt.sizes() == s.sizes(), "gradient must have the output's shape");
  const Rows yr = rows_of(dyt, rows, width), sr = rows_of(s, rows, width);
  Rows er{sr.t, 0};
  norm::Backward b;
  std::memset(&b, 0, sizeof(b));
  b.rows = rows, b.width = width;
  b.x_type = type_of(x_type), b.stream_type = type_of(s.scalar_type());
  b.dy = yr.p(), b.lddy = yr.ld;
  b.s = sr.p(), b.lds = sr.ld;
  if (ds.has_value()) {
    er = rows_of(ds->to(s.scalar_type()), rows, width);
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
    part = torch::empty({b.parts, width}, s.options().dtype(torch::kFloat32));
    b.partial = part.data_ptr<float>();
    b.dw = dw.data_ptr();
  }
  ck(norm::backward(b, sms, st), "rms_norm backward");
  return {dx, has_residual ? (split ? dres : dx) : torch::Tensor(), dw};
}

}  // namespace

void register_norm(pybind11::module& m) {
  m.def("rms_norm_forward", &rms_norm_forward);
  m.def("rms_norm_backward", &rms_norm_backward);
}

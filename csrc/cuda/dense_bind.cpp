// Torch bindings of the dense kernels (dense.h): argument checks, workspaces
// from torch's allocator, launches on the current stream of x's device.
#include "layer_bind.h"

#include <array>
#include <vector>

#include "dense.h"

namespace {
using namespace ngl::dense;
using namespace ngl::bind;

constexpr int64_t kMaxDim = (int64_t(1) << 31) - 1024;  // tile coordinates are 32-bit

// Operands that TMA can address: each as it is, or a copy with rows padded to
// whole 128 bytes (16 would do, but boxes that straddle lines load slower: 14 us
// against 10 for 1117 x 2312 x 776).  All copies of a product are one launch.
class Operands {
 public:
  Operands(std::vector<torch::Tensor>& keep, cudaStream_t s) : keep_(keep), s_(s) { copies_.n = 0; }
  Operand add(const Rows& r, int64_t rows, int64_t cols) {
    elem_ = (int)r.t.element_size();
    keep_.push_back(r.t);
    if (reinterpret_cast<uintptr_t>(r.p()) % 16 == 0 && (r.ld * elem_) % 16 == 0) return {r.p(), r.ld};
    const int64_t per = 128 / elem_, ldd = (cols + per - 1) / per * per;
    auto t = new_cuda({rows, ldd}, r.t.scalar_type(), r.t);
    copies_.m[copies_.n++] = {r.p(), r.ld, t.data_ptr(), ldd, rows, cols};
    keep_.push_back(t);
    return {t.data_ptr(), ldd};
  }
  void copy() {
    if (copies_.n > 0) ck(repack(copies_, elem_, s_), "repack");
    copies_.n = 0;
  }

 private:
  std::vector<torch::Tensor>& keep_;
  cudaStream_t s_;
  Copies copies_;
  int elem_ = 2;
};

// An earlier product gave up a wait: what follows would work on an incomplete output.
struct GaveUp : torch::PyTorchError {
  using PyTorchError::PyTorchError;
  PyObject* python_type() override {
    const pybind11::gil_scoped_acquire gil;
    return pybind11::module_::import("mini_nangila_b200.ops.dense").attr("DenseError").ptr();  // a class that stays
  }
};
int gave_up(int64_t device) {
  const volatile int* w = status_seen((int)device);
  return w == nullptr ? 0 : w[0];
}
void check_earlier(const torch::Tensor& x) {
  if (const int code = gave_up(x.get_device()))
    throw GaveUp("a dense product on cuda:" + text(x.get_device()) + " gave up a wait (status " + text(code) +
                 "): its output is incomplete; dense.check() clears the status");
}

void run_gemm(Gemm& g, const torch::Tensor& like, std::vector<torch::Tensor>& keep, cudaStream_t s) {
  const int sms = sm_count(like.get_device());
  plan(g, sms, true);
  g.partial = nullptr;
  if (const int64_t f = partial_floats(g)) {
    keep.push_back(new_cuda({f}, torch::kFloat32, like));
    g.partial = keep.back().data_ptr<float>();
  }
  ck(gemm(g, sms, s), "dense product");
}

struct Shape {
  int64_t m, k, n;
};
void check_weight(const torch::Tensor& x, const torch::Tensor& w, int64_t k, const char* what) {
  TORCH_CHECK(w.dim() == 2 && w.size(1) == k, what, " must be [out_features, ", text(k), "]; got ", text(w.sizes()));
  TORCH_CHECK(w.scalar_type() == x.scalar_type(), what, " must be ", x.scalar_type(), " like x; got ",
              w.scalar_type());
}
void check_scale(const OptTensor& s, bool fp8, int64_t n, const char* what) {
  TORCH_CHECK(fp8 == s.has_value(), what, fp8 ? " is needed with 8-bit operands" : " needs 8-bit operands");
  if (fp8)
    TORCH_CHECK(s->scalar_type() == torch::kFloat32 && s->numel() == n, what,
                " must be float32 with one value a row (", text(n), "); got ", text(s->sizes()));
}
// Checks shared by both forms; w2 undefined for the plain one.
Shape check_operands(const torch::Tensor& x, const torch::Tensor& w, const char* w_name, const torch::Tensor* w2) {
  TORCH_CHECK(x.dim() >= 1, "x needs at least one dimension");
  const auto t = x.scalar_type();
  TORCH_CHECK(t == at::kFloat8_e4m3fn || is_half(t), "x must be bfloat16, float16 or float8_e4m3fn; got ", t);
  Shape s;
  s.k = x.size(-1);
  TORCH_CHECK(s.k > 0, "x has no features (its last dimension is 0)");
  s.m = x.numel() / s.k;
  check_weight(x, w, s.k, w_name);
  s.n = w.size(0);
  if (w2 != nullptr) {
    check_weight(x, *w2, s.k, "w_up");
    TORCH_CHECK(w2->size(0) == s.n, "the two projections must have the same out_features; got ", text(s.n), " and ",
                text(w2->size(0)));
  }
  TORCH_CHECK(s.m <= kMaxDim && s.n <= kMaxDim && s.k <= kMaxDim, "a dimension exceeds ", text(kMaxDim));
  return s;
}

using Sizes = c10::SmallVector<int64_t, 6>;
Sizes out_shape(const torch::Tensor& x, int64_t n) {
  Sizes v(x.sizes().begin(), x.sizes().end());
  v.back() = n;
  return v;
}
bool has_shape(const torch::Tensor& t, const Sizes& v) { return t.sizes() == at::IntArrayRef(v); }

// Kept pre-activations of [m, n]: one buffer, the 16-bit plane first.
torch::Tensor kept_alloc(const Shape& sh, const torch::Tensor& like) {
  return new_cuda({sh.m * kept_ld(sh.n) * 3}, torch::kUInt8, like);
}
uint16_t* kept_hi(const torch::Tensor& t) { return static_cast<uint16_t*>(t.data_ptr()); }
uint8_t* kept_lo(const torch::Tensor& t, const Shape& sh) {
  return static_cast<uint8_t*>(t.data_ptr()) + 2 * sh.m * kept_ld(sh.n);
}

// The elements of t side by side.
const void* flat(const torch::Tensor& t, std::vector<torch::Tensor>& keep) {
  if (t.is_contiguous()) return t.data_ptr();
  keep.push_back(t.contiguous());
  return keep.back().data_ptr();
}

Epilogue empty_epilogue() {
  Epilogue e;
  std::memset(&e, 0, sizeof(e));
  return e;
}

// At most kSkinnyRows rows, whatever their alignment.
void run_skinny(const Shape& sh, const Rows& x, const Rows& w, const Rows* w2, const Epilogue& ep, cudaStream_t s) {
  Skinny g;
  std::memset(&g, 0, sizeof(g));
  g.m = sh.m, g.n = sh.n, g.k = sh.k;
  g.type = type_of(x.t.scalar_type());
  g.gated = w2 != nullptr;
  g.x = {x.p(), x.ld};
  g.w[0] = {w.p(), w.ld};
  if (w2 != nullptr) g.w[1] = {w2->p(), w2->ld};
  g.ep = ep;
  ck(skinny(g, sm_count(x.t.get_device()), s), "few-row product");
}

// y, and the kept pre-activations in *kept where it is not null.
torch::Tensor linear_forward(const torch::Tensor& x, const torch::Tensor& weight, const OptTensor& bias,
                             const OptTensor& residual, int act, const OptTensor& x_scale, const OptTensor& w_scale,
                             c10::optional<at::ScalarType> out_dtype, torch::Tensor* kept) {
  const Shape sh = check_operands(x, weight, "weight", nullptr);
  const bool fp8 = x.scalar_type() == at::kFloat8_e4m3fn;
  check_scale(x_scale, fp8, sh.m, "x_scale");
  check_scale(w_scale, fp8, sh.n, "w_scale");
  const Sizes shape = out_shape(x, sh.n);
  // 8-bit operands leave the 16-bit type open: out_dtype's, else the bias's, else the residual's, else bfloat16
  auto half = fp8 ? torch::kBFloat16 : x.scalar_type();
  if (fp8) {
    if (out_dtype.has_value() && is_half(*out_dtype))
      half = *out_dtype;
    else if (bias.has_value() && is_half(bias->scalar_type()))
      half = bias->scalar_type();
    else if (residual.has_value() && is_half(residual->scalar_type()))
      half = residual->scalar_type();
  }
  auto out_t = half;
  if (residual.has_value()) {
    out_t = residual->scalar_type();
    TORCH_CHECK(out_t == half || out_t == torch::kFloat32, "residual must be ", half, " or float32; got ", out_t);
    TORCH_CHECK(has_shape(*residual, shape), "residual must have the output's shape ", text(shape), "; got ",
                text(residual->sizes()));
  }
  if (out_dtype.has_value()) {
    TORCH_CHECK(*out_dtype == half || *out_dtype == torch::kFloat32, "out_dtype must be ", half, " or float32; got ",
                *out_dtype);
    TORCH_CHECK(!residual.has_value() || out_t == *out_dtype, "the output has the residual's type ", out_t,
                ", not out_dtype ", *out_dtype);
    out_t = *out_dtype;
  }
  if (bias.has_value()) {
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == sh.n, "bias must be [", text(sh.n), "]; got ",
                text(bias->sizes()));
    TORCH_CHECK(bias->scalar_type() == half, "bias must be ", half, "; got ", bias->scalar_type());
  }
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (there is no CPU path)");
  need_cuda(weight, x, "weight");
  if (bias.has_value()) need_cuda(*bias, x, "bias");
  if (residual.has_value()) need_cuda(*residual, x, "residual");
  if (fp8) {
    need_cuda(*x_scale, x, "x_scale");
    need_cuda(*w_scale, x, "w_scale");
  }
  check_earlier(x);
  const c10::cuda::CUDAGuard guard(x.device());
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  auto y = new_cuda(shape, out_t, x);
  if (kept != nullptr) *kept = kept_alloc(sh, x);
  if (y.numel() == 0) return y;

  std::vector<torch::Tensor> keep;
  const Rows xr = rows_of(x, sh.m, sh.k), wr = rows_of(weight, sh.n, sh.k);
  Epilogue ep = empty_epilogue();
  ep.act = act;
  ep.half_type = type_of(half);
  ep.out_type = type_of(out_t);
  ep.out[0] = y.data_ptr();
  ep.ldo = sh.n;
  ep.ldz = kept_ld(sh.n);
  if (kept != nullptr) {
    ep.z_hi[0] = kept_hi(*kept);
    ep.z_lo[0] = kept_lo(*kept, sh);
  }
  if (bias.has_value()) {
    ep.bias = flat(*bias, keep);
  }
  if (residual.has_value()) {
    const Rows rr = rows_of(*residual, sh.m, sh.n);
    if (!rr.t.is_same(*residual)) keep.push_back(rr.t);
    ep.residual = rr.p();
    ep.ldr = rr.ld;
  }
  if (fp8) {
    ep.row_scale = static_cast<const float*>(flat(*x_scale, keep));
    ep.col_scale[0] = static_cast<const float*>(flat(*w_scale, keep));
  }
  if (sh.m <= kSkinnyRows) {
    run_skinny(sh, xr, wr, nullptr, ep, s);
    return y;
  }
  Gemm g;
  std::memset(&g, 0, sizeof(g));
  g.m = sh.m, g.n = sh.n, g.k = sh.k;
  g.type = type_of(x.scalar_type());
  g.major_a = g.major_b = kMajorK;
  g.dual = kDualNone;
  Operands ops(keep, s);
  g.a[0] = ops.add(xr, sh.m, sh.k);
  g.b[0] = ops.add(wr, sh.n, sh.k);
  ops.copy();
  g.ep = ep;
  run_gemm(g, x, keep, s);
  return y;
}

// out [m, n] of like's type = A B^T with the given orders; plain epilogue.
void plain_product(Gemm& g, std::vector<torch::Tensor> outs, const torch::Tensor& like,
                   std::vector<torch::Tensor>& keep, cudaStream_t s) {
  g.type = type_of(like.scalar_type());
  g.ep = empty_epilogue();
  g.ep.half_type = g.ep.out_type = g.type;
  g.ep.ldo = g.n;
  for (size_t i = 0; i < outs.size(); ++i) g.ep.out[i] = outs[i].data_ptr();
  run_gemm(g, like, keep, s);
}

// dx, dw, db (undefined where not needed).
std::array<torch::Tensor, 3> linear_backward(const torch::Tensor& dy, const torch::Tensor& x,
                                             const torch::Tensor& weight, const torch::Tensor& z, int act, bool need_x,
                                             bool need_w, bool need_b) {
  const Shape sh = check_operands(x, weight, "weight", nullptr);
  TORCH_CHECK(is_half(x.scalar_type()), "no gradient through 8-bit operands");
  TORCH_CHECK(has_shape(dy, out_shape(x, sh.n)), "gradient must have the output's shape");
  TORCH_CHECK(dy.scalar_type() == x.scalar_type() || dy.scalar_type() == torch::kFloat32,
              "gradient must be ", x.scalar_type(), " or float32; got ", dy.scalar_type());
  TORCH_CHECK(act == kActNone || (z.defined() && z.numel() == 3 * sh.m * kept_ld(sh.n)), "the activation's gradient needs z");
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (there is no CPU path)");
  need_cuda(dy, x, "gradient");
  need_cuda(weight, x, "weight");
  check_earlier(x);
  const c10::cuda::CUDAGuard guard(x.device());
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  torch::Tensor dx, dw, db;
  if (sh.m == 0 || sh.n == 0) {
    if (need_x) dx = torch::zeros_like(x);
    if (need_w) dw = torch::zeros({sh.n, sh.k}, weight.options());
    if (need_b) db = torch::zeros({sh.n}, weight.options());
    return {dx, dw, db};
  }
  std::vector<torch::Tensor> keep;
  const int half = type_of(x.scalar_type());
  Rows dzr = rows_of(dy, sh.m, sh.n);
  const bool make_dz = act != kActNone || dy.scalar_type() != x.scalar_type();
  if (need_b || (make_dz && (need_x || need_w))) {
    torch::Tensor dz, part;
    const int64_t ldz = (sh.n + 63) / 64 * 64;  // rows that TMA can address, whatever n
    if (make_dz && (need_x || need_w)) dz = new_cuda({sh.m, ldz}, x.scalar_type(), x);
    const int parts = colsum_parts(sh.m, sh.n, sm_count(x.get_device()));
    if (need_b) {
      db = new_cuda({sh.n}, x.scalar_type(), x);
      part = new_cuda({parts, sh.n}, torch::kFloat32, x);
    }
    ck(act_backward(dzr.p(), type_of(dy.scalar_type()), dzr.ld, act != kActNone ? kept_hi(z) : nullptr,
                    act != kActNone ? kept_lo(z, sh) : nullptr, act, half, sh.m, sh.n, dz.defined() ? dz.data_ptr() : nullptr, ldz, need_b ? part.data_ptr<float>() : nullptr,
                    parts, need_b ? db.data_ptr() : nullptr, s),
       "activation gradient");
    keep.push_back(dzr.t);
    if (dz.defined()) dzr = {dz, ldz};
  }
  if (!need_x && !need_w) return {dx, dw, db};
  Operands ops(keep, s);
  const Operand dz = ops.add(dzr, sh.m, sh.n);
  Operand wo{}, xo{};
  if (need_x) wo = ops.add(rows_of(weight, sh.n, sh.k), sh.n, sh.k);
  if (need_w) xo = ops.add(rows_of(x, sh.m, sh.k), sh.m, sh.k);
  ops.copy();
  if (need_x) {
    dx = new_cuda(x.sizes(), x.scalar_type(), x);
    Gemm g;
    std::memset(&g, 0, sizeof(g));
    g.m = sh.m, g.n = sh.k, g.k = sh.n;
    g.major_a = kMajorK, g.major_b = kMajorMN;
    g.a[0] = dz;
    g.b[0] = wo;
    plain_product(g, {dx}, x, keep, s);
  }
  if (need_w) {
    dw = new_cuda({sh.n, sh.k}, x.scalar_type(), x);
    Gemm g;
    std::memset(&g, 0, sizeof(g));
    g.m = sh.n, g.n = sh.k, g.k = sh.m;
    g.major_a = g.major_b = kMajorMN;
    g.a[0] = dz;
    g.b[0] = xo;
    plain_product(g, {dw}, x, keep, s);
  }
  return {dx, dw, db};
}

// h, and the kept projections in kept[0] and kept[1] where it is not null.
torch::Tensor gated_forward(const torch::Tensor& x, const torch::Tensor& w_gate, const torch::Tensor& w_up, int act,
                            const OptTensor& x_scale, const OptTensor& gate_scale, const OptTensor& up_scale,
                            c10::optional<at::ScalarType> out_dtype, torch::Tensor* kept) {
  const Shape sh = check_operands(x, w_gate, "w_gate", &w_up);
  const bool fp8 = x.scalar_type() == at::kFloat8_e4m3fn;
  check_scale(x_scale, fp8, sh.m, "x_scale");
  check_scale(gate_scale, fp8, sh.n, "gate_scale");
  check_scale(up_scale, fp8, sh.n, "up_scale");
  auto half = fp8 ? torch::kBFloat16 : x.scalar_type();
  if (fp8 && out_dtype.has_value() && is_half(*out_dtype)) half = *out_dtype;
  auto out_t = half;
  if (out_dtype.has_value()) {
    TORCH_CHECK(*out_dtype == half || *out_dtype == torch::kFloat32, "out_dtype must be ", half, " or float32; got ",
                *out_dtype);
    out_t = *out_dtype;
  }
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (there is no CPU path)");
  need_cuda(w_gate, x, "w_gate");
  need_cuda(w_up, x, "w_up");
  if (fp8) {
    need_cuda(*x_scale, x, "x_scale");
    need_cuda(*gate_scale, x, "gate_scale");
    need_cuda(*up_scale, x, "up_scale");
  }
  check_earlier(x);
  const c10::cuda::CUDAGuard guard(x.device());
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  auto h = new_cuda(out_shape(x, sh.n), out_t, x);
  if (kept != nullptr) {
    kept[0] = kept_alloc(sh, x);
    kept[1] = kept_alloc(sh, x);
  }
  if (h.numel() == 0) return h;
  std::vector<torch::Tensor> keep;
  const Rows xr = rows_of(x, sh.m, sh.k), gr = rows_of(w_gate, sh.n, sh.k), ur = rows_of(w_up, sh.n, sh.k);
  Epilogue ep = empty_epilogue();
  ep.act = act;
  ep.half_type = type_of(half);
  ep.out_type = type_of(out_t);
  ep.out[0] = h.data_ptr();
  ep.ldo = sh.n;
  ep.ldz = kept_ld(sh.n);
  for (int i = 0; i < 2 && kept != nullptr; ++i) {
    ep.z_hi[i] = kept_hi(kept[i]);
    ep.z_lo[i] = kept_lo(kept[i], sh);
  }
  if (fp8) {
    ep.row_scale = static_cast<const float*>(flat(*x_scale, keep));
    ep.col_scale[0] = static_cast<const float*>(flat(*gate_scale, keep));
    ep.col_scale[1] = static_cast<const float*>(flat(*up_scale, keep));
  }
  if (sh.m <= kSkinnyRows) {
    run_skinny(sh, xr, gr, &ur, ep, s);
    return h;
  }
  Gemm g;
  std::memset(&g, 0, sizeof(g));
  g.m = sh.m, g.n = sh.n, g.k = sh.k;
  g.type = type_of(x.scalar_type());
  g.major_a = g.major_b = kMajorK;
  g.dual = kDualN;
  Operands ops(keep, s);
  g.a[0] = ops.add(xr, sh.m, sh.k);
  g.b[0] = ops.add(gr, sh.n, sh.k);
  g.b[1] = ops.add(ur, sh.n, sh.k);
  ops.copy();
  g.ep = ep;
  run_gemm(g, x, keep, s);
  return h;
}

// dx, dw_gate, dw_up (undefined where not needed).
std::array<torch::Tensor, 3> gated_gradients(const torch::Tensor& dh, const torch::Tensor& x,
                                             const torch::Tensor& w_gate, const torch::Tensor& w_up,
                                             const torch::Tensor& zg, const torch::Tensor& zu, int act, bool need_x,
                                             bool need_w) {
  const Shape sh = check_operands(x, w_gate, "w_gate", &w_up);
  TORCH_CHECK(is_half(x.scalar_type()), "no gradient through 8-bit operands");
  TORCH_CHECK(has_shape(dh, out_shape(x, sh.n)), "gradient must have the output's shape");
  TORCH_CHECK(dh.scalar_type() == x.scalar_type(), "gradient must be ", x.scalar_type(), "; got ", dh.scalar_type());
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (there is no CPU path)");
  need_cuda(dh, x, "gradient");
  check_earlier(x);
  const c10::cuda::CUDAGuard guard(x.device());
  cudaStream_t s = at::cuda::getCurrentCUDAStream();
  torch::Tensor dx, dwg, dwu;
  if (sh.m == 0 || sh.n == 0) {
    if (need_x) dx = torch::zeros_like(x);
    if (need_w) {
      dwg = torch::zeros({sh.n, sh.k}, w_gate.options());
      dwu = torch::zeros({sh.n, sh.k}, w_up.options());
    }
    return {dx, dwg, dwu};
  }
  std::vector<torch::Tensor> keep;
  const Rows dhr = rows_of(dh, sh.m, sh.n);
  const int64_t ldg = (sh.n + 63) / 64 * 64;
  auto dg = new_cuda({sh.m, ldg}, x.scalar_type(), x), du = new_cuda({sh.m, ldg}, x.scalar_type(), x);
  TORCH_CHECK(zg.numel() == 3 * sh.m * kept_ld(sh.n) && zu.numel() == 3 * sh.m * kept_ld(sh.n), "the gate's gradient needs g and u");
  const uint16_t* const hi[2] = {kept_hi(zg), kept_hi(zu)};
  const uint8_t* const lo[2] = {kept_lo(zg, sh), kept_lo(zu, sh)};
  ck(gated_backward(dhr.p(), dhr.ld, hi, lo, act, type_of(x.scalar_type()), sh.m, sh.n, dg.data_ptr(), du.data_ptr(), ldg,
                    sm_count(x.get_device()), s),
     "gate gradient");
  // dg and du in rows that TMA can address, whatever n
  Operands ops(keep, s);
  const Operand og{dg.data_ptr(), ldg}, ou{du.data_ptr(), ldg};
  Operand go{}, uo{}, xo{};
  if (need_x) {
    go = ops.add(rows_of(w_gate, sh.n, sh.k), sh.n, sh.k);
    uo = ops.add(rows_of(w_up, sh.n, sh.k), sh.n, sh.k);
  }
  if (need_w) xo = ops.add(rows_of(x, sh.m, sh.k), sh.m, sh.k);
  ops.copy();
  if (need_x) {
    dx = new_cuda(x.sizes(), x.scalar_type(), x);
    Gemm g;
    std::memset(&g, 0, sizeof(g));
    g.m = sh.m, g.n = sh.k, g.k = sh.n;
    g.major_a = kMajorK, g.major_b = kMajorMN;
    g.dual = kDualK;
    g.a[0] = og;
    g.a[1] = ou;
    g.b[0] = go;
    g.b[1] = uo;
    plain_product(g, {dx}, x, keep, s);
  }
  if (need_w) {
    dwg = new_cuda({sh.n, sh.k}, x.scalar_type(), x);
    dwu = new_cuda({sh.n, sh.k}, x.scalar_type(), x);
    Gemm g;
    std::memset(&g, 0, sizeof(g));
    g.m = sh.n, g.n = sh.k, g.k = sh.m;
    g.major_a = g.major_b = kMajorMN;
    g.dual = kDualM;
    g.a[0] = og;
    g.a[1] = ou;
    g.b[0] = xo;
    plain_product(g, {dwg, dwu}, x, keep, s);
  }
  return {dx, dwg, dwu};
}

// ---- gradients
namespace ag = torch::autograd;

class LinearFn : public ag::Function<LinearFn> {
 public:
  static torch::Tensor forward(ag::AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& w,
                               const OptTensor& bias, const OptTensor& residual, int64_t act) {
    torch::Tensor kept;
    auto y = linear_forward(x, w, bias, residual, (int)act, c10::nullopt, c10::nullopt, c10::nullopt,
                            act != kActNone ? &kept : nullptr);
    ctx->save_for_backward({x, w, kept});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    return y;
  }
  static ag::variable_list backward(ag::AutogradContext* ctx, ag::variable_list grads) {
    seen_by_all("the gradient of linear", grads[0]);
    const auto saved = ctx->get_saved_variables();
    const bool has_b = ctx->saved_data["bias"].toBool(), has_r = ctx->saved_data["residual"].toBool();
    // edges are those of the tensors given, in their order
    const bool nb = has_b && ctx->needs_input_grad(2), nr = has_r && ctx->needs_input_grad(has_b ? 3 : 2);
    auto g = linear_backward(grads[0], saved[0], saved[1], saved[2], (int)ctx->saved_data["act"].toInt(),
                             ctx->needs_input_grad(0), ctx->needs_input_grad(1), nb);
    return once({g[0], g[1], g[2], nr ? grads[0] : torch::Tensor(), torch::Tensor()}, "linear");
  }
};

class GatedFn : public ag::Function<GatedFn> {
 public:
  static torch::Tensor forward(ag::AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& w_gate,
                               const torch::Tensor& w_up, int64_t act) {
    torch::Tensor kept[2];
    auto h = gated_forward(x, w_gate, w_up, (int)act, c10::nullopt, c10::nullopt, c10::nullopt, c10::nullopt, kept);
    ctx->save_for_backward({x, w_gate, w_up, kept[0], kept[1]});
    ctx->saved_data["act"] = act;
    return h;
  }
  static ag::variable_list backward(ag::AutogradContext* ctx, ag::variable_list grads) {
    seen_by_all("the gradient of gated_linear", grads[0]);
    const auto s = ctx->get_saved_variables();
    const bool ng = ctx->needs_input_grad(1), nu = ctx->needs_input_grad(2);
    auto g = gated_gradients(grads[0], s[0], s[1], s[2], s[3], s[4], (int)ctx->saved_data["act"].toInt(),
                             ctx->needs_input_grad(0), ng || nu);
    return once({g[0], ng ? g[1] : torch::Tensor(), nu ? g[2] : torch::Tensor(), torch::Tensor()}, "gated_linear");
  }
};

// A tensor in autocast's type, as F.linear would make it (8-bit operands stay).
torch::Tensor cast(const torch::Tensor& t) {
  return t.scalar_type() == at::kFloat8_e4m3fn ? t
                                               : at::autocast::cached_cast(at::autocast::get_autocast_dtype(at::kCUDA), t);
}

int64_t check_act(int64_t act) {
  TORCH_CHECK(act >= kActNone && act <= kActSilu, "unknown activation");
  return act;
}

torch::Tensor linear(torch::Tensor x, torch::Tensor weight, OptTensor bias, int64_t act, OptTensor residual,
                     const OptTensor& x_scale, const OptTensor& w_scale, c10::optional<at::ScalarType> out_dtype) {
  seen_by_all("linear", x, weight, bias, residual, x_scale, w_scale);
  if (at::autocast::is_autocast_enabled(at::kCUDA)) {
    x = cast(x);
    weight = cast(weight);
    if (bias.has_value()) bias = cast(*bias);
    if (residual.has_value() && residual->scalar_type() != torch::kFloat32 && is_half(x.scalar_type()))
      residual = residual->to(x.scalar_type());
  }
  if (at::GradMode::is_enabled() &&
      (wants_grad(x) || wants_grad(weight) || wants_grad(bias) || wants_grad(residual))) {
    TORCH_CHECK_VALUE(!x_scale.has_value() && !w_scale.has_value() && x.scalar_type() != at::kFloat8_e4m3fn,
                      "linear: 8-bit operands have no gradient; call it under torch.no_grad()");
    TORCH_CHECK_VALUE(!out_dtype.has_value() ||
                          *out_dtype == (residual.has_value() ? residual->scalar_type() : x.scalar_type()),
                      "linear: out_dtype is fixed by x and residual where gradients are needed");
    return LinearFn::apply(x, weight, bias, residual, act);
  }
  return linear_forward(x, weight, bias, residual, (int)act, x_scale, w_scale, out_dtype, nullptr);
}

torch::Tensor gated_linear(torch::Tensor x, torch::Tensor w_gate, torch::Tensor w_up, int64_t act,
                           const OptTensor& x_scale, const OptTensor& gate_scale, const OptTensor& up_scale,
                           c10::optional<at::ScalarType> out_dtype) {
  seen_by_all("gated_linear", x, w_gate, w_up, x_scale, gate_scale, up_scale);
  if (at::autocast::is_autocast_enabled(at::kCUDA)) {
    x = cast(x);
    w_gate = cast(w_gate);
    w_up = cast(w_up);
  }
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w_gate) || wants_grad(w_up))) {
    TORCH_CHECK_VALUE(!x_scale.has_value() && x.scalar_type() != at::kFloat8_e4m3fn,
                      "gated_linear: 8-bit operands have no gradient; call it under torch.no_grad()");
    TORCH_CHECK_VALUE(!out_dtype.has_value() || *out_dtype == x.scalar_type(),
                      "gated_linear: out_dtype is x's type where gradients are needed");
    return GatedFn::apply(x, w_gate, w_up, act);
  }
  return gated_forward(x, w_gate, w_up, (int)act, x_scale, gate_scale, up_scale, out_dtype, nullptr);
}

// (CTAs of a tile, accumulator columns, splits of k) that a product of these
// sizes takes on `sms` SMs.
std::vector<int64_t> dense_plan(int64_t m, int64_t n, int64_t k, int64_t dual, bool fp8, int64_t sms) {
  TORCH_CHECK(m > 0 && n > 0 && k > 0 && sms > 1 && dual >= 0 && dual <= 3, "sizes must be positive, dual 0 to 3");
  Gemm g;
  std::memset(&g, 0, sizeof(g));
  g.m = m, g.n = n, g.k = k, g.dual = (int)dual, g.type = fp8 ? kE4M3 : kBF16;
  plan(g, (int)sms, true);
  return {g.cg, g.nb, g.splits};
}

// The words themselves, as a tensor on the CPU (tests write them).
torch::Tensor dense_status_words(int64_t device) {
  int* w = status_seen((int)device);
  TORCH_CHECK(w != nullptr, "no product has run on this device");
  return torch::from_blob(w, {4}, torch::kInt32);
}

void dense_force_plan(int64_t cg, int64_t nb, int64_t splits) {
  TORCH_CHECK(cg == 0 || ((cg == 1 || cg == 2) && (nb == 128 || nb == 256) && splits >= 1 && splits <= 64),
              "a plan has 1 or 2 CTAs, 128 or 256 columns, 1 to 64 splits");
  force_plan((int)cg, (int)nb, (int)splits);
}

std::vector<int64_t> dense_status(int64_t device, bool clear) {
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  int v[4] = {0, 0, 0, 0};
  ck(read_status(v, clear, at::cuda::getCurrentCUDAStream()), "dense status");
  return {v[0], v[1], v[2], v[3]};
}

// (x, weight, bias, activation, residual, x_scale, w_scale, out_dtype)
PyObject* py_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 8, "linear");
  return THPVariable_Wrap(linear(tensor_arg(a[0], "x"), tensor_arg(a[1], "weight"), opt_tensor_arg(a[2], "bias"),
                                 check_act(int_arg(a[3])), opt_tensor_arg(a[4], "residual"),
                                 opt_tensor_arg(a[5], "x_scale"), opt_tensor_arg(a[6], "w_scale"),
                                 opt_dtype_arg(a[7], "out_dtype")));
  END_HANDLE_TH_ERRORS
}
// (x, w_gate, w_up, activation, x_scale, gate_scale, up_scale, out_dtype)
PyObject* py_gated_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count_args(n, 8, "gated_linear");
  return THPVariable_Wrap(gated_linear(tensor_arg(a[0], "x"), tensor_arg(a[1], "w_gate"), tensor_arg(a[2], "w_up"),
                                       check_act(int_arg(a[3])), opt_tensor_arg(a[4], "x_scale"),
                                       opt_tensor_arg(a[5], "gate_scale"), opt_tensor_arg(a[6], "up_scale"),
                                       opt_dtype_arg(a[7], "out_dtype")));
  END_HANDLE_TH_ERRORS
}
PyMethodDef kMethods[] = {
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&py_linear)), METH_FASTCALL, nullptr},
    {"gated_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&py_gated_linear)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

void register_dense(pybind11::module& m) {
  if (PyModule_AddFunctions(m.ptr(), kMethods) != 0) throw pybind11::error_already_set();
  m.def("dense_plan", &dense_plan);
  m.def("dense_force_plan", &dense_force_plan);
  m.def("dense_status", &dense_status);
  m.def("dense_gave_up", &gave_up);
  m.def("dense_status_words", &dense_status_words);
}

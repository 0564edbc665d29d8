// Root-mean-square norm of rows with the residual's addition, its backward
// pass, and the output in e4m3 with one scale a row
// (csrc/cuda/norm_forward.cu, norm_backward.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ngl {
namespace norm {

constexpr int64_t kMaxWidth = 32768;  // elements of a row

// Types are those of dense.h.  s = round(x + residual) in stream_type (s = x
// where residual is null), y = s * rsqrt(mean(s^2) + eps) * w.
struct Forward {
  int64_t rows, width;
  int x_type, stream_type, w_type;
  const void* x;
  int64_t ldx;
  const void* residual;  // may be null
  int64_t ldr;
  const void* w;   // null: no norm, y = x (rows in 8 bits only)
  void* stream;    // [rows, width], written where residual is given
  void* y;         // [rows, width] of y_type, or e4m3 codes
  int y_type;      // x_type, or a 16-bit type where x is fp32
  float* scale;    // [rows]: the codes' scales; null: y of y_type
  float eps;
};
cudaError_t forward(const Forward& f, int sms, cudaStream_t st);

// dstream = ds + inv * (dy w - hat * mean(dy w hat)), written as dx (x_type)
// and as dres (stream_type, where given and of another type than x);
// dw = sum over rows of dy * hat, through partial [parts, width].
struct Backward {
  int64_t rows, width;
  int x_type, stream_type, w_type;
  const void* dy;  // x_type
  int64_t lddy;
  const void* ds;  // stream_type, may be null
  int64_t ldds;
  const void* s;   // stream_type
  int64_t lds;
  const void* w;
  void* dx;
  void* dres;      // may be null
  void* dw;        // w_type, may be null
  float* partial;
  int parts;
  float eps;
};
int backward_parts(int64_t rows, int64_t width, int sms);
cudaError_t backward(const Backward& b, cudaStream_t st);

}  // namespace norm
}  // namespace ngl

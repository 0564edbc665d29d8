// Root-mean-square norm of rows, forward and backward (norm.h).
//
// Bound by HBM bandwidth: a row is read once into registers (up to 32
// elements a thread, 16-byte runs), its sums go through shuffles, and where a
// row takes more than one warp through shared memory; everything else happens
// on the registers.  Sums and the norm are in fp32 whatever the types.  What
// is normalised is the stream as it is stored (x + residual rounded once to
// the stream's type), so the backward pass, which reads the stored stream,
// sees the same values.
#include "norm.h"

#include <algorithm>

#include "dense_math.cuh"
#include "ngl_cuda.cuh"

namespace ngl {
namespace norm {
namespace {

using namespace ngl::dev;
using namespace ngl::dense;

constexpr float kE4M3Max = 448.0f;
constexpr float kScaleMin = 1.17549435e-38f;  // 2^-126: a row of zeros keeps a finite inverse

template <int TPR>
constexpr int kCta = TPR < 128 ? 128 : TPR;

struct SumOp {
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct MaxOp {
  static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};
// Over the TPR threads of a row, N values at once; every thread gets them.
template <int TPR, int N, typename Op>
__device__ __forceinline__ void row_reduce(float (&v)[N], float* sm) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] = Op::of(v[i], __shfl_xor_sync(kFull, v[i], o));
  if (TPR > 32) {
    constexpr int kW = TPR / 32;
    const int warp = threadIdx.x >> 5;
    __syncthreads();  // the last reduction's readers are done
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) sm[warp * N + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float a = sm[i];
#pragma unroll
      for (int w = 1; w < kW; ++w) a = Op::of(a, sm[w * N + i]);
      v[i] = a;
    }
  }
}

// Four values to e4m3, saturating to +-448; a NaN stays one.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

template <int XT, int ST, int TPR, int VPT, bool kFp8>
__global__ void __launch_bounds__(kCta<TPR>, 1) k_forward(const __grid_constant__ Forward f) {
  constexpr int kRows = kCta<TPR> / TPR;
  __shared__ float sm[32];
  const int t = threadIdx.x % TPR;
  const bool vx = runs_aligned(f.x, f.ldx, type_bytes(XT)), vr = runs_aligned(f.residual, f.ldr, type_bytes(ST)),
             vs = runs_aligned(f.stream, f.width, type_bytes(ST)),
             vy = runs_aligned(f.y, f.width, kFp8 ? 1 : type_bytes(XT)) || (kFp8 && f.width % 8 == 0),
             vw = runs_aligned(f.w, 0, 4);
  const float inv_width = 1.0f / (float)f.width;
  // the loop runs the same number of times for all threads of a CTA
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < f.rows; r0 += (int64_t)gridDim.x * kRows) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool inside = row < f.rows;
    float v[VPT][8];
    float sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int64_t col = (int64_t)(i * TPR + t) * 8;
      const int valid = inside ? (int)max64(0, min64(8, f.width - col)) : 0;
      get_run<8>(f.x, row * f.ldx + col, XT, valid, vx, v[i]);
      if (f.residual != nullptr) {
        float r[8];
        get_run<8>(f.residual, row * f.ldr + col, ST, valid, vr, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[i][j] += r[j];
          if (ST != kF32) v[i][j] = half_to_float(float_to_half(v[i][j], ST), ST);
        }
        put_run<8>(f.stream, row * f.width + col, ST, valid, vs, v[i]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[0] += v[i][j] * v[i][j];
    }
    if (f.w != nullptr) {
      row_reduce<TPR, 1, SumOp>(sum, sm);
      const float inv = rsqrtf(sum[0] * inv_width + f.eps);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int64_t col = (int64_t)(i * TPR + t) * 8;
        float w[8];
        get_run<8>(f.w, col, f.w_type, (int)max64(0, min64(8, f.width - col)), vw, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * inv * w[j];
      }
    }
    float q = 1.0f;
    if (kFp8) {
      float top[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) top[0] = fmaxf(top[0], fabsf(v[i][j]));
      row_reduce<TPR, 1, MaxOp>(top, sm);
      const float scale = fmaxf(top[0] * (1.0f / kE4M3Max), kScaleMin);
      q = 1.0f / scale;
      if (inside && t == 0) f.scale[row] = scale;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int64_t col = (int64_t)(i * TPR + t) * 8;
      const int valid = inside ? (int)max64(0, min64(8, f.width - col)) : 0;
      if (kFp8) {
        const uint32_t lo = e4m3x4(v[i][0] * q, v[i][1] * q, v[i][2] * q, v[i][3] * q);
        const uint32_t hi = e4m3x4(v[i][4] * q, v[i][5] * q, v[i][6] * q, v[i][7] * q);
        uint8_t* p = static_cast<uint8_t*>(f.y) + row * f.width + col;
        if (valid == 8 && vy) {
          *reinterpret_cast<uint2*>(p) = make_uint2(lo, hi);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < valid) p[j] = (uint8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
        }
      } else {
        put_run<8>(f.y, row * f.width + col, XT, valid, vy, v[i]);
      }
    }
  }
}

template <int XT, int ST, int TPR, int VPT>
__global__ void __launch_bounds__(kCta<TPR>, 1) k_backward(const __grid_constant__ Backward b) {
  constexpr int kRows = kCta<TPR> / TPR;
  __shared__ float sm[64];
  const int t = threadIdx.x % TPR;
  const bool vdy = runs_aligned(b.dy, b.lddy, type_bytes(XT)), vds = runs_aligned(b.ds, b.ldds, type_bytes(ST)),
             vs = runs_aligned(b.s, b.lds, type_bytes(ST)), vx = runs_aligned(b.dx, b.width, type_bytes(XT)),
             vr = runs_aligned(b.dres, b.width, type_bytes(ST)), vw = runs_aligned(b.w, 0, 4);
  const float inv_width = 1.0f / (float)b.width;
  float dw[VPT][8] = {};
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < b.rows; r0 += (int64_t)gridDim.x * kRows) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool inside = row < b.rows;
    float s[VPT][8], g[VPT][8];
    float sum[2] = {0.0f, 0.0f};  // s^2, dy w s
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int64_t col = (int64_t)(i * TPR + t) * 8;
      const int valid = inside ? (int)max64(0, min64(8, b.width - col)) : 0;
      float w[8];
      get_run<8>(b.s, row * b.lds + col, ST, valid, vs, s[i]);
      get_run<8>(b.dy, row * b.lddy + col, XT, valid, vdy, g[i]);
      get_run<8>(b.w, col, b.w_type, (int)max64(0, min64(8, b.width - col)), vw, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum[0] += s[i][j] * s[i][j];
        sum[1] += g[i][j] * w[j] * s[i][j];
      }
    }
    row_reduce<TPR, 2, SumOp>(sum, sm);
    const float inv = rsqrtf(sum[0] * inv_width + b.eps);
    const float dot = sum[1] * inv * inv_width;  // mean(dy w hat)
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int64_t col = (int64_t)(i * TPR + t) * 8;
      const int valid = inside ? (int)max64(0, min64(8, b.width - col)) : 0;
      float w[8], e[8] = {};
      get_run<8>(b.w, col, b.w_type, (int)max64(0, min64(8, b.width - col)), vw, w);
      if (b.ds != nullptr) get_run<8>(b.ds, row * b.ldds + col, ST, valid, vds, e);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float hat = s[i][j] * inv;
        dw[i][j] += g[i][j] * hat;
        e[j] += inv * (g[i][j] * w[j] - hat * dot);
      }
      put_run<8>(b.dx, row * b.width + col, XT, valid, vx, e);
      if (b.dres != nullptr) put_run<8>(b.dres, row * b.width + col, ST, valid, vr, e);
    }
  }
  if (b.partial == nullptr) return;
  const int64_t part = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
  const bool vp = b.width % 4 == 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int64_t col = (int64_t)(i * TPR + t) * 8;
    put_run<8>(b.partial, part * b.width + col, kF32, (int)max64(0, min64(8, b.width - col)), vp, dw[i]);
  }
}

struct Split {
  int tpr, vpt;
};
// Threads and runs of a row: a warp a row while 32 elements a thread hold it,
// so that short rows need no block-wide reduction.
Split split_of(int64_t width) {
  const int64_t runs = (width + 7) / 8;
  if (runs <= 32) return {32, 1};
  if (runs <= 64) return {32, 2};
  if (runs <= 128) return {32, 4};
  if (runs <= 256) return {128, 2};
  if (runs <= 512) return {128, 4};
  if (runs <= 1024) return {256, 4};
  return {1024, 4};
}
int rows_per_cta(int tpr) { return tpr < 128 ? 128 / tpr : 1; }

template <int XT, int ST, int TPR, int VPT>
cudaError_t run_forward(const Forward& f, int sms, cudaStream_t st) {
  const int64_t ctas = (f.rows + rows_per_cta(TPR) - 1) / rows_per_cta(TPR);
  const int per_sm = 2048 / kCta<TPR>;
  const int grid = (int)std::min<int64_t>(ctas, (int64_t)sms * per_sm);
  if (f.scale != nullptr)
    k_forward<XT, ST, TPR, VPT, true><<<grid, kCta<TPR>, 0, st>>>(f);
  else
    k_forward<XT, ST, TPR, VPT, false><<<grid, kCta<TPR>, 0, st>>>(f);
  return cudaGetLastError();
}
template <int XT, int ST, int TPR, int VPT>
cudaError_t run_backward(const Backward& b, cudaStream_t st) {
  const int grid = b.parts / rows_per_cta(TPR);
  k_backward<XT, ST, TPR, VPT><<<grid, kCta<TPR>, 0, st>>>(b);
  return cudaGetLastError();
}

#define NGL_SPLITS(call)                                 \
  do {                                                   \
    const Split sp = split_of(p.width);                  \
    if (sp.tpr == 32 && sp.vpt == 1) return call(32, 1); \
    if (sp.tpr == 32 && sp.vpt == 2) return call(32, 2); \
    if (sp.tpr == 32) return call(32, 4);                \
    if (sp.tpr == 128 && sp.vpt == 2) return call(128, 2); \
    if (sp.tpr == 128) return call(128, 4);              \
    if (sp.tpr == 256) return call(256, 4);              \
    return call(1024, 4);                                \
  } while (0)

template <int XT, int ST>
cudaError_t forward_of(const Forward& p, int sms, cudaStream_t st) {
#define NGL_CALL(T, V) run_forward<XT, ST, T, V>(p, sms, st)
  NGL_SPLITS(NGL_CALL);
#undef NGL_CALL
}
template <int XT, int ST>
cudaError_t backward_of(const Backward& p, cudaStream_t st) {
#define NGL_CALL(T, V) run_backward<XT, ST, T, V>(p, st)
  NGL_SPLITS(NGL_CALL);
#undef NGL_CALL
}

}  // namespace

int backward_parts(int64_t rows, int64_t width, int sms) {
  const int per = rows_per_cta(split_of(width).tpr);
  const int64_t ctas = (rows + per - 1) / per;
  return (int)std::min<int64_t>(ctas, (int64_t)sms * 4) * per;
}

cudaError_t forward(const Forward& f, int sms, cudaStream_t st) {
  if (f.rows <= 0 || f.width <= 0 || f.width > kMaxWidth) return cudaErrorInvalidValue;
  if (f.x_type == kF32) return forward_of<kF32, kF32>(f, sms, st);
  if (f.x_type == kBF16)
    return f.stream_type == kF32 ? forward_of<kBF16, kF32>(f, sms, st) : forward_of<kBF16, kBF16>(f, sms, st);
  return f.stream_type == kF32 ? forward_of<kF16, kF32>(f, sms, st) : forward_of<kF16, kF16>(f, sms, st);
}

cudaError_t backward(const Backward& b, int sms, cudaStream_t st) {
  (void)sms;
  if (b.rows <= 0 || b.width <= 0 || b.width > kMaxWidth) return cudaErrorInvalidValue;
  cudaError_t e;
  if (b.x_type == kF32)
    e = backward_of<kF32, kF32>(b, st);
  else if (b.x_type == kBF16)
    e = b.stream_type == kF32 ? backward_of<kBF16, kF32>(b, st) : backward_of<kBF16, kBF16>(b, st);
  else
    e = b.stream_type == kF32 ? backward_of<kF16, kF32>(b, st) : backward_of<kF16, kF16>(b, st);
  if (e != cudaSuccess || b.dw == nullptr) return e;
  return colsum(b.partial, b.parts, b.width, b.dw, b.w_type, st);
}

}  // namespace norm
}  // namespace ngl

// Root-mean-square norm of rows, forward: with the residual's addition, and with
// an output of the rows' type or of e4m3 with one scale a row (norm.h;
// norm_common.cuh has the layout).
#include "norm_common.cuh"

namespace ngl {
namespace norm {
namespace {

constexpr float kE4M3Max = 448.0f;
constexpr float kScaleMin = 1.17549435e-38f;  // 2^-126: a row of zeros keeps a finite inverse

// Four values to e4m3, saturating to +-448; a NaN stays one.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Rows of more than 16384 elements spill whatever the bound; without the one CTA
// an SM said aloud, ptxas gave two of these kernels 32 registers a thread.
template <int XT, int ST, int TPR, int VPT, bool kFp8, int U>
__global__ void __launch_bounds__(kCta<TPR>, TPR == 512 && VPT == 8) k_forward(const __grid_constant__ Forward f) {
  pdl_begin();
  pdl_wait();
  constexpr int kRows = kCta<TPR> / TPR;
  __shared__ float sm[kRows][2 * (TPR / 32)];
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR, width = (int)f.width;
  const float inv_width = 1.0f / (float)width;
  const int64_t step = (int64_t)gridDim.x * kRows;
  int turn = 0;
  float w[VPT][8];
  Raw<XT> nx[VPT];
  Raw<ST> nr[VPT];
  constexpr int kStep = TPR * U;  // columns from one unit of a run to the next
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int col = run_col<TPR, U>(i, t), end = row < f.rows ? width : 0;
      nx[i].template load<U>(f.x, row * f.ldx, col, kStep, end);
      if (f.residual != nullptr) nr[i].template load<U>(f.residual, row * f.ldr, col, kStep, end);
    }
  };
  int64_t row = (int64_t)blockIdx.x * kRows + group;
  fetch(row);
#pragma unroll
  for (int i = 0; i < VPT; ++i) weight_run<U>(f.w, f.w_type, run_col<TPR, U>(i, t), kStep, width, w[i]);
  // the loop runs the same number of times for all threads of a CTA
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < f.rows; r0 += step, row += step) {
    const bool inside = row < f.rows;
    float v[VPT][8];
    float sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      nx[i].to(v[i]);
      if (f.residual != nullptr) {
        float r[8];
        nr[i].to(r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] += r[j];
        if (ST != kF32) {
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const uint32_t h = pack_half2(v[i][j], v[i][j + 1], ST);
            unpack_half2(h, ST, v[i][j], v[i][j + 1]);
          }
        }
        store_run<U>(f.stream, ST, row * f.width, run_col<TPR, U>(i, t), kStep, inside ? width : 0, v[i]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[0] += v[i][j] * v[i][j];
    }
    fetch(row + step);
    if (f.w != nullptr) {
      row_reduce<TPR, 1, SumOp>(sum, sm[group], turn, group);
      const float inv = rsqrtf(sum[0] * inv_width + f.eps);
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * inv * w[i][j];
    }
    float q = 1.0f;
    if (kFp8) {
      float top[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) top[0] = fmaxf(top[0], fabsf(v[i][j]));
      row_reduce<TPR, 1, MaxOp>(top, sm[group], turn, group);
      const float scale = fmaxf(top[0] * (1.0f / kE4M3Max), kScaleMin);
      q = 1.0f / scale;
      if (inside && t == 0) f.scale[row] = scale;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int col = run_col<TPR, U>(i, t), end = inside ? width : 0;
      if (kFp8) {
        const uint32_t b[2] = {e4m3x4(v[i][0] * q, v[i][1] * q, v[i][2] * q, v[i][3] * q),
                               e4m3x4(v[i][4] * q, v[i][5] * q, v[i][6] * q, v[i][7] * q)};
        uint8_t* p = static_cast<uint8_t*>(f.y) + row * f.width;
        if constexpr (U == 8) {
          if (col < end) *reinterpret_cast<uint2*>(p + col) = make_uint2(b[0], b[1]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; j += U) {
            const int c = col + (j / U) * kStep;
            const uint32_t code = b[j / 4] >> (8 * (j & 3));
            if (c >= end) continue;
            if (U == 2)
              *reinterpret_cast<uint16_t*>(p + c) = (uint16_t)code;
            else
              p[c] = (uint8_t)code;
          }
        }
      } else {
        store_run<U>(f.y, XT == kF32 ? f.y_type : XT, row * f.width, col, kStep, end, v[i]);
      }
    }
  }
}

template <int XT, int ST, int TPR, int VPT, bool kFp8, int U>
cudaError_t start(const Forward& f, int sms, cudaStream_t st) {
  constexpr int kRows = kCta<TPR> / TPR;
  auto* fn = &k_forward<XT, ST, TPR, VPT, kFp8, U>;
  static int fit = 0;  // CTAs of an SM, the same on every GPU this is built for
  if (fit == 0) {
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, fn, kCta<TPR>, 0);
    if (e != cudaSuccess) return e;
  }
  const int64_t ctas = (f.rows + kRows - 1) / kRows;
  return launch_dependent(fn, dim3((unsigned)std::min<int64_t>(ctas, (int64_t)sms * std::max(fit, 1))), dim3(kCta<TPR>),
                          0, 1, st, f);
}
template <int XT, int ST, int TPR, int VPT>
cudaError_t run_forward(const Forward& f, int sms, cudaStream_t st) {
  const int bytes = type_bytes(XT);
  const Side sides[] = {{f.x, f.ldx, bytes},
                        {f.residual, f.ldr, type_bytes(ST)},
                        {f.stream, f.width, type_bytes(ST)},
                        {f.y, f.width, f.scale != nullptr ? 1 : type_bytes(f.y_type)}};
  const int u = unit_of(f.width, sides);
  if (f.scale != nullptr)
    return u == 8   ? start<XT, ST, TPR, VPT, true, 8>(f, sms, st)
           : u == 2 ? start<XT, ST, TPR, VPT, true, 2>(f, sms, st)
                    : start<XT, ST, TPR, VPT, true, 1>(f, sms, st);
  return u == 8   ? start<XT, ST, TPR, VPT, false, 8>(f, sms, st)
         : u == 2 ? start<XT, ST, TPR, VPT, false, 2>(f, sms, st)
                  : start<XT, ST, TPR, VPT, false, 1>(f, sms, st);
}
template <int XT, int ST>
cudaError_t forward_of(const Forward& p, int sms, cudaStream_t st) {
#define NGL_CALL(T, V) run_forward<XT, ST, T, V>(p, sms, st)
  NGL_SPLITS(NGL_CALL);
#undef NGL_CALL
}

}  // namespace

cudaError_t forward(const Forward& f, int sms, cudaStream_t st) {
  if (f.rows <= 0 || f.width <= 0 || f.width > kMaxWidth) return cudaErrorInvalidValue;
  if (f.x_type == kF32) return forward_of<kF32, kF32>(f, sms, st);
  if (f.x_type == kBF16)
    return f.stream_type == kF32 ? forward_of<kBF16, kF32>(f, sms, st) : forward_of<kBF16, kBF16>(f, sms, st);
  return f.stream_type == kF32 ? forward_of<kF16, kF32>(f, sms, st) : forward_of<kF16, kF16>(f, sms, st);
}

}  // namespace norm
}  // namespace ngl

// Root-mean-square norm of rows, backward (norm.h; norm_common.cuh has the
// layout).  The norm's statistic is summed again from the stored stream, which is
// read anyway, so nothing but the stream is kept from the forward pass.  Each
// group of threads keeps the weight gradient of its own columns in registers
// over all its rows; groups, then CTAs, join in their order, so a call repeated
// gives the same bits.
#include "norm_common.cuh"

namespace ngl {
namespace norm {
namespace {

// Threads of a CTA: groups of TPR threads, a row each, that join their weight
// gradients at the end.
template <int TPR>
constexpr int kBackCta = TPR < 256 ? 256 : TPR;
// CTAs of an SM: 128 registers a thread.
constexpr int back_ctas(int tpr) { return tpr > 256 ? 1 : 2; }

template <int XT, int ST, int TPR, int VPT, int U>
__global__ void __launch_bounds__(kBackCta<TPR>, back_ctas(TPR)) k_backward(const __grid_constant__ Backward b) {
  pdl_begin();
  pdl_wait();
  constexpr int kGroups = kBackCta<TPR> / TPR;
  __shared__ float sm[kGroups][4 * (TPR / 32)];
  extern __shared__ float dw_sm[];  // [width], where kGroups > 1
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR, width = (int)b.width;
  const float inv_width = 1.0f / (float)width;
  const int64_t step = (int64_t)gridDim.x * kGroups;
  float dw[VPT][8] = {}, w[VPT][8];
  int turn = 0;
  Raw<ST> ns[VPT], ne[VPT];
  Raw<XT> ng[VPT];
  constexpr int kStep = TPR * U;  // columns from one unit of a run to the next
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int col = run_col<TPR, U>(i, t), end = row < b.rows ? width : 0;
      ns[i].template load<U>(b.s, row * b.lds, col, kStep, end);
      ng[i].template load<U>(b.dy, row * b.lddy, col, kStep, end);
      if (b.ds != nullptr) ne[i].template load<U>(b.ds, row * b.ldds, col, kStep, end);
    }
  };
  int64_t row = (int64_t)blockIdx.x * kGroups + group;
  fetch(row);
#pragma unroll
  for (int i = 0; i < VPT; ++i) weight_run<U>(b.w, b.w_type, run_col<TPR, U>(i, t), kStep, width, w[i]);
  for (; row < b.rows; row += step) {  // the same for all threads of a group
    Raw<ST> s_now[VPT], e_now[VPT];
    Raw<XT> g_now[VPT];
    float sum[2] = {0.0f, 0.0f};  // s^2, dy w s
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      s_now[i] = ns[i];
      g_now[i] = ng[i];
      e_now[i] = ne[i];
    }
    fetch(row + step);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float s[8], g[8];
      s_now[i].to(s);
      g_now[i].to(g);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum[0] += s[j] * s[j];
        sum[1] += g[j] * w[i][j] * s[j];
      }
    }
    row_reduce<TPR, 2, SumOp>(sum, sm[group], turn, group);
    const float inv = rsqrtf(sum[0] * inv_width + b.eps);
    const float dot = sum[1] * inv * inv_width;  // mean(dy w hat)
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int col = run_col<TPR, U>(i, t);
      float s[8], g[8], e[8] = {};
      s_now[i].to(s);
      g_now[i].to(g);
      if (b.ds != nullptr) e_now[i].to(e);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float hat = s[j] * inv;
        dw[i][j] += g[j] * hat;
        e[j] += inv * (g[j] * w[i][j] - hat * dot);
      }
      store_run<U>(b.dx, XT, row * b.width, col, kStep, width, e);
      if (b.dres != nullptr) store_run<U>(b.dres, ST, row * b.width, col, kStep, width, e);
    }
  }
  if (b.partial == nullptr) return;
  if (kGroups > 1) {
    for (int o = 0; o < kGroups; ++o) {
      if (o > 0) __syncthreads();
      if (group != o) continue;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = run_col<TPR, U>(i, t) + (j / U) * kStep + j % U;
          if (c < width) {
            if (o > 0) dw[i][j] += dw_sm[c];
            dw_sm[c] = dw[i][j];
          }
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += kBackCta<TPR>) b.partial[(int64_t)blockIdx.x * width + c] = dw_sm[c];
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = run_col<TPR, U>(i, t) + (j / U) * kStep + j % U;
        if (c < width) b.partial[(int64_t)blockIdx.x * width + c] = dw[i][j];
      }
  }
}

template <int XT, int ST, int TPR, int VPT>
cudaError_t run_backward(const Backward& b, cudaStream_t st) {
  const Side sides[] = {{b.dy, b.lddy, type_bytes(XT)},
                        {b.ds, b.ldds, type_bytes(ST)},
                        {b.s, b.lds, type_bytes(ST)},
                        {b.dx, b.width, type_bytes(XT)},
                        {b.dres, b.width, type_bytes(ST)}};
  const int u = unit_of(b.width, sides);
  auto* fn = u == 8   ? &k_backward<XT, ST, TPR, VPT, 8>
             : u == 2 ? &k_backward<XT, ST, TPR, VPT, 2>
                      : &k_backward<XT, ST, TPR, VPT, 1>;
  // at most 8 KB: several groups only up to rows of 2048 elements
  const int smem = b.partial != nullptr && kBackCta<TPR> / TPR > 1 ? (int)b.width * 4 : 0;
  return launch_dependent(fn, dim3((unsigned)b.parts), dim3(kBackCta<TPR>), smem, 1, st, b);
}
template <int XT, int ST>
cudaError_t backward_of(const Backward& p, cudaStream_t st) {
#define NGL_CALL(T, V) run_backward<XT, ST, T, V>(p, st)
  NGL_SPLITS(NGL_CALL);
#undef NGL_CALL
}

}  // namespace

int backward_parts(int64_t rows, int64_t width, int sms) {
  const int tpr = split_of(width).tpr, groups = tpr < 256 ? 256 / tpr : 1;
  return (int)std::min<int64_t>((rows + groups - 1) / groups, (int64_t)sms * back_ctas(tpr));
}

cudaError_t backward(const Backward& b, cudaStream_t st) {
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

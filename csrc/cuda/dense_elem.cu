// Elementwise parts of the dense backward passes, and repacking of operands
// whose rows TMA cannot address.  All are bound by HBM bandwidth: each input
// is read once and each output written once in 16-byte runs.
#include "dense.h"

#include <algorithm>

#include "dense_math.cuh"
#include "ngl_cuda.cuh"

namespace ngl {
namespace dense {
namespace {

using namespace ngl::dev;

constexpr int kColGroup = 8;     // columns of one thread
constexpr int kLanesX = 32;      // threads along the columns of a CTA
constexpr int kLanesY = 8;       // threads along the rows

// dz = dy act'(z), rounded once to the type that the products read; sums of
// its columns from the unrounded values.  CTA (bx, by): 256 columns, every
// gridDim.y-th group of 8 rows.
__global__ void __launch_bounds__(kLanesX* kLanesY) k_act_backward(const void* dy, int dy_type, int64_t ldy,
                                                                   const void* z, int act, int half_type, int64_t m,
                                                                   int64_t n, void* dz, float* partial) {
  const int64_t col = ((int64_t)blockIdx.x * kLanesX + threadIdx.x) * kColGroup;
  const int valid = (int)max64(0, min64(kColGroup, n - col));
  const bool vdy = runs_aligned(dy, ldy, type_bytes(dy_type)), vz = runs_aligned(z, n, 2), vo = runs_aligned(dz, n, 2);
  float sum[kColGroup] = {};
  if (valid > 0) {
#pragma unroll 2
    for (int64_t r = (int64_t)blockIdx.y * kLanesY + threadIdx.y; r < m; r += (int64_t)gridDim.y * kLanesY) {
      float d[kColGroup], t[kColGroup];
      get_run<kColGroup>(dy, r * ldy + col, dy_type, valid, vdy, d);
      if (z != nullptr) {
        get_run<kColGroup>(z, r * n + col, half_type, valid, vz, t);
#pragma unroll
        for (int j = 0; j < kColGroup; ++j) {
          float v, g;
          act_both(act, t[j], v, g);
          d[j] *= g;
        }
      }
      if (dz != nullptr) put_run<kColGroup>(dz, r * n + col, half_type, valid, vo, d);
#pragma unroll
      for (int j = 0; j < kColGroup; ++j) sum[j] += d[j];
    }
  }
  if (partial == nullptr) return;
  __shared__ float s[kLanesY][kLanesX * kColGroup + 1];
#pragma unroll
  for (int j = 0; j < kColGroup; ++j) s[threadIdx.y][threadIdx.x * kColGroup + j] = sum[j];
  __syncthreads();
  const int c = threadIdx.y * kLanesX + threadIdx.x;  // 256 threads, 256 columns
  const int64_t out = (int64_t)blockIdx.x * kLanesX * kColGroup + c;
  if (out < n) {
    float a = 0.0f;
#pragma unroll
    for (int y = 0; y < kLanesY; ++y) a += s[y][c];
    partial[(int64_t)blockIdx.y * n + out] = a;
  }
}

// Column sums of [parts, n]: 32 columns a CTA, 16 threads along the parts, joined in their order.
constexpr int kSumY = 16;
__global__ void __launch_bounds__(32 * kSumY) k_colsum(const float* partial, int parts, int64_t n, void* out, int type) {
  __shared__ float s[kSumY][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float a = 0.0f;
  if (c < n) {
#pragma unroll 8
    for (int p = threadIdx.y; p < parts; p += kSumY) a += partial[(int64_t)p * n + c];
  }
  s[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.y == 0 && c < n) {
    a = 0.0f;
#pragma unroll
    for (int y = 0; y < kSumY; ++y) a += s[y][threadIdx.x];
    put(out, c, a, type);
  }
}

__global__ void __launch_bounds__(256) k_gated_backward(const void* dh, int64_t ldh, const void* g, const void* u,
                                                        int act, int half_type, int64_t m, int64_t n, void* dg,
                                                        void* du) {
  const int64_t nc = (n + 7) / 8;
  const bool vh = runs_aligned(dh, ldh, 2),
             vs = runs_aligned(g, n, 2) && runs_aligned(u, n, 2) && runs_aligned(dg, n, 2) && runs_aligned(du, n, 2);
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < nc * m; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / nc, col = (i - row * nc) * 8;
    const int valid = (int)min64(8, n - col);
    float d[8], a[8], b[8];
    get_run<8>(dh, row * ldh + col, half_type, valid, vh, d);
    get_run<8>(g, row * n + col, half_type, valid, vs, a);
    get_run<8>(u, row * n + col, half_type, valid, vs, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float v, s;
      act_both(act, a[j], v, s);
      a[j] = d[j] * b[j] * s;
      b[j] = d[j] * v;
    }
    put_run<8>(dg, row * n + col, half_type, valid, vs, a);
    put_run<8>(du, row * n + col, half_type, valid, vs, b);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) k_repack(const T* src, int64_t lds, T* dst, int64_t ldd, int64_t rows,
                                                int64_t cols) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < rows * ldd;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / ldd, c = i - r * ldd;
    dst[i] = c < cols ? src[r * lds + c] : T(0);
  }
}

int blocks_for(int64_t items) { return (int)std::max<int64_t>(1, std::min<int64_t>((items + 255) / 256, 148 * 16)); }

}  // namespace

int colsum_parts(int64_t m, int64_t n, int sms) {
  const int64_t bx = (n + kLanesX * kColGroup - 1) / (kLanesX * kColGroup);
  const int64_t want = (int64_t)sms * 6 / std::max<int64_t>(bx, 1);
  return (int)std::max<int64_t>(1, std::min<int64_t>(want, (m + kLanesY - 1) / kLanesY));
}

cudaError_t colsum(const float* partial, int parts, int64_t n, void* out, int type, cudaStream_t s) {
  k_colsum<<<(unsigned)((n + 31) / 32), dim3(32, kSumY), 0, s>>>(partial, parts, n, out, type);
  return cudaGetLastError();
}

cudaError_t act_backward(const void* dy, int dy_type, int64_t ldy, const void* z, int act, int half_type, int64_t m,
                         int64_t n, void* dz, float* partial, int parts, void* db, cudaStream_t s) {
  if (m <= 0 || n <= 0) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)((n + kLanesX * kColGroup - 1) / (kLanesX * kColGroup)), (unsigned)parts);
  k_act_backward<<<grid, dim3(kLanesX, kLanesY), 0, s>>>(dy, dy_type, ldy, z, act, half_type, m, n, dz,
                                                         db != nullptr ? partial : nullptr);
  const cudaError_t e = cudaGetLastError();
  return e != cudaSuccess || db == nullptr ? e : colsum(partial, parts, n, db, half_type, s);
}

cudaError_t gated_backward(const void* dh, int64_t ldh, const void* g, const void* u, int act, int half_type,
                           int64_t m, int64_t n, void* dg, void* du, cudaStream_t s) {
  if (m <= 0 || n <= 0) return cudaErrorInvalidValue;
  k_gated_backward<<<blocks_for(m * ((n + 7) / 8)), 256, 0, s>>>(dh, ldh, g, u, act, half_type, m, n, dg, du);
  return cudaGetLastError();
}

cudaError_t repack(const void* src, int64_t lds, void* dst, int64_t ldd, int64_t rows, int64_t cols, int elem,
                   cudaStream_t s) {
  if (rows <= 0 || cols <= 0) return cudaErrorInvalidValue;
  const int grid = blocks_for(rows * ldd);
  if (elem == 1)
    k_repack<uint8_t><<<grid, 256, 0, s>>>(static_cast<const uint8_t*>(src), lds, static_cast<uint8_t*>(dst), ldd,
                                           rows, cols);
  else
    k_repack<uint16_t><<<grid, 256, 0, s>>>(static_cast<const uint16_t*>(src), lds, static_cast<uint16_t*>(dst), ldd,
                                            rows, cols);
  return cudaGetLastError();
}

}  // namespace dense
}  // namespace ngl

// Elementwise parts of the dense backward passes, and repacking of operands
// whose rows TMA cannot address.  Each input is read once and each output
// written once in 16-byte runs.  The gate's gradient is bound by HBM bandwidth:
// 8192 x 5632 takes 94 us for its 553 MB (5.9 TB/s, 90 % of the copy rate).  An
// activation's with its column sums is not: 8192 x 2048 takes 28 us for 117 MB
// (4.1 TB/s) with 65 % of the issue slots and 40 % of DRAM busy, one wave of five
// CTAs an SM, whose warps wait for their loads about half of the time.  Two rows
// of a thread loaded before either is computed took 56 us (94 of the gate's 144):
// 110 to 128 registers a thread for 48.
#include "dense.h"

#include <algorithm>

#include "dense_math.cuh"
#include "layer_launch.cuh"
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
template <int kAct>
__global__ void __launch_bounds__(kLanesX* kLanesY) k_act_backward(const void* dy, int dy_type, int64_t ldy,
                                                                   const uint16_t* z_hi, const uint8_t* z_lo,
                                                                   int half_type, int64_t m, int64_t n, void* dz,
                                                                   int64_t ldd, float* partial) {
  pdl_begin();
  pdl_wait();
  const int64_t col = ((int64_t)blockIdx.x * kLanesX + threadIdx.x) * kColGroup;
  const int valid = (int)max64(0, min64(kColGroup, n - col));
  const bool vdy = runs_aligned(dy, ldy, type_bytes(dy_type)), vo = runs_aligned(dz, ldd, 2);
  const int64_t ldz = (n + 15) / 16 * 16;
  float sum[kColGroup] = {};
  if (valid > 0) {
#pragma unroll 2
    for (int64_t r = (int64_t)blockIdx.y * kLanesY + threadIdx.y; r < m; r += (int64_t)gridDim.y * kLanesY) {
      float d[kColGroup], t[kColGroup];
      get_run<kColGroup>(dy, r * ldy + col, dy_type, valid, vdy, d);
      if (kAct != kActNone) {
        get_kept8(z_hi, z_lo, r * ldz + col, t);
#pragma unroll
        for (int j = 0; j < kColGroup; ++j) {
          float v, g;
          act_both<kAct>(t[j], v, g);
          d[j] *= g;
        }
      }
      if (dz != nullptr) put_run<kColGroup>(dz, r * ldd + col, half_type, valid, vo, d);
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

// Column sums of [parts, n]: 32 columns a CTA, 32 threads along the parts, joined in their order.
constexpr int kSumY = 32;
__global__ void __launch_bounds__(32 * kSumY) k_colsum(const float* partial, int parts, int64_t n, void* out, int type) {
  pdl_begin();
  pdl_wait();
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

template <int kAct>
__global__ void __launch_bounds__(kLanesX* kLanesY) k_gated_backward(const void* dh, int64_t ldh, const uint16_t* g_hi,
                                                                     const uint8_t* g_lo, const uint16_t* u_hi,
                                                                     const uint8_t* u_lo, int half_type, int64_t m,
                                                                     int64_t n, void* dg, void* du, int64_t ldd) {
  pdl_begin();
  pdl_wait();
  const int64_t col = ((int64_t)blockIdx.x * kLanesX + threadIdx.x) * kColGroup;
  const int valid = (int)max64(0, min64(kColGroup, n - col));
  if (valid <= 0) return;
  const bool vh = runs_aligned(dh, ldh, 2), vs = runs_aligned(dg, ldd, 2) && runs_aligned(du, ldd, 2);
  const int64_t ldz = (n + 15) / 16 * 16;
#pragma unroll 2
  for (int64_t r = (int64_t)blockIdx.y * kLanesY + threadIdx.y; r < m; r += (int64_t)gridDim.y * kLanesY) {
    float d[kColGroup], a[kColGroup], b[kColGroup];
    get_run<kColGroup>(dh, r * ldh + col, half_type, valid, vh, d);
    get_kept8(g_hi, g_lo, r * ldz + col, a);
    get_kept8(u_hi, u_lo, r * ldz + col, b);
#pragma unroll
    for (int j = 0; j < kColGroup; ++j) {
      float v, s;
      act_both<kAct>(a[j], v, s);
      a[j] = d[j] * b[j] * s;
      b[j] = d[j] * v;
    }
    put_run<kColGroup>(dg, r * ldd + col, half_type, valid, vs, a);
    put_run<kColGroup>(du, r * ldd + col, half_type, valid, vs, b);
  }
}

// CTA (bx, by, bz): 8 elements a thread of the rows by, by + gridDim.y, ... of
// matrix bz.  The sources come here because their rows are not 16-byte aligned,
// so loads are single elements (adjacent threads share the sectors through L1);
// stores are 8 elements wide.
template <typename T>
__global__ void __launch_bounds__(256) k_repack(const __grid_constant__ Copies all) {
  pdl_begin();
  pdl_wait();
  const Copy& m = all.m[blockIdx.z];
  const T* src = static_cast<const T*>(m.src);
  T* dst = static_cast<T*>(m.dst);
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (c >= m.ldd) return;  // ldd is a multiple of 8
  for (int64_t r = blockIdx.y; r < m.rows; r += gridDim.y) {
    alignas(16) T v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < m.cols ? src[r * m.lds + c + j] : T(0);
    if (sizeof(T) == 2)
      *reinterpret_cast<uint4*>(dst + r * m.ldd + c) = *reinterpret_cast<const uint4*>(v);
    else
      *reinterpret_cast<uint2*>(dst + r * m.ldd + c) = *reinterpret_cast<const uint2*>(v);
  }
}

// Rows of the grid for the 256-column kernels, for about per_sm CTAs an SM.
int row_ctas(int64_t m, int64_t n, int sms, int per_sm) {
  const int64_t bx = (n + kLanesX * kColGroup - 1) / (kLanesX * kColGroup);
  const int64_t want = (int64_t)sms * per_sm / std::max<int64_t>(bx, 1);
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, 65535), (m + kLanesY - 1) / kLanesY));
}

#define NGL_BY_ACT(call)              \
  switch (act) {                      \
    case kActRelu: call(kActRelu); break;         \
    case kActGelu: call(kActGelu); break;         \
    case kActGeluTanh: call(kActGeluTanh); break; \
    case kActSilu: call(kActSilu); break;         \
    default: call(kActNone); break;               \
  }

}  // namespace

int colsum_parts(int64_t m, int64_t n, int sms) {
  return row_ctas(m, n, sms, 5);  // those that fit at once: each writes a row of partial sums
}

cudaError_t colsum(const float* partial, int parts, int64_t n, void* out, int type, cudaStream_t s) {
  return launch_dependent(&k_colsum, dim3((unsigned)((n + 31) / 32)), dim3(32, kSumY), 0, 1, s, partial, parts, n, out,
                          type);
}

cudaError_t act_backward(const void* dy, int dy_type, int64_t ldy, const uint16_t* z_hi, const uint8_t* z_lo, int act,
                         int half_type, int64_t m, int64_t n, void* dz, int64_t ldd, float* partial, int parts, void* db,
                         cudaStream_t s) {
  if (m <= 0 || n <= 0) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)((n + kLanesX * kColGroup - 1) / (kLanesX * kColGroup)), (unsigned)parts);
#define NGL_CALL(a)                                                                                          \
  e = launch_dependent(&k_act_backward<a>, grid, dim3(kLanesX, kLanesY), 0, 1, s, dy, dy_type, ldy, z_hi, z_lo, \
                       half_type, m, n, dz, ldd, db != nullptr ? partial : nullptr)
  cudaError_t e = cudaSuccess;
  NGL_BY_ACT(NGL_CALL)
#undef NGL_CALL
  return e != cudaSuccess || db == nullptr ? e : colsum(partial, parts, n, db, half_type, s);
}

cudaError_t gated_backward(const void* dh, int64_t ldh, const uint16_t* const z_hi[2], const uint8_t* const z_lo[2],
                           int act, int half_type, int64_t m, int64_t n, void* dg, void* du, int64_t ldd, int sms,
                           cudaStream_t s) {
  if (m <= 0 || n <= 0) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)((n + kLanesX * kColGroup - 1) / (kLanesX * kColGroup)), (unsigned)row_ctas(m, n, sms, 8));
#define NGL_CALL(a)                                                                                             \
  e = launch_dependent(&k_gated_backward<a>, grid, dim3(kLanesX, kLanesY), 0, 1, s, dh, ldh, z_hi[0], z_lo[0], \
                       z_hi[1], z_lo[1], half_type, m, n, dg, du, ldd)
  cudaError_t e = cudaSuccess;
  NGL_BY_ACT(NGL_CALL)
#undef NGL_CALL
  return e;
}

cudaError_t repack(const Copies& c, int elem, cudaStream_t s) {
  if (c.n <= 0 || c.n > 4) return cudaErrorInvalidValue;
  int64_t wide = 0, rows = 0;
  for (int i = 0; i < c.n; ++i) {
    if (c.m[i].rows <= 0 || c.m[i].cols <= 0) return cudaErrorInvalidValue;
    wide = std::max(wide, c.m[i].ldd);
    rows = std::max(rows, c.m[i].rows);
  }
  const dim3 grid((unsigned)((wide + 2047) / 2048), (unsigned)std::min<int64_t>(rows, 65535), (unsigned)c.n);
  return elem == 1 ? launch_dependent(&k_repack<uint8_t>, grid, dim3(256), 0, 1, s, c)
                   : launch_dependent(&k_repack<uint16_t>, grid, dim3(256), 0, 1, s, c);
}

}  // namespace dense
}  // namespace ngl

// Parts shared by the norm's forward and backward kernels (norm.h).
//
// Bound by HBM bandwidth: a row is read once into registers (16-byte runs, 16
// elements a thread up to rows of 8192), its sums go through shuffles, and
// where a row takes more than one warp through shared memory; everything else
// happens on the registers.  The next row's runs are loaded before this row's
// sums are joined, so that loads are in flight all the time.  Sums and the norm
// are in fp32 whatever the types.  What is normalised is the stream as it is
// stored (x + residual rounded once to the stream's type), so the backward
// pass, which reads the stored stream, sees the same values.
// 8192 x 2048 bf16 with a residual: forward 20.7 us (6.5 TB/s, the copy rate),
// in 8 bits 20.0 us, backward 29 us and 4 us for the weight's column sums.
#pragma once
#include "norm.h"

#include <algorithm>

#include "dense_math.cuh"
#include "layer_launch.cuh"
#include "ngl_cuda.cuh"

namespace ngl {
namespace norm {

using namespace ngl::dev;
using namespace ngl::dense;

// Threads of a forward CTA (several rows where a row takes one warp).
template <int TPR>
constexpr int kCta = TPR < 128 ? 128 : TPR;
struct SumOp {
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct MaxOp {
  static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};
// Barrier of the TPR threads of a row's group.
template <int TPR>
__device__ __forceinline__ void group_sync(int group) {
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(TPR) : "memory");
}
// Over the TPR threads of a row, N values at once; every thread gets them in
// the same order of operations.  sm: 2 * N * (TPR / 32) floats of this group;
// `turn` alternates, so that one barrier is enough (the readers of a turn are
// past it before the turn after next writes).
template <int TPR, int N, typename Op>
__device__ __forceinline__ void row_reduce(float (&v)[N], float* sm, int& turn, int group) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] = Op::of(v[i], __shfl_xor_sync(kFull, v[i], o));
  if (TPR > 32) {
    constexpr int kW = TPR / 32;
    float* buf = sm + turn * N * kW;
    turn ^= 1;
    const int warp = (threadIdx.x % TPR) >> 5;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) buf[warp * N + i] = v[i];
    group_sync<TPR>(group);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float a = buf[i];
#pragma unroll
      for (int w = 1; w < kW; ++w) a = Op::of(a, buf[w * N + i]);
      v[i] = a;
    }
  }
}

// A run of 8 elements as it lies in memory.
template <int T>
struct Raw {
  uint4 q[T == kF32 ? 2 : 1];
  // The elements of a run lie in units of U adjacent ones: 8 (16 bytes and
  // more at a time), 2 or 1 where rows are not aligned for more.  c0 is the run's
  // first column, d the distance from one unit to the next; elements from `end`
  // on are 0.
  template <int U>
  __device__ __forceinline__ void load(const void* p, int64_t row, int c0, int d, int end) {
    if constexpr (U == 8) {
      const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + (row + c0) * (T == kF32 ? 4 : 2));
      q[0] = c0 < end ? s[0] : make_uint4(0, 0, 0, 0);
      if constexpr (T == kF32) q[1] = c0 < end ? s[1] : make_uint4(0, 0, 0, 0);
    } else {
      uint32_t w[8] = {};
#pragma unroll
      for (int j = 0; j < 8; j += U) {
        const int c = c0 + (j / U) * d;
        if (c < end) {
          if constexpr (T == kF32) {
            if constexpr (U == 2) {
              const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const float*>(p) + row + c);
              w[j] = u.x;
              w[j + 1] = u.y;
            } else {
              w[j] = static_cast<const uint32_t*>(p)[row + c];
            }
          } else if constexpr (U == 2) {
            w[j / 2] = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p) + row + c);
          } else {
            w[j / 2] |= (uint32_t)static_cast<const uint16_t*>(p)[row + c] << (16 * (j & 1));
          }
        }
      }
      q[0] = make_uint4(w[0], w[1], w[2], w[3]);
      if constexpr (T == kF32) q[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
  __device__ __forceinline__ void to(float (&v)[8]) const {
    if constexpr (T == kF32) {
      v[0] = __uint_as_float(q[0].x); v[1] = __uint_as_float(q[0].y);
      v[2] = __uint_as_float(q[0].z); v[3] = __uint_as_float(q[0].w);
      v[4] = __uint_as_float(q[1].x); v[5] = __uint_as_float(q[1].y);
      v[6] = __uint_as_float(q[1].z); v[7] = __uint_as_float(q[1].w);
    } else {
      unpack_half2(q[0].x, T, v[0], v[1]);
      unpack_half2(q[0].y, T, v[2], v[3]);
      unpack_half2(q[0].z, T, v[4], v[5]);
      unpack_half2(q[0].w, T, v[6], v[7]);
    }
  }
};

template <int U>
__device__ __forceinline__ void store_run(void* p, int type, int64_t row, int c0, int d, int end,
                                          const float (&v)[8]) {
  if constexpr (U == 8) {
    if (c0 < end) put_run<8>(p, row + c0, type, 8, true, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j += U) {
      const int c = c0 + (j / U) * d;
      if (c >= end) continue;
      if (U == 2 && type == kF32)
        *reinterpret_cast<float2*>(static_cast<float*>(p) + row + c) = make_float2(v[j], v[j + 1]);
      else if (U == 2)
        *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p) + row + c) = pack_half2(v[j], v[j + 1], type);
      else
        put(p, row + c, v[j], type);
    }
  }
}
// Columns of thread t's run i: the first, and the distance of its units.
template <int TPR, int U>
__device__ __forceinline__ int run_col(int i, int t) {
  return (i * (8 / U) * TPR + t) * U;
}

// The weight's run in fp32: the same for every row, so read once a thread.
template <int U>
__device__ __forceinline__ void weight_run(const void* w, int type, int c0, int d, int width, float (&v)[8]) {
  if (w == nullptr) return;
  if constexpr (U == 8) {
    get_run<8>(w, c0, type, max(0, min(8, width - c0)), runs_aligned(w, 0, 4), v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = c0 + (j / U) * d + j % U;
      v[j] = c < width ? get(w, c, type) : 0.0f;
    }
  }
}

// Units of a row's elements: 8, 2 or 1 (see Raw::load), from what all matrices allow.
struct Side {
  const void* p;
  int64_t ld;
  int bytes;
};
template <int N>
int unit_of(int64_t width, const Side (&m)[N]) {
  int u = width % 8 == 0 ? 8 : width % 2 == 0 ? 2 : 1;
  for (const Side& s : m) {
    if (s.p == nullptr) continue;
    const uintptr_t a = reinterpret_cast<uintptr_t>(s.p) | (uintptr_t)(s.ld * s.bytes);
    if (u == 8 && a % (s.bytes == 1 ? 8 : 16) != 0) u = 2;
    if (u == 2 && a % (2 * s.bytes) != 0) u = 1;
  }
  return u;
}

struct Split {
  int tpr, vpt;
};
// Threads and runs of a row: two runs a thread as long as there are threads, so
// that this row, the next and the weight's gradient stay in registers.
inline Split split_of(int64_t width) {
  const int64_t runs = (width + 7) / 8;
  if (runs <= 32) return {32, 1};
  if (runs <= 64) return {32, 2};
  if (runs <= 128) return {64, 2};
  if (runs <= 256) return {128, 2};
  if (runs <= 512) return {256, 2};
  if (runs <= 1024) return {512, 2};
  if (runs <= 2048) return {512, 4};
  return {512, 8};
}

#define NGL_SPLITS(call)                                   \
  do {                                                     \
    const Split sp = split_of(p.width);                    \
    if (sp.tpr == 32 && sp.vpt == 1) return call(32, 1);   \
    if (sp.tpr == 32) return call(32, 2);                  \
    if (sp.tpr == 64) return call(64, 2);                  \
    if (sp.tpr == 128) return call(128, 2);                \
    if (sp.tpr == 256) return call(256, 2);                \
    if (sp.vpt == 2) return call(512, 2);                  \
    if (sp.vpt == 4) return call(512, 4);                  \
    return call(512, 8);                                   \
  } while (0)

}  // namespace norm
}  // namespace ngl

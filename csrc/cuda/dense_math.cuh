// Arithmetic shared by the dense kernels: activations and their derivatives in
// fp32, conversions, and the epilogue over a run of consecutive columns.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dense.h"
#include "ngl_cuda.cuh"

namespace ngl {
namespace dense {

// 1 / (1 + exp(-z)) from the hardware's base-2 exponential and reciprocal: a few
// ulp of fp32, two orders below the rounding of a 16-bit result.  An overflowing
// exponential gives 0.
__device__ __forceinline__ float logistic(float z) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}

constexpr float kGeluA = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluC = 0.044715f;

template <int kAct>
__device__ __forceinline__ float act_value(float z) {
  if (kAct == kActRelu) return z < 0.0f ? 0.0f : z;  // a NaN stays one
  if (kAct == kActGelu) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  // 0.5 (1 + tanh(u)) is the logistic function of 2 u
  if (kAct == kActGeluTanh) return z * logistic(2.0f * kGeluA * (z + kGeluC * z * z * z));
  if (kAct == kActSilu) return z * logistic(z);
  return z;
}

// Value and derivative together.  Beyond |z| = 100 the logistic function is 0 or
// 1 in fp32, and with it each derivative; the clamp keeps 0 * inf out and changes
// no value.  A NaN passes.
template <int kAct>
__device__ __forceinline__ void act_both(float z, float& v, float& d) {
  const float c = z != z ? z : fminf(fmaxf(z, -100.0f), 100.0f);
  if (kAct == kActRelu) {
    v = z < 0.0f ? 0.0f : z;
    d = z != z ? z : (z > 0.0f ? 1.0f : 0.0f);
  } else if (kAct == kActGelu) {
    const float phi = 0.5f * (1.0f + erff(c * 0.70710678118654752f));
    v = z * phi;
    d = phi + c * 0.3989422804014327f * __expf(-0.5f * c * c);
  } else if (kAct == kActGeluTanh) {
    const float s = logistic(2.0f * kGeluA * (c + kGeluC * c * c * c));
    v = z * s;
    d = s + c * s * (1.0f - s) * (2.0f * kGeluA) * (1.0f + 3.0f * kGeluC * c * c);
  } else if (kAct == kActSilu) {
    const float s = logistic(c);
    v = z * s;
    d = s + c * s * (1.0f - s);
  } else {
    v = z;
    d = 1.0f;
  }
}

// One branch for a run of values, not one a value.
template <int C>
__device__ __forceinline__ void act_run(int act, float (&v)[C]) {
#define NGL_ACT(a)                                       \
  case a:                                                \
    _Pragma("unroll") for (int j = 0; j < C; ++j) v[j] = act_value<a>(v[j]); \
    break
  switch (act) {
    NGL_ACT(kActRelu);
    NGL_ACT(kActGelu);
    NGL_ACT(kActGeluTanh);
    NGL_ACT(kActSilu);
    default:
      break;
  }
#undef NGL_ACT
}

__device__ __forceinline__ float half_to_float(uint16_t h, int type) {
  return type == kBF16 ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
}
__device__ __forceinline__ uint16_t float_to_half(float v, int type) {
  return type == kBF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi, int type) {
  uint32_t r;
  if (type == kBF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void unpack_half2(uint32_t w, int type, float& lo, float& hi) {
  if (type == kBF16) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
  }
}

// One element at index i of an array of `type` (kF32, kBF16 or kF16).
__device__ __forceinline__ float get(const void* p, int64_t i, int type) {
  return type == kF32 ? static_cast<const float*>(p)[i] : half_to_float(static_cast<const uint16_t*>(p)[i], type);
}
__device__ __forceinline__ void put(void* p, int64_t i, float v, int type) {
  if (type == kF32)
    static_cast<float*>(p)[i] = v;
  else
    static_cast<uint16_t*>(p)[i] = float_to_half(v, type);
}

// C consecutive elements (C a multiple of 8) from index i, `valid` of them
// inside; `vec` says that the address is 16-byte aligned.
template <int C>
__device__ __forceinline__ void get_run(const void* p, int64_t i, int type, int valid, bool vec, float (&v)[C]) {
  if (valid >= C && vec) {
    if (type == kF32) {
      const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
#pragma unroll
      for (int j = 0; j < C / 4; ++j) {
        const float4 f = q[j];
        v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
      }
    } else {
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
      for (int j = 0; j < C / 8; ++j) {
        const uint4 u = q[j];
        unpack_half2(u.x, type, v[8 * j], v[8 * j + 1]);
        unpack_half2(u.y, type, v[8 * j + 2], v[8 * j + 3]);
        unpack_half2(u.z, type, v[8 * j + 4], v[8 * j + 5]);
        unpack_half2(u.w, type, v[8 * j + 6], v[8 * j + 7]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] = j < valid ? get(p, i + j, type) : 0.0f;
  }
}
template <int C>
__device__ __forceinline__ void put_run(void* p, int64_t i, int type, int valid, bool vec, const float (&v)[C]) {
  if (valid >= C && vec) {
    if (type == kF32) {
      float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
#pragma unroll
      for (int j = 0; j < C / 4; ++j) q[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    } else {
      uint4* q = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i);
#pragma unroll
      for (int j = 0; j < C / 8; ++j)
        q[j] = make_uint4(pack_half2(v[8 * j], v[8 * j + 1], type), pack_half2(v[8 * j + 2], v[8 * j + 3], type),
                          pack_half2(v[8 * j + 4], v[8 * j + 5], type), pack_half2(v[8 * j + 6], v[8 * j + 7], type));
    }
  } else {
#pragma unroll
    for (int j = 0; j < C; ++j)
      if (j < valid) put(p, i + j, v[j], type);
  }
}

// Pre-activations kept for the backward pass: the upper 24 bits of fp32, 16 in
// one plane and 8 in another.  Kept in 16 bits, their rounding would double the
// error of the gradients, whose own rounding to 16 bits before the products
// cannot be avoided; 24 bits cost half as much again in bytes and leave an
// error below 2^-15, without a trace.  The rest is cut off, not rounded, so that
// no NaN turns into a number.  Both planes have rows of a multiple of 16
// elements (kept_ld) and 16-byte aligned bases.
__device__ __forceinline__ uint32_t kept_bits(float v) { return __float_as_uint(v); }
template <int C>
__device__ __forceinline__ void put_kept(uint16_t* hi, uint8_t* lo, int64_t i, int valid, bool vec,
                                         const float (&v)[C]) {
  uint32_t u[C];
#pragma unroll
  for (int j = 0; j < C; ++j) u[j] = kept_bits(v[j]);
  if (valid >= C && vec) {
    uint4* h = reinterpret_cast<uint4*>(hi + i);
    uint2* l = reinterpret_cast<uint2*>(lo + i);
#pragma unroll
    for (int j = 0; j < C / 8; ++j) {
      const uint32_t* w = u + 8 * j;
      h[j] = make_uint4(__byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632),
                        __byte_perm(w[4], w[5], 0x7632), __byte_perm(w[6], w[7], 0x7632));
      l[j] = make_uint2(__byte_perm(__byte_perm(w[0], w[1], 0x0051), __byte_perm(w[2], w[3], 0x0051), 0x5410),
                        __byte_perm(__byte_perm(w[4], w[5], 0x0051), __byte_perm(w[6], w[7], 0x0051), 0x5410));
    }
  } else {
#pragma unroll
    for (int j = 0; j < C; ++j)
      if (j < valid) {
        hi[i + j] = (uint16_t)(u[j] >> 16);
        lo[i + j] = (uint8_t)(u[j] >> 8);
      }
  }
}
__device__ __forceinline__ void put_kept1(uint16_t* hi, uint8_t* lo, int64_t i, float v) {
  const uint32_t u = kept_bits(v);
  hi[i] = (uint16_t)(u >> 16);
  lo[i] = (uint8_t)(u >> 8);
}
// 8 elements from a multiple of 8.  Those behind the row's last are whatever
// the padding holds: the caller stores none of them.
__device__ __forceinline__ void get_kept8(const uint16_t* hi, const uint8_t* lo, int64_t i, float (&v)[8]) {
  const uint4 h = *reinterpret_cast<const uint4*>(hi + i);
  const uint2 l = *reinterpret_cast<const uint2*>(lo + i);
  const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[2] = {l.x, l.y};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = lw[j / 2] >> (16 * (j & 1));  // bytes: the even element's 8 bits, the odd one's
    v[2 * j] = __uint_as_float(__byte_perm(hw[j], w << 8, 0x1054) & 0xffffff00u);
    v[2 * j + 1] = __uint_as_float(__byte_perm(hw[j], w, 0x3254) & 0xffffff00u);
  }
}

// Whether runs that start at multiples of 8 columns are 16-byte aligned in
// every row of a matrix.
__host__ __device__ inline bool runs_aligned(const void* p, int64_t ld, int elem) {
  return (reinterpret_cast<uintptr_t>(p) % 16) == 0 && (ld * elem) % 16 == 0;
}
__host__ __device__ inline int type_bytes(int type) { return type == kF32 ? 4 : type == kE4M3 ? 1 : 2; }

// Alignment of what an epilogue reads and writes, worked out once a thread.
struct EpiVec {
  bool out, res, bias, scale;
};
__device__ __forceinline__ EpiVec epi_vec(const Epilogue& e) {
  EpiVec v;
  v.out = runs_aligned(e.out[0], e.ldo, type_bytes(e.out_type)) &&
          runs_aligned(e.out[1], e.ldo, type_bytes(e.out_type));
  v.res = runs_aligned(e.residual, e.ldr, type_bytes(e.out_type));
  v.bias = runs_aligned(e.bias, 0, 2);
  v.scale = runs_aligned(e.col_scale[0], 0, 4) && runs_aligned(e.col_scale[1], 0, 4);
  return v;
}

// The epilogue on columns col .. col + C - 1 of one row, in three parts, so
// that z can be kept between them.  Sums to z: scales of projection `which`, bias.
template <int C>
__device__ __forceinline__ void epi_sums(const Epilogue& e, const EpiVec& ev, int which, int64_t row, int64_t col,
                                         int valid, float (&v)[C]) {
  float t[C];
  if (e.row_scale != nullptr) {
    const float rs = e.row_scale[row];
    get_run<C>(e.col_scale[which], col, kF32, valid, ev.scale, t);
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] *= rs * t[j];
  }
  if (e.bias != nullptr) {
    get_run<C>(e.bias, col, e.half_type, valid, ev.bias, t);
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] += t[j];
  }
}
template <int C>
__device__ __forceinline__ void epi_finish(const Epilogue& e, const EpiVec& ev, int64_t row, int64_t col, int valid,
                                           float (&v)[C]) {
  act_run<C>(e.act, v);
  if (e.residual != nullptr) {
    float t[C];
    get_run<C>(e.residual, row * e.ldr + col, e.out_type, valid, ev.res, t);
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] += t[j];
  }
}
// All of it, stored by this thread.
template <int C>
__device__ __forceinline__ void epilogue_run(const Epilogue& e, const EpiVec& ev, int which, int64_t row, int64_t col,
                                             int64_t n, float (&v)[C]) {
  const int valid = (int)::ngl::dev::min64(C, n - col);
  epi_sums<C>(e, ev, 0, row, col, valid, v);
  if (e.z_hi[0] != nullptr) put_kept<C>(e.z_hi[0], e.z_lo[0], row * e.ldz + col, valid, true, v);
  epi_finish<C>(e, ev, row, col, valid, v);
  put_run<C>(e.out[which], row * e.ldo + col, e.out_type, valid, ev.out, v);
}
template <int C>
__device__ __forceinline__ void epilogue_gated_run(const Epilogue& e, const EpiVec& ev, int64_t row, int64_t col,
                                                   int64_t n, float (&g)[C], float (&u)[C]) {
  const int valid = (int)::ngl::dev::min64(C, n - col);
  epi_sums<C>(e, ev, 0, row, col, valid, g);
  epi_sums<C>(e, ev, 1, row, col, valid, u);
  if (e.z_hi[0] != nullptr) {
    put_kept<C>(e.z_hi[0], e.z_lo[0], row * e.ldz + col, valid, true, g);
    put_kept<C>(e.z_hi[1], e.z_lo[1], row * e.ldz + col, valid, true, u);
  }
  act_run<C>(e.act, g);
#pragma unroll
  for (int j = 0; j < C; ++j) g[j] *= u[j];
  put_run<C>(e.out[0], row * e.ldo + col, e.out_type, valid, ev.out, g);
}

}  // namespace dense
}  // namespace ngl

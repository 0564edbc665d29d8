// Products of few rows (decoding): bound by one pass over the weights.
//
// Mathematics: the epilogue of dense.h over z[i, j] = sum_k x[i, k] w[j, k]
// for up to 32 rows i.  A warp takes 16 weight rows as the 16-row operand of
// mma m16n8k16 and groups of 8 rows of x as its 8-column operand; the CTA's
// 8 warps split k and join their sums in shared memory in warp order.  The
// sum over k may run in any order as long as both operands agree, so each
// thread loads 16 contiguous bytes of a row straight into its fragment: no
// shared memory between the weights and the products.
#include "dense.h"

#include <algorithm>

#include "dense_math.cuh"
#include "ngl_cuda.cuh"

namespace ngl {
namespace dense {
namespace {

using namespace ngl::dev;

constexpr int kWarps = 8;
constexpr int kWRows = 16;

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool bf16) {
  if (bf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 bytes of row `row` from byte `at` of its k; zero beyond the row's end.
template <bool kVec>
__device__ __forceinline__ uint4 load16(const uint8_t* p, int64_t row_bytes, int64_t at, int64_t k_bytes, bool inside,
                                        int elem) {
  if (!inside || at >= k_bytes) return make_uint4(0, 0, 0, 0);
  const uint8_t* q = p + row_bytes + at;
  if (kVec) return __ldg(reinterpret_cast<const uint4*>(q));
  uint32_t w[4] = {0, 0, 0, 0};
  if (elem == 2) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at + 2 * j < k_bytes) w[j / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(q)[j] << (16 * (j & 1));
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (at + j < k_bytes) w[j / 4] |= (uint32_t)q[j] << (8 * (j & 3));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Two e4m3 values as two fp16 (exact).
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t v) {
  uint32_t r;
  asm("{\n .reg .b16 h;\n cvt.u16.u32 h, %1;\n cvt.rn.f16x2.e4m3x2 %0, h;\n}\n" : "=r"(r) : "r"(v & 0xffffu));
  return r;
}

// MT groups of 8 rows of x; kVec: rows 16-byte aligned and k a multiple of 16 bytes.
template <int MT, bool kGated, bool kFp8, bool kVec>
__global__ void __launch_bounds__(kWarps * 32) k_skinny(const __grid_constant__ Skinny g) {
  constexpr int NW = kGated ? 2 : 1;
  constexpr int elem = kFp8 ? 1 : 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gq = lane >> 2, t = lane & 3;
  const int64_t j0 = (int64_t)blockIdx.x * kWRows;
  const int64_t kbytes = g.k * elem;
  const int64_t nblk = (kbytes + 63) / 64;
  const bool bf16 = g.type == kBF16;
  const uint8_t* x = static_cast<const uint8_t*>(g.x.p);
  float acc[NW][MT][4];
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[w][m][i] = 0.0f;

  const bool in0 = j0 + gq < g.n, in1 = j0 + gq + 8 < g.n;
#pragma unroll 2
  for (int64_t b = warp; b < nblk; b += kWarps) {
    const int64_t at = b * 64 + t * 16;
    uint4 a[NW][2], xb[MT];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const uint8_t* p = static_cast<const uint8_t*>(g.w[w].p);
      a[w][0] = load16<kVec>(p, (j0 + gq) * g.w[w].ld * elem, at, kbytes, in0, elem);
      a[w][1] = load16<kVec>(p, (j0 + gq + 8) * g.w[w].ld * elem, at, kbytes, in1, elem);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
      xb[m] = load16<kVec>(x, (int64_t)(m * 8 + gq) * g.x.ld * elem, at, kbytes, m * 8 + gq < g.m, elem);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const uint32_t r0[4] = {a[w][0].x, a[w][0].y, a[w][0].z, a[w][0].w};
      const uint32_t r1[4] = {a[w][1].x, a[w][1].y, a[w][1].z, a[w][1].w};
#pragma unroll
      for (int h = 0; h < (kFp8 ? 4 : 2); ++h) {
        uint32_t f[4];
        if (kFp8) {
          f[0] = e4m3x2_to_half2(r0[h]);
          f[1] = e4m3x2_to_half2(r1[h]);
          f[2] = e4m3x2_to_half2(r0[h] >> 16);
          f[3] = e4m3x2_to_half2(r1[h] >> 16);
        } else {
          f[0] = r0[2 * h];
          f[1] = r1[2 * h];
          f[2] = r0[2 * h + 1];
          f[3] = r1[2 * h + 1];
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint32_t xr[4] = {xb[m].x, xb[m].y, xb[m].z, xb[m].w};
          if (kFp8)
            mma16816(acc[w][m], f, e4m3x2_to_half2(xr[h]), e4m3x2_to_half2(xr[h] >> 16), false);
          else
            mma16816(acc[w][m], f, xr[2 * h], xr[2 * h + 1], bf16);
        }
      }
    }
  }

  // acc[.][m][i]: weight row gq + 8 (i / 2), x row m * 8 + 2 t + (i & 1)
  __shared__ float part[kWarps][NW][MT * 8][kWRows + 1];
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[warp][w][m * 8 + 2 * t + (i & 1)][gq + 8 * (i >> 1)] = acc[w][m][i];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 8 * kWRows; i += kWarps * 32) {
    const int r = i / kWRows, c = i % kWRows;
    const int64_t row = r, col = j0 + c;
    if (row >= g.m || col >= g.n) continue;
    float s[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      s[w] = 0.0f;
#pragma unroll
      for (int q = 0; q < kWarps; ++q) s[w] += part[q][w][r][c];
    }
    const Epilogue& e = g.ep;
    float z = s[0], u = s[NW - 1];
    if (e.row_scale != nullptr) {
      z *= e.row_scale[row] * e.col_scale[0][col];
      if (kGated) u *= e.row_scale[row] * e.col_scale[1][col];
    }
    if (!kGated && e.bias != nullptr) z += get(e.bias, col, e.half_type);
    if (e.z[0] != nullptr) {
      put(e.z[0], row * g.n + col, z, e.half_type);
      if (kGated) put(e.z[1], row * g.n + col, u, e.half_type);
    }
    float y = act_value(e.act, z);
    if (kGated) y *= u;
    if (!kGated && e.residual != nullptr) y += get(e.residual, row * e.ldr + col, e.out_type);
    put(e.out[0], row * e.ldo + col, y, e.out_type);
  }
}

template <int MT, bool kGated, bool kFp8>
cudaError_t launch_mt(const Skinny& g, bool vec, cudaStream_t s) {
  const unsigned grid = (unsigned)((g.n + kWRows - 1) / kWRows);
  if (vec)
    k_skinny<MT, kGated, kFp8, true><<<grid, kWarps * 32, 0, s>>>(g);
  else
    k_skinny<MT, kGated, kFp8, false><<<grid, kWarps * 32, 0, s>>>(g);
  return cudaGetLastError();
}
template <bool kGated, bool kFp8>
cudaError_t launch_skinny(const Skinny& g, bool vec, cudaStream_t s) {
  if (g.m <= 8) return launch_mt<1, kGated, kFp8>(g, vec, s);
  if (g.m <= 16) return launch_mt<2, kGated, kFp8>(g, vec, s);
  return launch_mt<4, kGated, kFp8>(g, vec, s);
}

}  // namespace

cudaError_t skinny(const Skinny& g, cudaStream_t s) {
  if (g.m <= 0 || g.m > kSkinnyRows || g.n <= 0 || g.k <= 0) return cudaErrorInvalidValue;
  const int elem = type_bytes(g.type);
  bool vec = (g.k * elem) % 16 == 0 && runs_aligned(g.x.p, g.x.ld, elem) && runs_aligned(g.w[0].p, g.w[0].ld, elem);
  if (g.gated) vec = vec && runs_aligned(g.w[1].p, g.w[1].ld, elem);
  if (g.type == kE4M3) return g.gated ? launch_skinny<true, true>(g, vec, s) : launch_skinny<false, true>(g, vec, s);
  return g.gated ? launch_skinny<true, false>(g, vec, s) : launch_skinny<false, false>(g, vec, s);
}

}  // namespace dense
}  // namespace ngl

// Products of few rows (decoding): bound by one pass over the weights.
//
// Mathematics: the epilogue of dense.h over z[i, j] = sum_k x[i, k] w[j, k]
// for up to 16 rows i.  The rows of x are the 16-row operand of mma m16n8k16
// and 8 weight rows its 8-column operand; the CTA's warps split k and join
// their sums in shared memory in warp order.  The sum over k may run in any
// order as long as both operands agree, so each thread loads 16 contiguous
// bytes of a row straight into its fragment: no shared memory between the
// weights and the products, and every load of a batch is in flight before the
// first product.  Weights that nothing has cached: 2 x 5632 x 2048 in 9.4 us
// (4.9 TB/s), 2048 x 5632 in 6.2 us (3.7 TB/s), where the latency of starting,
// of one or two rounds of loads and of the join is half of the time.
#include "dense.h"

#include <algorithm>

#include "dense_math.cuh"
#include "layer_launch.cuh"
#include "ngl_cuda.cuh"

namespace ngl {
namespace dense {
namespace {

using namespace ngl::dev;

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, bool bf16) {
  if (bf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of a row from byte `at` of its k.  Weights, which nothing reads
// again, do not go through L1.
__device__ __forceinline__ uint4 load_once(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
// The same from any address, zero beyond the row's end: the aligned words that
// hold its bytes, shifted into place.  Only words with a byte of the row in them
// are read, so no load leaves the row's first and last word.
__device__ __forceinline__ uint4 load_any(const uint8_t* row, int64_t at, int64_t k_bytes) {
  const int n = (int)min64(16, k_bytes - at);  // bytes of the row
  if (n <= 0) return make_uint4(0, 0, 0, 0);
  const uintptr_t p = reinterpret_cast<uintptr_t>(row + at);
  const uint32_t* q = reinterpret_cast<const uint32_t*>(p & ~(uintptr_t)3);
  const int off = (int)(p & 3);
  uint32_t w[5];
#pragma unroll
  for (int j = 0; j < 5; ++j) w[j] = 4 * j < off + n ? q[j] : 0u;
  uint32_t v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = __funnelshift_r(w[j], w[j + 1], 8 * off);
    const int left = n - 4 * j;  // bytes of this word inside the row
    v[j] = left >= 4 ? v[j] : left <= 0 ? 0u : v[j] & (0xffffffffu >> (32 - 8 * left));
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// Two e4m3 values as two fp16 (exact).
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t v) {
  uint32_t r;
  asm("{\n .reg .b16 h;\n cvt.u16.u32 h, %1;\n cvt.rn.f16x2.e4m3x2 %0, h;\n}\n" : "=r"(r) : "r"(v & 0xffffu));
  return r;
}

// NT groups of 8 weight rows a CTA (of each projection); a warp takes U
// consecutive 64-byte blocks of k at a time, all in flight at once.  kHigh: x
// has more than 8 rows; kVec: rows 16-byte aligned and k a multiple of 16
// bytes.  Rows beyond the last are read as the last: their sums go nowhere.
// W warps, OCC CTAs an SM.
template <int W, int OCC, int NT, int U, bool kHigh, bool kGated, bool kFp8, bool kVec>
__global__ void __launch_bounds__(W * 32, OCC) k_skinny(const __grid_constant__ Skinny g) {
  pdl_begin();
  constexpr int NW = kGated ? 2 : 1;
  constexpr int elem = kFp8 ? 1 : 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q = lane >> 2, t = lane & 3;
  const int64_t j0 = (int64_t)blockIdx.x * (8 * NT);
  const int64_t kbytes = g.k * elem;
  const bool bf16 = g.type == kBF16;
  const uint8_t* x0 = static_cast<const uint8_t*>(g.x.p) + min64(q, g.m - 1) * g.x.ld * elem;
  const uint8_t* x1 = static_cast<const uint8_t*>(g.x.p) + min64(q + 8, g.m - 1) * g.x.ld * elem;
  const uint8_t* wr[NW][NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int w = 0; w < NW; ++w)
      wr[w][n] = static_cast<const uint8_t*>(g.w[w].p) + min64(j0 + 8 * n + q, g.n - 1) * g.w[w].ld * elem;
  float acc[NW][NT][4];
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[w][n][i] = 0.0f;

  // The CTA's weights on their way into L2 while the kernel before this one ends
  // (L2 is where all writes meet, so whatever it writes is still seen).
  if (kVec && warp == 0 && lane < 8 * NT * NW) {
    const int64_t row = j0 + lane % (8 * NT);
    const int w = lane / (8 * NT);
    if (row < g.n)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(static_cast<const uint8_t*>(g.w[w].p) +
                                                                    row * g.w[w].ld * elem),
                   "r"((uint32_t)min64(kbytes, 1 << 16))
                   : "memory");
  }
  pdl_wait();
  for (int64_t b0 = (int64_t)warp * (U * 64); b0 < kbytes; b0 += W * U * 64) {
    uint4 wv[U][NW][NT], xa[U], xb[U];
    if (kVec && b0 + U * 64 <= kbytes) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = b0 + u * 64 + t * 16;
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
          for (int n = 0; n < NT; ++n) wv[u][w][n] = load_once(wr[w][n] + at);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = b0 + u * 64 + t * 16;
        xa[u] = *reinterpret_cast<const uint4*>(x0 + at);
        if (kHigh) xb[u] = *reinterpret_cast<const uint4*>(x1 + at);
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = b0 + u * 64 + t * 16;
        const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            wv[u][w][n] = kVec ? (at < kbytes ? load_once(wr[w][n] + at) : none) : load_any(wr[w][n], at, kbytes);
        xa[u] = kVec ? (at < kbytes ? *reinterpret_cast<const uint4*>(x0 + at) : none)
                     : load_any(x0, at, kbytes);
        if (kHigh)
          xb[u] = kVec ? (at < kbytes ? *reinterpret_cast<const uint4*>(x1 + at) : none)
                       : load_any(x1, at, kbytes);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t p[4] = {xa[u].x, xa[u].y, xa[u].z, xa[u].w};
      uint32_t r[4] = {0, 0, 0, 0};
      if (kHigh) {
        r[0] = xb[u].x;
        r[1] = xb[u].y;
        r[2] = xb[u].z;
        r[3] = xb[u].w;
      }
#pragma unroll
      for (int h = 0; h < (kFp8 ? 4 : 2); ++h) {
        uint32_t a0, a1, a2, a3;
        if (kFp8) {
          a0 = e4m3x2_to_half2(p[h]);
          a2 = e4m3x2_to_half2(p[h] >> 16);
          a1 = kHigh ? e4m3x2_to_half2(r[h]) : 0u;
          a3 = kHigh ? e4m3x2_to_half2(r[h] >> 16) : 0u;
        } else {
          a0 = p[2 * h];
          a2 = p[2 * h + 1];
          a1 = r[2 * h];
          a3 = r[2 * h + 1];
        }
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 v = wv[u][w][n];
            const uint32_t s[4] = {v.x, v.y, v.z, v.w};
            if (kFp8)
              mma16816(acc[w][n], a0, a1, a2, a3, e4m3x2_to_half2(s[h]), e4m3x2_to_half2(s[h] >> 16), false);
            else
              mma16816(acc[w][n], a0, a1, a2, a3, s[2 * h], s[2 * h + 1], bf16);
          }
      }
    }
  }

  // acc[.][n][i]: x row q + 8 (i / 2), weight row 8 n + 2 t + (i & 1)
  constexpr int kX = kHigh ? 16 : 8;
  __shared__ float part[W][NW][kX][8 * NT + 1];
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < (kHigh ? 4 : 2); ++i) part[warp][w][q + 8 * (i >> 1)][8 * n + 2 * t + (i & 1)] = acc[w][n][i];
  __syncthreads();
  for (int i = threadIdx.x; i < kX * 8 * NT; i += W * 32) {
    const int r = i / (8 * NT), c = i % (8 * NT);
    const int64_t row = r, col = j0 + c;
    if (row >= g.m || col >= g.n) continue;
    float s[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      s[w] = 0.0f;
#pragma unroll
      for (int o = 0; o < W; ++o) s[w] += part[o][w][r][c];
    }
    const Epilogue& e = g.ep;
    float z = s[0], u = s[NW - 1];
    if (e.row_scale != nullptr) {
      z *= e.row_scale[row] * e.col_scale[0][col];
      if (kGated) u *= e.row_scale[row] * e.col_scale[1][col];
    }
    if (!kGated && e.bias != nullptr) z += get(e.bias, col, e.half_type);
    if (e.z_hi[0] != nullptr) {
      put_kept1(e.z_hi[0], e.z_lo[0], row * e.ldz + col, z);
      if (kGated) put_kept1(e.z_hi[1], e.z_lo[1], row * e.ldz + col, u);
    }
    float y[1] = {z};
    act_run<1>(e.act, y);
    if (kGated) y[0] *= u;
    if (!kGated && e.residual != nullptr) y[0] += get(e.residual, row * e.ldr + col, e.out_type);
    put(e.out[0], row * e.ldo + col, y[0], e.out_type);
  }
}

template <int W, int OCC, int NT, int U, bool kHigh, bool kGated, bool kFp8>
cudaError_t launch_nt(const Skinny& g, bool vec, cudaStream_t s) {
  const unsigned grid = (unsigned)((g.n + 8 * NT - 1) / (8 * NT));
  return launch_dependent(vec ? &k_skinny<W, OCC, NT, U, kHigh, kGated, kFp8, true>
                              : &k_skinny<W, OCC, NT, 2, kHigh, kGated, kFp8, false>,
                          dim3(grid), dim3(W * 32), 0, 1, s, g);
}
// With more CTAs than fit at once, small ones that leave room for the next; else
// 16 warps share a CTA's k, so that its loads go out together.  Times of weights
// from HBM, 8 warps against 16: 5632 x 2048 6.8 and 8.0 us, 32000 x 2048 28.5 and
// 34.0 us, gated 2 x 5632 x 2048 9.9 and 12.5 us; 2048 x 5632 8.9 and 6.2 us,
// gated 2 x 2048 x 768 3.2 and 2.7 us.
template <bool kGated, bool kFp8>
cudaError_t launch_skinny(const Skinny& g, bool vec, int sms, cudaStream_t s) {
  if (g.m > 8)
    return kGated ? launch_nt<8, 2, 1, 4, true, kGated, kFp8>(g, vec, s)
                  : launch_nt<8, 2, 2, 4, true, kGated, kFp8>(g, vec, s);
  if ((g.n + 7) / 8 > 2 * sms) return launch_nt<8, 3, 1, kGated ? 4 : 8, false, kGated, kFp8>(g, vec, s);
  return launch_nt<16, 2, 1, kGated ? 2 : 4, false, kGated, kFp8>(g, vec, s);
}

}  // namespace

cudaError_t skinny(const Skinny& g, int sms, cudaStream_t s) {
  if (g.m <= 0 || g.m > kSkinnyRows || g.n <= 0 || g.k <= 0) return cudaErrorInvalidValue;
  const int elem = type_bytes(g.type);
  bool vec = (g.k * elem) % 16 == 0 && runs_aligned(g.x.p, g.x.ld, elem) && runs_aligned(g.w[0].p, g.w[0].ld, elem);
  if (g.gated) vec = vec && runs_aligned(g.w[1].p, g.w[1].ld, elem);
  if (g.type == kE4M3) return g.gated ? launch_skinny<true, true>(g, vec, sms, s) : launch_skinny<false, true>(g, vec, sms, s);
  return g.gated ? launch_skinny<true, false>(g, vec, sms, s) : launch_skinny<false, false>(g, vec, sms, s);
}

}  // namespace dense
}  // namespace ngl

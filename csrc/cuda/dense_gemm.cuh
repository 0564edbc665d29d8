// Matrix products on the tensor cores with the epilogues of a dense layer.
//
// Mathematics: D[i, j] = sum_k A[i, k] B[j, k] for 16-bit or e4m3 operands,
// sums in fp32, followed by the epilogue of dense.h in the same kernel.  One
// kernel serves the forward product (both operands with k contiguous), the
// gradient of the input (B stored as [k, j]) and the gradient of the weight
// (both stored with k as the slow axis): tcgen05.mma reads either order from
// shared memory, so no operand is transposed in memory.
//
// Layout: persistent CTAs, one per SM (or pairs on one tile).  Warp 0 moves
// 128-byte-wide tiles with TMA, warp 1 issues the products of 128-byte k
// blocks, warps 4 on take finished accumulators from tensor memory through
// the epilogue while the next tile's products run into the other half of
// tensor memory.  A tile of 256 x 256 by a pair of CTAs reads 32 KB of operands
// a CTA for 512 cycles of products, a tile of 128 columns 32 KB for 256.
//
// Bound by the tensor cores, and on a GPU that is busy for milliseconds by its
// power: 4096^3 bf16 takes 96 us (1.43 PFLOP/s, tensor pipe active 90 % of the
// time), 8192 x 5632 x 2048 127 us, with zeros for operands 98 us; the gated
// form 2 x 5632 with its kept projections 260 us (1.45 PFLOP/s), the input's
// gradient of the same size 265 us (tensor pipe 96 %).  Small products are
// bound by what does not overlap: 1.2 us to the first operands, 1.5 us (128
// columns) or 2.6 us (256) for the last epilogue, 0.19 us a k block between.
#pragma once
#include "dense.h"

#include <algorithm>

#include "dense_math.cuh"
#include "layer_launch.cuh"
#include "ngl_cuda.cuh"

namespace ngl {
namespace dense {

using namespace ngl::dev;

constexpr int kRowsA = 128;       // A rows of one CTA
constexpr int kBlockBytes = 128;  // bytes of k in one stage
constexpr int kStageBytes = 2048;  // staging of an epilogue warp
constexpr uint64_t kWaitNs = 4000000000ull;
constexpr uint64_t kDrainNs = 100000000ull;

struct alignas(64) Maps {
  CUtensorMap a[2], b[2];
};
struct Args {
  int64_t m, n;
  int mt, nt;        // tiles of one problem along m and n
  int kb;            // k blocks of one operand pair
  int* status;       // this device's status words
  int* status_host;  // their copy in host memory
  int dual;
  int splits;        // pieces of k of each tile
  uint32_t idesc;
  uint32_t stage_bytes;  // of TMA's boxes in one stage, both CTAs of a pair
  float* partial;    // [tiles, splits, rows of a tile, NB] sums, where splits > 1
  Epilogue ep;
};

// ------------------------------------------------------------------- PTX
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// One lane of a warp whose 32 lanes are all here.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// kCluster: what the other CTA of a pair did before it arrived is to be seen.
// That costs a fence, so the waits inside a tile, on TMA's bytes and on finished
// products, go without (8192 x 5632 x 2048: 134 us with it, 131 without).
template <bool kCluster>
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  if (kCluster)
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
  return ok != 0;
}
template <bool kCluster = false>
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, uint64_t limit_ns) {
  if (try_wait<kCluster>(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  while (!try_wait<kCluster>(bar, parity))
    if (globaltimer() - t0 > limit_ns) return false;
  return true;
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
template <int CG>
__device__ __forceinline__ void arrive_leader(uint32_t bar) {
  if (CG == 1)
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
  else
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(map_to_rank(bar, 0))
                 : "memory");
}
// A box of a 2-D tensor map into this CTA's shared memory; the bytes are
// counted by the pair's first CTA.
template <int CG>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, "
        "{%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t cols) {
  if (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
  if (CG == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
template <int CG, bool kFp8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
#define NGL_MMA(group, kind)                                                                                       \
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::" group ".kind::" kind           \
               " [%0], %1, %2, %3, p;\n}\n" ::"r"(d),                                                              \
               "l"(a), "l"(b), "r"(idesc), "r"(accumulate)                                                         \
               : "memory")
  if (CG == 1) {
    if (kFp8) NGL_MMA("1", "f8f6f4"); else NGL_MMA("1", "f16");
  } else {
    if (kFp8) NGL_MMA("2", "f8f6f4"); else NGL_MMA("2", "f16");
  }
#undef NGL_MMA
}
// Arrive on `bar` (in both CTAs of a pair) once this thread's products are done.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Record that a wait ran out, the first since the words were cleared, for
// check() and, in host memory, for the next call.
__device__ __forceinline__ void give_up(const Args& g, int code, int role) {
  if (atomicCAS(g.status, 0, code) != 0) return;
  g.status[1] = (int)blockIdx.x;
  g.status[2] = role;
  volatile int* h = g.status_host;
  h[1] = (int)blockIdx.x;
  h[2] = role;
  __threadfence_system();
  h[0] = code;
}

// 32 columns of this warp's 32 lanes.  The load and its wait are one statement:
// nothing may touch the registers between them.
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Shared-memory matrix descriptor, 128-byte swizzle.  A tile with k contiguous
// has groups of 8 rows 1024 bytes apart; a tile with rows contiguous holds
// chunks of 64 rows of 8192 bytes (64 k of 128 bytes each), 8 k 1024 bytes
// apart.
template <int kMaj>
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
  constexpr uint64_t lead = kMaj == kMajorK ? 1 : (8192 >> 4);
  return (uint64_t)((addr >> 4) & 0x3fff) | (lead << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Bytes from one product's k to the next inside a stage (32 bytes of k).
template <int kMaj>
constexpr uint32_t kStep = kMaj == kMajorK ? 32u : 2048u;

// EW: warps of the epilogue.  16 where a tile's products take less time than an
// epilogue with an activation (up to 16 k blocks), else 8, whose registers hold
// everything.  16 against 8 warps, bias and GELU: 8192 x 2048 x 256 31 and 33.5 us
// (with kept z 37 and 45), x 512 33 and 36, 300 x 5632 x 1024 10.5 and 12, 8192 x
// 2048 x 1024 level at 54; without an epilogue's work 16 warps lose: 14.6 and 13.8,
// 20.3 and 19.1, 7.9 and 7.5, 36 and 27.5 us.
template <int CG, int NB, int EW>
struct Shape {
  static constexpr int kThreads = 128 + 32 * EW;
  static constexpr int kRowsB = NB / CG;  // B rows of one CTA
  static constexpr int kBytesA = kRowsA * kBlockBytes;
  static constexpr int kBytesB = kRowsB * kBlockBytes;
  static constexpr int kStage = kBytesA + kBytesB;
  static constexpr int kStages = (192 * 1024) / kStage > 8 ? 8 : (192 * 1024) / kStage;
  static constexpr int kCols = 2 * NB;  // tensor memory: two accumulators
  static constexpr int kBarBytes = 256;
  static constexpr int kSmem = kStages * kStage + kBarBytes + EW * kStageBytes + 1024 /* alignment */;
  static_assert(kSmem <= 227 * 1024, "shared memory of one CTA");
};

// ---- writing a warp's 32 x 32 pieces
// The accumulator's layout gives a lane one row; stored so, every store is half
// a sector in each of 32 rows, and slows the operands' loads (8192 x 5632 x
// 2048 took 145 us so, 121 without any stores).  A piece goes through 2 KB of shared
// memory a warp instead, and each store writes 64 adjacent bytes of 8 rows
// (138 us at that step; TMA stores from the same staging took as long, and need a
// tensor map for each output on the host).
struct Piece {
  uint32_t smem;
  int64_t row0, col;
  int rows;  // rows inside the matrix, 1 to 32
  int cols;  // columns inside, 1 to 32
  int lane;
};
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
// Rows of R 16-byte units (R = 2 or 4): this lane's row from p, then lanes
// side by side along the rows of `out`, whose rows are 16-byte aligned.  The
// units of a row are permuted so that both passes are free of bank conflicts.
template <int R>
__device__ __forceinline__ void write_units(const Piece& w, void* out, int64_t ld_bytes, int unit_cols,
                                            const uint32_t (&p)[4 * R], int skip = 0) {
  auto at = [&](int row, int unit) {
    const int swap = R == 4 ? (row >> 1) & 3 : (row >> 2) & 1;
    return w.smem + (uint32_t)(row * R + (unit ^ swap)) * 16u;
  };
  __syncwarp();  // the last piece has been read
#pragma unroll
  for (int c = 0; c < R; ++c) sts16(at(w.lane, c), p[4 * c], p[4 * c + 1], p[4 * c + 2], p[4 * c + 3]);
  __syncwarp();
  constexpr int kRowsAtOnce = 32 / R;
  const int unit = w.lane % R, r0 = w.lane / R;
  if (skip + unit * unit_cols >= w.cols) return;
  uint8_t* q = static_cast<uint8_t*>(out) + (w.row0 + r0) * ld_bytes + ((w.col + skip) / unit_cols + unit) * 16;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = i * kRowsAtOnce + r0;
    const uint4 v = lds16(at(row, unit));
    if (row < w.rows) *reinterpret_cast<uint4*>(q + (int64_t)i * kRowsAtOnce * ld_bytes) = v;
  }
}
// A piece of the residual, 32 rows of 64 bytes (32 columns of 16 bits, or half h
// of 32 of fp32): fetched as it is written, a row's units side by side, so that
// it can be under way before the sums are ready.
__device__ __forceinline__ void fetch_units(const Piece& w, const void* src, int64_t ld_bytes, int unit_cols, int h,
                                            uint4 (&r)[4]) {
  const int unit = w.lane & 3, r0 = w.lane >> 2, c = 4 * unit_cols * h + unit * unit_cols;
  const uint8_t* q =
      static_cast<const uint8_t*>(src) + (w.row0 + r0) * ld_bytes + (w.col + c) * (int64_t)(16 / unit_cols);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = c < w.cols && i * 8 + r0 < w.rows ? *reinterpret_cast<const uint4*>(q + (int64_t)i * 8 * ld_bytes)
                                             : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ void add_units(const Piece& w, const uint4 (&r)[4], int type, int h, float (&v)[32]) {
  auto at = [&](int row, int unit) { return w.smem + (uint32_t)(row * 4 + (unit ^ ((row >> 1) & 3))) * 16u; };
  const int unit = w.lane & 3, r0 = w.lane >> 2;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) sts16(at(i * 8 + r0, unit), r[i].x, r[i].y, r[i].z, r[i].w);
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint4 u = lds16(at(w.lane, c));
    const uint32_t p[4] = {u.x, u.y, u.z, u.w};
    if (type == kF32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (h == 0) v[4 * c + j] += __uint_as_float(p[j]);
        else v[16 + 4 * c + j] += __uint_as_float(p[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float lo, hi;
        unpack_half2(p[j], type, lo, hi);
        v[8 * c + 2 * j] += lo;
        v[8 * c + 2 * j + 1] += hi;
      }
    }
  }
}
// Staging of 16 fp32 columns of 32 rows for matrices whose rows are not 16-byte
// aligned: a lane's own row on one side, two rows of 16 adjacent columns on the other.
__device__ __forceinline__ uint32_t plain_at(const Piece& w, int row, int c) {
  return w.smem + 4u * (uint32_t)(row * 16 + ((c + (row >> 1)) & 15));
}
__device__ __forceinline__ void add_plain(const Piece& w, const void* src, int64_t ld, int type, float (&v)[32]) {
  const int c = w.lane & 15, sub = w.lane >> 4;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    __syncwarp();
    const bool in = 16 * h + c < w.cols;
    const int64_t first = (w.row0 + sub) * ld + w.col + 16 * h + c;
    uint32_t t[16];  // all under way before the first is stored
    if (type == kF32) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        t[i] = in && sub + 2 * i < w.rows ? static_cast<const uint32_t*>(src)[first + 2 * i * ld] : 0u;
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        t[i] = in && sub + 2 * i < w.rows ? static_cast<const uint16_t*>(src)[first + 2 * i * ld] : 0u;
      if (type == kBF16) {
#pragma unroll
        for (int i = 0; i < 16; ++i) t[i] <<= 16;
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) t[i] = __float_as_uint(half_to_float((uint16_t)t[i], kF16));
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(plain_at(w, sub + 2 * i, c)), "r"(t[i]) : "memory");
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float f;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(plain_at(w, w.lane, j)) : "memory");
      v[16 * h + j] += f;
    }
  }
}
__device__ __forceinline__ void write_kept(const Piece& w, uint16_t* hi, uint8_t* lo, int64_t ld,
                                           const float (&v)[32]) {
  uint32_t p[16], q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t a = kept_bits(v[4 * j]), b = kept_bits(v[4 * j + 1]), c = kept_bits(v[4 * j + 2]),
                   d = kept_bits(v[4 * j + 3]);
    p[2 * j] = __byte_perm(a, b, 0x7632);
    p[2 * j + 1] = __byte_perm(c, d, 0x7632);
    q[j] = __byte_perm(__byte_perm(a, b, 0x0051), __byte_perm(c, d, 0x0051), 0x5410);
  }
  write_units<4>(w, hi, ld * 2, 8, p);
  write_units<2>(w, lo, ld, 16, q);
}
// `aligned`: rows of out start on 16 bytes (then n is a multiple of a unit).
// Otherwise (kAny) two rows of 16 adjacent columns a store.
template <bool kAny>
__device__ __forceinline__ void write_piece(const Piece& w, void* out, int64_t ld, int type, bool aligned,
                                            const float (&v)[32]) {
  if (aligned && type == kF32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // 16 columns at a time
      uint32_t p[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) p[j] = __float_as_uint(v[16 * h + j]);
      write_units<4>(w, out, ld * 4, 4, p, 16 * h);
    }
  } else if (aligned) {
    uint32_t p[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) p[j] = pack_half2(v[2 * j], v[2 * j + 1], type);
    write_units<4>(w, out, ld * 2, 8, p);
  } else if constexpr (kAny) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // 16 columns of 32 rows, two rows a store
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 16; ++j)
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(plain_at(w, w.lane, j)), "f"(v[16 * h + j]) : "memory");
      __syncwarp();
      const int c = w.lane & 15, sub = w.lane >> 4;
      if (16 * h + c < w.cols) {
        float t[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(t[i]) : "r"(plain_at(w, sub + 2 * i, c)) : "memory");
        const int64_t first = (w.row0 + sub) * ld + w.col + 16 * h + c;
        if (type == kF32) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (sub + 2 * i < w.rows) static_cast<float*>(out)[first + 2 * i * ld] = t[i];
        } else {
          uint16_t u[16];
          if (type == kBF16) {
#pragma unroll
            for (int i = 0; i < 16; ++i) u[i] = float_to_half(t[i], kBF16);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) u[i] = float_to_half(t[i], kF16);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (sub + 2 * i < w.rows) static_cast<uint16_t*>(out)[first + 2 * i * ld] = u[i];
        }
      }
    }
  }
}

struct Item {
  int prob;     // kDualM: which product
  int mt, nt;   // tile
  int k0, k1;   // k blocks
  int part;     // slot of `partial`, or -1
};
__device__ __forceinline__ uint32_t tiles_of(const Args& g) {
  return (uint32_t)g.mt * (g.dual == kDualM ? 2u : 1u) * (uint32_t)g.nt;
}
// Tile t.  Groups of 8 rows of tiles sweep the columns together, so that the
// tiles that run at one time share their operands in L2.  32-bit arithmetic: the
// host refuses more tiles, and every warp divides once a tile.
__device__ __forceinline__ void tile_of(const Args& g, uint32_t t, Item& it) {
  const uint32_t rows = (uint32_t)g.mt * (g.dual == kDualM ? 2u : 1u);
  const uint32_t per = 8u * (uint32_t)g.nt;
  const uint32_t grp = t / per, in = t - grp * per;
  const uint32_t h = min(8u, rows - grp * 8u);
  const uint32_t nt = h == 8u ? in >> 3 : in / h;
  const uint32_t r = grp * 8u + (in - nt * h);
  it.nt = (int)nt;
  it.prob = r >= (uint32_t)g.mt ? 1 : 0;
  it.mt = (int)r - it.prob * g.mt;
}
// Work item w: a tile, or one of its pieces of k.
__device__ __forceinline__ Item item_of(const Args& g, uint32_t w) {
  Item it;
  const int kb = g.kb * (g.dual == kDualK ? 2 : 1);
  if (g.splits == 1) {
    tile_of(g, w, it);
    it.k0 = 0;
    it.k1 = kb;
    it.part = -1;
    return it;
  }
  const uint32_t t = w / (uint32_t)g.splits;
  const int sp = (int)(w - t * (uint32_t)g.splits);
  tile_of(g, t, it);
  it.k0 = (int)((int64_t)kb * sp / g.splits);
  it.k1 = (int)((int64_t)kb * (sp + 1) / g.splits);
  it.part = (int)w;
  return it;
}

// kAny: outputs and residuals whose rows may lie at any address; without it they
// are 16-byte aligned, which the kernels that most calls take are built for.
template <int CG, int NB, int EW, bool kAny, int MA, int MB, bool kFp8, bool kGated>
__global__ void __launch_bounds__(128 + 32 * EW, 1) k_gemm(const __grid_constant__ Maps maps, const __grid_constant__ Args g) {
  using S = Shape<CG, NB, EW>;
  constexpr int kBk = kFp8 ? 128 : 64;  // k of one stage
  constexpr int kTileN = kGated ? NB / 2 : NB;
  constexpr int kGroups = kTileN / 32 < EW / 4 ? kTileN / 32 : EW / 4;  // epilogue warps share a tile's columns
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = base + S::kStages * S::kStage;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (S::kStages + s); };
  auto tfull = [&](int b) { return bars + 8u * (2 * S::kStages + b); };
  auto tempty = [&](int b) { return bars + 8u * (2 * S::kStages + 2 + b); };
  const uint32_t drained = bars + 8u * (2 * S::kStages + 4);
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;

  // The warp's number in a uniform register: the loads' and products' warps run
  // their loops as whole warps with uniform operands and elect a lane only to
  // issue.  With one lane in a branch of its own each operand of each product is
  // moved on its way: 0.31 us a k block whatever its size, against 0.19 us (128
  // columns) and 0.28 us (256).
  pdl_begin();
  const int warp = __shfl_sync(kFull, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cta_rank() : 0u;
  if (threadIdx.x == 0) {
    abort_s = 0;
    for (int s = 0; s < S::kStages; ++s) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full(s)) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(empty(s)) : "memory");
    }
    for (int b = 0; b < 2; ++b) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(tfull(b)) : "memory");
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(tempty(b)), "r"(CG * 4 * kGroups) : "memory");
    }
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(drained) : "memory");
    fence_mbar_init();
  }
  if (warp == 2) tmem_alloc<CG>(smem_u32(&tmem_base_s), S::kCols);
  fence_before();
  if (CG == 2) cluster_sync(); else __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_base_s;
  pdl_wait();

  const uint32_t items = tiles_of(g) * (uint32_t)g.splits;
  const uint32_t first = blockIdx.x / CG, step = gridDim.x / CG;
  volatile int* const aborted = &abort_s;

  if (warp == 0) {
    // ---- loads
    int s = 0;
    uint32_t ph = 0;
    int64_t loads = 0;
    bool ok = true;
    for (uint32_t w = first; ok && w < items; w += step) {
      const Item it = item_of(g, w);
      const int row_a = (it.mt * CG + (int)rank) * kRowsA;
      for (int kb = it.k0; kb < it.k1; ++kb) {
        ok = __all_sync(kFull, *aborted == 0 && wait_bar(empty(s), ph ^ 1u, kWaitNs));
        if (!ok) break;
        const uint32_t bar = CG == 2 ? map_to_rank(full(s), 0) : full(s);
        const int seg = g.dual == kDualK && kb >= g.kb ? 1 : 0;
        const int k = (kb - seg * g.kb) * kBk;
        const CUtensorMap* ma = &maps.a[g.dual == kDualM ? it.prob : seg];
        const CUtensorMap* mb = &maps.b[seg];
        const uint32_t da = base + s * S::kStage, db = da + S::kBytesA;
        if (elect_one()) {
          if (rank == 0) expect_bytes(full(s), g.stage_bytes);
          if (MA == kMajorK) {
            tma_load<CG>(da, ma, k, row_a, bar);
          } else {
#pragma unroll
            for (int c = 0; c < kRowsA / 64; ++c) tma_load<CG>(da + c * 8192, ma, row_a + 64 * c, k, bar);
          }
          if (kGated) {
            // gate rows in the accumulator's first half, up rows in its second
            if (CG == 2) {
              tma_load<CG>(db, &maps.b[rank], k, it.nt * kTileN, bar);
            } else {
              tma_load<CG>(db, &maps.b[0], k, it.nt * kTileN, bar);
              tma_load<CG>(db + S::kBytesB / 2, &maps.b[1], k, it.nt * kTileN, bar);
            }
          } else {
            const int row_b = it.nt * NB + (int)rank * S::kRowsB;
            if (MB == kMajorK) {
              tma_load<CG>(db, mb, k, row_b, bar);
            } else {
#pragma unroll
              for (int c = 0; c < S::kRowsB / 64; ++c) tma_load<CG>(db + c * 8192, mb, row_b + 64 * c, k, bar);
            }
          }
        }
        __syncwarp();
        ++loads;
        if (++s == S::kStages) {
          s = 0;
          ph ^= 1u;
        }
      }
    }
    // Until the products have read the last copies: none is in flight into a CTA
    // that has left.
    for (int64_t l = loads > S::kStages ? loads - S::kStages : 0; ok && l < loads; ++l)
      ok = __all_sync(kFull, *aborted == 0 && wait_bar(empty((int)(l % S::kStages)),
                                                       (uint32_t)((l / S::kStages) & 1), kWaitNs));
    if (!ok) {
      *aborted = 1;
      if (lane == 0) give_up(g, kTimeoutCopy, 0);
      // Products that gave up read no more, so the copies' arrival cannot be waited
      // for there, nor in a pair at the first CTA's barriers, whose count needs
      // both CTAs' loads: they have landed long before this has passed.
      for (const uint64_t t0 = globaltimer(); globaltimer() - t0 < kDrainNs;) __nanosleep(1000);
    }
  } else if (warp == 1 && rank == 0) {
    // ---- products
    int s = 0;
    uint32_t ph = 0;
    int buf = 0;
    uint32_t bph = 0;
    bool ok = true;
    const uint64_t desc_a = smem_desc<MA>(base), desc_b = smem_desc<MB>(base + S::kBytesA);
    for (uint32_t w = first; ok && w < items; w += step) {
      const Item it = item_of(g, w);
      ok = __all_sync(kFull, *aborted == 0 && wait_bar<CG == 2>(tempty(buf), bph ^ 1u, kWaitNs));
      if (!ok) break;
      fence_after();
      const uint32_t d = tmem + buf * NB;
      for (int kb = it.k0; kb < it.k1; ++kb) {
        ok = __all_sync(kFull, wait_bar(full(s), ph, kWaitNs));
        if (!ok) break;
        fence_after();
        // addresses are the low bits of a descriptor, in units of 16 bytes
        const uint64_t sa = desc_a + (uint64_t)(s * (S::kStage >> 4)), sb = desc_b + (uint64_t)(s * (S::kStage >> 4));
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma<CG, kFp8>(d, sa + j * (kStep<MA> >> 4), sb + j * (kStep<MB> >> 4), g.idesc,
                          (kb > it.k0 || j > 0) ? 1u : 0u);
          commit<CG>(empty(s));
        }
        __syncwarp();
        if (++s == S::kStages) {
          s = 0;
          ph ^= 1u;
        }
      }
      if (elect_one()) commit<CG>(tfull(buf));
      __syncwarp();
      if (++buf == 2) {
        buf = 0;
        bph ^= 1u;
      }
    }
    if (!ok) {
      *aborted = 1;
      if (lane == 0) give_up(g, kTimeoutPayload, 1);
      if (elect_one()) commit<CG>(drained);
      __syncwarp();
      wait_bar(drained, 0, kDrainNs);
    }
  } else if (warp >= 4 && warp < 4 + 4 * kGroups) {
    // ---- epilogue
    const int quad = warp & 3, part = (warp - 4) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    const EpiVec ev = epi_vec(g.ep);
    Piece pc;
    pc.smem = base + S::kStages * S::kStage + S::kBarBytes + (uint32_t)(warp - 4) * kStageBytes;
    pc.lane = lane;
    const int unit_cols = g.ep.out_type == kF32 ? 4 : 8;  // of the residual in 16 bytes
    const bool res_units = !kGated && g.ep.residual != nullptr && ev.res && g.n % unit_cols == 0;
    const int64_t res_ld = g.ep.ldr * (g.ep.out_type == kF32 ? 4 : 2);
    int buf = 0;
    uint32_t bph = 0;
    for (uint32_t w = first; w < items; w += step) {
      const Item it = item_of(g, w);
      const int64_t row0 = (int64_t)(it.mt * CG + (int)rank) * kRowsA + quad * 32, row = row0 + lane;
      const bool inside = row < g.m;
      auto place = [&](int c) {
        pc.row0 = row0;
        pc.col = (int64_t)it.nt * kTileN + c;
        pc.rows = (int)max64(0, min64(32, g.m - row0));
        pc.cols = (int)max64(0, min64(32, g.n - pc.col));
      };
      constexpr int kColsW = kTileN / kGroups;  // columns of a warp
      uint4 res[4];
      if (res_units) {
        place(part * kColsW);
        fetch_units(pc, g.ep.residual, res_ld, unit_cols, 0, res);
      }
      // the whole warp's decision: what follows reads tensor memory as a whole warp
      if (!__all_sync(kFull, *aborted == 0 && wait_bar(tfull(buf), bph, kWaitNs))) {
        *aborted = 1;
        if (lane == 0) give_up(g, kTimeoutResult, 2);
        break;
      }
      __syncwarp();
      fence_after();
      const uint32_t acc = lanes + buf * NB;
#pragma unroll 1
      for (int c = part * kColsW; c < (part + 1) * kColsW; c += 32) {
        place(c);
        if (pc.rows <= 0 || pc.cols <= 0) break;  // the same for the whole warp
        const int64_t col = pc.col;
        const int valid = inside ? pc.cols : 0;
        float v[32];
        tmem_load32(acc + c, v);
        if (it.part >= 0) {
          // this CTA's rows of the slot, all of them: the join looks at the sizes
          Piece q = {pc.smem, (int64_t)((int)rank * kRowsA + quad * 32), c, 32, 32, lane};
          float* p = g.partial + (int64_t)it.part * (CG * kRowsA * NB);
          write_piece<false>(q, p, NB, kF32, true, v);
          if constexpr (kGated) {
            tmem_load32(acc + kTileN + c, v);
            q.col += kTileN;
            write_piece<false>(q, p, NB, kF32, true, v);
          }
          continue;
        }
        epi_sums<32>(g.ep, ev, 0, inside ? row : 0, col, valid, v);
        if (g.ep.z_hi[0] != nullptr) write_kept(pc, g.ep.z_hi[0], g.ep.z_lo[0], g.ep.ldz, v);
        if constexpr (kGated) {
          float u[32];
          tmem_load32(acc + kTileN + c, u);
          act_run<32>(g.ep.act, v);
          epi_sums<32>(g.ep, ev, 1, inside ? row : 0, col, valid, u);
          if (g.ep.z_hi[1] != nullptr) write_kept(pc, g.ep.z_hi[1], g.ep.z_lo[1], g.ep.ldz, u);
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= u[j];
        } else {
          act_run<32>(g.ep.act, v);
          if (res_units) {
            add_units(pc, res, g.ep.out_type, 0, v);
            if (g.ep.out_type == kF32) {
              fetch_units(pc, g.ep.residual, res_ld, unit_cols, 1, res);
              add_units(pc, res, kF32, 1, v);
            }
            if (c + 32 < (part + 1) * kColsW) {  // the next piece's, while this one is written
              place(c + 32);
              fetch_units(pc, g.ep.residual, res_ld, unit_cols, 0, res);
              place(c);
            }
          } else if (kAny && g.ep.residual != nullptr) {
            add_plain(pc, g.ep.residual, g.ep.ldr, g.ep.out_type, v);
          }
        }
        write_piece<kAny>(pc, g.ep.out[it.prob], g.ep.ldo, g.ep.out_type, ev.out, v);
      }
      fence_before();
      __syncwarp();
      if (lane == 0) arrive_leader<CG>(tempty(buf));
      if (++buf == 2) {
        buf = 0;
        bph ^= 1u;
      }
    }
  }
  __syncwarp();
  fence_before();
  if (CG == 2) cluster_sync(); else __syncthreads();
  fence_after();
  if (warp == 2) tmem_free<CG>(tmem, S::kCols);
}

template <int CG, int NB, int EW, bool kAny, int MA, int MB, bool kFp8, bool kGated>
cudaError_t launch(const Maps& maps, const Args& args, int sms, cudaStream_t s) {
  using S = Shape<CG, NB, EW>;
  auto* fn = &k_gemm<CG, NB, EW, kAny, MA, MB, kFp8, kGated>;
  // holds for the current device alone, so every launch sets it
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (e != cudaSuccess) return e;
  const int64_t tiles = (int64_t)args.mt * (args.dual == kDualM ? 2 : 1) * args.nt;
  const int64_t items = tiles * args.splits;
  return launch_dependent(fn, dim3((unsigned)(CG * std::min<int64_t>(items, sms / CG))), dim3(S::kThreads), S::kSmem, CG,
                          s, maps, args);
}

template <int EW, bool kAny, int MA, int MB, bool kFp8, bool kGated>
cudaError_t launch_shape(const Gemm& g, const Maps& maps, const Args& args, int sms, cudaStream_t s) {
  if (g.cg == 2)
    return g.nb == 256 ? launch<2, 256, EW, kAny, MA, MB, kFp8, kGated>(maps, args, sms, s)
                       : launch<2, 128, EW, kAny, MA, MB, kFp8, kGated>(maps, args, sms, s);
  return g.nb == 256 ? launch<1, 256, EW, kAny, MA, MB, kFp8, kGated>(maps, args, sms, s)
                     : launch<1, 128, EW, kAny, MA, MB, kFp8, kGated>(maps, args, sms, s);
}

// The families of kernels, a source file each.  busy: the epilogue takes as long
// as the products; aligned: rows of outputs and residual on 16 bytes.
struct Call {
  const Maps* maps;
  const Args* args;
  int sms;
  bool busy, aligned;
  cudaStream_t s;
};
cudaError_t launch_linear(const Gemm& g, const Call& c);  // both operands with k contiguous
cudaError_t launch_gated(const Gemm& g, const Call& c);
cudaError_t launch_8bit(const Gemm& g, const Call& c);    // linear and gated
cudaError_t launch_gradient(const Gemm& g, const Call& c);  // B, or both, with rows contiguous

}  // namespace dense
}  // namespace ngl

// Dense half of a decoder layer (csrc/cuda/dense_gemm.cuh, dense_skinny.cu,
// dense_elem.cu): the matrix product with bias, activation and residual in
// its epilogue, the gated product of two projections, and their backward
// passes.  No counterpart in the reference, whose models run stock layers.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ngl {
namespace dense {

enum Type : int { kF32 = 0, kBF16 = 1, kF16 = 2, kE4M3 = 3 };
enum Act : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };

// How an operand [rows, k] lies in memory: kMajorK with k contiguous,
// kMajorMN with rows contiguous (that is, stored as [k, rows]).
enum Major : int { kMajorK = 0, kMajorMN = 1 };

// A matrix product reads one operand of each side, or two (see Dual).
//   kDualNone  D = A0 B0^T
//   kDualN     D = (A0 B0^T, A0 B1^T): the two projections of the gated form
//   kDualK     D = A0 B0^T + A1 B1^T
//   kDualM     D0 = A0 B0^T and D1 = A1 B0^T
enum Dual : int { kDualNone = 0, kDualN = 1, kDualK = 2, kDualM = 3 };

// What follows the sums.  z = acc * row_scale[i] * col_scale[j] + bias[j];
// out = act(z) + residual, or act(z) * z1 in the gated form, whose z1 is the
// second projection's.  Null pointers leave their part out.
struct Epilogue {
  int act;
  int half_type;   // kBF16 or kF16: type of bias, z, and of out/residual where not fp32
  int out_type;    // of out and residual: half_type or kF32
  void* out[2];    // [m, n] each, row stride ldo; the second for kDualM
  int64_t ldo;
  uint16_t* z_hi[2];  // pre-activations kept for the backward pass: the upper 16
  uint8_t* z_lo[2];   // bits of fp32 and the next 8, row stride ldz = kept_ld(n)
  int64_t ldz;
  const void* bias;
  const void* residual;
  int64_t ldr;
  const float* row_scale;     // [m], 8-bit operands only
  const float* col_scale[2];  // [n]
};

inline int64_t kept_ld(int64_t n) { return (n + 15) / 16 * 16; }

struct Operand {
  const void* p;
  int64_t ld;  // elements between consecutive rows of the stored matrix
};

struct Gemm {
  int64_t m, n, k;
  int type;  // kBF16, kF16, kE4M3
  int major_a, major_b;
  int dual;
  Operand a[2], b[2];
  Epilogue ep;
  float* partial;  // partial_floats(): sums of the pieces of k, when splits > 1
  int splits;
  int cg, nb;      // CTAs per tile (1 or 2), accumulator columns of a tile
};

// Choose cg, nb and splits of a product for `sms` SMs (g.m, n, k, dual set);
// may_split allows splits > 1.
void plan(Gemm& g, int sms, bool may_split);
// Every following product takes this plan (tests and measurements of one tile
// shape); cg = 0 returns to plan().
void force_plan(int cg, int nb, int splits);
int64_t partial_floats(const Gemm& g);

// Enqueue the product.  Every operand must be fit for TMA: base 16-byte
// aligned, row stride a multiple of 16 bytes.  Returns a CUDA
// error, or cudaErrorInvalidValue when a tensor map cannot be made.
cudaError_t gemm(const Gemm& g, int sms, cudaStream_t s);

// Few rows (m <= kSkinnyRows): one pass over the weights, any alignment.
// x [m, k] ldx, w [n, k] ldw (two for the gated form).
constexpr int kSkinnyRows = 16;
struct Skinny {
  int64_t m, n, k;
  int type;
  bool gated;
  Operand x, w[2];
  Epilogue ep;
};
cudaError_t skinny(const Skinny& g, int sms, cudaStream_t s);

// ---- elementwise parts of the backward passes
// dz = dy * act'(z) in half_type (act none: dz = dy, a cast; z is not read),
// db[j] = sum_i dz: partial [parts, n] is scratch for db (null: no db).  dy of
// dy_type; dz null: only db.
int colsum_parts(int64_t m, int64_t n, int sms);
cudaError_t act_backward(const void* dy, int dy_type, int64_t ldy, const uint16_t* z_hi, const uint8_t* z_lo, int act,
                         int half_type, int64_t m, int64_t n, void* dz, int64_t ldd, float* partial, int parts, void* db,
                         cudaStream_t s);
// out[j] = sum of partial[p, j] over p < parts.
cudaError_t colsum(const float* partial, int parts, int64_t n, void* out, int type, cudaStream_t s);
// dg = dh * u * act'(g), du = dh * act(g); z_hi/z_lo[0] hold g, [1] u.
cudaError_t gated_backward(const void* dh, int64_t ldh, const uint16_t* const z_hi[2], const uint8_t* const z_lo[2],
                           int act, int half_type, int64_t m, int64_t n, void* dg, void* du, int64_t ldd, int sms,
                           cudaStream_t s);
// Matrices of `elem`-byte elements copied, up to four in one launch: cols
// elements a row to a row stride of ldd (a multiple of 128 bytes), the tail zeroed.
struct Copy {
  const void* src;
  int64_t lds;
  void* dst;
  int64_t ldd, rows, cols;
};
struct Copies {
  Copy m[4];
  int n;
};
cudaError_t repack(const Copies& c, int elem, cudaStream_t s);

// Status of the current device's products since it was cleared: {code, CTA, role, 0},
// the code of ngl_cuda.cuh; waits for stream s.
cudaError_t read_status(int* out4, bool clear, cudaStream_t s);
// The copy of those words that kernels write into host memory, or null where no
// product has been started on the device; reading it waits for nothing.
int* status_seen(int dev);

}  // namespace dense
}  // namespace ngl

// Matrix products on the tensor cores: plans, tensor maps and launches, and the
// join of products whose k is split (dense_gemm.cuh has the kernel).
#include "dense_gemm.cuh"

#include <atomic>
#include <cstring>
#include <mutex>

namespace ngl {
namespace dense {
namespace {

__device__ int g_status[4];

// A device's status words, and their copy in host memory, which a kernel that
// gives up writes too: the host sees it at its next call, without asking the GPU.
struct Words {
  int* device;
  int* host;
};
constexpr int kMaxDevices = 64;
Words g_words[kMaxDevices];
std::atomic<bool> g_words_known[kMaxDevices];

// Those of device dev, the current one; found and allocated once a device.
cudaError_t status_words(int dev, Words* w) {
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (!g_words_known[dev].load(std::memory_order_acquire)) {
    static std::mutex m;
    const std::lock_guard<std::mutex> lock(m);
    if (!g_words_known[dev].load(std::memory_order_relaxed)) {
      void *d = nullptr, *h = nullptr;
      // allowed while a graph is captured: it is no work on a stream
      cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
      cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
      if (e == cudaSuccess) {
        e = cudaGetSymbolAddress(&d, g_status);
        if (e == cudaSuccess) e = cudaHostAlloc(&h, 4 * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
        const cudaError_t back = cudaThreadExchangeStreamCaptureMode(&mode);
        if (e == cudaSuccess) e = back;
      }
      if (e != cudaSuccess) return e;
      std::memset(h, 0, 4 * sizeof(int));
      g_words[dev] = {static_cast<int*>(d), static_cast<int*>(h)};
      g_words_known[dev].store(true, std::memory_order_release);
    }
  }
  *w = g_words[dev];
  return cudaSuccess;
}

// Sum of a tile's pieces in their order, then the epilogue.  One thread takes 8
// columns of one row; rows x nb: a slot of `partial`.
template <bool kGated>
__global__ void __launch_bounds__(256) k_join(const __grid_constant__ Args g, int rows, int nb) {
  pdl_begin();
  pdl_wait();
  const int tile_n = kGated ? nb / 2 : nb, runs = tile_n / 8;
  const EpiVec ev = epi_vec(g.ep);
  const int64_t total = (int64_t)tiles_of(g) * rows * runs;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / runs;
    const int c = (int)(i - r * runs) * 8;
    const int64_t tile = r / rows;
    const int rr = (int)(r - tile * rows);
    Item it;
    tile_of(g, (uint32_t)tile, it);
    const int64_t row = (int64_t)it.mt * rows + rr, col = (int64_t)it.nt * tile_n + c;
    if (row >= g.m || col >= g.n) continue;
    float v[8] = {}, u[8] = {};
    const float* p = g.partial + tile * g.splits * rows * nb + (int64_t)rr * nb + c;
    for (int s = 0; s < g.splits; ++s, p += (int64_t)rows * nb) {
      float t[8];
      get_run<8>(p, 0, kF32, 8, true, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += t[j];
      if (kGated) {
        get_run<8>(p, tile_n, kF32, 8, true, t);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] += t[j];
      }
    }
    if (kGated)
      epilogue_gated_run<8>(g.ep, ev, row, col, g.n, v, u);
    else
      epilogue_run<8>(g.ep, ev, it.prob, row, col, g.n, v);
  }
}

// ------------------------------------------------------------------ host
// The driver's tensor-map encoder, found at run time: the library loads on
// machines without a driver (builds, CPU tests).
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

bool make_map(CUtensorMap* map, const Operand& o, int type, int major, int64_t rows, int64_t k, int box_rows) {
  const int elem = type_bytes(type);
  const cuuint64_t dims[2] = {(cuuint64_t)(major == kMajorK ? k : rows), (cuuint64_t)(major == kMajorK ? rows : k)};
  const cuuint64_t strides[1] = {(cuuint64_t)(o.ld * elem)};
  const cuuint32_t box[2] = {(cuuint32_t)(kBlockBytes / elem), (cuuint32_t)(major == kMajorK ? box_rows : 64)};
  const cuuint32_t es[2] = {1, 1};
  const CUtensorMapDataType dt = type == kBF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                 : type == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const EncodeFn encode = encoder();
  return encode(map, dt, 2, const_cast<void*>(o.p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Instruction descriptor: fp32 sums, operand types and orders, tile size.
uint32_t make_idesc(const Gemm& g) {
  const uint32_t t = g.type == kBF16 ? 1u : 0u;  // f16 and e4m3 are both 0 in their kinds
  return (1u << 4) | (t << 7) | (t << 10) | ((uint32_t)(g.major_a == kMajorMN) << 15) |
         ((uint32_t)(g.major_b == kMajorMN) << 16) | ((uint32_t)(g.nb / 8) << 17) | ((uint32_t)(128 * g.cg / 16) << 24);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

namespace {
int64_t tile_count(const Gemm& g) {
  return ceil_div(g.m, kRowsA * g.cg) * (g.dual == kDualM ? 2 : 1) * ceil_div(g.n, g.dual == kDualN ? g.nb / 2 : g.nb);
}
int g_force[3] = {0, 0, 0};
}  // namespace

int64_t partial_floats(const Gemm& g) {
  return g.splits > 1 ? tile_count(g) * g.splits * g.cg * kRowsA * g.nb : 0;
}

void force_plan(int cg, int nb, int splits) {
  g_force[0] = cg;
  g_force[1] = nb;
  g_force[2] = splits;
}

void plan(Gemm& g, int sms, bool may_split) {
  const int bk = g.type == kE4M3 ? 128 : 64;
  const int64_t kb = ceil_div(g.k, bk) * (g.dual == kDualK ? 2 : 1);
  if (g_force[0] != 0) {
    g.cg = g_force[0];
    g.nb = g_force[1];
    // at least one k block a piece: a piece without any has no sums to store
    g.splits = may_split ? (int)std::min<int64_t>(g_force[2], kb) : 1;
    return;
  }
  // Time of a plan = waves of tiles x the longer of their products and their
  // epilogue + the first fill and the last epilogue + the join of pieces of k.
  // Microseconds of a k block and of an epilogue as measured on a busy GPU with
  // 8192 x 5632 x 2048 and 8192 x 2048 x 256: tiles of 128 columns take 0.6 of
  // the time of 256 columns for half of the work, so they win where they fill
  // the last wave, or where the epilogue rules; a pair of CTAs saves a third of
  // the operand bytes, but its epilogues wait for one another.  The join is a
  // launch of its own (128 x 5632 x 2048 in three pieces 12.9 us, whole 11.4;
  // 64 x 2048 x 5632 in four 12.6 us, whole 22.5), so k is split only where tiles
  // leave most SMs idle.  Splitting the tiles behind
  // the last full wave gained nothing: a busy GPU runs at its power limit, and a
  // wave half empty at a higher clock.  Products of 8 bits take the same times for
  // twice the k of a block; planned and best plan there: 2048 x 5632 x 2048 25.0
  // and 25.0 us, 2048 x 2048 x 5632 23.3 and 23.3, 8192 x 5632 x 2048 96 and 92,
  // 777 x 5632 x 2048 21.5 and 18.3.
  double best = 1e30;
  Gemm c = g;
  for (c.cg = 2; c.cg >= 1; --c.cg)
    for (c.nb = 256; c.nb >= 128; c.nb -= 128) {
      const double t_kb = c.nb == 256 ? (c.cg == 2 ? 0.36 : 0.39) : (c.cg == 2 ? 0.23 : 0.24);
      const double t_epi = c.nb == 256 ? (c.cg == 2 ? 5.2 : 3.6) : (c.cg == 2 ? 3.0 : 2.1);
      const int64_t slots = sms / c.cg, tiles = tile_count(c);
      for (c.splits = 1; c.splits <= 32 && c.splits <= std::max<int64_t>(1, kb / 4); ++c.splits) {
        if (c.splits > 1 && (!may_split || tiles * c.splits > slots)) break;
        double t = ceil_div(tiles * c.splits, slots) * std::max(ceil_div(kb, c.splits) * t_kb + 0.3, t_epi) + t_epi;
        if (c.splits > 1) t += 6.0 + 2.0 * 4 * tiles * c.splits * c.cg * kRowsA * c.nb / 5e6;
        if (t < best * 0.999) {
          best = t;
          g.cg = c.cg;
          g.nb = c.nb;
          g.splits = c.splits;
        }
      }
    }
}

cudaError_t gemm(const Gemm& g, int sms, cudaStream_t s) {
  if (g.m <= 0 || g.n <= 0 || g.k <= 0) return cudaErrorInvalidValue;
  if (tile_count(g) * g.splits >= (int64_t(1) << 30)) return cudaErrorInvalidValue;  // 2^44 outputs
  if (encoder() == nullptr) return cudaErrorNotSupported;
  // The encoder is a driver call and needs a current context, which a thread
  // of autograd's may not have yet: setting the device makes it current.
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaSetDevice(dev);
  if (e != cudaSuccess) return e;
  const int bk = g.type == kE4M3 ? 128 : 64;
  const bool gated = g.dual == kDualN;
  const int tn = gated ? g.nb / 2 : g.nb;
  // Few rows: a box of 32 rows instead of 128, whose other rows of shared memory
  // then hold anything; they are rows of the accumulator that nothing reads.
  // (With 128, fewer than 32 rows took 3 us longer than 32 of them.)
  const int box_a = g.cg == 1 && g.major_a == kMajorK && g.m <= 32 ? 32 : kRowsA;
  Maps maps;
  std::memset(&maps, 0, sizeof(maps));
  const int na = g.dual == kDualK || g.dual == kDualM ? 2 : 1, nbm = g.dual == kDualK || gated ? 2 : 1;
  for (int i = 0; i < 2; ++i) {
    if (i < na && !make_map(&maps.a[i], g.a[i], g.type, g.major_a, g.m, g.k, box_a))
      return cudaErrorInvalidValue;
    if (i < nbm && !make_map(&maps.b[i], g.b[i], g.type, g.major_b, g.n, g.k, gated ? g.nb / 2 : g.nb / g.cg))
      return cudaErrorInvalidValue;
  }
  Args args;
  args.m = g.m;
  args.n = g.n;
  args.mt = (int)ceil_div(g.m, kRowsA * g.cg);
  args.nt = (int)ceil_div(g.n, tn);
  args.kb = (int)ceil_div(g.k, bk);
  args.dual = g.dual;
  args.splits = g.splits;
  args.idesc = make_idesc(g);
  args.stage_bytes = (uint32_t)(g.cg * kBlockBytes * (box_a + g.nb / g.cg));
  args.partial = g.partial;
  args.ep = g.ep;
  Words words;
  e = status_words(dev, &words);
  if (e != cudaSuccess) return e;
  args.status = words.device;
  args.status_host = words.host;
  // 16 k blocks take about as long as an epilogue with an activation
  const int out_bytes = type_bytes(g.ep.out_type);
  Call call;
  call.maps = &maps;
  call.args = &args;
  call.sms = sms;
  call.s = s;
  call.aligned = g.splits > 1 || (g.n % (16 / out_bytes) == 0 && runs_aligned(g.ep.out[0], g.ep.ldo, out_bytes) &&
                 runs_aligned(g.ep.out[1], g.ep.ldo, out_bytes) && runs_aligned(g.ep.residual, g.ep.ldr, out_bytes));
  call.busy = args.kb <= 16;
  if (g.type == kE4M3)
    e = launch_8bit(g, call);
  else if (gated)
    e = launch_gated(g, call);
  else if (g.major_a == kMajorK && g.major_b == kMajorK)
    e = launch_linear(g, call);
  else if (g.major_b == kMajorMN)
    e = launch_gradient(g, call);
  else
    return cudaErrorInvalidValue;
  if (e != cudaSuccess || g.splits == 1) return e;
  const int64_t runs = tile_count(g) * g.cg * kRowsA * tn / 8;
  const int grid = (int)std::min<int64_t>(ceil_div(runs, 256), (int64_t)sms * 8);
  return launch_dependent(gated ? &k_join<true> : &k_join<false>, dim3(grid), dim3(256), 0, 1, s, args,
                          g.cg * kRowsA, g.nb);
}

cudaError_t read_status(int* out4, bool clear, cudaStream_t s) {
  int dev = 0;
  Words w;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = status_words(dev, &w);
  if (e != cudaSuccess) return e;
  e = cudaMemcpyAsync(out4, w.device, 4 * sizeof(int), cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess && clear) e = cudaMemsetAsync(w.device, 0, 4 * sizeof(int), s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return e;
  volatile int* h = w.host;
  if (out4[0] == 0)
    for (int i = 0; i < 4; ++i) out4[i] = h[i];
  if (clear)
    for (int i = 0; i < 4; ++i) h[i] = 0;
  return cudaSuccess;
}

int* status_seen(int dev) {
  if (dev < 0 || dev >= kMaxDevices || !g_words_known[dev].load(std::memory_order_acquire)) return nullptr;
  return g_words[dev].host;
}

}  // namespace dense
}  // namespace ngl

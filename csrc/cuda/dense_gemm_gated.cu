// The gated product of two projections, 16-bit (dense_gemm.cuh).
#include "dense_gemm.cuh"

namespace ngl {
namespace dense {

cudaError_t launch_gated(const Gemm& g, const Call& c) {
  return c.aligned ? launch_shape<8, false, kMajorK, kMajorK, false, true>(g, *c.maps, *c.args, c.sms, c.s)
                   : launch_shape<8, true, kMajorK, kMajorK, false, true>(g, *c.maps, *c.args, c.sms, c.s);
}

}  // namespace dense
}  // namespace ngl

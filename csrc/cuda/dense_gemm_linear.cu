// Products of two operands with k contiguous, 16-bit (dense_gemm.cuh).
#include "dense_gemm.cuh"

namespace ngl {
namespace dense {

cudaError_t launch_linear(const Gemm& g, const Call& c) {
  if (!c.aligned) return launch_shape<8, true, kMajorK, kMajorK, false, false>(g, *c.maps, *c.args, c.sms, c.s);
  return c.busy ? launch_shape<16, false, kMajorK, kMajorK, false, false>(g, *c.maps, *c.args, c.sms, c.s)
                : launch_shape<8, false, kMajorK, kMajorK, false, false>(g, *c.maps, *c.args, c.sms, c.s);
}

}  // namespace dense
}  // namespace ngl

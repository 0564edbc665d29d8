// Products of the backward passes: an operand with its rows contiguous (dense_gemm.cuh).
#include "dense_gemm.cuh"

namespace ngl {
namespace dense {

cudaError_t launch_gradient(const Gemm& g, const Call& c) {
  if (g.major_a == kMajorK)
    return c.aligned ? launch_shape<8, false, kMajorK, kMajorMN, false, false>(g, *c.maps, *c.args, c.sms, c.s)
                     : launch_shape<8, true, kMajorK, kMajorMN, false, false>(g, *c.maps, *c.args, c.sms, c.s);
  return c.aligned ? launch_shape<8, false, kMajorMN, kMajorMN, false, false>(g, *c.maps, *c.args, c.sms, c.s)
                   : launch_shape<8, true, kMajorMN, kMajorMN, false, false>(g, *c.maps, *c.args, c.sms, c.s);
}

}  // namespace dense
}  // namespace ngl

// Products of 8-bit operands (dense_gemm.cuh).
#include "dense_gemm.cuh"

namespace ngl {
namespace dense {

cudaError_t launch_8bit(const Gemm& g, const Call& c) {
  if (g.dual == kDualN)
    return c.aligned ? launch_shape<8, false, kMajorK, kMajorK, true, true>(g, *c.maps, *c.args, c.sms, c.s)
                     : launch_shape<8, true, kMajorK, kMajorK, true, true>(g, *c.maps, *c.args, c.sms, c.s);
  if (!c.aligned) return launch_shape<8, true, kMajorK, kMajorK, true, false>(g, *c.maps, *c.args, c.sms, c.s);
  return c.busy ? launch_shape<16, false, kMajorK, kMajorK, true, false>(g, *c.maps, *c.args, c.sms, c.s)
                : launch_shape<8, false, kMajorK, kMajorK, true, false>(g, *c.maps, *c.args, c.sms, c.s);
}

}  // namespace dense
}  // namespace ngl

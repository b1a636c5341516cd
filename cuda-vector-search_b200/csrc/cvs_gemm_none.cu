// The linear layer's product without an activation.
#include "cvs_gemm.cuh"

namespace cvs {

cudaError_t gemm_launch_none(int cg, int bn, const GemmMaps& maps, const GemmArgs& a, int ctas, cudaStream_t stream) {
  return gemm_launch_act<kActNone>(cg, bn, maps, a, ctas, stream);
}

}  // namespace cvs

// The linear layer's product with GELU.
#include "cvs_gemm.cuh"

namespace cvs {

cudaError_t gemm_launch_gelu(int cg, int bn, const GemmMaps& maps, const GemmArgs& a, int ctas, cudaStream_t stream) {
  return gemm_launch_act<kActGelu>(cg, bn, maps, a, ctas, stream);
}

}  // namespace cvs

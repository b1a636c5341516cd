// The linear layer's product with SiLU.
#include "cvs_gemm.cuh"

namespace cvs {

cudaError_t gemm_launch_silu(int cg, int bn, const GemmMaps& maps, const GemmArgs& a, int ctas, cudaStream_t stream) {
  return gemm_launch_act<kActSilu>(cg, bn, maps, a, ctas, stream);
}

}  // namespace cvs

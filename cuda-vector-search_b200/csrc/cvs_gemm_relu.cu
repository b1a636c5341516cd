// The linear layer's product with ReLU.
#include "cvs_gemm.cuh"

namespace cvs {

cudaError_t gemm_launch_relu(int cg, int bn, const GemmMaps& maps, const GemmArgs& a, int ctas, cudaStream_t stream) {
  return gemm_launch_act<kActRelu>(cg, bn, maps, a, ctas, stream);
}

}  // namespace cvs

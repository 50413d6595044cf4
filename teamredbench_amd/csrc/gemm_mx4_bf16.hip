// The pipelined MX4 products with bf16 output (gemm_mx4_kernels.hpp).
#include "gemm_mx4_kernels.hpp"

namespace mb {

int gemm_mx4_tiled_bf16(const Mx4Call& c, const Mx4Plan& plan, int cus, void* workspace, hipStream_t stream) {
    return launch_mx4_config<MB_DT_BFLOAT16>(c, plan, cus, workspace, stream);
}

}  // namespace mb

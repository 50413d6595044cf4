// The pipelined grouped products for one input type.
#include "gemm_grouped_kernels.hpp"

namespace mb {

int gemm_grouped_tiled_bf16(const GroupedCall& c, const GroupedPlan& plan, void* workspace, hipStream_t stream) {
    return launch_grouped_dtype<MB_DT_BFLOAT16>(c, plan, workspace, stream);
}

}  // namespace mb

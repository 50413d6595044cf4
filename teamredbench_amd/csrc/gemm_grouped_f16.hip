// The pipelined grouped products for one input type.
#include "gemm_grouped_kernels.hpp"

namespace mb {

int gemm_grouped_tiled_f16(const GroupedCall& c, int config, hipStream_t stream) {
    return launch_grouped_dtype<MB_DT_FLOAT16>(c, config, stream);
}

}  // namespace mb

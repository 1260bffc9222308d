// gemm_grouped16.cu — the f16 / bf16 instantiations of gemm_blk_kernel.
#include "gemm_blk_launch.cuh"

namespace futon {
cudaError_t launch_blk_16(const BlkLaunch& g) { return launch_blk_any<false>(g); }
}  // namespace futon

// gemm_f8.cu — the block-scaled e4m3 instantiations of gemm_blk_kernel.
#include "gemm_blk_launch.cuh"

namespace futon {
cudaError_t launch_blk_f8(const BlkLaunch& g) { return launch_blk_any<true>(g); }
}  // namespace futon

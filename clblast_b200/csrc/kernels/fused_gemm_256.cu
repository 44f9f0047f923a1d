// Instances of the fused product kernel: one CTA per 128 x 256 tile.
#include "fused_gemm.cuh"

namespace b200 {

cudaError_t launch_fused_256(int type, int d_type, int c_type, const CUtensorMap* maps, const FusedParams& p, int grid,
                            int smem, cudaStream_t stream) {
  return fused::launch_by_type<1, 256>(type, d_type, c_type, maps, p, grid, smem, stream);
}

}  // namespace b200

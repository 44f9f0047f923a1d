// Instances of the fused product kernel: pairs of CTAs, 256 x 128 tiles.
#include "fused_gemm.cuh"

namespace b200 {

cudaError_t launch_fused_pair128(int type, int d_type, int c_type, const CUtensorMap* maps, const FusedParams& p, int grid,
                            int smem, cudaStream_t stream) {
  return fused::launch_by_type<2, 128>(type, d_type, c_type, maps, p, grid, smem, stream);
}

}  // namespace b200

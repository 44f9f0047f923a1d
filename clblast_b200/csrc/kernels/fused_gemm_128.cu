// Instances of the fused product kernel: one CTA per 128 x 128 tile.
#include "fused_gemm.cuh"

namespace b200 {

cudaError_t launch_fused_128(int type, int d_type, int c_type, const CUtensorMap* maps, const FusedParams& p, int grid,
                            int smem, cudaStream_t stream) {
  return fused::launch_by_type<1, 128>(type, d_type, c_type, maps, p, grid, smem, stream);
}

int fused_resident_clusters(int cluster) {
  if (cluster <= 1) return sm_count();
  static std::atomic<int> tables[3][kMaxDevices];
  if (cluster == 2) return per_device(tables[0], [] { return fused::resident_clusters<1, 128>(2, 200 * 1024); });
  if (cluster == 4) return per_device(tables[1], [] { return fused::resident_clusters<1, 128>(4, 200 * 1024); });
  return per_device(tables[2], [] { return fused::resident_clusters<1, 128>(8, 200 * 1024); });
}

}  // namespace b200

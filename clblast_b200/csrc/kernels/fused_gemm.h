// Launch interface of the fused 16-bit products: bias, activation, residual and their gradients in the epilogue, and
// ragged groups of rows (csrc/fused_abi.cpp holds the entry points, csrc/fused_host.cpp the selection).
#pragma once

#include <cuda.h>
#include <cuda_runtime_api.h>

namespace b200 {

constexpr int kBFloat16 = 1016;  // precision code of bfloat16, known to the fused routines only

// What the ragged extent of a grouped call is.
enum FusedKind : int {
  kFusedPlain = 0,        // one problem, or `problems` of equal size at constant strides
  kFusedRaggedCols = 1,   // group g owns the columns [offsets[g], offsets[g + 1]) of C and of op(B), and its own op(A)
  kFusedRaggedInner = 2,  // group g sums over the inner indices [offsets[g], offsets[g + 1]) and has its own C
};

// Most groups of a call: the table of the groups' tiles lives in shared memory.
constexpr int kFusedMaxGroups = 1024;

// Inner elements per accumulator of results in 16 bits. What the tensor cores cut off below it is a fifth of half's rounding
// at most, of bfloat16's a fortieth.
constexpr int kChunkHalf = 16384;

// Kernel arguments. C is m x n with m contiguous: rows are the features of a caller's contiguous vectors, columns the
// vectors (tokens).
struct FusedParams {
  unsigned int* status;
  int m, n, k;                // kFusedRaggedCols: n is the bound on the offsets; kFusedRaggedInner: k is
  int kind, problems;
  const long long* offsets;   // problems + 1 entries in device memory (ragged kinds)
  int tiles_m, tiles_n;       // per problem (tiles_n unused for kFusedRaggedCols)
  int raster;                 // tile rows walked together
  int tri;                    // C is symmetric: tiles on and below the diagonal are computed, the others mirrored
  int a_mn, b_mn;             // operand is contiguous along m / n (else along k)
  unsigned int idesc;
  int a_batched, b_batched;
  int stages;                 // depth of the operand ring
  int parts;                  // every matrix is a sum of two halves in consecutive planes (see kModeParts)
  int chained;                // the launch may be set up before the one in front of it in the stream has finished
  int split;                  // CTAs of a cluster that share one tile's inner extent (kernels of one CTA per tile)
  float alpha, beta;
  const void* bias;           // one value per row of C, or null
  long long bias_stride;      // between problems
  int act, grad;              // grad: C = (alpha AB + beta D) * slope(Z); else Z = alpha AB + bias, C = act(Z) + beta D
  void* c;
  const void* d;              // null without residual
  void* z;                    // written (grad == 0) or read; null without
  long long ldc, ldd, ldz, c_stride, d_stride, z_stride;
  int vec;                    // C, D and Z: bases, leading dimensions and strides are multiples of 16 bytes
  int prefetch;               // D and Z have tensor maps and are asked for ahead
  float* partial;             // row sums of C per column tile (bias gradient), or null
  float* sums;                // one tile per CTA, where a result in 16 bits has more than kChunkHalf inner elements; or null
};

#ifdef __CUDACC__
#define B200_HD __host__ __device__
#else
#define B200_HD
#endif
// Inner elements per operand stage, in swizzle rows of 64. The loops over the stages take about 700 cycles whatever a stage
// holds, more than the MMAs of one swizzle row (8192 x 8192 x 2048 on 256 x 256 pairs: 220 us with one row per stage, 212
// with two; 32 groups of 512 x 2048 x 2048 into single precision 287 and 236). 128 x 256 on a single SM has no room for
// more than two stages of two rows.
B200_HD constexpr int fused_stage_rows(int ctas, int bn) { return ctas == 2 || bn <= 128 ? 2 : 1; }

// Sizes of one kernel variant as the selection sees it.
struct FusedVariant {
  int ctas;           // CTAs per tile: 2 for the pair kernel
  int bn;             // columns per tile; rows are 128 * ctas
  int stage_bytes;
};
// Epilogue groups of four warps that share a tile's columns, next to four warps with other roles.
// (Four groups on 128 columns halve the registers of a thread: 25 % slower where stores go element by element.)
B200_HD constexpr int fused_groups(int bn) { return bn >= 64 ? 2 : 1; }
B200_HD constexpr int fused_threads(int bn) { return 128 + 128 * fused_groups(bn); }
// Shared memory of an epilogue warp: a block of 16 columns x 32 rows of C or D and one of Z.
B200_HD constexpr int fused_warp_bytes(bool single, bool aux) { return (single ? 2048 : 1024) + (aux ? 1024 : 0); }
// Shared memory behind the operand ring: the epilogue warps', or the fp32 sums of a split tile; then barriers, then the
// group table.
B200_HD constexpr int fused_staging_bytes(int bn, bool single, bool aux, int split) {
  return split > 1 ? bn * 512 : 4 * fused_groups(bn) * fused_warp_bytes(single, aux);
}
constexpr int kFusedBarBytes = 512;
constexpr int kFusedVariants = 6;
constexpr FusedVariant kFusedTable[kFusedVariants] = {
    {2, 256, 65536}, {1, 256, 49152}, {1, 128, 65536}, {1, 64, 49152}, {1, 32, 40960}, {2, 128, 49152}};

// Enqueues variant `v` with operand type / D type / C type. `grid` counts CTAs, `smem` bytes of dynamic shared memory.
cudaError_t launch_fused_variant(int v, int type, int d_type, int c_type, const CUtensorMap* maps, const FusedParams& p,
                                 int grid, int smem, cudaStream_t stream);
// Clusters of `cluster` (1, 2, 4 or 8) CTAs with nearly all of an SM's shared memory each that the current device
// holds at once.
int fused_resident_clusters(int cluster);
cudaError_t launch_fused_pair(int type, int d_type, int c_type, const CUtensorMap* maps, const FusedParams& p, int grid,
                              int smem, cudaStream_t stream);
cudaError_t launch_fused_pair128(int type, int d_type, int c_type, const CUtensorMap* maps, const FusedParams& p, int grid,
                                 int smem, cudaStream_t stream);
cudaError_t launch_fused_256(int type, int d_type, int c_type, const CUtensorMap* maps, const FusedParams& p, int grid,
                             int smem, cudaStream_t stream);
cudaError_t launch_fused_128(int type, int d_type, int c_type, const CUtensorMap* maps, const FusedParams& p, int grid,
                             int smem, cudaStream_t stream);
cudaError_t launch_fused_64(int type, int d_type, int c_type, const CUtensorMap* maps, const FusedParams& p, int grid,
                            int smem, cudaStream_t stream);
cudaError_t launch_fused_32(int type, int d_type, int c_type, const CUtensorMap* maps, const FusedParams& p, int grid,
                            int smem, cudaStream_t stream);

}  // namespace b200

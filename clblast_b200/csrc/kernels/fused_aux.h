// Launch interface of the small kernels around the fused products: operand copies, element-wise epilogues, sums of
// partial bias gradients, and the normalisation in front of the Newton-Schulz products.
#pragma once

#include <cuda_runtime_api.h>

namespace b200 {

// Copies `planes` matrices of `two` lines of `one` contiguous 2-byte elements each (any alignment, leading dimension and
// plane stride) to lines of `pitch` elements (a multiple of 8, the rest zero), planes two * pitch apart. Two jobs go in one
// launch; one with planes == 0 is skipped. With `offsets` (device, planes + 1 of them) a plane whose group has no rows is
// left out.
struct PackJob {
  const void* src;
  void* dst;
  long long one, two, planes, src_ld, src_stride, pitch;
  const long long* offsets;
};
cudaError_t launch_pack(const PackJob (&jobs)[2], cudaStream_t stream);

// Element-wise tail of a product P (m x n, m contiguous; n vectors of m features):
//   grad == 0: Z = P + bias, C = act(Z) + beta D;   grad == 1: C = (P + beta D) * slope(Z), partial sums over vectors.
// `type` 16 / 1016 / 32 is the type of every matrix. Null: bias, D, Z, partial are optional.
struct PointwiseJob {
  int type, act, grad;
  long long m, n;
  const void* p; long long ldp;
  const void* bias;
  const void* d; long long ldd; float beta;
  void* z; long long ldz;
  void* c; long long ldc;
  const long long* offsets;  // device table of `groups` + 1 offsets: only the vectors between the first and the last
  int groups;                // one (offsets null) or the number of groups
  float* partial;            // pointwise_chunks() lines of m sums, grouped by group
};
constexpr int kPointwiseChunk = 64;  // vectors per line of partial sums
long long pointwise_chunks(const PointwiseJob& job);
cudaError_t launch_pointwise(const PointwiseJob& job, cudaStream_t stream);

// out[g][row] (type 16 / 1016 / 32, groups out_stride apart) = sum of the group's lines of `partial`. A group has
// ceil(vectors / per_tile) * lines_per_tile lines, in order; without offsets there is one group of `tiles` tiles.
struct SumJob {
  const float* partial;
  long long m;
  int type;
  void* out;
  long long out_stride;
  const long long* offsets;
  int groups;
  long long bound;     // upper bound of the offsets
  int per_tile, lines_per_tile;
  long long tiles;
};
cudaError_t launch_sum_partials(const SumJob& job, cudaStream_t stream);

// Newton-Schulz input: X = scale * G / (|G|_F + eps) for `batch` matrices (lines of `one` contiguous elements, `two`
// lines), X dense with `lines` lines of `pitch` elements (what G does not have is zero), planes lines * pitch apart, in half (x_type 16) or single
// (32) precision, or (x_type kParts) as a sum of two halves in consecutive planes. `sums` is scratch of batch * kNormBlocks
// doubles.
constexpr int kNormBlocks = 256;  // blocks per matrix
constexpr int kParts = 1616;
struct NormaliseJob {
  int type, x_type;
  const void* g;
  long long one, two, ld, stride, batch;
  void* x;
  long long pitch, lines;
  double eps, scale;
  double* sums;
};
cudaError_t launch_normalise(const NormaliseJob& job, cudaStream_t stream);

// B = scale * X, `batch` matrices to the caller's type. x_type 32: X in single precision; kParts: planes 2z and 2z + 1 of
// x (lines x pitch halves each) hold hi and lo, X = hi + lo.
struct JoinJob {
  int type, x_type;
  const void* x;
  long long lines, pitch;
  void* b;
  long long one, two, ld, stride, batch;
  float scale;
};
cudaError_t launch_join(const JoinJob& job, cudaStream_t stream);

}  // namespace b200

// Host side of the fused products: description of one normalised call, kernel selection and launch.
#pragma once

#include <cuda_runtime_api.h>

#include "kernels/fused_gemm.h"

namespace b200 {

// C (m x n, m contiguous) = epilogue of op(A) (m x k) * op(B) (k x n); pointers are to first elements. `type` is that of
// A, B, bias and Z (16 or kBFloat16), d_type / c_type those of D and C (16, kBFloat16 or 32).
struct FusedDesc {
  int type, d_type, c_type;
  int kind;
  long long problems;          // 1, a batch, or the number of groups
  const long long* offsets;
  long long m, n, k;
  const void* a; long long lda, a_stride; int a_mn;  // strides between problems (kFusedRaggedCols: of A alone)
  const void* b; long long ldb, b_stride; int b_mn;
  double alpha, beta;
  const void* bias; long long bias_stride;
  int act, grad, tri, parts;   // parts: all matrices are pairs of halves, planes `stride` apart, problems two of them
  int chained;                 // one of a chain of launches that read each other's results
  const void* d; long long ldd, d_stride;
  void* z; long long ldz, z_stride;
  void* c; long long ldc, c_stride;
  void* bias_grad; long long bias_grad_stride;
};

// Copies operands that TMA cannot address, picks a variant, enqueues the product and the sum of its bias gradient.
cudaError_t launch_fused(const FusedDesc& d, cudaStream_t stream, const char** name);

}  // namespace b200

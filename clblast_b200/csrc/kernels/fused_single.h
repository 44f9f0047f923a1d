// Products with an epilogue in single precision whose tiles alone would leave most of the GPU idle.
#pragma once

#include <cuda_runtime_api.h>

namespace b200 {

// C (n vectors of m features) = act(alpha op(A) op(B) + bias) + beta D, or its gradient form. A: m features, B: n vectors;
// a_mn / b_mn: the features (vectors) are contiguous, otherwise k is. D and a Z that is read may be C.
struct SingleJob {
  long long m, n, k;
  const float* a; long long lda; int a_mn;
  const float* b; long long ldb; int b_mn;
  float alpha, beta;
  const float* bias;
  int act, grad;
  const float* d; long long ldd;
  float* z; long long ldz;
  float* c; long long ldc;
};
// Whether the kernel below is expected to take less time than the tensor-core product and a pass over its result.
bool single_fits(long long m, long long n, long long k);
cudaError_t launch_single(const SingleJob& job, cudaStream_t stream);

}  // namespace b200

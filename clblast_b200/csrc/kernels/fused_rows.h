// Products of very few vectors with one weight matrix, on the CUDA cores.
#pragma once

#include <cuda_runtime_api.h>

namespace b200 {

// C (n vectors of m features) = act(alpha W x + bias) + beta D or its gradient form; W is m x k with k contiguous, 16-byte
// aligned rows. One kernel for up to kFewRows vectors.
constexpr int kFewRows = 4;
struct FewRowsJob {
  int type, c_type;  // operands (16, bfloat16's code or 32), C and D (the same or 32)
  int m, n, k;
  const void* w; long long ldw;
  const void* x; long long ldx;
  float alpha, beta;
  const void* bias;
  int act, grad;
  const void* d; long long ldd;
  void* z; long long ldz;
  void* c; long long ldc;
};
cudaError_t launch_few_rows(const FewRowsJob& job, cudaStream_t stream);

}  // namespace b200

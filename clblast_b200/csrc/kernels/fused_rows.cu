// One to four vectors times a weight matrix: the time is that of reading the matrix once. A tensor-core tile would carry
// 32 columns for them and, with so few tiles, split the inner extent over clusters that meet again at the end (4096 x 4096,
// one vector: 14 us); here every warp reads one row of the matrix, or a part of it, with all its 16-byte loads in flight
// and the vectors come out of L1 (8.5 us with the matrix in memory, 3.9 TB/s; 4.9 us with it in L2).
//
// Sums run in fp32: one per lane and vector, then over the lanes by shuffles, then over the parts in order.
#include "fused_rows.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../runtime_state.h"
#include "activation.cuh"
#include "fused_gemm.h"

namespace b200 {

namespace {

constexpr int kWarps = 8;
constexpr int kDeep = 4;  // 16-byte loads of W that a lane has in flight

// Elements of a 16-byte piece.
template <class T>
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(w[i]);
    } else {
      const unsigned short lo = static_cast<unsigned short>(w[i]), hi = static_cast<unsigned short>(w[i] >> 16);
      f[2 * i] = to_float(*reinterpret_cast<const T*>(&lo));
      f[2 * i + 1] = to_float(*reinterpret_cast<const T*>(&hi));
    }
  }
}

// PARTS warps of the block share a row's inner extent. VX: the vectors can be read 16 bytes at a time.
template <class T, class OT, int ROWS, int PARTS, bool VX>
__global__ void __launch_bounds__(kWarps * 32) few_rows_kernel(const FewRowsJob job) {
  constexpr bool FAST = sizeof(OT) == 2;
  constexpr int PV = 16 / sizeof(T);
  __shared__ float sums[kWarps][ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x * (kWarps / PARTS) + warp / PARTS;
  const int part = warp % PARTS;
  float acc[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) acc[r] = 0.f;
  if (row < job.m) {
    const T* const w = static_cast<const T*>(job.w) + static_cast<long long>(row) * job.ldw;
    const T* const x = static_cast<const T*>(job.x);
    const int vectors = job.k / PV;  // whole 16-byte pieces
    const int begin = static_cast<int>(static_cast<long long>(vectors) * part / PARTS);
    const int end = static_cast<int>(static_cast<long long>(vectors) * (part + 1) / PARTS);
    auto multiply = [&](const uint4& wv, int i) {
      float a[PV];
      unpack<T>(wv, a);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (r >= job.n) break;
        float b[PV];
        const T* const xr = x + static_cast<long long>(r) * job.ldx + PV * i;
        if (VX) {
          unpack<T>(__ldg(reinterpret_cast<const uint4*>(xr)), b);
        } else {
#pragma unroll
          for (int j = 0; j < PV; ++j) b[j] = to_float(xr[j]);
        }
#pragma unroll
        for (int j = 0; j < PV; ++j) acc[r] = fmaf(a[j], b[j], acc[r]);
      }
    };
    int i = begin + lane;
    for (; i + 32 * (kDeep - 1) < end; i += 32 * kDeep) {
      uint4 v[kDeep];
#pragma unroll
      for (int u = 0; u < kDeep; ++u) v[u] = __ldcs(reinterpret_cast<const uint4*>(w) + i + 32 * u);
#pragma unroll
      for (int u = 0; u < kDeep; ++u) multiply(v[u], i + 32 * u);
    }
    for (; i < end; i += 32) multiply(__ldcs(reinterpret_cast<const uint4*>(w) + i), i);
    if (part == PARTS - 1) {  // what is left behind the last whole piece
      const int j = vectors * PV + lane;
      if (j < job.k) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
          if (r < job.n) acc[r] = fmaf(to_float(w[j]), to_float(x[static_cast<long long>(r) * job.ldx + j]), acc[r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) acc[r] += __shfl_xor_sync(0xFFFFFFFFu, acc[r], d);
    if (lane == 0) sums[warp][r] = acc[r];
  }
  __syncthreads();
  // thread (feature of the block, vector)
  const int feature = threadIdx.x % (kWarps / PARTS), r = threadIdx.x / (kWarps / PARTS);
  const int f = blockIdx.x * (kWarps / PARTS) + feature;
  if (r >= ROWS || r >= job.n || f >= job.m) return;
  float y = 0.f;
#pragma unroll
  for (int q = 0; q < PARTS; ++q) y += sums[feature * PARTS + q][r];
  y *= job.alpha;
  const float add = job.d != nullptr ? job.beta * to_float(static_cast<const OT*>(job.d)[r * job.ldd + f]) : 0.f;
  T* const z = static_cast<T*>(job.z) + r * job.ldz + f;
  if (job.grad) {
    y += add;
    if (job.z != nullptr) {
      const float zz = to_float(*z);
      with_act(job.act, [&](auto tag) { y *= act_slope<FAST, decltype(tag)::value>(zz); });
    }
  } else {
    if (job.bias != nullptr) y += to_float(static_cast<const T*>(job.bias)[f]);
    if (job.z != nullptr) *z = from_float<T>(y);
    with_act(job.act, [&](auto tag) { y = act_value<FAST, decltype(tag)::value>(y); });
    y += add;
  }
  static_cast<OT*>(job.c)[r * job.ldc + f] = from_float<OT>(y);
}

template <class T, class OT, int ROWS, int PARTS>
cudaError_t launch_parts(const FewRowsJob& job, cudaStream_t stream) {
  const int per_block = kWarps / PARTS;
  const unsigned blocks = static_cast<unsigned>((job.m + per_block - 1) / per_block);
  const bool vx = (reinterpret_cast<uintptr_t>(job.x) & 15) == 0 && (job.n == 1 || job.ldx % (16 / static_cast<int>(sizeof(T))) == 0);
  if (vx) few_rows_kernel<T, OT, ROWS, PARTS, true><<<blocks, kWarps * 32, 0, stream>>>(job);
  else few_rows_kernel<T, OT, ROWS, PARTS, false><<<blocks, kWarps * 32, 0, stream>>>(job);
  return cudaGetLastError();
}

template <class T, class OT, int ROWS>
cudaError_t launch_rows(const FewRowsJob& job, cudaStream_t stream) {
  // enough warps to keep every SM's memory pipeline full, each with at least one round of deep loads
  const long long wanted = 24LL * sm_count();
  const int round = 32 * kDeep * 16 / static_cast<int>(sizeof(T));  // elements of one
  if (job.m >= wanted || job.k < 2 * round) return launch_parts<T, OT, ROWS, 1>(job, stream);
  if (2LL * job.m >= wanted || job.k < 4 * round) return launch_parts<T, OT, ROWS, 2>(job, stream);
  if (4LL * job.m >= wanted || job.k < 8 * round) return launch_parts<T, OT, ROWS, 4>(job, stream);
  return launch_parts<T, OT, ROWS, 8>(job, stream);
}

template <class T, class OT>
cudaError_t launch_types(const FewRowsJob& job, cudaStream_t stream) {
  if (job.n == 1) return launch_rows<T, OT, 1>(job, stream);
  if (job.n == 2) return launch_rows<T, OT, 2>(job, stream);
  return launch_rows<T, OT, 4>(job, stream);
}

}  // namespace

cudaError_t launch_few_rows(const FewRowsJob& job, cudaStream_t stream) {
  if (job.n < 1 || job.n > kFewRows) return cudaErrorInvalidValue;
  if (job.type == 16) {
    if (job.c_type == 16) return launch_types<__half, __half>(job, stream);
    if (job.c_type == 32) return launch_types<__half, float>(job, stream);
  } else if (job.type == kBFloat16) {
    if (job.c_type == kBFloat16) return launch_types<__nv_bfloat16, __nv_bfloat16>(job, stream);
    if (job.c_type == 32) return launch_types<__nv_bfloat16, float>(job, stream);
  }
  if (job.type == 32 && job.c_type == 32) return launch_types<float, float>(job, stream);
  return cudaErrorInvalidValue;
}

}  // namespace b200

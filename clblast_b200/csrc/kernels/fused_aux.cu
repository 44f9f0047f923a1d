// The small kernels around the fused products. All of them are bound by memory traffic or by launch latency.
#include "fused_aux.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "activation.cuh"
#include "fused_gemm.h"
#include "group_table.cuh"

namespace b200 {

namespace {

// ---- copies to TMA's alignment ---------------------------------------------------------------------------------------

constexpr int kPackThreads = 256, kPackVec = 8;

// A block covers kPackThreads * kPackVec elements of one line: element loads that are consecutive across the lanes (the
// source may start at any element), one exchange through shared memory, 16-byte stores.
struct PackPair {
  PackJob job[2];
  int segments[2];
  unsigned first_of_second;
};
__global__ void __launch_bounds__(kPackThreads) pack_kernel(const PackPair pair) {
  __shared__ __align__(16) unsigned short buf[kPackThreads * kPackVec];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the product behind it may be set up meanwhile
  const int which = blockIdx.x >= pair.first_of_second ? 1 : 0;
  const unsigned block = blockIdx.x - (which ? pair.first_of_second : 0u);
  const PackJob& job = pair.job[which];
  const unsigned segments = static_cast<unsigned>(pair.segments[which]);
  const long long line = block / segments;
  const int x0 = static_cast<int>(block % segments) * (kPackThreads * kPackVec);
  const long long plane = line / job.two, in_plane = line - plane * job.two;
  if (job.offsets != nullptr && job.offsets[plane + 1] <= job.offsets[plane]) return;
  const unsigned short* const src = static_cast<const unsigned short*>(job.src) + plane * job.src_stride + in_plane * job.src_ld + x0;
  const long long left = job.one - x0;
#pragma unroll
  for (int j = 0; j < kPackVec; ++j) {
    const int i = threadIdx.x + j * kPackThreads;
    buf[i] = i < left ? src[i] : static_cast<unsigned short>(0);
  }
  __syncthreads();
  const int i = threadIdx.x * kPackVec;
  if (x0 + i < job.pitch)
    *reinterpret_cast<uint4*>(static_cast<unsigned short*>(job.dst) + line * job.pitch + x0 + i) = *reinterpret_cast<const uint4*>(buf + i);
}

// ---- element-wise tails ------------------------------------------------------------------------------------------------

constexpr int kPwLanes = 32, kPwRows = 8;  // threads along the features and along the vectors

template <class T, int VEC>
struct alignas(VEC * sizeof(T)) Pack { T v[VEC]; };

// A block covers 32 * VEC features of kPointwiseChunk vectors of one group. VEC > 1 needs every line 16-byte aligned.
template <class T, int VEC>
__global__ void __launch_bounds__(kPwLanes * kPwRows) pointwise_kernel(const PointwiseJob job) {
  constexpr bool FAST = sizeof(T) == 2;
  extern __shared__ int table[];
  __shared__ float sums[kPwRows][kPwLanes * VEC];
  long long first = static_cast<long long>(blockIdx.y) * kPointwiseChunk;
  long long last = first + kPointwiseChunk < job.n ? first + kPointwiseChunk : job.n;
  int group = 0;
  if (job.offsets != nullptr) {
    int* const start = table;
    int* const tiles = table + job.groups + 1;
    if (threadIdx.y == 0) build_table(job.offsets, job.groups, static_cast<int>(job.n), kPointwiseChunk, start, tiles);
    __syncthreads();
    const int want = static_cast<int>(blockIdx.y);
    if (want >= tiles[job.groups]) return;  // the grid is an upper bound
    int lo = 0, hi = job.groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tiles[mid] <= want) lo = mid; else hi = mid;
    }
    group = lo;
    first = start[lo] + static_cast<long long>(want - tiles[lo]) * kPointwiseChunk;
    last = first + kPointwiseChunk < start[lo + 1] ? first + kPointwiseChunk : start[lo + 1];
  }
  (void)group;
  const long long f0 = (static_cast<long long>(blockIdx.x) * kPwLanes + threadIdx.x) * VEC;
  const bool in = f0 < job.m;  // VEC > 1: m is a multiple of VEC
  float total[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) total[j] = 0.f;
  if (in) {
    using P = Pack<T, VEC>;
    float bias[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      bias[j] = job.bias != nullptr ? to_float(static_cast<const T*>(job.bias)[f0 + j]) : 0.f;
    for (long long t = first + threadIdx.y; t < last; t += kPwRows) {
      const P p = *reinterpret_cast<const P*>(static_cast<const T*>(job.p) + t * job.ldp + f0);
      P d = {}, z = {}, c;
      if (job.d != nullptr) d = *reinterpret_cast<const P*>(static_cast<const T*>(job.d) + t * job.ldd + f0);
      if (job.grad && job.z != nullptr) z = *reinterpret_cast<const P*>(static_cast<const T*>(job.z) + t * job.ldz + f0);
      with_act(job.grad && job.z == nullptr ? static_cast<int>(kActIdentity) : job.act, [&](auto tag) {
        constexpr int ACT = decltype(tag)::value;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float add = job.d != nullptr ? job.beta * to_float(d.v[j]) : 0.f;
          float y = to_float(p.v[j]) + bias[j];
          if (job.grad) {
            y = (y + add) * act_slope<FAST, ACT>(to_float(z.v[j]));
            total[j] += y;
          } else {
            z.v[j] = from_float<T>(y);
            y = act_value<FAST, ACT>(y) + add;
          }
          c.v[j] = from_float<T>(y);
        }
      });
      if (!job.grad && job.z != nullptr) *reinterpret_cast<P*>(static_cast<T*>(job.z) + t * job.ldz + f0) = z;
      if (job.c != nullptr) *reinterpret_cast<P*>(static_cast<T*>(job.c) + t * job.ldc + f0) = c;
    }
  }
  if (job.partial == nullptr) return;
#pragma unroll
  for (int j = 0; j < VEC; ++j) sums[threadIdx.y][threadIdx.x * VEC + j] = total[j];
  __syncthreads();
  for (int i = threadIdx.y * kPwLanes + threadIdx.x; i < kPwLanes * VEC; i += kPwLanes * kPwRows) {
    const long long f = static_cast<long long>(blockIdx.x) * kPwLanes * VEC + i;
    if (f >= job.m) continue;
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < kPwRows; ++r) s += sums[r][i];
    job.partial[static_cast<long long>(blockIdx.y) * job.m + f] = s;
  }
}

// ---- sums of partial bias gradients ------------------------------------------------------------------------------------

// Block: 32 features x 8 lines at a time; the eight running sums are added in a fixed order.
template <class T>
__global__ void __launch_bounds__(256) sum_partials_kernel(const SumJob job) {
  extern __shared__ int table[];
  __shared__ float sums[8][33];
  const int group = static_cast<int>(blockIdx.y);
  long long first = 0, last = job.tiles;
  if (job.offsets != nullptr) {
    int* const start = table;
    int* const tiles = table + job.groups + 1;
    if (threadIdx.y == 0) build_table(job.offsets, job.groups, static_cast<int>(job.bound), job.per_tile, start, tiles);
    __syncthreads();
    first = tiles[group];
    last = tiles[group + 1];
  }
  first *= job.lines_per_tile;
  last *= job.lines_per_tile;
  const long long row = static_cast<long long>(blockIdx.x) * 32 + threadIdx.x;
  float s = 0.f;
  if (row < job.m) {
#pragma unroll 4
    for (long long i = first + threadIdx.y; i < last; i += 8) s += job.partial[i * job.m + row];
  }
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && row < job.m) {
#pragma unroll
    for (int r = 1; r < 8; ++r) s += sums[r][threadIdx.x];
    static_cast<T*>(job.out)[group * job.out_stride + row] = from_float<T>(s);
  }
}

// ---- Newton-Schulz normalisation -----------------------------------------------------------------------------------------

// Squares are summed in 64 bits: neither gradients of 1e-30 nor of 1e30 leave the range, and the kernel waits for memory
// either way. Block sums are added in order, so the result does not vary.
template <class T>
__global__ void __launch_bounds__(256) norm_kernel(const NormaliseJob job) {
  __shared__ double part[8];
  const T* const g = static_cast<const T*>(job.g) + static_cast<long long>(blockIdx.y) * job.stride;
  double s = 0.0;
  for (long long line = blockIdx.x; line < job.two; line += gridDim.x) {
    const T* const row = g + line * job.ld;
#pragma unroll 4
    for (long long i = threadIdx.x; i < job.one; i += 256) {
      const double v = static_cast<double>(to_float(row[i]));
      s += v * v;
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < 8; ++w) t += part[w];
    job.sums[static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x] = t;
  }
}

template <class T, class X, bool PARTS>
__global__ void __launch_bounds__(256) scale_kernel(const NormaliseJob job, int blocks) {
  __shared__ double factor;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x < 32) {
    double t = 0.0;
    for (int i = threadIdx.x; i < blocks; i += 32) t += job.sums[static_cast<long long>(blockIdx.y) * blocks + i];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, d);
    if (threadIdx.x == 0) factor = job.scale / (sqrt(t) + job.eps);
  }
  __syncthreads();
  const double f = factor;
  const T* const g = static_cast<const T*>(job.g) + static_cast<long long>(blockIdx.y) * job.stride;
  X* const x = static_cast<X*>(job.x) + static_cast<long long>(blockIdx.y) * (PARTS ? 2 : 1) * job.lines * job.pitch;
  for (long long line = blockIdx.x; line < job.lines; line += gridDim.x) {
    const T* const row = g + line * job.ld;
#pragma unroll 4
    for (long long i = threadIdx.x; i < job.pitch; i += 256) {
      const float v = i < job.one && line < job.two ? static_cast<float>(static_cast<double>(to_float(row[i])) * f) : 0.f;
      const X high = from_float<X>(v);
      x[line * job.pitch + i] = high;
      if (PARTS) x[(job.lines + line) * job.pitch + i] = from_float<X>(v - to_float(high));
    }
  }
}

template <class T, bool PARTS>
__global__ void __launch_bounds__(256) join_kernel(const JoinJob job) {
  using S = typename std::conditional<PARTS, __half, float>::type;
  const long long plane = job.lines * job.pitch;
  const S* const x = static_cast<const S*>(job.x) + static_cast<long long>(blockIdx.y) * (PARTS ? 2 : 1) * plane;
  T* const b = static_cast<T*>(job.b) + static_cast<long long>(blockIdx.y) * job.stride;
  for (long long line = blockIdx.x; line < job.two; line += gridDim.x) {
    const S* const from = x + line * job.pitch;
#pragma unroll 4
    for (long long i = threadIdx.x; i < job.one; i += 256) {
      float v = to_float(from[i]);
      if constexpr (PARTS) v += to_float(from[plane + i]);
      b[line * job.ld + i] = from_float<T>(job.scale * v);
    }
  }
}

template <class F>
cudaError_t by_type(int type, F&& f) {
  switch (type) {
    case 16: return f(static_cast<__half*>(nullptr));
    case kBFloat16: return f(static_cast<__nv_bfloat16*>(nullptr));
    case 32: return f(static_cast<float*>(nullptr));
    default: return cudaErrorInvalidValue;
  }
}

bool aligned16(const void* p, long long ld, long long elem) {
  return p == nullptr || (((reinterpret_cast<uintptr_t>(p) & 15) == 0) && ((ld * elem) % 16 == 0));
}

int table_smem(const long long* offsets, int groups) { return offsets != nullptr ? 8 * (groups + 1) : 0; }

}  // namespace

cudaError_t launch_pack(const PackJob (&jobs)[2], cudaStream_t stream) {
  const long long seg = kPackThreads * kPackVec;
  PackPair pair = {};
  long long total = 0;
  for (int i = 0; i < 2; ++i) {
    const PackJob& job = jobs[i];
    pair.job[i] = job;
    if (i == 1) pair.first_of_second = static_cast<unsigned>(total);
    const long long segments = (job.pitch + seg - 1) / seg;
    const long long blocks = job.planes > 0 ? segments * job.two * job.planes : 0;
    if (blocks > 0x3FFFFFFFLL || job.pitch > 0x7FFFFFFFLL || (job.pitch & 7)) return cudaErrorInvalidValue;
    pair.segments[i] = blocks > 0 ? static_cast<int>(segments) : 1;
    total += blocks;
  }
  if (total <= 0) return cudaSuccess;
  pack_kernel<<<static_cast<unsigned>(total), kPackThreads, 0, stream>>>(pair);
  return cudaGetLastError();
}

long long pointwise_chunks(const PointwiseJob& job) {
  const long long whole = (job.n + kPointwiseChunk - 1) / kPointwiseChunk;
  return job.offsets != nullptr ? whole + job.groups : whole;
}

cudaError_t launch_pointwise(const PointwiseJob& job, cudaStream_t stream) {
  return by_type(job.type, [&](auto* tag) {
    using T = typename std::remove_pointer<decltype(tag)>::type;
    constexpr int VEC = 16 / static_cast<int>(sizeof(T));
    constexpr long long elem = sizeof(T);
    const bool vec = job.m % VEC == 0 && aligned16(job.p, job.ldp, elem) && aligned16(job.d, job.ldd, elem) &&
                     aligned16(job.z, job.ldz, elem) && aligned16(job.c, job.ldc, elem);
    const long long cover = kPwLanes * (vec ? VEC : 1);
    const long long gx = (job.m + cover - 1) / cover, gy = pointwise_chunks(job);
    if (gx > 0x7FFFFFFFLL) return cudaErrorInvalidValue;
    // the second grid dimension ends at 65535 blocks: longer calls go in pieces of that many chunks
    if (job.offsets == nullptr) {
      for (long long at = 0; at < gy; at += 65535) {
        PointwiseJob part = job;
        const long long skip = at * kPointwiseChunk;
        part.n = job.n - skip < 65535LL * kPointwiseChunk ? job.n - skip : 65535LL * kPointwiseChunk;
        auto move = [&](const void* q, long long ld) { return q ? static_cast<const T*>(q) + skip * ld : nullptr; };
        part.p = move(job.p, job.ldp);
        part.d = move(job.d, job.ldd);
        part.z = const_cast<T*>(move(job.z, job.ldz));
        part.c = const_cast<T*>(move(job.c, job.ldc));
        if (job.partial) part.partial = job.partial + at * job.m;
        const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(pointwise_chunks(part))), block(kPwLanes, kPwRows);
        if (vec) pointwise_kernel<T, VEC><<<grid, block, 0, stream>>>(part);
        else pointwise_kernel<T, 1><<<grid, block, 0, stream>>>(part);
      }
      return cudaGetLastError();
    }
    if (gy > 65535) return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy)), block(kPwLanes, kPwRows);
    const int smem = table_smem(job.offsets, job.groups);
    if (vec) pointwise_kernel<T, VEC><<<grid, block, smem, stream>>>(job);
    else pointwise_kernel<T, 1><<<grid, block, smem, stream>>>(job);
    return cudaGetLastError();
  });
}

cudaError_t launch_sum_partials(const SumJob& job, cudaStream_t stream) {
  const long long gx = (job.m + 31) / 32;
  if (gx > 0x7FFFFFFFLL || job.groups > 65535) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(job.offsets ? job.groups : 1)), block(32, 8);
  const int smem = table_smem(job.offsets, job.groups);
  return by_type(job.type, [&](auto* tag) {
    using T = typename std::remove_pointer<decltype(tag)>::type;
    sum_partials_kernel<T><<<grid, block, smem, stream>>>(job);
    return cudaGetLastError();
  });
}

cudaError_t launch_normalise(const NormaliseJob& job, cudaStream_t stream) {
  if (job.batch > 65535) return cudaErrorInvalidValue;
  const int blocks = static_cast<int>(job.two < kNormBlocks ? job.two : kNormBlocks);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(job.batch));
  const long long wide = job.lines < 4096 ? job.lines : 4096;
  const dim3 scale_grid(static_cast<unsigned>(wide), static_cast<unsigned>(job.batch));
  return by_type(job.type, [&](auto* tag) {
    using T = typename std::remove_pointer<decltype(tag)>::type;
    norm_kernel<T><<<grid, 256, 0, stream>>>(job);
    if (job.x_type == 16) scale_kernel<T, __half, false><<<scale_grid, 256, 0, stream>>>(job, blocks);
    else if (job.x_type == kParts) scale_kernel<T, __half, true><<<scale_grid, 256, 0, stream>>>(job, blocks);
    else scale_kernel<T, float, false><<<scale_grid, 256, 0, stream>>>(job, blocks);
    return cudaGetLastError();
  });
}

cudaError_t launch_join(const JoinJob& job, cudaStream_t stream) {
  if (job.batch > 65535) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(job.two < 4096 ? job.two : 4096), static_cast<unsigned>(job.batch));
  return by_type(job.type, [&](auto* tag) {
    using T = typename std::remove_pointer<decltype(tag)>::type;
    if (job.x_type == kParts) join_kernel<T, true><<<grid, 256, 0, stream>>>(job);
    else join_kernel<T, false><<<grid, 256, 0, stream>>>(job);
    return cudaGetLastError();
  });
}

}  // namespace b200

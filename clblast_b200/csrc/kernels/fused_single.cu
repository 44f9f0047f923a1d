// Single-precision products of few vectors or of small matrices, with the epilogue in the same kernel, on the CUDA cores.
//
// The tensor-core product in single precision works on 128 x 128 tiles over the whole inner extent: with few tiles most
// SMs have nothing to do, and a pass over the result follows. Here a tile is 64 x 64 or 32 x 16, and the inner extent is
// split over up to eight blocks of a cluster. Each keeps a ring of cp.async copies in flight; the partial sums meet through
// the cluster's shared memory, in a fixed order, and every block finishes its share of the tile.
//
// Within a block the operands stay in shared memory as they lie in memory. A thread reads four inner elements at a time:
// along k as 16-byte pieces of its features' lines (lines are padded by four words, so the eight lines that lanes read at a
// time fall into different banks), or, where features are contiguous, four features of each of the four. Either way TM + TN
// 16-byte reads feed 4 * TM * TN multiply-adds. Shared memory bounds it: 12 reads of a warp, four cycles each, for 128
// multiply-adds that four schedulers share (25 of the 74 TFLOP/s; tiles of 8 x 8 per thread leave too few warps and are
// slower). Sums run in fp32, one running sum per element, block and warp.
#include "fused_single.h"

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../runtime_state.h"
#include "activation.cuh"

namespace b200 {

namespace {

namespace cg = cooperative_groups;

constexpr int kStages = 4;
constexpr int kEach = 4;
constexpr int kMaxSplit = 8;  // blocks of a cluster that any launch may have

// TM x TN elements per thread, 8 x 4 threads per warp; WN warps side by side along the vectors, WK warps on different parts
// of a stage's KT inner elements.
template <int TM_, int TN_, int WN_, int WK_, int KT_>
struct Shape {
  static constexpr int TM = TM_, TN = TN_, WN = WN_, WK = WK_, KT = KT_;
  static constexpr int BM = 8 * TM, BN = 4 * TN * WN, THREADS = 32 * WN * WK;
  static_assert(KT % (4 * WK) == 0, "");
};
using Wide = Shape<8, 4, 4, 2, 32>;     // 64 x 64
using Slim = Shape<4, 4, 1, 4, 64>;     // 32 x 16

// Words of one operand's stage: `rows` lines of KT, or KT lines of `rows`.
template <bool MN>
__host__ __device__ constexpr int pitch_of(int rows, int kt) { return (MN ? rows : kt) + 4; }
template <bool MN>
__host__ __device__ constexpr int words_of(int rows, int kt) { return pitch_of<MN>(rows, kt) * (MN ? kt : rows); }

template <class S, bool AMN, bool BMN>
constexpr int ring_words() { return kStages * (words_of<AMN>(S::BM, S::KT) + words_of<BMN>(S::BN, S::KT)); }
template <class S, bool AMN, bool BMN>
constexpr int smem_bytes() {
  return 4 * (ring_words<S, AMN, BMN>() > S::WK * S::BM * S::BN ? ring_words<S, AMN, BMN>() : S::WK * S::BM * S::BN);
}

// Copies BYTES to shared memory of which the last BYTES - `valid` are zero; nothing is read when `valid` is 0.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from, int valid) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(valid) : "memory");
}

// One operand's stage: rows [r0, r0 + ROWS) of `count`, inner elements [k0, k0 + KT) of those before `end`.
template <bool MN, int ROWS, int KT, int VEC, int THREADS>
__device__ __forceinline__ void load_stage(uint32_t to, const float* base, long long ld, long long r0, long long count, long long k0,
                                           long long end) {
  constexpr int LINE = MN ? ROWS : KT, LINES = MN ? KT : ROWS, PITCH = pitch_of<MN>(ROWS, KT);
  constexpr int PIECES = LINE / VEC * LINES;
  static_assert(PIECES % THREADS == 0, "");
  const long long one0 = MN ? r0 : k0, one_end = MN ? count : end;
  const long long two0 = MN ? k0 : r0, two_end = MN ? end : count;
#pragma unroll
  for (int i = 0; i < PIECES / THREADS; ++i) {
    const int p = i * THREADS + static_cast<int>(threadIdx.x);
    const int line = p / (LINE / VEC), word = p % (LINE / VEC) * VEC;
    const long long one = one0 + word, two = two0 + line;
    long long left = one_end - one;
    left = two < two_end ? (left < 0 ? 0 : (left > VEC ? VEC : left)) : 0;
    copy_async<VEC * 4>(to + 4u * static_cast<uint32_t>(line * PITCH + word), left > 0 ? base + two * ld + one : base,
                        static_cast<int>(left) * 4);
  }
}

// Row of a tile that is a thread's i-th, out of N = count / lanes of them; `lane` counts over `LANES`.
template <bool MN, int LANES>
__device__ __forceinline__ int row_of(int lane, int i) {
  return MN ? (i >> 2) * 4 * LANES + lane * 4 + (i & 3) : lane + LANES * i;
}

// v[i][kk]: element kk of four inner elements for the thread's i-th row.
template <bool MN, int N, int LANES>
__device__ __forceinline__ void read_operand(float (&v)[N][4], const float* stage, int pitch, int first, int lane, int k) {
  if constexpr (MN) {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 q = *reinterpret_cast<const float4*>(stage + (k + kk) * pitch + first + row_of<true, LANES>(lane, i));
        v[i][kk] = q.x; v[i + 1][kk] = q.y; v[i + 2][kk] = q.z; v[i + 3][kk] = q.w;
      }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float4 q = *reinterpret_cast<const float4*>(stage + (first + row_of<false, LANES>(lane, i)) * pitch + k);
      v[i][0] = q.x; v[i][1] = q.y; v[i][2] = q.z; v[i][3] = q.w;
    }
  }
}

template <class S, bool AMN, bool BMN, int VEC>
__global__ void __launch_bounds__(S::THREADS) single_kernel(const SingleJob job, const long long k_per_block) {
  constexpr int A_WORDS = words_of<AMN>(S::BM, S::KT), B_WORDS = words_of<BMN>(S::BN, S::KT);
  constexpr int A_PITCH = pitch_of<AMN>(S::BM, S::KT), B_PITCH = pitch_of<BMN>(S::BN, S::KT);
  extern __shared__ __align__(16) float ring[];
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lane_m = lane & 7, lane_n = lane >> 3;
  const int warp_n = warp % S::WN, warp_k = warp / S::WN;
  const long long m0 = static_cast<long long>(blockIdx.x) * S::BM, n0 = static_cast<long long>(blockIdx.y) * S::BN;
  const long long begin = blockIdx.z * k_per_block;
  const long long end = begin + k_per_block < job.k ? begin + k_per_block : job.k;
  const int stages = begin < end ? static_cast<int>((end - begin + S::KT - 1) / S::KT) : 0;

  auto load = [&](int s) {
    if (s < stages) {
      const uint32_t at = ring_at + 4u * static_cast<uint32_t>((s % kStages) * (A_WORDS + B_WORDS));
      const long long k0 = begin + static_cast<long long>(s) * S::KT;
      load_stage<AMN, S::BM, S::KT, VEC, S::THREADS>(at, job.a, job.lda, m0, job.m, k0, end);
      load_stage<BMN, S::BN, S::KT, VEC, S::THREADS>(at + 4u * A_WORDS, job.b, job.ldb, n0, job.n, k0, end);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  float acc[S::TM][S::TN];
#pragma unroll
  for (int i = 0; i < S::TM; ++i)
#pragma unroll
    for (int j = 0; j < S::TN; ++j) acc[i][j] = 0.f;

#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load(s);
  for (int s = 0; s < stages; ++s) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncthreads();  // the stage has arrived for every thread, and the one to be overwritten has been read by every thread
    load(s + kStages - 1);
    const float* const a = ring + (s % kStages) * (A_WORDS + B_WORDS);
    const float* const b = a + A_WORDS;
    constexpr int PART = S::KT / S::WK;
#pragma unroll 2
    for (int k = warp_k * PART; k < (warp_k + 1) * PART; k += 4) {
      float av[S::TM][4], bv[S::TN][4];
      read_operand<AMN, S::TM, 8>(av, a, A_PITCH, 0, lane_m, k);
      read_operand<BMN, S::TN, 4>(bv, b, B_PITCH, warp_n * 4 * S::TN, lane_n, k);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int i = 0; i < S::TM; ++i)
#pragma unroll
          for (int j = 0; j < S::TN; ++j) acc[i][j] = fmaf(av[i][kk], bv[j][kk], acc[i][j]);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();

  // partial sums as [warp_k][vector][feature] in this block's shared memory
#pragma unroll
  for (int i = 0; i < S::TM; ++i)
#pragma unroll
    for (int j = 0; j < S::TN; ++j) {
      const int f = row_of<AMN, 8>(lane_m, i), v = warp_n * 4 * S::TN + row_of<BMN, 4>(lane_n, j);
      ring[(warp_k * S::BN + v) * S::BM + f] = acc[i][j];
    }
  cg::cluster_group cluster = cg::this_cluster();
  const int split = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  cluster.sync();
  constexpr int TILE = S::BM * S::BN;
  const int share = TILE / split;  // split is a power of two up to eight
  // kEach elements of a thread at a time, so that their reads overlap
  for (int first = rank * share + static_cast<int>(threadIdx.x); first < (rank + 1) * share; first += kEach * S::THREADS) {
    float y[kEach], add[kEach], z[kEach], bias[kEach];
    bool in[kEach];
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int e = first + u * S::THREADS;
      const long long f = m0 + e % S::BM, v = n0 + e / S::BM;
      in[u] = e < (rank + 1) * share && f < job.m && v < job.n;
      add[u] = in[u] && job.d != nullptr ? job.d[v * job.ldd + f] : 0.f;
      z[u] = in[u] && job.grad && job.z != nullptr ? job.z[v * job.ldz + f] : 0.f;
      bias[u] = in[u] && job.bias != nullptr ? job.bias[f] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int e = first + u * S::THREADS;
      y[u] = 0.f;
      if (!in[u]) continue;
#pragma unroll
      for (int q = 0; q < kMaxSplit; ++q) {
        if (q >= split) break;
        const float* const other = cluster.map_shared_rank(ring, q);
#pragma unroll
        for (int w = 0; w < S::WK; ++w) y[u] += other[w * TILE + e];
      }
      y[u] = job.alpha * y[u] + bias[u];
    }
    with_act(job.grad && job.z == nullptr ? static_cast<int>(kActIdentity) : job.act, [&](auto tag) {
      constexpr int ACT = decltype(tag)::value;
#pragma unroll
      for (int u = 0; u < kEach; ++u) {
        const int e = first + u * S::THREADS;
        const long long f = m0 + e % S::BM, v = n0 + e / S::BM;
        const float more = job.beta * add[u];
        if (job.grad) {
          y[u] = (y[u] + more) * act_slope<false, ACT>(z[u]);
        } else {
          if (in[u] && job.z != nullptr) job.z[v * job.ldz + f] = y[u];
          y[u] = act_value<false, ACT>(y[u]) + more;
        }
        if (in[u]) job.c[v * job.ldc + f] = y[u];
      }
    });
  }
  cluster.sync();  // nobody leaves while its sums are being read
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// Blocks that share a tile's inner extent: enough for two blocks per SM, each with at least 128 inner elements.
template <class S>
int split_of(long long m, long long n, long long k) {
  const long long tiles = ceil_div(m, S::BM) * ceil_div(n, S::BN);
  int split = 1;
  while (split < kMaxSplit && tiles * split < 2 * sm_count() && k / (2 * split) >= 128) split *= 2;
  return split;
}

template <class S, bool AMN, bool BMN, int VEC>
cudaError_t launch_as(const SingleJob& job, cudaStream_t stream) {
  constexpr int smem = smem_bytes<S, AMN, BMN>();
  const auto kernel = &single_kernel<S, AMN, BMN, VEC>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const long long gx = ceil_div(job.m, S::BM), gy = ceil_div(job.n, S::BN);
  if (gx > 0x7FFFFFFFLL || gy > 65535) return cudaErrorInvalidValue;
  const int split = split_of<S>(job.m, job.n, job.k);
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy), static_cast<unsigned>(split));
  config.blockDim = dim3(S::THREADS);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 1;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = static_cast<unsigned>(split);
  config.attrs = &attr;
  config.numAttrs = 1;
  // whole 16-byte pieces of k per block, so that pieces stay aligned
  return cudaLaunchKernelEx(&config, kernel, job, ceil_div(ceil_div(job.k, split), 4) * 4);
}

template <class S, bool AMN, bool BMN>
cudaError_t launch_width(const SingleJob& job, cudaStream_t stream) {
  const auto aligned = [](const float* p, long long ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 4 == 0; };
  return aligned(job.a, job.lda) && aligned(job.b, job.ldb) ? launch_as<S, AMN, BMN, 4>(job, stream)
                                                            : launch_as<S, AMN, BMN, 1>(job, stream);
}

template <class S>
cudaError_t launch_shape(const SingleJob& job, cudaStream_t stream) {
  if (job.a_mn) return job.b_mn ? launch_width<S, true, true>(job, stream) : launch_width<S, true, false>(job, stream);
  return job.b_mn ? launch_width<S, false, true>(job, stream) : launch_width<S, false, false>(job, stream);
}

}  // namespace

// The tensor-core product takes 24 to 31 us for anything up to two waves of its tiles, the kernels here run at 20 to 27
// TFLOP/s: 0.5e9 operations are where they meet (300 x 1000 x 1000: 29 us against 38; 256 x 1000 x 1000: 29 against 26).
// With fewer than 128 vectors it does not run at all, and the CUDA-core kernels without a split take 148 to 970 us where
// these take 85 to 153 (64 x 8192 x 2048 to 16 x 8192 x 8192); with fewer than 128 features its narrow form does, from
// 2e9 operations on better than this.
bool single_fits(long long m, long long n, long long k) {
  if (m > 65535LL * 16 || n > 65535LL * 16) return false;
  const double work = 2.0 * m * n * k;
  return n < 128 || work < (m < 128 ? 2e9 : 5e8);
}

cudaError_t launch_single(const SingleJob& job, cudaStream_t stream) {
  // The wide tile reads shared memory less often (100 x 4096 x 4096: 153 us against 174), the slim one wastes less on
  // ragged edges (33 x 1000 x 4096: 24 us against 40) and makes more blocks of a small product (64 x 400 x 300: 6.0 us
  // against 12.8).
  const auto covered = [&](long long bm, long long bn) { return static_cast<double>(ceil_div(job.m, bm) * bm) * (ceil_div(job.n, bn) * bn); };
  const long long wide_blocks = ceil_div(job.m, Wide::BM) * ceil_div(job.n, Wide::BN) * split_of<Wide>(job.m, job.n, job.k);
  if (wide_blocks >= sm_count() && 0.8 * covered(Wide::BM, Wide::BN) < covered(Slim::BM, Slim::BN)) return launch_shape<Wide>(job, stream);
  return launch_shape<Slim>(job, stream);
}

}  // namespace b200

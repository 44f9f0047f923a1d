// C = act(alpha op(A) op(B) + bias) + beta D and its backward form (alpha op(A) op(B) + beta D) * slope(Z), fp16 or
// bf16 operands, fp32 accumulation and epilogue arithmetic, one rounding per stored value. One kernel template serves
// plain and strided-batched products, products whose column extent is cut into ragged groups (experts' rows), and
// products whose inner extent is (experts' weight gradients).
//
// C is m x n with m contiguous. Rows are the features of the caller's vectors and columns the vectors, so a thread of
// the epilogue owns one feature (one tensor-memory lane) and walks along the vectors: the bias is one register, the
// bias gradient a running sum, and a 32-lane store covers consecutive addresses.
//
// Warp roles: warp 0 issues the TMA loads of the operand ring, warp 1 the MMAs (and clears what a ragged inner extent
// leaves behind its end), warp 2 builds the group table, warp 3 asks for D and Z of the next tile, warps 4.. drain the
// accumulators in groups of four warps, each group its own range of the tile's columns. Two accumulators alternate, so a
// tile is drained under the next one's MMAs.
//   CTAS == 2: a cluster of two CTAs works on 256 x BN tiles with cta_group::2, each CTA staging half of op(B).
//   CTAS == 1: tiles of 128 x BN; a cluster of p.split CTAs may share a tile's inner extent. Each CTA then leaves its
//   fp32 sums in its own shared memory and the CTAs add them up for a range of columns each, in the order of the ranks
//   (the result does not depend on which CTA came first).
//
// The epilogue goes by blocks of 16 columns x 32 rows, each warp by itself. A lane holds one row of a block while memory
// runs along the rows, so blocks are turned round in 1 to 2 KB of the warp's own shared memory and leave as 16-byte
// stores, four lanes to a column (C in half precision); D and Z come in the same way, one block ahead in registers.
// Columns and rows that end inside a block are cut off lane by lane. (Staging through TMA with a barrier among the warps
// per block, the form of the half-precision GEMM kernels, took 115 us for 8192 x 8192 x 512 and could not cut a group's
// columns.)
//
// Sums: the tensor cores cut off instead of rounding when they add to an accumulator, an error that all points towards zero
// and grows by 1e-7 of the result per 16 inner elements where all products have one sign. For results in single precision
// an accumulator therefore takes a few blocks at most and is then added, rounded, to sums in further columns of tensor
// memory (which the widest tile has room for only with one accumulator instead of two). The same sums in registers spill:
// 286 us against 247 for 32 weight gradients of 512 rows, 2048 x 2048 each, on 128 x 128 tiles. Results in 16 bits see the
// error beyond some ten thousand inner elements (half, 131072 products of one sign: 2.6 half steps of rounding, a million:
// 13): from kChunkHalf on an accumulator is handed over and the sums wait in global memory, one tile's per CTA (2048 x 2048
// x 65536 in half 394 -> 410 to 418 us, 4096 x 4096 x 32768 in bfloat16 1193 -> 1194 to 1222; shorter extents as before).
//
// What bounds it: products of 10^11 operations and more first the tensor pipe and, run for seconds, the board's power. 8192 x
// 8192 x 2048 in bfloat16 with bias, gelu and Z kept takes 208 us in a short run at full clock (1.32 PFLOP/s, tensor pipe
// busy 77 % of the cycles). Back to back at the power limit it takes 248, where a library product without any epilogue takes
// 210 and this one without any 218: the epilogue's work and its 268 MB of stores draw on the same power. Groups of rows: their last tiles
// run over the full width (256 columns round 16384 rows of 32 experts up to 1.2 times as many). Weight gradients in single
// precision: the MMAs wait while the one accumulator of 256 columns is being emptied (244 us for 32 of 2048 x 2048, 2.8 TB/s).
// Decoding: the reads of the weights (48 x 4096 x 8192 20.5 us with the weights in memory, 3.4 TB/s; 16.4 with them in L2),
// of which 5 us are the start and the meeting of the split tiles.
//
// All waits are bounded; on expiry a code is left in the status word and every role leaves its loop.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../runtime_state.h"
#include "activation.cuh"
#include "fused_gemm.h"
#include "group_table.cuh"
#include "tc_common.cuh"

namespace b200 {
namespace fused {

using namespace tc;

constexpr int BM = 128;   // rows of op(A) per CTA
constexpr int ROW_K = 64; // inner elements of a 128-byte swizzle row
constexpr int CB = 16;    // columns per epilogue block
// inner elements per accumulator: results in single precision; sums of two halves, whose users (the Newton-Schulz steps)
// amplify an error that all entries share
constexpr int kChunkSingle = 256, kChunkParts = 128;
static_assert(kChunkHalf % 128 == 0, "whole stages");

// Two values rounded to 16 bits in one word (the packed conversion runs on the full-rate pipe, the single one does not).
template <class E>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A block of 32 rows x CB columns of a 16-bit matrix between memory and the lanes. In memory order lane l has the rows
// 8 (l % 4) .. + 7 of the columns 2 (l / 4) and 2 (l / 4) + 1; in row order it has row l of all columns. Between the two the
// block lies in shared memory as [column pair][row] words of two columns.
template <class E>
struct Block16 {
  static constexpr int WORDS = CB * 16;  // shared memory
  uint4 v[2];

  // base: the block's first element; rows_left (a multiple of 8) and cols_left: how many of its rows and columns exist.
  __device__ __forceinline__ void load(const E* base, long long ld, int rows_left, int cols_left, int lane) {
    const int c0 = 2 * (lane >> 2), r0 = 8 * (lane & 3);
    const bool in = r0 < rows_left;
    const E* const at = base + static_cast<long long>(c0) * ld + r0;
    v[0] = v[1] = make_uint4(0, 0, 0, 0);
    if (in && c0 < cols_left) v[0] = *reinterpret_cast<const uint4*>(at);
    if (in && c0 + 1 < cols_left) v[1] = *reinterpret_cast<const uint4*>(at + ld);
  }
  // memory order -> row order: f[j] is column j of this lane's row. The buffer is free before and after.
  __device__ __forceinline__ void to_rows(uint32_t* smem, float (&f)[CB], int lane) const {
    const uint4 a = v[0], b = v[1];
    uint4* const at = reinterpret_cast<uint4*>(smem + (lane >> 2) * 32 + (lane & 3) * 8);
    at[0] = make_uint4(__byte_perm(a.x, b.x, 0x5410), __byte_perm(a.x, b.x, 0x7632), __byte_perm(a.y, b.y, 0x5410),
                       __byte_perm(a.y, b.y, 0x7632));
    at[1] = make_uint4(__byte_perm(a.z, b.z, 0x5410), __byte_perm(a.z, b.z, 0x7632), __byte_perm(a.w, b.w, 0x5410),
                       __byte_perm(a.w, b.w, 0x7632));
    __syncwarp();
#pragma unroll
    for (int q = 0; q < CB / 2; ++q) {
      const uint32_t w = smem[q * 32 + lane];
      const unsigned short lo = static_cast<unsigned short>(w), hi = static_cast<unsigned short>(w >> 16);
      f[2 * q] = to_float(*reinterpret_cast<const E*>(&lo));
      f[2 * q + 1] = to_float(*reinterpret_cast<const E*>(&hi));
    }
    __syncwarp();
  }
  // row order -> memory
  static __device__ __forceinline__ void store(E* base, long long ld, int rows_left, int cols_left, uint32_t* smem,
                                               const float (&f)[CB], int lane) {
#pragma unroll
    for (int q = 0; q < CB / 2; ++q) smem[q * 32 + lane] = pack2<E>(f[2 * q], f[2 * q + 1]);
    __syncwarp();
    const int c0 = 2 * (lane >> 2), r0 = 8 * (lane & 3);
    const bool in = r0 < rows_left;
    E* const at = base + static_cast<long long>(c0) * ld + r0;
    const uint4* const from = reinterpret_cast<const uint4*>(smem + (lane >> 2) * 32 + r0);
    const uint4 w0 = from[0], w1 = from[1];
    if (in && c0 < cols_left)
      *reinterpret_cast<uint4*>(at) = make_uint4(__byte_perm(w0.x, w0.y, 0x5410), __byte_perm(w0.z, w0.w, 0x5410),
                                                 __byte_perm(w1.x, w1.y, 0x5410), __byte_perm(w1.z, w1.w, 0x5410));
    if (in && c0 + 1 < cols_left)
      *reinterpret_cast<uint4*>(at + ld) = make_uint4(__byte_perm(w0.x, w0.y, 0x7632), __byte_perm(w0.z, w0.w, 0x7632),
                                                      __byte_perm(w1.x, w1.y, 0x7632), __byte_perm(w1.z, w1.w, 0x7632));
    __syncwarp();
  }
};

// The same for single precision: in memory order lane l has the rows 4 (l % 8) .. + 3 of the columns l / 8 + 4 h.
struct Block32 {
  static constexpr int WORDS = CB * 32;
  uint4 v[CB / 4];

  __device__ __forceinline__ void load(const float* base, long long ld, int rows_left, int cols_left, int lane) {
    const int r0 = 4 * (lane & 7), c0 = lane >> 3;
    const float* at = base + static_cast<long long>(c0) * ld + r0;
#pragma unroll
    for (int h = 0; h < CB / 4; ++h, at += 4 * ld) {
      v[h] = make_uint4(0, 0, 0, 0);
      if (r0 < rows_left && c0 + 4 * h < cols_left) v[h] = *reinterpret_cast<const uint4*>(at);
    }
  }
  __device__ __forceinline__ void to_rows(uint32_t* smem, float (&f)[CB], int lane) const {
#pragma unroll
    for (int h = 0; h < CB / 4; ++h) *reinterpret_cast<uint4*>(smem + ((lane >> 3) + 4 * h) * 32 + 4 * (lane & 7)) = v[h];
    __syncwarp();
#pragma unroll
    for (int j = 0; j < CB; ++j) f[j] = __uint_as_float(smem[j * 32 + lane]);
    __syncwarp();
  }
  static __device__ __forceinline__ void store(float* base, long long ld, int rows_left, int cols_left, uint32_t* smem,
                                               const float (&f)[CB], int lane) {
#pragma unroll
    for (int j = 0; j < CB; ++j) smem[j * 32 + lane] = __float_as_uint(f[j]);
    __syncwarp();
    const int r0 = 4 * (lane & 7), c0 = lane >> 3;
    float* at = base + static_cast<long long>(c0) * ld + r0;
#pragma unroll
    for (int h = 0; h < CB / 4; ++h, at += 4 * ld) {
      const uint4 w = *reinterpret_cast<const uint4*>(smem + (c0 + 4 * h) * 32 + r0);
      if (r0 < rows_left && c0 + 4 * h < cols_left) *reinterpret_cast<uint4*>(at) = w;
    }
    __syncwarp();
  }
};
template <class E>
struct BlockOf { using type = Block16<E>; };
template <>
struct BlockOf<float> { using type = Block32; };

// Starts the load of 16 accumulator columns; the values may be used after tmem_wait.
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// The registers are operands, so that no use of them moves above the wait.
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}

__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tma_load_3d_hint(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z,
                                                 uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5}], [%2], %6;"
      :
      : "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "l"(policy)
      : "memory");
}
// Arrival on a barrier of another CTA that orders this CTA's own accesses only: what it announces are tensor-memory
// reads, ordered by their own wait and fence. A release at cluster scope would first wait for the epilogue's global
// stores (1500 cycles per tile).
__device__ __forceinline__ void mbar_arrive_peer(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// Asks L2 for a tile of an epilogue matrix.
__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* map, int x, int y, int z) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x),
               "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
// True in one lane of a converged warp. Instructions of the tensor and TMA units take their operands from uniform
// registers; behind this predicate the compiler knows that one lane is active, behind `lane == 0` it does not and walks
// through the lanes (measured: 550 cycles for the four MMAs of a stage, whatever their width).
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one)::"memory");
  return one != 0;
}
// Bounded wait of a whole converged warp: one lane polls.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, unsigned code,
                                          unsigned int* status) {
  int ok = 1;
  if ((threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity, abort_flag, code, status) ? 1 : 0;
  return __shfl_sync(0xFFFFFFFFu, ok, 0) != 0;
}
// The same for the epilogue's long waits: sleeping between polls leaves the issue slots and the power to the MMAs (1.5 % of
// 8192^3, which runs at the power limit).
__device__ __forceinline__ bool warp_wait_relaxed(uint32_t bar, uint32_t parity, volatile int* abort_flag, unsigned code,
                                                  unsigned int* status) {
  int ok = 1;
  if ((threadIdx.x & 31) == 0) {
    for (int i = 0; i < 10000 && !mbar_try_wait(bar, parity); ++i) __nanosleep(200);
    ok = mbar_wait(bar, parity, abort_flag, code, status) ? 1 : 0;
  }
  return __shfl_sync(0xFFFFFFFFu, ok, 0) != 0;
}
// The same for the inner loops of the producer and of the MMA issuer: a try by all lanes and a vote take 30 ns less per
// stage than one lane's poll and its broadcast where the barrier is ready, as it mostly is (128 x 128 tiles 344 -> 303 ns).
__device__ __forceinline__ bool loop_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, unsigned code,
                                          unsigned int* status) {
  const bool ready = mbar_try_wait(bar, parity);
  if (__all_sync(0xFFFFFFFFu, ready)) return true;
  return warp_wait(bar, parity, abort_flag, code, status);
}
__device__ __forceinline__ bool warp_wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, unsigned code,
                                                  unsigned int* status) {
  int ok = 1;
  if ((threadIdx.x & 31) == 0) ok = mbar_wait_cluster(bar, parity, abort_flag, code, status) ? 1 : 0;
  return __shfl_sync(0xFFFFFFFFu, ok, 0) != 0;
}

// The same value as the compiler sees it in every lane: what the tensor and TMA units take from uniform registers is
// computed there if it stems from such values, and moved there operand by operand if not.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xFFFFFFFFu, x, 0); }

// One tile of the walk.
struct Tile {
  int z;             // problem
  int tm, tn;        // tile row / column inside the problem
  int col0, col_end; // first column of the tile, end of the problem's columns
  int k0, k_len;     // inner extent
  int col_tile;      // running number of the column tile over all groups
};

__device__ __forceinline__ int total_tiles(const FusedParams& p, const int* tiles) {
  if (p.kind == kFusedRaggedCols) return tiles[p.problems] * p.tiles_m;
  if (p.tri) return p.tiles_m * (p.tiles_m + 1) / 2 * p.problems;
  return p.tiles_m * p.tiles_n * p.problems;
}

// a / b for 0 <= a < 2^30 and b > 0 by a float quotient and a correction; exact.
__device__ __forceinline__ int divide(int a, int b) {
  if (a < b) return 0;
  if (a >= (1 << 22)) return a / b;  // the quotient's error stays below one for smaller numerators
  int q = __float2int_rz(__fdividef(__int2float_rn(a), __int2float_rn(b)));
  const int r = a - q * b;
  q += (r >= b) - (r < 0);
  return q;
}

template <int BN>
__device__ __forceinline__ Tile locate(const FusedParams& p, int tile, const int* start, const int* tiles) {
  Tile t;
  int in_problem, cols;
  if (p.kind == kFusedRaggedCols) {
    const int want = divide(tile, p.tiles_m);  // the group with tiles[g] <= want < tiles[g + 1]
    int lo = 0, hi = p.problems;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tiles[mid] <= want) lo = mid; else hi = mid;
    }
    t.z = lo;
    in_problem = tile - tiles[lo] * p.tiles_m;
    cols = tiles[lo + 1] - tiles[lo];
  } else if (p.tri) {
    const int per = p.tiles_m * (p.tiles_m + 1) / 2;
    t.z = divide(tile, per);
    in_problem = tile - t.z * per;
    cols = p.tiles_n;
  } else {
    const int per = p.tiles_m * p.tiles_n;
    t.z = divide(tile, per);
    in_problem = tile - t.z * per;
    cols = p.tiles_n;
  }
  if (p.tri) {
    int r = static_cast<int>((sqrtf(8.f * static_cast<float>(in_problem) + 1.f) - 1.f) * 0.5f);
    while (r * (r + 1) / 2 > in_problem) --r;
    while ((r + 1) * (r + 2) / 2 <= in_problem) ++r;
    t.tm = r;
    t.tn = in_problem - r * (r + 1) / 2;
  } else {
    const int per_group = p.raster * cols;
    const int group = divide(in_problem, per_group);
    const int first = group * p.raster;
    const int rows = min(p.raster, p.tiles_m - first);
    const int in_group = in_problem - group * per_group;
    t.tn = divide(in_group, rows);
    t.tm = first + in_group - t.tn * rows;
  }
  t.k0 = 0;
  t.k_len = p.k;
  t.col_tile = t.tn;
  if (p.kind == kFusedRaggedCols) {
    t.col0 = start[t.z] + t.tn * BN;
    t.col_end = start[t.z + 1];
    t.col_tile += tiles[t.z];
  } else {
    t.col0 = t.tn * BN;
    t.col_end = p.n;
    if (p.kind == kFusedRaggedInner) {
      t.k0 = start[t.z];
      t.k_len = start[t.z + 1] - t.k0;
    }
  }
  return t;
}

// What the epilogue is compiled for. The first two need 16-byte accesses to C, D and Z; the third takes everything else,
// tiles shared by a cluster included.
// The fourth multiplies matrices that are kept as a sum of two halves, hi + lo: about 22 bits. Planes 2z and 2z + 1 of every
// matrix are the two parts of problem z. The product takes three terms one after the other, hi hi + hi lo + lo hi (lo lo
// lies below the rounding), C and D are split and joined in the epilogue.
enum FusedMode : int { kModeForward = 0, kModeGrad = 1, kModeGeneral = 2, kModeParts = 3 };

template <int CTAS, int BN, class T, class DT, class OT, int MODE>
__global__ void __launch_bounds__(fused_threads(BN), 1)
fused_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                  const __grid_constant__ CUtensorMap map_d, const __grid_constant__ CUtensorMap map_z,
                  const FusedParams p) {
  static_assert(sizeof(DT) == sizeof(OT), "D and C share the staging buffers");
  constexpr bool CHUNKED = sizeof(OT) == 4 || MODE == kModeParts;  // sums beyond what the accumulators give
  constexpr int CHUNK = (MODE == kModeParts ? kChunkParts : kChunkSingle) / (ROW_K * fused_stage_rows(CTAS, BN));  // stages
  constexpr int EG = fused_groups(BN);
  constexpr int B_ROWS = BN / CTAS;
  constexpr int SUBS = fused_stage_rows(CTAS, BN);  // a stage holds SUBS blocks of 64 inner elements, one after the other
  constexpr int BK = ROW_K * SUBS;
  constexpr int A_BYTES = BM * ROW_K * 2;
  constexpr int SUB_BYTES = A_BYTES + B_ROWS * ROW_K * 2;
  constexpr int STAGE_BYTES = SUB_BYTES * SUBS;
  constexpr int GROUP_COLS = BN / EG;
  // accumulators, then the sums of results in single precision; a power of two
  constexpr int ACCS = (CHUNKED && BN == 256) ? 1 : 2;
  constexpr uint32_t SUMS_AT = ACCS * BN;
  constexpr uint32_t TMEM_COLS = CHUNKED ? (BN == 256 ? 512 : 4 * BN) : 2 * BN;
  constexpr bool FAST = sizeof(OT) == 2;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t tiles_base = (raw + 1023u) & ~1023u;
  uint8_t* const base_ptr = smem_raw + (tiles_base - raw);
  const bool aux = p.z != nullptr;
  const int stages = p.stages;
  const int split = (CTAS == 1 && MODE == kModeGeneral) ? p.split : 1;
  const int chunk = CHUNKED ? CHUNK : (p.sums != nullptr ? kChunkHalf / BK : 0x7FFFFFFF);  // stages per accumulator
  uint8_t* const staging = base_ptr + stages * STAGE_BYTES;
  uint8_t* const behind = staging + fused_staging_bytes(BN, CHUNKED, aux, split);
  const uint32_t bar_base = smem_u32(behind);
  // full [0, 16), empty [16, 32), accumulator full / empty [32, 36), sums ready / free [36, 38), tail [40, 56)
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (16 + s); };
  auto acc_full_bar = [&](int a) { return bar_base + 8u * (32 + a); };
  auto acc_empty_bar = [&](int a) { return bar_base + 8u * (34 + a); };
  const uint32_t sums_ready = bar_base + 8u * 36, sums_free = bar_base + 8u * 37;
  // Pairs with a ragged inner extent: the second CTA has cleared the end of the block in this stage. (That the block has
  // landed there it learns from its own full barrier.) One barrier per stage: of groups shorter than the ring several
  // last blocks are under way at once.
  auto tail_bar = [&](int s) { return bar_base + 8u * (40 + s); };
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(behind + 8 * 56);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* const progress = abort_flag + 1;  // tiles that the epilogue has begun
  int* const start = reinterpret_cast<int*>(behind + kFusedBarBytes);
  int* const tiles = start + p.problems + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = (CTAS == 2 || split > 1) ? cluster_ctarank() : 0u;
  const int team = CTAS == 2 ? 2 : split;          // CTAs that work on one tile
  const int first_tile = static_cast<int>(blockIdx.x) / team;
  const int tile_step = static_cast<int>(gridDim.x) / team;

  if (threadIdx.x == 32) {
    prefetch_map(&map_a);
    prefetch_map(&map_b);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full_bar(a), 1);
      mbar_init(acc_empty_bar(a), 4 * EG * CTAS);
    }
    mbar_init(sums_ready, 4 * EG * split);
    mbar_init(sums_free, 4 * EG * split);
    for (int s = 0; s < stages; ++s) mbar_init(tail_bar(s), 1);
    *abort_flag = 0;
    *progress = 0;
    fence_barrier_init();
  }
  // this CTA's share of a tile's inner blocks
  auto k_range = [&](const Tile& t, int& kb0, int& kb1) {
    const int blocks = (t.k_len + BK - 1) / BK * (MODE == kModeParts ? 3 : 1);
    if (split > 1) {
      kb0 = blocks * static_cast<int>(rank) / split;
      kb1 = blocks * (static_cast<int>(rank) + 1) / split;
    } else {
      kb0 = 0;
      kb1 = blocks;
    }
  };


  // Loads of one inner block into a stage of the ring, by one lane.
  auto issue_block = [&](const Tile& t, int kb, int stage, uint64_t policy) {
    const int a_row0 = (t.tm * CTAS + (CTAS == 2 ? static_cast<int>(rank) : 0)) * BM;
    const int b_row0 = t.col0 + (CTAS == 2 ? static_cast<int>(rank) * B_ROWS : 0);
    int az = p.a_batched ? t.z : 0, bz = p.b_batched ? t.z : 0;
    if constexpr (MODE == kModeParts) {
      const int per_term = (t.k_len + BK - 1) / BK;
      const int term = kb >= 2 * per_term ? 2 : (kb >= per_term ? 1 : 0);
      kb -= term * per_term;
      az = 2 * t.z + (term == 2 ? 1 : 0);
      bz = 2 * t.z + (term == 1 ? 1 : 0);
    }
    uint32_t bar;
    if constexpr (CTAS == 2) {
      // a block whose end has to be cleared is counted by each CTA for itself
      const bool tail = p.kind == kFusedRaggedInner && t.k_len - kb * BK < BK;
      if (rank == 0) {
        bar = map_to_cta(full_bar(stage), 0);
        mbar_arrive_expect_tx(full_bar(stage), (tail ? 1 : 2) * STAGE_BYTES);  // otherwise the bytes of both CTAs
      } else if (tail) {
        bar = map_to_cta(full_bar(stage), 1);
        mbar_arrive_expect_tx(full_bar(stage), STAGE_BYTES);
      } else {
        bar = map_to_cta(full_bar(stage), 0);
      }
    } else {
      bar = full_bar(stage);
      mbar_arrive_expect_tx(bar, STAGE_BYTES);
    }
    auto load = [&](uint32_t dst, const CUtensorMap* map, int cx, int cy, int cz) {
      if constexpr (CTAS == 2) tma_load_3d_pair_hint(dst, map, bar, cx, cy, cz, policy);
      else tma_load_3d_hint(dst, map, bar, cx, cy, cz, policy);
    };
#pragma unroll
    for (int sub = 0; sub < SUBS; ++sub) {
      const uint32_t a_dst = tiles_base + stage * STAGE_BYTES + sub * SUB_BYTES;
      const uint32_t b_dst = a_dst + A_BYTES;
      const int x = t.k0 + kb * BK + sub * ROW_K;
      if (p.a_mn) {
#pragma unroll
        for (int j = 0; j < BM / 64; ++j) load(a_dst + j * 8192, &map_a, a_row0 + j * 64, x, az);
      } else {
        load(a_dst, &map_a, x, a_row0, az);
      }
      if (p.b_mn) {
#pragma unroll
        for (int j = 0; j < B_ROWS / 64; ++j) load(b_dst + j * 8192, &map_b, b_row0 + j * 64, x, bz);
      } else {
        load(b_dst, &map_b, x, b_row0, bz);
      }
    }
  };

  if (warp == 1) {
    if constexpr (CTAS == 2) tmem_alloc_pair(smem_u32(tmem_slot), TMEM_COLS);
    else tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
  }
  if (warp == 2 && p.kind != kFusedPlain)
    build_table(p.offsets, p.problems, p.kind == kFusedRaggedCols ? p.n : p.k, BN, start, tiles);
  // A launch that follows another one closely is set up under the end of that one; from here on its results are read.
  if (p.chained) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  if (CTAS == 2 || split > 1) cluster_sync_all();  // all barriers exist before anyone signals across CTAs
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int num_tiles = total_tiles(p, tiles);

  // accumulator number n of this CTA: which one, and the parity of its use
  auto acc_of = [](int n) { return ACCS == 1 ? 0 : (n & 1); };
  auto acc_parity = [](int n) { return static_cast<uint32_t>(ACCS == 1 ? n : (n >> 1)) & 1u; };

  if (warp == 0) {
    // ---- TMA producer: the warp walks along, one lane issues ----
    {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint64_t policy = l2_policy(2);  // operands stay in L2: other tiles read them too
      const int last_tile = uniform(num_tiles);
      for (int tile = first_tile; tile < last_tile && ok; tile += tile_step) {
        Tile t = locate<BN>(p, tile, start, tiles);
        t.z = uniform(t.z);
        t.tm = uniform(t.tm);
        t.col0 = uniform(t.col0);
        t.k0 = uniform(t.k0);
        t.k_len = uniform(t.k_len);
        int kb0, kb1;
        k_range(t, kb0, kb1);
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = loop_wait(empty_bar(stage), phase ^ 1u, abort_flag, 1u, p.status);
          if (!ok) break;
          if (elect_one()) issue_block(t, kb, stage, policy);
          __syncwarp();
          if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) {
        // copies already issued still land in this CTA's shared memory: wait far longer than any copy takes
        const long long begin = clock64();
        while (clock64() - begin < 2000000LL) {}
      }
    }
  } else if (warp == 1) {
    // Of a ragged inner extent the last block holds inner indices of the next group (or whatever lies behind the matrix).
    // Both operands have one 128-byte row per inner index and 64 elements of m / n; rows up to the next multiple of an
    // MMA's 16 are cleared in both (0 * NaN would not be 0), the MMAs behind that are left out. Called by the whole warp.
    auto clear_tail = [&](int stage, int valid) {
      const int steps = (valid + 15) / 16, rows = steps * 16 - valid;
      // (a block that ends at a swizzle row's end has nothing to clear; otherwise the end lies inside one)
      const int in_row = valid % ROW_K;
      uint8_t* const s = base_ptr + stage * STAGE_BYTES + valid / ROW_K * SUB_BYTES;
      constexpr int TILES = BM / 64 + B_ROWS / 64;
      // eight lanes to a row, four rows at a time
      for (int r = lane >> 3; r < rows; r += 4) {
#pragma unroll
        for (int j = 0; j < TILES; ++j)
          *reinterpret_cast<uint4*>(s + j * 8192 + (in_row + r) * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async();
      __syncwarp();
      return steps;
    };
    if (CTAS == 2 && rank == 1 && p.kind == kFusedRaggedInner) {
      // ---- second CTA of a pair: clears the end of its own operands and tells the leader ----
      int blocks_before = 0;
      uint32_t phases = 0;  // of the full barriers, one bit per stage
      for (int tile = first_tile; tile < num_tiles; tile += tile_step) {
        const Tile t = locate<BN>(p, tile, start, tiles);
        blocks_before += (t.k_len + BK - 1) / BK;
        if (t.k_len % BK == 0) continue;
        const int stage = (blocks_before - 1) % stages;
        if (!warp_wait(full_bar(stage), (phases >> stage) & 1u, abort_flag, 10u, p.status)) break;
        phases ^= 1u << stage;
        clear_tail(stage, t.k_len % BK);
        if (lane == 0) mbar_arrive_remote(map_to_cta(tail_bar(stage), 0));
      }
    }
    // ---- MMA issuer (of a pair: the leader, for both SMs): the warp walks along, one lane issues ----
    if (CTAS == 1 || rank == 0) {
      auto wait = [&](uint32_t bar, uint32_t parity, unsigned code) { return loop_wait(bar, parity, abort_flag, code, p.status); };
      auto commit = [&](uint32_t bar) {
        if constexpr (CTAS == 2) umma_commit_pair(bar);
        else umma_commit(bar);
      };
      // K-major: 128-byte rows along K (stride offset 1024 = eight rows), 32 B per MMA step. MN-major: one 128-byte row of
      // 64 elements per k, blocks 8192 B apart, 2048 B per MMA step.
      const uint64_t a_form = smem_desc(0, p.a_mn ? 8192 : 16, 1024, kLayoutSw128);
      const uint64_t b_form = smem_desc(0, p.b_mn ? 8192 : 16, 1024, kLayoutSw128);
      const uint32_t a_step = p.a_mn ? (2048u >> 4) : 2u, b_step = p.b_mn ? (2048u >> 4) : 2u;
      const uint32_t idesc = p.idesc;
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      uint32_t tail_phases = 0;
      bool ok = true;
      const int last_tile = uniform(num_tiles);
      const uint32_t tmem = static_cast<uint32_t>(uniform(static_cast<int>(tmem_base)));
      for (int tile = first_tile; tile < last_tile && ok; tile += tile_step, ++local) {
        Tile t = locate<BN>(p, tile, start, tiles);
        t.k_len = uniform(t.k_len);
        int kb0, kb1;
        k_range(t, kb0, kb1);
        int acc = acc_of(local);
        ok = wait(acc_empty_bar(acc), acc_parity(local) ^ 1u, 2u);
        if (!ok) break;
        tcgen05_fence_after();
        uint32_t d_tmem = tmem + static_cast<uint32_t>(acc * BN);
        int first_kb = kb0;  // first block of the current accumulator
        for (int kb = kb0; kb < kb1; ++kb) {
          if (kb - first_kb == chunk) {  // hand this accumulator over and go on in the other one
            if (elect_one()) commit(acc_full_bar(acc));
            __syncwarp();
            ++local;
            first_kb = kb;
            acc = acc_of(local);
            ok = wait(acc_empty_bar(acc), acc_parity(local) ^ 1u, 2u);
            if (!ok) break;
            tcgen05_fence_after();
            d_tmem = tmem + static_cast<uint32_t>(acc * BN);
          }
          ok = wait(full_bar(stage), phase, 3u);
          if (!ok) break;
          int steps = BK / 16;
          if (p.kind == kFusedRaggedInner && t.k_len - kb * BK < BK) {
            steps = clear_tail(stage, t.k_len - kb * BK);
            if (CTAS == 2) {
              ok = warp_wait_cluster(tail_bar(stage), (tail_phases >> stage) & 1u, abort_flag, 11u, p.status);
              if (!ok) break;
              tail_phases ^= 1u << stage;
            }
          }
          tcgen05_fence_after();
          if (elect_one()) {
            // (an address in a cluster carries the CTA's rank above the 18 bits that the descriptor takes)
            const uint32_t a_src = tiles_base + stage * STAGE_BYTES;
            const uint64_t da = a_form | ((a_src >> 4) & 0x3FFFu), db = b_form | (((a_src + A_BYTES) >> 4) & 0x3FFFu);
            const uint32_t fresh = kb == first_kb ? 0u : 1u;
            auto mma = [&](int ks) {
              const uint32_t sub = static_cast<uint32_t>(ks / 4) * (SUB_BYTES >> 4), in_sub = static_cast<uint32_t>(ks % 4);
              const uint64_t ma = da + sub + a_step * in_sub, mb = db + sub + b_step * in_sub;
              if constexpr (CTAS == 2) umma_f16_pair(d_tmem, ma, mb, idesc, ks == 0 ? fresh : 1u);
              else umma_f16(d_tmem, ma, mb, idesc, ks == 0 ? fresh : 1u);
            };
            if (steps == BK / 16) {
#pragma unroll
              for (int ks = 0; ks < BK / 16; ++ks) mma(ks);
            } else {
              for (int ks = 0; ks < steps; ++ks) mma(ks);
            }
            commit(empty_bar(stage));
          }
          __syncwarp();
          if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
        if (ok && elect_one()) commit(acc_full_bar(acc));  // without inner blocks this arrives at once: zeros are taken
      }
    }
  } else if (warp == 3) {
    // ---- D and Z of the next tile on their way to L2 while this one's operands are multiplied ----
    if (MODE != kModeGeneral && p.prefetch && lane == 0) {
      for (int tile = first_tile; tile < num_tiles; tile += tile_step) {
        // at most two tiles ahead of the epilogue; a hint, so it does not insist
        const int n = (tile - first_tile) / tile_step;
        for (int spin = 0; spin < 20000 && *progress < n - 1 && !*abort_flag; ++spin) __nanosleep(200);
        const Tile t = locate<BN>(p, tile, start, tiles);
        const int row0 = (t.tm * CTAS + (CTAS == 2 ? static_cast<int>(rank) : 0)) * BM;
        const int zc = p.kind == kFusedRaggedCols ? 0 : (MODE == kModeParts ? 2 * t.z : t.z);
        if (row0 < p.m) {
#pragma unroll
          for (int c = 0; c < BN; c += 32) {
            if (t.col0 + c >= t.col_end) break;
            if (p.d != nullptr) tma_prefetch_3d(&map_d, row0, t.col0 + c, zc);
            if (MODE == kModeParts && p.d != nullptr) tma_prefetch_3d(&map_d, row0, t.col0 + c, zc + 1);
            if (MODE == kModeGrad && aux) tma_prefetch_3d(&map_z, row0, t.col0 + c, zc);
          }
        }
      }
    }
  } else if (warp >= 4) {
    // ---- epilogue ----
    using BlockC = typename BlockOf<OT>::type;
    using BlockD = typename BlockOf<DT>::type;
    using BlockZ = Block16<T>;
    constexpr int BLOCKS = GROUP_COLS / CB;
    const int group = (warp - 4) >> 2;
    const int quad = warp & 3;  // tensor-memory lanes this warp may read
    const int row_in_cta = quad * 32 + lane;
    const bool has_d = p.d != nullptr;
    const bool grad = MODE == kModeGrad || (MODE == kModeGeneral && p.grad);
    const bool z_in = aux && grad, z_out = aux && !grad;
    const bool one_tile = num_tiles <= tile_step;  // a short kernel: its end is what counts
    int local = 0;   // accumulators taken so far
    int tiles_done = 0;
    bool ok = true;

    for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step, ++tiles_done) {
      if (threadIdx.x == 128) *progress = tiles_done + 1;
      const Tile t = locate<BN>(p, tile, start, tiles);
      const int cta_row0 = (t.tm * CTAS + (CTAS == 2 ? static_cast<int>(rank) : 0)) * BM;
      const int warp_row0 = cta_row0 + quad * 32;
      const int row = cta_row0 + row_in_cta;
      const int rows_left = p.m - warp_row0;  // may be negative: the tile's last warps may lie wholly below C
      const bool in_rows = row < p.m;
      const int zc = p.kind == kFusedRaggedCols ? 0 : (MODE == kModeParts ? 2 * t.z : t.z);  // plane of C, D, Z
      const float bias = (p.bias != nullptr && in_rows) ? to_float(static_cast<const T*>(p.bias)[t.z * p.bias_stride + row]) : 0.f;
      const int group_col0 = t.col0 + group * GROUP_COLS;
      const int group_cols = t.col_end - group_col0;  // columns that exist from this group's first one on
      // first element of this warp's part
      OT* const c_ptr = static_cast<OT*>(p.c) + zc * p.c_stride + static_cast<long long>(group_col0) * p.ldc + warp_row0;
      const DT* const d_ptr = static_cast<const DT*>(p.d) + zc * p.d_stride + static_cast<long long>(group_col0) * p.ldd + warp_row0;
      T* const z_ptr = static_cast<T*>(p.z) + zc * p.z_stride + static_cast<long long>(group_col0) * p.ldz + warp_row0;
      float row_sum = 0.f;
      int kb0, kb1;
      k_range(t, kb0, kb1);
      const bool empty = kb1 <= kb0;
      auto accumulator = [&](int number) {
        return tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(acc_of(number) * BN + group * GROUP_COLS);
      };
      auto wait_accumulator = [&](int number) {
        return one_tile ? warp_wait(acc_full_bar(acc_of(number)), acc_parity(number), abort_flag, 4u, p.status)
                        : warp_wait_relaxed(acc_full_bar(acc_of(number)), acc_parity(number), abort_flag, 4u, p.status);
      };
      auto release_accumulator = [&](int number) {
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CTAS == 2) mbar_arrive_peer(map_to_cta(acc_empty_bar(acc_of(number)), 0));
          else mbar_arrive(acc_empty_bar(acc_of(number)));
        }
      };

      // Results in single precision: the accumulators are added up in further columns, which only this warp touches.
      const uint32_t sums_tmem = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + SUMS_AT + static_cast<uint32_t>(group * GROUP_COLS);
      if constexpr (CHUNKED) {
        const int chunks = empty ? 1 : (kb1 - kb0 + CHUNK - 1) / CHUNK;
        for (int c = 0; c < chunks; ++c) {
          ok = wait_accumulator(local);
          if (!ok) break;
          tcgen05_fence_after();
          if (!empty) {
            // two blocks at a time: all their loads under way before the first wait
            constexpr int PAIR = BLOCKS % 2 == 0 ? 2 : 1;
            const uint32_t from = accumulator(local);
#pragma unroll 2
            for (int cb = 0; cb < BLOCKS; cb += PAIR) {
              uint32_t r[PAIR][CB], s[PAIR][CB];
#pragma unroll
              for (int i = 0; i < PAIR; ++i) {
                tmem_ld(from + (cb + i) * CB, r[i]);
                if (c > 0) tmem_ld(sums_tmem + (cb + i) * CB, s[i]);
              }
#pragma unroll
              for (int i = 0; i < PAIR; ++i) tmem_wait(r[i]);
              if (c > 0) {
#pragma unroll
                for (int i = 0; i < PAIR; ++i) {
                  tmem_wait(s[i]);
#pragma unroll
                  for (int j = 0; j < CB; ++j) r[i][j] = __float_as_uint(__uint_as_float(s[i][j]) + __uint_as_float(r[i][j]));
                }
              }
#pragma unroll
              for (int i = 0; i < PAIR; ++i) tmem_st(sums_tmem + (cb + i) * CB, r[i]);
            }
            tmem_st_wait();
          }
          release_accumulator(local);
          ++local;
        }
        if (!ok) break;
      } else if (kb1 - kb0 > chunk) {
        // A long inner extent in 16 bits: all accumulators but the last are added up in global memory, where a thread meets
        // only what it has written itself; the last takes them in and is used like the only one of a short extent.
        float* const sums = p.sums + (static_cast<long long>(blockIdx.x) * BN + group * GROUP_COLS) * BM + row_in_cta;
        const int chunks = (kb1 - kb0 + chunk - 1) / chunk;
        for (int c = 0; c < chunks; ++c) {
          ok = wait_accumulator(local);
          if (!ok) break;
          tcgen05_fence_after();
          const bool last = c == chunks - 1;
#pragma unroll 1
          for (int cb = 0; cb < BLOCKS; ++cb) {
            uint32_t r[CB];
            tmem_ld(accumulator(local) + cb * CB, r);
            tmem_wait(r);
            float* const at = sums + cb * CB * BM;
#pragma unroll
            for (int j = 0; j < CB; ++j) {
              const float sum = c > 0 ? at[j * BM] + __uint_as_float(r[j]) : __uint_as_float(r[j]);
              if (last) r[j] = __float_as_uint(sum);
              else at[j * BM] = sum;
            }
            if (last) tmem_st(accumulator(local) + cb * CB, r);
          }
          if (last) {
            tmem_st_wait();
          } else {
            release_accumulator(local);
            ++local;
          }
        }
        if (!ok) break;
      }
      const uint32_t values = CHUNKED ? sums_tmem : accumulator(local);  // where the finished values lie

      if constexpr (MODE == kModeGeneral) {
        if (split > 1) {
          // -- tile shared by a cluster: sums meet in shared memory, every CTA finishes a range of columns --
          float* const sums = reinterpret_cast<float*>(staging);  // [column][128 rows]
          // This CTA's columns in steps of STEP per group; D and Z of the next step are under way while one is finished.
          constexpr int STEP = 4;
          const int mine = BN / split;  // a multiple of STEP
          const int first_col = static_cast<int>(rank) * mine;
          float d_ahead[STEP], z_ahead[STEP];
#pragma unroll
          for (int j = 0; j < STEP; ++j) d_ahead[j] = z_ahead[j] = 0.f;
          auto fetch = [&](int q) {
            const int rel = first_col + q * STEP - group * GROUP_COLS;
            const int cols_left = t.col_end - (t.col0 + first_col + q * STEP);
#pragma unroll
            for (int j = 0; j < STEP; ++j) {
              const bool in = in_rows && j < cols_left;
              d_ahead[j] = has_d && in ? to_float(d_ptr[static_cast<long long>(rel + j) * p.ldd + lane]) : 0.f;
              z_ahead[j] = z_in && in ? to_float(z_ptr[static_cast<long long>(rel + j) * p.ldz + lane]) : 0.f;
            }
          };
          if (tiles_done > 0) fetch(group);
          // Step -1 of a CTA's first tile requests that and brings the code into the instruction caches (see run_blocks).
#pragma unroll 1
          for (int step = tiles_done == 0 ? -1 : 0; ok; ++step) {
            if (step == 0) {
              if constexpr (!CHUNKED) {
                ok = wait_accumulator(local);
                if (!ok) break;
                tcgen05_fence_after();
              }
              if (tiles_done > 0) {
                ok = warp_wait_cluster(sums_free, (tiles_done - 1) & 1u, abort_flag, 7u, p.status);
                if (!ok) break;
              }
#pragma unroll 1
              for (int cb = 0; cb < BLOCKS; ++cb) {
                const int col = group * GROUP_COLS + cb * CB;
                uint32_t r[CB];
                if (!empty) {
                  tmem_ld(values + cb * CB, r);
                  tmem_wait(r);
                }
#pragma unroll
                for (int j = 0; j < CB; ++j) sums[(col + j) * BM + row_in_cta] = empty ? 0.f : __uint_as_float(r[j]);
              }
              if constexpr (!CHUNKED) {
                release_accumulator(local);
                ++local;
              }
              __syncwarp();
              if (lane == 0) {
                for (int q = 0; q < split; ++q) mbar_arrive_remote(map_to_cta(sums_ready, q));
              }
              ok = warp_wait_cluster(sums_ready, tiles_done & 1u, abort_flag, 8u, p.status);
              if (!ok) break;
            }
            const bool dry = step < 0;
            const int q = group + step * EG;
            if (!dry && q >= mine / STEP) break;
            const int in_tile = dry ? 0 : first_col + q * STEP;
            const int rel = in_tile - group * GROUP_COLS;  // column relative to group_col0
            const int cols_left = dry ? 0 : t.col_end - (t.col0 + in_tile);
            if (!dry && cols_left <= 0) break;
            const uint32_t at = smem_u32(sums + in_tile * BM + row_in_cta);
            float v[STEP], d4[STEP], z4[STEP];
            // all reads of a pair of ranks before their sum; the order of the additions is that of the ranks
#pragma unroll
            for (int j = 0; j < STEP; ++j) v[j] = 0.f;
#pragma unroll 1
            for (int s = 0; s < split; s += 2) {
              const uint32_t src0 = map_to_cta(at, s), src1 = map_to_cta(at, s + 1);
              float u0[STEP], u1[STEP];
#pragma unroll
              for (int j = 0; j < STEP; ++j) {
                u0[j] = ld_cluster_f32(src0 + j * BM * 4);
                u1[j] = ld_cluster_f32(src1 + j * BM * 4);
              }
#pragma unroll
              for (int j = 0; j < STEP; ++j) v[j] = (v[j] + u0[j]) + u1[j];
            }
#pragma unroll
            for (int j = 0; j < STEP; ++j) { d4[j] = d_ahead[j]; z4[j] = z_ahead[j]; }
            if (q + EG < mine / STEP) fetch(q + EG);
#pragma unroll
            for (int j = 0; j < STEP; ++j) v[j] = fmaf(p.alpha, v[j], bias);
            if (grad) {
              if (has_d) {
#pragma unroll
                for (int j = 0; j < STEP; ++j) v[j] = fmaf(p.beta, d4[j], v[j]);
              }
              if (z_in) {
                with_act(p.act, [&](auto tag) {
#pragma unroll
                  for (int j = 0; j < STEP; ++j) v[j] *= act_slope<FAST, decltype(tag)::value>(z4[j]);
                });
              }
#pragma unroll
              for (int j = 0; j < STEP; ++j) row_sum += j < cols_left ? v[j] : 0.f;
            } else {
              if (z_out) {
#pragma unroll
                for (int j = 0; j < STEP; ++j)
                  if (in_rows && j < cols_left) z_ptr[static_cast<long long>(rel + j) * p.ldz + lane] = from_float<T>(v[j]);
              }
              with_act(p.act, [&](auto tag) {
#pragma unroll
                for (int j = 0; j < STEP; ++j) v[j] = act_value<FAST, decltype(tag)::value>(v[j]);
              });
              if (has_d) {
#pragma unroll
                for (int j = 0; j < STEP; ++j) v[j] = fmaf(p.beta, d4[j], v[j]);
              }
            }
#pragma unroll
            for (int j = 0; j < STEP; ++j)
              if (in_rows && j < cols_left) c_ptr[static_cast<long long>(rel + j) * p.ldc + lane] = from_float<OT>(v[j]);
          }
          if (!ok) break;
          __syncwarp();
          // (the arrival is a release that waits for the stores above, so the last tile goes without)
          if (lane == 0 && tile + tile_step < num_tiles) {
            for (int q = 0; q < split; ++q) mbar_arrive_remote(map_to_cta(sums_free, q));
          }
          if (p.partial != nullptr && in_rows)
            p.partial[(static_cast<long long>(t.col_tile * split + static_cast<int>(rank)) * EG + group) * p.m + row] = row_sum;
          continue;
        }
      }

      // accumulator values of block cb; the load of the next block starts as this one's arrives
      uint32_t r_next[CB];
      auto take = [&](int cb, float (&v)[CB]) {
        if (empty || cb < 0) {
#pragma unroll
          for (int j = 0; j < CB; ++j) v[j] = bias;
        } else {
          tmem_wait(r_next);
#pragma unroll
          for (int j = 0; j < CB; ++j) v[j] = fmaf(p.alpha, __uint_as_float(r_next[j]), bias);
          if (cb + 1 < BLOCKS) tmem_ld(values + (cb + 1) * CB, r_next);
        }
      };
      auto begin = [&]() {
        if constexpr (!CHUNKED) {
          ok = wait_accumulator(local);
          if (!ok) return false;
          tcgen05_fence_after();
        }
        if (!empty) tmem_ld(values, r_next);
        return true;
      };
      // All blocks of the tile. On a CTA's first tile they are preceded by a dry one without columns: it brings the code
      // into the instruction caches and requests the first block's D and Z while the operands are still on their way.
      // (Cold code cost 15000 cycles at the end of a kernel of one tile per CTA.)
      auto run_blocks = [&](auto& block, auto& request) {
        int cb = -1;
        if (tiles_done > 0) {
          request(0);
          cb = 0;
        }
#pragma unroll 1
        for (; cb < BLOCKS; ++cb) {
          if (cb == 0 && !begin()) break;
          if (cb >= 0 && cb * CB >= group_cols) break;
          block(cb);
        }
      };
      auto end = [&]() {
        if (!empty) tmem_wait(r_next);  // a load may have started for a block that does not exist
        if constexpr (!CHUNKED) {
          release_accumulator(local);
          ++local;
        }
      };

      if constexpr (MODE != kModeGeneral) {
        // D and Z of a block are requested while the block before it is worked on
        BlockD d_next = {}, d_low = {};
        BlockZ z_next = {};
        auto request = [&](int cb) {
          if (has_d) d_next.load(d_ptr + static_cast<long long>(cb * CB) * p.ldd, p.ldd, rows_left, group_cols - cb * CB, lane);
          if (MODE == kModeParts && has_d)
            d_low.load(d_ptr + p.d_stride + static_cast<long long>(cb * CB) * p.ldd, p.ldd, rows_left, group_cols - cb * CB, lane);
          if (MODE == kModeGrad && aux) z_next.load(z_ptr + static_cast<long long>(cb * CB) * p.ldz, p.ldz, rows_left, group_cols - cb * CB, lane);
        };
        uint8_t* const own = staging + (warp - 4) * fused_warp_bytes(CHUNKED, aux);
        uint32_t* const turn_c = reinterpret_cast<uint32_t*>(own);
        uint32_t* const turn_z = turn_c + BlockC::WORDS;
        auto block = [&](int cb) {
          const int cols_left = cb < 0 ? 0 : group_cols - cb * CB;
          float v[CB];
          take(cb, v);
          auto add_d = [&]() {
            float add[CB];
            d_next.to_rows(turn_c, add, lane);
#pragma unroll
            for (int j = 0; j < CB; ++j) v[j] = fmaf(p.beta, add[j], v[j]);
            if constexpr (MODE == kModeParts) {
              d_low.to_rows(turn_c, add, lane);
#pragma unroll
              for (int j = 0; j < CB; ++j) v[j] = fmaf(p.beta, add[j], v[j]);
            }
          };
          if constexpr (MODE == kModeGrad) {
            if (has_d) add_d();
            if (aux) {
              float zz[CB];
              z_next.to_rows(turn_z, zz, lane);
              if (cb + 1 < BLOCKS) request(cb + 1);
              with_act(p.act, [&](auto tag) {
#pragma unroll
                for (int j = 0; j < CB; ++j) v[j] *= act_slope<FAST, decltype(tag)::value>(zz[j]);
              });
            } else if (cb + 1 < BLOCKS) {
              request(cb + 1);
            }
            if (p.partial != nullptr) {
              if (cols_left >= CB) {
                float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < CB; ++j) s4[j & 3] += v[j];
                row_sum += (s4[0] + s4[1]) + (s4[2] + s4[3]);
              } else {
#pragma unroll
                for (int j = 0; j < CB; ++j) row_sum += j < cols_left ? v[j] : 0.f;
              }
            }
          } else {
            if (aux) BlockZ::store(z_ptr + static_cast<long long>(cb * CB) * p.ldz, p.ldz, rows_left, cols_left, turn_z, v, lane);
            with_act(p.act, [&](auto tag) {
#pragma unroll
              for (int j = 0; j < CB; ++j) v[j] = act_value<FAST, decltype(tag)::value>(v[j]);
            });
            if (has_d) add_d();
            if (cb + 1 < BLOCKS) request(cb + 1);
          }
          // stores the block, and its mirror image where the result is symmetric
          auto put = [&](long long plane) {
            BlockC::store(c_ptr + plane + static_cast<long long>(cb * CB) * p.ldc, p.ldc, rows_left, cols_left, turn_c, v, lane);
            if constexpr ((MODE == kModeForward || MODE == kModeParts) && sizeof(OT) == 2 && BN == CTAS * BM) {
              if (p.tri && t.tm != t.tn && in_rows) {
                // this lane's columns are consecutive rows there
                OT* const dst = static_cast<OT*>(p.c) + zc * p.c_stride + plane + static_cast<long long>(row) * p.ldc + group_col0 + cb * CB;
                uint32_t w[CB / 2];
#pragma unroll
                for (int q = 0; q < CB / 2; ++q) w[q] = pack2<OT>(v[2 * q], v[2 * q + 1]);
#pragma unroll
                for (int q = 0; q < CB / 8; ++q)
                  if (cols_left >= 8 * (q + 1))
                    *reinterpret_cast<uint4*>(dst + 8 * q) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
              }
            }
          };
          put(0);
          if constexpr (MODE == kModeParts) {
#pragma unroll
            for (int j = 0; j < CB; ++j) v[j] -= to_float(from_float<OT>(v[j]));
            put(p.c_stride);
          }
        };
        run_blocks(block, request);
        if (!ok) break;
        end();
      } else {
        // row by row, element by element; D and Z of a block are requested while the block before it is worked on
        DT d_next[CB];
        T z_next[CB];
        auto request = [&](int cb) {
          const int cols_left = in_rows ? group_cols - cb * CB : 0;
          const DT* d_at = d_ptr + static_cast<long long>(cb * CB) * p.ldd + lane;
          const T* z_at = z_ptr + static_cast<long long>(cb * CB) * p.ldz + lane;
          if (has_d) {
#pragma unroll
            for (int j = 0; j < CB; ++j, d_at += p.ldd) d_next[j] = j < cols_left ? *d_at : from_float<DT>(0.f);
          }
          if (z_in) {
#pragma unroll
            for (int j = 0; j < CB; ++j, z_at += p.ldz) z_next[j] = j < cols_left ? *z_at : from_float<T>(0.f);
          }
        };
#pragma unroll
        for (int j = 0; j < CB; ++j) {
          d_next[j] = from_float<DT>(0.f);
          z_next[j] = from_float<T>(0.f);
        }
        auto block = [&](int cb) {
          const int cols_left = in_rows && cb >= 0 ? group_cols - cb * CB : 0;
          float v[CB];
          take(cb, v);
          if (grad) {
            if (has_d) {
#pragma unroll
              for (int j = 0; j < CB; ++j) v[j] = fmaf(p.beta, to_float(d_next[j]), v[j]);
            }
            if (z_in) {
              with_act(p.act, [&](auto tag) {
#pragma unroll
                for (int j = 0; j < CB; ++j) v[j] *= act_slope<FAST, decltype(tag)::value>(to_float(z_next[j]));
              });
            }
#pragma unroll
            for (int j = 0; j < CB; ++j) row_sum += j < cols_left ? v[j] : 0.f;
          } else {
            if (z_out) {
              T* at = z_ptr + static_cast<long long>(cb * CB) * p.ldz + lane;
#pragma unroll
              for (int j = 0; j < CB; ++j, at += p.ldz)
                if (j < cols_left) *at = from_float<T>(v[j]);
            }
            with_act(p.act, [&](auto tag) {
#pragma unroll
              for (int j = 0; j < CB; ++j) v[j] = act_value<FAST, decltype(tag)::value>(v[j]);
            });
            if (has_d) {
#pragma unroll
              for (int j = 0; j < CB; ++j) v[j] = fmaf(p.beta, to_float(d_next[j]), v[j]);
            }
          }
          if (cb + 1 < BLOCKS) request(cb + 1);
          OT* at = c_ptr + static_cast<long long>(cb * CB) * p.ldc + lane;
#pragma unroll
          for (int j = 0; j < CB; ++j, at += p.ldc)
            if (j < cols_left) *at = from_float<OT>(v[j]);
        };
        run_blocks(block, request);
        if (!ok) break;
        end();
      }
      if (MODE != kModeForward && MODE != kModeParts && p.partial != nullptr && in_rows)
        p.partial[(static_cast<long long>(t.col_tile) * EG + group) * p.m + row] = row_sum;
    }
  }

  tcgen05_fence_before();
  __syncthreads();
  if (CTAS == 2 || split > 1) cluster_sync_all();  // nobody exits while a peer may still signal or read
  if (warp == 1) {
    tcgen05_fence_after();
    if constexpr (CTAS == 2) tmem_dealloc_pair(tmem_base, TMEM_COLS);
    else tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <int CTAS, int BN, class T, class DT, class OT, int MODE>
cudaError_t launch_mode(const CUtensorMap* maps, const FusedParams& p, int grid, int smem, cudaStream_t stream) {
  auto kernel = fused_gemm_kernel<CTAS, BN, T, DT, OT, MODE>;
  const cudaError_t e = kernel_ready(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(fused_threads(BN), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  const int cluster = CTAS == 2 ? 2 : p.split;
  unsigned attrs = 0;
  if (cluster > 1) {
    attr[attrs].id = cudaLaunchAttributeClusterDimension;
    attr[attrs].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[attrs].val.clusterDim.y = 1;
    attr[attrs].val.clusterDim.z = 1;
    ++attrs;
  }
  if (p.chained) {
    attr[attrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[attrs].val.programmaticStreamSerializationAllowed = 1;
    ++attrs;
  }
  cfg.attrs = attrs ? attr : nullptr;
  cfg.numAttrs = attrs;
  return cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], maps[2], maps[3], p);
}

template <int CTAS, int BN, class T, class DT, class OT>
cudaError_t launch_typed(const CUtensorMap* maps, const FusedParams& p, int grid, int smem, cudaStream_t stream) {
  if constexpr (BN == 128 && CTAS == 1) {
    if constexpr (std::is_same<T, __half>::value && std::is_same<OT, __half>::value) {
      if (p.parts) return launch_mode<CTAS, BN, T, DT, OT, kModeParts>(maps, p, grid, smem, stream);
    }
  }
  if (p.parts) return cudaErrorInvalidValue;
  if (!p.vec || p.split > 1) return launch_mode<CTAS, BN, T, DT, OT, kModeGeneral>(maps, p, grid, smem, stream);
  if (!p.grad) return launch_mode<CTAS, BN, T, DT, OT, kModeForward>(maps, p, grid, smem, stream);
  // gradients are stored in the operands' type
  if constexpr (std::is_same<T, OT>::value) return launch_mode<CTAS, BN, T, DT, OT, kModeGrad>(maps, p, grid, smem, stream);
  return cudaErrorInvalidValue;
}

// Clusters of `cluster` CTAs that the device holds at once (one CTA per SM; a cluster sits in one GPC).
template <int CTAS, int BN>
int resident_clusters(int cluster, int smem) {
  auto kernel = fused_gemm_kernel<CTAS, BN, __half, __half, __half, kModeGeneral>;
  if (kernel_ready(reinterpret_cast<const void*>(kernel), smem) != cudaSuccess) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(sm_count() / cluster * cluster), 1, 1);
  cfg.blockDim = dim3(fused_threads(BN), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return clusters;
}

template <int CTAS, int BN>
cudaError_t launch_by_type(int type, int d_type, int c_type, const CUtensorMap* maps, const FusedParams& p, int grid,
                           int smem, cudaStream_t stream) {
  using H = __half;
  using B = __nv_bfloat16;
  if (type == 16) {
    if (c_type == 16 && d_type == 16) return launch_typed<CTAS, BN, H, H, H>(maps, p, grid, smem, stream);
    if (c_type == kBFloat16 && d_type == 16) return launch_typed<CTAS, BN, H, H, B>(maps, p, grid, smem, stream);
    if (c_type == 32 && d_type == 32) return launch_typed<CTAS, BN, H, float, float>(maps, p, grid, smem, stream);
  } else if (type == kBFloat16) {
    if (c_type == kBFloat16 && d_type == kBFloat16) return launch_typed<CTAS, BN, B, B, B>(maps, p, grid, smem, stream);
    if (c_type == 32 && d_type == 32) return launch_typed<CTAS, BN, B, float, float>(maps, p, grid, smem, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace fused
}  // namespace b200

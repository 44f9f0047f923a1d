// C = act(alpha op(A) op(B) + bias) + beta D and its backward form (alpha op(A) op(B) + beta D) * slope(Z), fp16 or
// bf16 operands, fp32 accumulation and epilogue arithmetic, one rounding per stored value. One kernel template serves
// plain and strided-batched products, products whose column extent is cut into ragged groups (experts' rows), and
// products whose inner extent is (experts' weight gradients).
//
// C is m x n with m contiguous. Rows are the features of the caller's vectors and columns the vectors, so a thread of
// the epilogue owns one feature (one tensor-memory lane) and walks along the vectors: the bias is one register, the
// bias gradient a running sum, and a 32-lane store covers consecutive addresses.
//
// Warp roles: warp 0 lane 0 issues the TMA loads of the operand ring, warp 1 the MMAs (and clears what a ragged inner
// extent leaves behind its end), warps 2.. drain the accumulators in groups of four warps, each group its own range
// of the tile's columns. Two accumulators alternate, so a tile is drained under the next one's MMAs.
//   CTAS == 2: a cluster of two CTAs works on 256 x BN tiles with cta_group::2, each CTA staging half of op(B).
//   CTAS == 1: tiles of 128 x BN; a cluster of p.split CTAs may share a tile's inner extent. Each CTA then leaves its
//   fp32 sums in its own shared memory and the CTAs add them up for a range of columns each, in the order of the ranks
//   (the result does not depend on which CTA came first).
//
// The epilogue goes by blocks of 32 bytes of columns x 128 rows (4 KB). D and Z come in and C and Z go out by TMA
// through rings of four buffers per group; see write_block's counterpart in hgemm_epilogue.cuh for why one named barrier
// per block orders everything. Columns behind a group's last one are cut off by storing column by column with bulk copies.
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
constexpr int BK = 64;    // inner elements per stage: 128-byte swizzle rows
constexpr int SLOT = 4096;
constexpr int RING = 4;   // staging buffers per epilogue group and matrix
constexpr int BAR_BYTES = 512;

// Shared memory behind the operand ring: staging (or the fp32 sums of a split tile), barriers, group table.
__host__ __device__ constexpr int staging_bytes(int groups, bool aux) { return groups * RING * SLOT * (aux ? 2 : 1); }
__host__ __device__ constexpr int sums_bytes(int bn) { return bn * BM * 4; }
__host__ __device__ inline int table_bytes(int kind, int problems) {
  return kind == kFusedRaggedCols ? 8 * (problems + 1) : 0;
}

__device__ __forceinline__ void group_barrier(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool group_all(int id, bool mine) {
  uint32_t out;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.and.pred p, %2, 128, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(out)
      : "r"(static_cast<uint32_t>(mine)), "r"(id)
      : "memory");
  return out != 0;
}

template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[N]) {
  static_assert(N == 8 || N == 16, "block width");
  if constexpr (N == 16) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
  } else {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
  }
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tma_load_3d_hint(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z,
                                                 uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5}], [%2], %6;"
      :
      : "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}

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

template <int BN>
__device__ __forceinline__ Tile locate(const FusedParams& p, int tile, const int* start, const int* tiles) {
  Tile t;
  int in_problem, cols;
  if (p.kind == kFusedRaggedCols) {
    const int want = tile / p.tiles_m;  // the group with tiles[g] <= want < tiles[g + 1]
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
    t.z = tile / per;
    in_problem = tile - t.z * per;
    cols = p.tiles_n;
  } else {
    const int per = p.tiles_m * p.tiles_n;
    t.z = tile / per;
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
    const int group = in_problem / per_group;
    const int first = group * p.raster;
    const int rows = min(p.raster, p.tiles_m - first);
    const int in_group = in_problem - group * per_group;
    t.tn = in_group / rows;
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
      long long lo = p.offsets[t.z], hi = p.offsets[t.z + 1];
      lo = lo < 0 ? 0 : (lo > p.k ? p.k : lo);
      hi = hi < lo ? lo : (hi > p.k ? p.k : hi);
      t.k0 = static_cast<int>(lo);
      t.k_len = static_cast<int>(hi - lo);
    }
  }
  return t;
}

template <class T, class DT, class OT>
struct Types {
  static constexpr int CB = 32 / static_cast<int>(sizeof(OT));  // columns per block: 32 bytes of a column-of-columns
  static constexpr int C_BYTES = CB * BM * static_cast<int>(sizeof(OT));
  static constexpr int Z_BYTES = CB * BM * 2;
};

template <int CTAS, int BN, class T, class DT, class OT>
__global__ void __launch_bounds__(64 + 128 * (BN >= 128 ? 2 : 1), 1)
fused_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                  const __grid_constant__ CUtensorMap map_c, const __grid_constant__ CUtensorMap map_d,
                  const __grid_constant__ CUtensorMap map_z, const FusedParams p) {
  static_assert(sizeof(DT) == sizeof(OT), "D and C share the staging buffers");
  constexpr int EG = BN >= 128 ? 2 : 1;
  constexpr int CB = Types<T, DT, OT>::CB;
  constexpr int B_ROWS = BN / CTAS;
  constexpr int A_BYTES = BM * BK * 2;
  constexpr int STAGE_BYTES = A_BYTES + B_ROWS * BK * 2;
  constexpr int GROUP_COLS = BN / EG;
  constexpr uint32_t TMEM_COLS = 2 * BN;
  constexpr bool FAST = sizeof(OT) == 2;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t tiles_base = (raw + 1023u) & ~1023u;
  uint8_t* const base_ptr = smem_raw + (tiles_base - raw);
  const bool aux = p.z != nullptr;
  const int stages = p.stages;
  uint8_t* const staging = base_ptr + stages * STAGE_BYTES;
  const int sb = staging_bytes(EG, aux);
  uint8_t* const behind = staging + (p.split > 1 && sums_bytes(BN) > sb ? sums_bytes(BN) : sb);
  const uint32_t bar_base = smem_u32(behind);
  // full [0, 16), empty [16, 32), accumulator full / empty [32, 36), sums ready / free [36, 38), loads [40, 40 + 8)
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (16 + s); };
  auto acc_full_bar = [&](int a) { return bar_base + 8u * (32 + a); };
  auto acc_empty_bar = [&](int a) { return bar_base + 8u * (34 + a); };
  const uint32_t sums_ready = bar_base + 8u * 36, sums_free = bar_base + 8u * 37;
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(behind + 8 * 48);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* const start = reinterpret_cast<int*>(behind + BAR_BYTES);
  int* const tiles = start + p.problems + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = (CTAS == 2 || p.split > 1) ? cluster_ctarank() : 0u;
  const int team = CTAS == 2 ? 2 : p.split;          // CTAs that work on one tile
  const int first_tile = static_cast<int>(blockIdx.x) / team;
  const int tile_step = static_cast<int>(gridDim.x) / team;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full_bar(a), 1);
      mbar_init(acc_empty_bar(a), 4 * EG * CTAS);
    }
    mbar_init(sums_ready, 4 * EG * p.split);
    mbar_init(sums_free, 4 * EG * p.split);
    for (int b = 0; b < EG * RING; ++b) mbar_init(bar_base + 8u * (40 + b), 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (CTAS == 2) tmem_alloc_pair(smem_u32(tmem_slot), TMEM_COLS);
    else tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
  }
  if (warp == 2 && p.kind == kFusedRaggedCols) build_table(p.offsets, p.problems, p.n, BN, start, tiles);
  tcgen05_fence_before();
  __syncthreads();
  if (CTAS == 2 || p.split > 1) cluster_sync_all();  // all barriers exist before anyone signals across CTAs
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int num_tiles = total_tiles(p, tiles);

  // this CTA's share of a tile's inner blocks
  auto k_range = [&](const Tile& t, int& kb0, int& kb1) {
    const int blocks = (t.k_len + BK - 1) / BK;
    if (CTAS == 1 && p.split > 1) {
      kb0 = blocks * static_cast<int>(rank) / p.split;
      kb1 = blocks * (static_cast<int>(rank) + 1) / p.split;
    } else {
      kb0 = 0;
      kb1 = blocks;
    }
  };

  if (warp == 0) {
    // ---- TMA producer ----
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint64_t pol_a = l2_policy(p.hint_a), pol_b = l2_policy(p.hint_b);
      for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
        const Tile t = locate<BN>(p, tile, start, tiles);
        const int a_row0 = (t.tm * CTAS + (CTAS == 2 ? static_cast<int>(rank) : 0)) * BM;
        const int b_row0 = t.col0 + (CTAS == 2 ? static_cast<int>(rank) * B_ROWS : 0);
        const int az = p.a_batched ? t.z : 0, bz = p.b_batched ? t.z : 0;
        int kb0, kb1;
        k_range(t, kb0, kb1);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, 1u, p.status)) { ok = false; break; }
          const uint32_t a_dst = tiles_base + stage * STAGE_BYTES;
          const uint32_t b_dst = a_dst + A_BYTES;
          const int x = t.k0 + kb * BK;
          uint32_t bar;
          if constexpr (CTAS == 2) {
            bar = map_to_cta(full_bar(stage), 0);
            if (rank == 0) mbar_arrive_expect_tx(full_bar(stage), 2 * STAGE_BYTES);  // the bytes of both CTAs
          } else {
            bar = full_bar(stage);
            mbar_arrive_expect_tx(bar, STAGE_BYTES);
          }
          auto load = [&](uint32_t dst, const CUtensorMap* map, int cx, int cy, int cz, uint64_t pol) {
            if constexpr (CTAS == 2) tma_load_3d_pair_hint(dst, map, bar, cx, cy, cz, pol);
            else tma_load_3d_hint(dst, map, bar, cx, cy, cz, pol);
          };
          if (p.a_mn) {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) load(a_dst + j * 8192, &map_a, a_row0 + j * 64, x, az, pol_a);
          } else {
            load(a_dst, &map_a, x, a_row0, az, pol_a);
          }
          if (p.b_mn) {
#pragma unroll
            for (int j = 0; j < B_ROWS / 64; ++j) load(b_dst + j * 8192, &map_b, b_row0 + j * 64, x, bz, pol_b);
          } else {
            load(b_dst, &map_b, x, b_row0, bz, pol_b);
          }
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
    // ---- MMA issuer (of a pair: the leader, for both SMs). The whole warp walks along; lane 0 issues. ----
    if (CTAS == 1 || rank == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step, ++local) {
        const Tile t = locate<BN>(p, tile, start, tiles);
        int kb0, kb1;
        k_range(t, kb0, kb1);
        const int acc = local & 1;
        const uint32_t acc_phase = (local >> 1) & 1u;
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(acc_empty_bar(acc), acc_phase ^ 1u, abort_flag, 2u, p.status));
        if (!ok) break;
        tcgen05_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = __all_sync(0xFFFFFFFFu, mbar_wait(full_bar(stage), phase, abort_flag, 3u, p.status));
          if (!ok) break;
          const uint32_t a_src = tiles_base + stage * STAGE_BYTES;
          const uint32_t b_src = a_src + A_BYTES;
          int steps = BK / 16;
          if (CTAS == 1 && p.kind == kFusedRaggedInner) {
            // The last block of a group holds inner indices of the next one (or whatever lies behind the matrix). Both
            // operands have one 128-byte row per inner index and 64 elements of m / n; rows up to the next multiple
            // of an MMA's 16 are cleared in both (0 * NaN would not be 0), the MMAs behind that are left out.
            const int valid = t.k_len - kb * BK;
            if (valid < BK) {
              steps = (valid + 15) / 16;
              const int rows = steps * 16 - valid;
              uint8_t* const s = base_ptr + stage * STAGE_BYTES;
              constexpr int BLOCKS = BM / 64 + B_ROWS / 64;
              for (int i = lane; i < rows * BLOCKS * 8; i += 32) {
                const int chunk = i & 7, r = (i >> 3) % rows, j = (i >> 3) / rows;
                *reinterpret_cast<uint4*>(s + j * 8192 + (valid + r) * 128 + chunk * 16) = make_uint4(0, 0, 0, 0);
              }
              fence_proxy_async();
              __syncwarp();
            }
          }
          tcgen05_fence_after();
          if (lane == 0) {
            // K-major: 128-byte rows along K (stride offset 1024 = eight rows), 32 B per MMA step. MN-major: one
            // 128-byte row of 64 elements per k, blocks 8192 B apart, 2048 B per MMA step.
            const uint64_t da = p.a_mn ? smem_desc(a_src, 8192, 1024, kLayoutSw128) : smem_desc(a_src, 16, 1024, kLayoutSw128);
            const uint64_t db = p.b_mn ? smem_desc(b_src, 8192, 1024, kLayoutSw128) : smem_desc(b_src, 16, 1024, kLayoutSw128);
            const uint32_t a_step = p.a_mn ? (2048u >> 4) : 2u, b_step = p.b_mn ? (2048u >> 4) : 2u;
#pragma unroll
            for (int ks = 0; ks < BK / 16; ++ks) {
              if (ks < steps) {
                const uint32_t accumulate = (kb != kb0 || ks != 0) ? 1u : 0u;
                if constexpr (CTAS == 2) umma_f16_pair(d_tmem, da + a_step * ks, db + b_step * ks, p.idesc, accumulate);
                else umma_f16(d_tmem, da + a_step * ks, db + b_step * ks, p.idesc, accumulate);
              }
            }
            if constexpr (CTAS == 2) umma_commit_pair(empty_bar(stage));
            else umma_commit(empty_bar(stage));
          }
          if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
        if (ok && lane == 0) {  // without inner blocks this arrives at once and the epilogue takes zeros
          if constexpr (CTAS == 2) umma_commit_pair(acc_full_bar(acc));
          else umma_commit(acc_full_bar(acc));
        }
      }
    }
  } else {
    // ---- epilogue ----
    const int group = EG == 1 ? 0 : (warp - 2) >> 2;
    const int quad = warp & 3;  // tensor-memory lanes this warp may read
    const int row_in_cta = quad * 32 + lane;
    const int bar_id = 1 + group;
    const bool elected = (threadIdx.x & 127) == 64;  // first thread of each group
    uint8_t* const ring_c = staging + group * RING * SLOT * (aux ? 2 : 1);
    uint8_t* const ring_z = ring_c + RING * SLOT;
    const uint32_t load_bars = bar_base + 8u * (40 + group * RING);
    const bool has_d = p.d != nullptr;
    const bool z_in = aux && p.grad, z_out = aux && !p.grad;
    const uint32_t load_bytes = (has_d ? Types<T, DT, OT>::C_BYTES : 0) + (z_in ? Types<T, DT, OT>::Z_BYTES : 0);
    int local = 0, blocks_done = 0;
    uint32_t load_phases = 0;
    bool ok = true;

    // requests D and Z of the block that will be number `block` (elected thread only)
    auto request = [&](int block, int row0, int col, int z) {
      const int b = block & (RING - 1);
      const uint32_t bar = load_bars + 8u * b;
      mbar_arrive_expect_tx(bar, load_bytes);
      if (has_d) tma_load_3d(smem_u32(ring_c + b * SLOT), &map_d, bar, row0, col, z);
      if (z_in) tma_load_3d(smem_u32(ring_z + b * SLOT), &map_z, bar, row0, col, z);
    };

    for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step, ++local) {
      const Tile t = locate<BN>(p, tile, start, tiles);
      const int cta_row0 = (t.tm * CTAS + (CTAS == 2 ? static_cast<int>(rank) : 0)) * BM;
      const int row = cta_row0 + row_in_cta;
      const bool live = cta_row0 < p.m;  // the second CTA of a pair may lie wholly below C
      const bool in_rows = row < p.m;
      const int zc = p.kind == kFusedRaggedCols ? 0 : t.z;  // third coordinate of C, D, Z
      const float bias = (p.bias != nullptr && in_rows) ? to_float(static_cast<const T*>(p.bias)[t.z * p.bias_stride + row]) : 0.f;
      OT* const c_ptr = static_cast<OT*>(p.c) + zc * p.c_stride;
      const DT* const d_ptr = static_cast<const DT*>(p.d) + zc * p.d_stride;
      T* const z_ptr = static_cast<T*>(p.z) + zc * p.z_stride;
      float row_sum = 0.f;
      const int acc = local & 1;
      const uint32_t acc_phase = (local >> 1) & 1u;
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(acc * BN);
      int kb0, kb1;
      k_range(t, kb0, kb1);
      const bool empty = kb1 <= kb0;

      if (CTAS == 1 && p.split > 1) {
        // -- tile shared by a cluster: sums meet in shared memory, every CTA finishes a range of columns --
        float* const sums = reinterpret_cast<float*>(staging);  // [column][128 rows]
        ok = mbar_wait(acc_full_bar(acc), acc_phase, abort_flag, 4u, p.status);
        if (ok && local > 0) ok = mbar_wait_cluster(sums_free, (local - 1) & 1u, abort_flag, 7u, p.status);
        ok = group_all(bar_id, ok);
        if (!ok) break;
        tcgen05_fence_after();
#pragma unroll 1
        for (int cb = 0; cb < GROUP_COLS / 16; ++cb) {
          const int col = group * GROUP_COLS + cb * 16;
          uint32_t r[16];
          if (!empty) tmem_ld<16>(t_row + col, r);
#pragma unroll
          for (int j = 0; j < 16; ++j) sums[(col + j) * BM + row_in_cta] = empty ? 0.f : __uint_as_float(r[j]);
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(acc_empty_bar(acc));
          for (int q = 0; q < p.split; ++q) mbar_arrive_remote(map_to_cta(sums_ready, q));
        }
        ok = mbar_wait_cluster(sums_ready, local & 1u, abort_flag, 8u, p.status);
        ok = group_all(bar_id, ok);
        if (!ok) break;
        const int mine = BN / p.split;  // a multiple of four
        for (int q = group; q < mine / 4; q += EG) {
          const int in_tile = static_cast<int>(rank) * mine + q * 4;
          const int col = t.col0 + in_tile;
          if (col >= t.col_end) break;
          float v[4] = {0.f, 0.f, 0.f, 0.f};
          for (int s = 0; s < p.split; ++s) {
            const uint32_t src = map_to_cta(smem_u32(sums + in_tile * BM + row_in_cta), s);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += ld_cluster_f32(src + j * BM * 4);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (!in_rows || col + j >= t.col_end) continue;
            const long long cj = col + j;
            const float add = has_d ? p.beta * to_float(d_ptr[cj * p.ldd + row]) : 0.f;
            float y = p.alpha * v[j] + bias;
            if (p.grad) {
              y += add;
              if (z_in) y *= act_slope<FAST>(p.act, to_float(z_ptr[cj * p.ldz + row]));
              row_sum += y;
            } else {
              if (z_out) z_ptr[cj * p.ldz + row] = from_float<T>(y);
              y = act_value<FAST>(p.act, y) + add;
            }
            c_ptr[cj * p.ldc + row] = from_float<OT>(y);
          }
        }
        __syncwarp();
        if (lane == 0) {
          for (int q = 0; q < p.split; ++q) mbar_arrive_remote(map_to_cta(sums_free, q));
        }
        if (p.partial != nullptr && in_rows)
          p.partial[(static_cast<long long>(t.col_tile * p.split + static_cast<int>(rank)) * EG + group) * p.m + row] = row_sum;
        continue;
      }

      const int group_col0 = t.col0 + group * GROUP_COLS;
      const bool loads = p.tma && live && load_bytes != 0;
      if (elected && loads) {
        if (group_col0 < t.col_end) request(blocks_done, cta_row0, group_col0, zc);
        if (group_col0 + CB < t.col_end) request(blocks_done + 1, cta_row0, group_col0 + CB, zc);
      }
      ok = mbar_wait(acc_full_bar(acc), acc_phase, abort_flag, 4u, p.status);
      ok = group_all(bar_id, ok);  // all four warps go on, or none
      if (!ok) break;
      tcgen05_fence_after();
#pragma unroll 1
      for (int cb = 0; cb < GROUP_COLS / CB; ++cb) {
        const int col = group_col0 + cb * CB;
        if (col >= t.col_end) break;  // uniform over the group
        uint32_t r[CB];
        if (empty) {
#pragma unroll
          for (int j = 0; j < CB; ++j) r[j] = 0u;
        } else {
          tmem_ld<CB>(t_row + group * GROUP_COLS + cb * CB, r);
        }
        const int valid = min(CB, t.col_end - col);
        float v[CB];
        const int b = blocks_done & (RING - 1);
        OT* const slot_c = reinterpret_cast<OT*>(ring_c + b * SLOT) + row_in_cta;
        T* const slot_z = reinterpret_cast<T*>(ring_z + b * SLOT) + row_in_cta;
        if (p.tma) {
          if (loads) {
            ok = wait_old_block(load_bars + 8u * b, (load_phases >> b) & 1u, p.status);
            load_phases ^= 1u << b;
            if (!ok) break;
          }
#pragma unroll
          for (int j = 0; j < CB; ++j) v[j] = p.alpha * __uint_as_float(r[j]) + bias;
          if (p.grad) {
            if (has_d) {
#pragma unroll
              for (int j = 0; j < CB; ++j) v[j] += p.beta * to_float(reinterpret_cast<const DT*>(slot_c)[j * BM]);
            }
            if (z_in) {
#pragma unroll
              for (int j = 0; j < CB; ++j) v[j] *= act_slope<FAST>(p.act, to_float(slot_z[j * BM]));
            }
          } else {
            if (z_out) {
#pragma unroll
              for (int j = 0; j < CB; ++j) slot_z[j * BM] = from_float<T>(v[j]);
            }
            if (p.act != kActIdentity) {
#pragma unroll
              for (int j = 0; j < CB; ++j) v[j] = act_value<FAST>(p.act, v[j]);
            }
            if (has_d) {
#pragma unroll
              for (int j = 0; j < CB; ++j) v[j] += p.beta * to_float(reinterpret_cast<const DT*>(slot_c)[j * BM]);
            }
          }
#pragma unroll
          for (int j = 0; j < CB; ++j) slot_c[j * BM] = from_float<OT>(v[j]);
          fence_proxy_async();  // the TMA unit reads the buffers through the async proxy
          group_barrier(bar_id);
          if (elected) {
            if (live) {
              if (p.kind == kFusedRaggedCols && valid < CB) {
                // the next columns belong to another group: column by column, 16-byte multiples (m is one of 8 / 4)
                const uint32_t rows = static_cast<uint32_t>(min(BM, p.m - cta_row0));
                for (int j = 0; j < valid; ++j) {
                  const long long cj = col + j;
                  bulk_store(c_ptr + cj * p.ldc + cta_row0, smem_u32(ring_c + b * SLOT) + j * BM * sizeof(OT), rows * sizeof(OT));
                  if (z_out) bulk_store(z_ptr + cj * p.ldz + cta_row0, smem_u32(ring_z + b * SLOT) + j * BM * 2, rows * 2);
                }
              } else {
                tma_store_3d(&map_c, smem_u32(ring_c + b * SLOT), cta_row0, col, zc);
                if (z_out) tma_store_3d(&map_z, smem_u32(ring_z + b * SLOT), cta_row0, col, zc);
              }
            }
            bulk_commit();
            bulk_wait_read<2>();  // the stores of two blocks ago have left their buffers, where block + 2 lands
            if (loads && cb + 2 < GROUP_COLS / CB && col + 2 * CB < t.col_end)
              request(blocks_done + 2, cta_row0, col + 2 * CB, zc);
          }
        } else {
#pragma unroll
          for (int j = 0; j < CB; ++j) v[j] = p.alpha * __uint_as_float(r[j]) + bias;
          if (in_rows) {
            float old[CB];
#pragma unroll
            for (int j = 0; j < CB; ++j)
              old[j] = (has_d && j < valid) ? p.beta * to_float(d_ptr[static_cast<long long>(col + j) * p.ldd + row]) : 0.f;
            if (p.grad) {
              float zz[CB];
#pragma unroll
              for (int j = 0; j < CB; ++j)
                zz[j] = (z_in && j < valid) ? to_float(z_ptr[static_cast<long long>(col + j) * p.ldz + row]) : 0.f;
#pragma unroll
              for (int j = 0; j < CB; ++j) v[j] = (v[j] + old[j]) * (z_in ? act_slope<FAST>(p.act, zz[j]) : 1.f);
            } else {
              if (z_out) {
#pragma unroll
                for (int j = 0; j < CB; ++j)
                  if (j < valid) z_ptr[static_cast<long long>(col + j) * p.ldz + row] = from_float<T>(v[j]);
              }
#pragma unroll
              for (int j = 0; j < CB; ++j) v[j] = act_value<FAST>(p.act, v[j]) + old[j];
            }
#pragma unroll
            for (int j = 0; j < CB; ++j)
              if (j < valid) c_ptr[static_cast<long long>(col + j) * p.ldc + row] = from_float<OT>(v[j]);
          }
        }
        if (p.partial != nullptr) {
#pragma unroll
          for (int j = 0; j < CB; ++j) row_sum += j < valid ? v[j] : 0.f;
        }
        if constexpr (sizeof(OT) == 2) {
          if (p.tri && t.tm != t.tn && in_rows) {
            // mirror image: this thread's columns are consecutive rows there
            OT packed[CB];
#pragma unroll
            for (int j = 0; j < CB; ++j) packed[j] = from_float<OT>(v[j]);
            OT* const dst = c_ptr + static_cast<long long>(row) * p.ldc + col;
            if (p.tma && valid == CB) {
              reinterpret_cast<uint4*>(dst)[0] = reinterpret_cast<const uint4*>(packed)[0];
              reinterpret_cast<uint4*>(dst)[1] = reinterpret_cast<const uint4*>(packed)[1];
            } else {
              for (int j = 0; j < valid; ++j) dst[j] = packed[j];
            }
          }
        }
        ++blocks_done;
      }
      if (!ok) break;
      if (p.partial != nullptr && in_rows)
        p.partial[(static_cast<long long>(t.col_tile) * EG + group) * p.m + row] = row_sum;
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CTAS == 2) mbar_arrive_remote(map_to_cta(acc_empty_bar(acc), 0));
        else mbar_arrive(acc_empty_bar(acc));
      }
    }
    if (elected) bulk_wait_all();  // shared memory stays valid until the last store has read it
  }

  tcgen05_fence_before();
  __syncthreads();
  if (CTAS == 2 || p.split > 1) cluster_sync_all();  // nobody exits while a peer may still signal or read
  if (warp == 1) {
    tcgen05_fence_after();
    if constexpr (CTAS == 2) tmem_dealloc_pair(tmem_base, TMEM_COLS);
    else tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <int CTAS, int BN, class T, class DT, class OT>
cudaError_t launch_typed(const CUtensorMap* maps, const FusedParams& p, int grid, int smem, cudaStream_t stream) {
  auto kernel = fused_gemm_kernel<CTAS, BN, T, DT, OT>;
  const cudaError_t e = kernel_ready(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(64 + 128 * (BN >= 128 ? 2 : 1), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  const int cluster = CTAS == 2 ? 2 : p.split;
  if (cluster > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], maps[2], maps[3], maps[4], p);
}

// Clusters of `cluster` CTAs that the device holds at once (one CTA per SM; a cluster sits in one GPC).
template <int CTAS, int BN>
int resident_clusters(int cluster, int smem) {
  auto kernel = fused_gemm_kernel<CTAS, BN, __half, __half, __half>;
  if (kernel_ready(reinterpret_cast<const void*>(kernel), smem) != cudaSuccess) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(sm_count() / cluster * cluster), 1, 1);
  cfg.blockDim = dim3(64 + 128 * (BN >= 128 ? 2 : 1), 1, 1);
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

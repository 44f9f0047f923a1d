#include "fused_host.h"

#include <cuda.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "driver_api.h"
#include "kernels/fused_aux.h"
#include "kernels/fused_rows.h"
#include "kernels/launchers.h"
#include "runtime_state.h"
#include "scratch.h"
#include "tc_host.h"

namespace b200 {

namespace {

constexpr int kMaxSmem = 232448;  // 227 KB
constexpr int kAlign = 1024;

int elem_size(int type) { return type == 32 ? 4 : 2; }

bool aligned16(const void* base, long long ld, long long planes, long long stride, int elem) {
  return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && (ld * elem) % 16 == 0 && (planes <= 1 || (stride * elem) % 16 == 0);
}

// Tensor map of an epilogue matrix (m contiguous), used to bring tiles of 128 rows x 32 columns into L2.
bool encode_prefetch_map(CUtensorMap* map, int elem, const void* base, long long m, long long n, long long ld, long long planes,
                         long long stride) {
  const DriverApi& drv = driver_api();
  if (!drv.ok) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(m), static_cast<cuuint64_t>(n), static_cast<cuuint64_t>(planes > 1 ? planes : 1)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld * elem), static_cast<cuuint64_t>((planes > 1 ? stride : ld) * elem)};
  if (strides[0] >= (1ULL << 40) || strides[1] >= (1ULL << 40)) return false;
  const cuuint32_t box[3] = {128, 32, 1}, estr[3] = {1, 1, 1};
  const CUtensorMapDataType dt = elem == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  return drv.TensorMapEncodeTiled(map, dt, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                  CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Choice {
  int variant, split;
};

// Rows and columns of a tile; a stage's inner elements are fused_stage_rows() swizzle rows of 64.
constexpr const char* kNames[kFusedVariants] = {"fused_pair_256x256", "fused_128x256", "fused_128x128",
                                                "fused_128x64", "fused_128x32", "fused_pair_256x128"};

// Upper bound of the column tiles of a call (exact for the plain kinds).
long long column_tiles(const FusedDesc& d, int bn) {
  const long long whole = (d.n + bn - 1) / bn;
  return d.kind == kFusedRaggedCols ? whole + d.problems : whole;
}

// Shared memory that a variant needs besides the operand ring: alignment, staging or the sums of split tiles, barriers and
// the group table (8 bytes per group; a thousand groups take 8 KB).
int fixed_smem(const FusedDesc& d, int v, int split) {
  const bool single = d.c_type == 32 || d.parts;
  const int table = d.kind != kFusedPlain ? 8 * (static_cast<int>(d.problems) + 1) : 0;
  return kAlign + fused_staging_bytes(kFusedTable[v].bn, single, d.z != nullptr, split) + kFusedBarBytes + table;
}
// Stages of the ring in what is left; the kernel works from two on.
int ring_stages(const FusedDesc& d, int v, int split) {
  const int stages = (kMaxSmem - fixed_smem(d, v, split)) / kFusedTable[v].stage_bytes;
  return stages < 12 ? stages : 12;
}

bool variant_fits(const FusedDesc& d, int v, int split) {
  const FusedVariant& t = kFusedTable[v];
  if (ring_stages(d, v, split) < 2) return false;  // 128 x 256 with a split from 192 groups on
  const int team = t.ctas * split;
  if (team > 1 && sm_budget() > 0 && team > sm_budget()) return false;  // a tile's CTAs run at once
  if (t.ctas == 2 && split > 1) return false;
  if (d.b_mn && t.bn / t.ctas < 64) return false;                               // a 128-byte row is 64 columns
  if (d.tri && t.ctas * 128 != t.bn) return false;                               // square tiles meet their mirror image
  if (split > 1 && (t.bn / split) % 4 != 0) return false;
  if (split > 1 && (d.tri || d.parts)) return false;
  // Sums of two halves: 256 columns leave one accumulator beside the sums, a pair's block takes 2244 cycles against 1400 for
  // its four blocks of 128 x 128 on two SMs.
  if (d.parts && v != 2) return false;
  return true;
}

// Teams of `team` CTAs that run at once, within the caller's limit on SMs.
int resident_teams(int team) {
  int n = fused_resident_clusters(team);
  if (sm_budget() > 0 && sm_budget() / team < n) n = sm_budget() / team;
  return n > 0 ? n : 1;
}

// Time in SM cycles by a small model: waves of tiles, each the slower of its inner blocks and its epilogue, against the
// memory traffic of the whole call, and what nothing hides at both ends. The constants were fitted to 727 problems with
// every variant timed on each (sizes 1 to 8192, all kinds and types): the choice is within 3 % of the best one in the mean.
// A stage holds 128 inner elements, of 128 x 256 on single SMs 64. Results in single precision wait for their
// one accumulator on 256 columns.
double estimate(const FusedDesc& d, int v, int split, bool vec) {
  static constexpr double kBlock[kFusedVariants] = {1320.0, 743.0, 700.0, 704.0, 700.0, 1000.0};
  const FusedVariant& t = kFusedTable[v];
  const auto whole = [](double x) { return std::ceil(x); };
  const bool single = d.c_type == 32 || d.parts;
  const double rows = static_cast<double>(d.m), cols = static_cast<double>(d.n);
  const double tm = whole(rows / (128 * t.ctas));
  const double active = static_cast<double>(d.problems < d.n ? d.problems : d.n);  // groups that can have vectors
  double tn = whole(cols / t.bn), problems = 1.0, k = static_cast<double>(d.k);
  if (d.kind == kFusedRaggedCols) {
    tn = active * whole(cols / active / t.bn);
  } else {
    problems = static_cast<double>(d.problems);
    if (d.kind == kFusedRaggedInner) k /= problems;
  }
  const double tiles = d.tri ? tm * (tm + 1.0) / 2.0 * problems : tm * tn * problems;
  const double block = kBlock[v] * (single && t.bn == 256 ? 1.7 : 1.0);
  const double load = t.stage_bytes / 71.6;
  const double waves = whole(tiles / resident_teams(t.ctas * split));
  const double main = whole((d.parts ? 3.0 : 1.0) * whole(k / (64.0 * fused_stage_rows(t.ctas, t.bn))) / split) * (block > load ? block : load) + 2350.0;
  // per column of a tile
  const bool reads_z = d.z != nullptr && d.grad, writes_z = d.z != nullptr && !d.grad;
  const bool adds = d.beta != 0.0 && d.d != nullptr;
  double column = 10.1 + (d.act != 161 ? 7.5 : 0.0) + (adds ? 4.3 : 0.0) + (d.z != nullptr ? 4.3 : 0.0);
  if (single) column *= 1.5;
  if (!vec) column += 4.65 * (1.0 + (writes_z ? 1.0 : 0.0) + (reads_z ? 0.5 : 0.0) + (adds ? 0.5 : 0.0));
  double epilogue = column * t.bn;
  if (split > 1) epilogue = 3.0 * epilogue / split + 5500.0 + 10.0 * t.bn;
  // each operand read once and C written once
  const double a_planes = d.kind == kFusedRaggedCols ? active : (d.a_stride != 0 ? problems : 1.0);
  const double c_planes = d.kind == kFusedRaggedCols ? 1.0 : static_cast<double>(d.problems);
  const double bytes = 2.0 * d.k * (a_planes * rows + cols * (d.kind == kFusedPlain ? problems : 1.0)) +
                       c_planes * rows * cols * (single ? 4.0 : 2.0);
  const double work = waves * (main > epilogue ? main : epilogue), memory = bytes / 4136.0;
  return (work > memory ? work : memory) + 6000.0 + epilogue;
}

// B200BLAS_FUSED=<variant>[,<split>] forces one for measurements and tests where it can serve the call.
bool forced_variant(int* variant, int* split) {
  const char* const env = std::getenv("B200BLAS_FUSED");
  if (env == nullptr) return false;
  int v = -1, s = 1;
  if (std::sscanf(env, "%d,%d", &v, &s) < 1 || v < 0 || v >= kFusedVariants || s < 1 || s > 8 || (s & (s - 1)) != 0) return false;
  if (variant) *variant = v;
  if (split) *split = s;
  return true;
}

Choice choose(const FusedDesc& d, bool vec) {
  Choice best = {2, 1};
  double best_time = 1e300;
  for (int v = 0; v < kFusedVariants; ++v) {
    for (int split = 1; split <= 8; split *= 2) {
      if (!variant_fits(d, v, split)) continue;
      const double time = estimate(d, v, split, vec);
      if (time < best_time * 0.999) {
        best_time = time;
        best = {v, split};
      }
    }
  }
  int v, split;
  if (forced_variant(&v, &split) && variant_fits(d, v, split)) best = {v, split};
  return best;
}

// Addresses and strides of a tensor map are multiples of 16 bytes, strides below 2^40.
bool unaddressable(const void* base, long long ld, long long planes, long long stride) {
  constexpr long long kFar = 1LL << 39;
  return (reinterpret_cast<uintptr_t>(base) & 15) != 0 || (ld % 8) != 0 || ld >= kFar ||
         (planes > 1 && ((stride % 8) != 0 || stride >= kFar));
}

}  // namespace

cudaError_t launch_fused(const FusedDesc& d, cudaStream_t stream, const char** name) {
  // A handful of vectors and a matrix whose rows are read along the inner extent. The bias gradient is a sum over the
  // vectors: those calls stay with the kernels that leave partial sums.
  if (d.kind == kFusedPlain && d.problems == 1 && !d.tri && d.n <= kFewRows && !d.a_mn && !d.b_mn && !d.bias_grad &&
      d.c_type == d.d_type && !unaddressable(d.a, d.lda, 1, 0) && !forced_variant(nullptr, nullptr)) {
    FewRowsJob job = {};
    job.type = d.type; job.c_type = d.c_type;
    job.m = static_cast<int>(d.m); job.n = static_cast<int>(d.n); job.k = static_cast<int>(d.k);
    job.w = d.a; job.ldw = d.lda; job.x = d.b; job.ldx = d.ldb;
    job.alpha = static_cast<float>(d.alpha); job.beta = static_cast<float>(d.beta);
    job.bias = d.bias; job.act = d.act; job.grad = d.grad;
    job.d = d.beta != 0.0 ? d.d : nullptr; job.ldd = d.ldd; job.z = d.z; job.ldz = d.ldz; job.c = d.c; job.ldc = d.ldc;
    *name = "fused_few_rows";
    return launch_few_rows(job, stream);
  }
  // an operand with stride 0 is shared by all problems
  const long long per_problem = d.parts ? 2 : 1;
  const long long a_planes = d.kind == kFusedRaggedInner || d.a_stride == 0 ? 1 : d.problems * per_problem;
  const long long b_planes = d.kind == kFusedPlain && d.b_stride != 0 ? d.problems * per_problem : 1;
  // Operands that TMA cannot address are copied once to an aligned pitch.
  PoolScratch copies, partial, sums;
  FusedDesc r = d;
  PackJob jobs[2] = {};
  const auto plan = [&](PackJob& job, const void* base, long long ld, long long stride, bool mn, long long rows,
                        long long planes) -> size_t {
    if (!unaddressable(base, ld, planes, stride)) return 0;
    job.one = mn ? rows : d.k;
    job.two = mn ? d.k : rows;
    job.planes = planes;
    job.src = base;
    job.src_ld = ld;
    job.src_stride = planes > 1 ? stride : 0;
    job.pitch = (job.one + 7) / 8 * 8;
    return (static_cast<size_t>(job.pitch) * job.two * planes * 2 + 255) / 256 * 256;
  };
  const size_t a_bytes = plan(jobs[0], d.a, d.lda, d.a_stride, d.a_mn != 0, d.m, a_planes);
  const size_t b_bytes = plan(jobs[1], d.b, d.ldb, d.b_stride, d.b_mn != 0, d.n, b_planes);
  if (d.kind == kFusedRaggedCols && a_planes > 1) jobs[0].offsets = d.offsets;
  cudaError_t e = cudaSuccess;
  if (a_bytes + b_bytes > 0) {
    e = copies.get(a_bytes + b_bytes, stream);
    if (e != cudaSuccess) return e;
    if (a_bytes) {
      jobs[0].dst = copies.ptr();
      r.a = jobs[0].dst; r.lda = jobs[0].pitch; r.a_stride = jobs[0].pitch * jobs[0].two;
    }
    if (b_bytes) {
      jobs[1].dst = copies.ptr() + a_bytes;
      r.b = jobs[1].dst; r.ldb = jobs[1].pitch; r.b_stride = jobs[1].pitch * jobs[1].two;
    }
    e = launch_pack(jobs, stream);
    if (e != cudaSuccess) return e;
  }

  const void* const residual = d.beta != 0.0 ? d.d : nullptr;
  const long long c_planes = d.kind == kFusedRaggedCols ? 1 : d.problems * per_problem;
  const bool vec = d.m % 8 == 0 && aligned16(d.c, d.ldc, c_planes, d.c_stride, elem_size(d.c_type)) &&
                   (!residual || aligned16(residual, d.ldd, c_planes, d.d_stride, elem_size(d.d_type))) &&
                   (!d.z || aligned16(d.z, d.ldz, c_planes, d.z_stride, 2));
  const Choice choice = choose(d, vec);
  const FusedVariant& t = kFusedTable[choice.variant];
  FusedParams p = {};
  p.status = tc_status_device();
  p.m = static_cast<int>(d.m);
  p.n = static_cast<int>(d.n);
  p.k = static_cast<int>(d.k);
  p.kind = d.kind;
  p.problems = static_cast<int>(d.problems);
  p.offsets = d.offsets;
  p.tiles_m = static_cast<int>((d.m + 128 * t.ctas - 1) / (128 * t.ctas));
  p.tiles_n = static_cast<int>((d.n + t.bn - 1) / t.bn);
  p.raster = t.ctas == 2 ? 8 : 16;
  p.tri = d.tri;
  p.parts = d.parts;
  p.chained = d.chained || a_bytes + b_bytes > 0;  // right behind the copies
  p.a_mn = d.a_mn;
  p.b_mn = d.b_mn;
  const unsigned format = d.type == 16 ? 0u : 1u;  // fp32 accumulator; f16 or bf16 operands
  p.idesc = (1u << 4) | (format << 7) | (format << 10) | (static_cast<unsigned>(d.a_mn != 0) << 15) |
            (static_cast<unsigned>(d.b_mn != 0) << 16) | (static_cast<unsigned>(t.bn >> 3) << 17) |
            (static_cast<unsigned>((128 * t.ctas) >> 4) << 24);
  p.a_batched = a_planes > 1;
  p.b_batched = b_planes > 1;
  p.split = choice.split;
  p.alpha = static_cast<float>(d.alpha);
  p.beta = static_cast<float>(d.beta);
  p.bias = d.bias;
  p.bias_stride = d.bias_stride;
  p.act = d.act;
  p.grad = d.grad;
  p.c = d.c; p.ldc = d.ldc; p.c_stride = d.c_stride;
  p.d = residual; p.ldd = d.ldd; p.d_stride = d.d_stride;
  p.z = d.z; p.ldz = d.ldz; p.z_stride = d.z_stride;
  p.vec = vec ? 1 : 0;

  CUtensorMap maps[4];
  std::memset(maps + 2, 0, 2 * sizeof(CUtensorMap));
  if (!encode_operand_map(&maps[0], 2, r.a, d.m, d.k, r.lda, d.a_mn != 0, 128, a_planes, r.a_stride) ||
      !encode_operand_map(&maps[1], 2, r.b, d.n, d.k, r.ldb, d.b_mn != 0, t.bn / t.ctas, b_planes, r.b_stride))
    return cudaErrorInvalidValue;
  const bool reads_z = p.z && d.grad;
  if (p.vec && choice.split == 1 && (p.d || reads_z))
    p.prefetch = (!p.d || encode_prefetch_map(&maps[2], elem_size(d.d_type), p.d, d.m, d.n, d.ldd, c_planes, d.d_stride)) &&
                 (!reads_z || encode_prefetch_map(&maps[3], 2, p.z, d.m, d.n, d.ldz, c_planes, d.z_stride));
  if ((d.tri || d.parts) && (!p.vec || p.z)) return cudaErrorInvalidValue;  // 16-byte stores only
  if (d.tri && d.n != d.m) return cudaErrorInvalidValue;

  const long long col_tiles = column_tiles(d, t.bn);
  long long tiles = col_tiles * p.tiles_m;
  if (d.kind != kFusedRaggedCols) tiles *= d.problems;
  if (d.tri) tiles = static_cast<long long>(p.tiles_m) * (p.tiles_m + 1) / 2 * d.problems;
  if (tiles > 0x3FFFFFFF) return cudaErrorInvalidValue;
  const int lines_per_tile = fused_groups(t.bn) * choice.split;
  if (d.bias_grad != nullptr) {
    e = partial.get(static_cast<size_t>(col_tiles) * lines_per_tile * d.m * sizeof(float), stream);
    if (e != cudaSuccess) return e;
    p.partial = reinterpret_cast<float*>(partial.ptr());
  }

  p.stages = ring_stages(d, choice.variant, choice.split);
  const int smem = fixed_smem(d, choice.variant, choice.split) + p.stages * t.stage_bytes;

  const int team = t.ctas * choice.split;
  long long teams = resident_teams(team);
  if (tiles < teams) teams = tiles;
  if (d.c_type != 32 && !d.parts) {
    const long long stage_k = 64LL * fused_stage_rows(t.ctas, t.bn), in_all = (d.k + stage_k - 1) / stage_k;
    if ((in_all + choice.split - 1) / choice.split > kChunkHalf / stage_k) {
      e = sums.get(static_cast<size_t>(teams) * team * 128 * t.bn * sizeof(float), stream);
      if (e != cudaSuccess) return e;
      p.sums = reinterpret_cast<float*>(sums.ptr());
    }
  }
  e = launch_fused_variant(choice.variant, d.type, d.d_type, d.c_type, maps, p, static_cast<int>(teams) * team, smem, stream);
  static thread_local char label[64];
  if (choice.split > 1) std::snprintf(label, sizeof(label), "%s_split%d", kNames[choice.variant], choice.split);
  else std::snprintf(label, sizeof(label), "%s", kNames[choice.variant]);
  *name = label;
  if (e == cudaSuccess && d.bias_grad != nullptr) {
    SumJob job = {};
    job.partial = p.partial;
    job.m = d.m;
    job.type = d.type;
    job.out = d.bias_grad;
    job.out_stride = d.bias_grad_stride;
    job.offsets = d.kind == kFusedRaggedCols ? d.offsets : nullptr;
    job.groups = p.problems;
    job.bound = d.n;
    job.per_tile = t.bn;
    job.lines_per_tile = lines_per_tile;
    job.tiles = col_tiles;
    e = launch_sum_partials(job, stream);
  }
  return e;
}

cudaError_t launch_fused_variant(int v, int type, int d_type, int c_type, const CUtensorMap* maps, const FusedParams& p,
                                 int grid, int smem, cudaStream_t stream) {
  switch (v) {
    case 0: return launch_fused_pair(type, d_type, c_type, maps, p, grid, smem, stream);
    case 1: return launch_fused_256(type, d_type, c_type, maps, p, grid, smem, stream);
    case 2: return launch_fused_128(type, d_type, c_type, maps, p, grid, smem, stream);
    case 3: return launch_fused_64(type, d_type, c_type, maps, p, grid, smem, stream);
    case 5: return launch_fused_pair128(type, d_type, c_type, maps, p, grid, smem, stream);
    case 4: return launch_fused_32(type, d_type, c_type, maps, p, grid, smem, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace b200

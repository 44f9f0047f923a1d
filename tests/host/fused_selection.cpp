// Host half of the fused products without a device: csrc/fused_host.cpp over launchers that only note what they are given.
// Reads one call per line from standard input and prints what would be launched.
//   kind problems m n k type c_type grad z bias_grad beta a_mn b_mn tri parts budget
//   -> error variant split stages smem grid
#include <cstdio>
#include <cstdint>

#include "driver_api.h"
#include "fused_host.h"
#include "kernels/fused_aux.h"
#include "kernels/fused_rows.h"
#include "kernels/launchers.h"
#include "runtime_state.h"
#include "scratch.h"
#include "tc_host.h"

namespace b200 {

namespace {

int g_budget = 0;
struct Launch { int variant, split, stages, smem, grid; } g_last;

CUresult encode(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
  return CUDA_SUCCESS;
}
cudaError_t note(int variant, const FusedParams& p, int grid, int smem) {
  g_last = {variant, p.split, p.stages, smem, grid};
  return cudaSuccess;
}

}  // namespace

const DriverApi& driver_api() {
  static DriverApi api = {};
  api.TensorMapEncodeTiled = encode;
  api.ok = true;
  return api;
}
unsigned int* tc_status_device() { return nullptr; }
int sm_count() { return 148; }
int sm_budget() { return g_budget; }
cudaError_t PoolScratch::get(size_t, cudaStream_t) {
  static unsigned char page[256];
  ptr_ = page;
  return cudaSuccess;
}
PoolScratch::~PoolScratch() {}
bool encode_operand_map(CUtensorMap*, int, const void*, long long, long long, long long, bool, int, long long, long long) { return true; }
cudaError_t launch_pack(const PackJob (&)[2], cudaStream_t) { return cudaSuccess; }
cudaError_t launch_few_rows(const FewRowsJob&, cudaStream_t) { g_last = {-1, 1, 2, 0, 1}; return cudaSuccess; }
cudaError_t launch_sum_partials(const SumJob&, cudaStream_t) { return cudaSuccess; }
// the clusters that a B200 holds at once
int fused_resident_clusters(int cluster) { return cluster <= 1 ? 148 : cluster == 2 ? 74 : cluster == 4 ? 36 : 16; }
#define VARIANT(name, v)                                                                                                \
  cudaError_t name(int, int, int, const CUtensorMap*, const FusedParams& p, int grid, int smem, cudaStream_t) {        \
    return note(v, p, grid, smem);                                                                                      \
  }
VARIANT(launch_fused_pair, 0)
VARIANT(launch_fused_256, 1)
VARIANT(launch_fused_128, 2)
VARIANT(launch_fused_64, 3)
VARIANT(launch_fused_32, 4)
VARIANT(launch_fused_pair128, 5)

}  // namespace b200

int main() {
  using namespace b200;
  int kind, type, c_type, grad, z, bias_grad, a_mn, b_mn, tri, parts, budget;
  long long problems, m, n, k;
  double beta;
  while (std::scanf("%d %lld %lld %lld %lld %d %d %d %d %d %lf %d %d %d %d %d", &kind, &problems, &m, &n, &k, &type, &c_type, &grad, &z,
                    &bias_grad, &beta, &a_mn, &b_mn, &tri, &parts, &budget) == 16) {
    g_budget = budget;
    g_last = {-2, 0, 0, 0, 0};
    const auto up = [](long long x) { return (x + 7) / 8 * 8; };
    void* const somewhere = reinterpret_cast<void*>(uintptr_t(1) << 32);  // never read
    FusedDesc d = {};
    d.type = type; d.c_type = d.d_type = c_type; d.kind = kind; d.problems = problems;
    d.offsets = kind != kFusedPlain ? static_cast<const long long*>(somewhere) : nullptr;
    d.m = m; d.n = n; d.k = k; d.alpha = 1.0; d.beta = beta; d.act = 161; d.grad = grad; d.tri = tri; d.parts = parts;
    d.a = somewhere; d.lda = up(a_mn ? m : k); d.a_mn = a_mn;
    d.b = somewhere; d.ldb = up(b_mn ? n : k); d.b_mn = b_mn;
    if (kind == kFusedRaggedCols || (kind == kFusedPlain && problems > 1)) d.a_stride = d.lda * (a_mn ? k : m);
    if (kind == kFusedPlain && problems > 1) d.b_stride = d.ldb * (b_mn ? k : n);
    d.c = somewhere; d.ldc = up(m);
    if (kind != kFusedRaggedCols) d.c_stride = d.ldc * n;
    if (beta != 0.0) { d.d = somewhere; d.ldd = d.ldc; d.d_stride = d.c_stride; }
    if (z) { d.z = somewhere; d.ldz = up(m); d.z_stride = d.c_stride; }
    if (bias_grad) d.bias_grad = somewhere;
    const char* name = "";
    const cudaError_t e = launch_fused(d, nullptr, &name);
    std::printf("%d %d %d %d %d %d\n", static_cast<int>(e), g_last.variant, g_last.split, g_last.stages, g_last.smem, g_last.grid);
  }
  return 0;
}

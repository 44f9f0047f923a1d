// Entry points of the products with an epilogue, the products grouped by expert, their backward forms and the
// Newton-Schulz orthogonalisation.
//
// All of them see memory order only: "features" are the elements of a contiguous vector (the unit-stride extent of C),
// "vectors" are its lines. A row-major call is the column-major call on the transposed matrices, as in the GEMM family.
#include "b200blas.h"

#include <cuda.h>
#include <cuda_runtime_api.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include <type_traits>

#include "driver_api.h"
#include "fused_host.h"
#include "host_common.h"
#include "kernels/fused_aux.h"
#include "kernels/fused_rows.h"
#include "kernels/fused_single.h"
#include "kernels/launchers.h"
#include "scratch.h"

namespace b200 {

void note_launch(const char* name, cudaError_t err);

namespace {

constexpr int kInvalidVectorX = -1019, kInvalidVectorY = -1018, kInsufficientMemoryX = -1008, kInsufficientMemoryY = -1007;
constexpr int kActIdentityCode = 161;
constexpr size_t kMaxExtent = 0x7FFFFFFFull - 4096;  // extents and tile ends stay inside 32 bits
constexpr size_t kMaxElements = size_t(1) << 46;     // offsets, leading dimensions, strides: no product overflows

int elem_of(int type) { return type == 32 ? 4 : 2; }
bool valid_activation(int a) { return a >= 161 && a <= 165; }
bool valid_transpose(int t) { return t == kNo || t == kYes || t == kConjugate; }
bool half_type(int t) { return t == 16 || t == kBFloat16; }

// kSuccess for the types the routines are built for, kNotImplemented for the library's other precisions.
int check_types(int dtype, int c_dtype, bool single_too) {
  if (half_type(dtype)) return (c_dtype == dtype || c_dtype == 32) ? kSuccess : kNotImplemented;
  if (dtype == 32 && single_too) return c_dtype == 32 ? kSuccess : kNotImplemented;
  if (dtype == 32 || dtype == 64 || dtype == 3232 || dtype == 6464) return kNotImplemented;
  return kUnexpectedError;
}

// `planes` matrices, `stride` apart, of `two` lines of `one` elements each: leading dimension, then the allocation that
// holds them, which has to lie on the current device.
int check(size_t one, size_t two, size_t planes, const void* buf, size_t offset, size_t ld, size_t stride, int elem,
          int bad_ld, int too_small, int invalid) {
  if (ld < one) return bad_ld;
  if (!buf || (reinterpret_cast<uintptr_t>(buf) % elem) != 0) return invalid;
  if (ld > kMaxElements || offset > kMaxElements || stride > kMaxElements || two > kMaxElements / ld ||
      planes > kMaxElements / (stride + 1))
    return too_small;
  const DriverApi& drv = driver_api();
  if (!drv.ok) return invalid;
  CUdeviceptr base = 0;
  size_t size = 0;
  const CUdeviceptr at = reinterpret_cast<CUdeviceptr>(buf);
  if (drv.MemGetAddressRange(&base, &size, at) != CUDA_SUCCESS) {
    // a host thread's first call finds no context: that binds the device's own (backward passes run on such threads)
    unsigned long long key = 0;
    if (context_key(&key) != 0 || drv.MemGetAddressRange(&base, &size, at) != CUDA_SUCCESS) return invalid;
  }
  if (drv.PointerGetAttribute) {
    int owner = -1, current = -2;
    if (drv.PointerGetAttribute(&owner, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL, at) == CUDA_SUCCESS &&
        cudaGetDevice(&current) == cudaSuccess && owner != current)
      return invalid;
  }
  const size_t have = size - (at - base);
  const size_t need = ((planes - 1) * stride + ld * (two - 1) + one + offset) * elem;
  return have < need ? too_small : static_cast<int>(kSuccess);
}

int check_a(size_t one, size_t two, size_t planes, const void* p, size_t off, size_t ld, size_t stride, int elem) {
  return check(one, two, planes, p, off, ld, stride, elem, kInvalidLeadDimA, kInsufficientMemoryA, kInvalidMatrixA);
}
int check_b(size_t one, size_t two, size_t planes, const void* p, size_t off, size_t ld, size_t stride, int elem) {
  return check(one, two, planes, p, off, ld, stride, elem, kInvalidLeadDimB, kInsufficientMemoryB, kInvalidMatrixB);
}
int check_c(size_t one, size_t two, size_t planes, const void* p, size_t off, size_t ld, size_t stride, int elem) {
  return check(one, two, planes, p, off, ld, stride, elem, kInvalidLeadDimC, kInsufficientMemoryC, kInvalidMatrixC);
}

template <class P>
P at(P base, size_t offset, int elem) {
  using Byte = typename std::conditional<std::is_const<typename std::remove_pointer<P>::type>::value, const unsigned char, unsigned char>::type;
  return base ? static_cast<P>(static_cast<Byte*>(base) + offset * elem) : nullptr;
}

// Bytes [first, last) that a matrix spans.
struct Span {
  const unsigned char *first, *last;
};
Span span_of(const void* p, size_t one, size_t two, size_t ld, int elem) {
  const unsigned char* b = static_cast<const unsigned char*>(p);
  return {b, b ? b + (ld * (two - 1) + one) * elem : b};
}
bool overlap(const Span& a, const Span& b) { return a.first && b.first && a.first < b.last && b.first < a.last; }

// A matrix in memory: `two` lines of `one` elements.
struct Area {
  const void* p;
  size_t one, two, ld;
  int elem;
  Span span() const { return span_of(p, one, two, ld, elem); }
};

// Whether a matrix may lie where it does beside one that is written: apart from it, as other columns of the same lines, or
// (where `same_allowed`) as the very same elements, each read before it is written.
bool beside(const Area& x, const Area& c, bool same_allowed) {
  if (!x.p || !c.p || !overlap(x.span(), c.span())) return true;
  const size_t pitch = c.ld * c.elem;
  if (x.ld * x.elem != pitch) return false;
  if (same_allowed && x.p == c.p && x.elem == c.elem) return true;
  const unsigned char *p = static_cast<const unsigned char*>(x.p), *q = static_cast<const unsigned char*>(c.p);
  const size_t x_line = x.one * x.elem, c_line = c.one * c.elem;
  // where x's lines begin relative to c's, within a pitch
  const size_t gap = p >= q ? static_cast<size_t>(p - q) % pitch : (pitch - static_cast<size_t>(q - p) % pitch) % pitch;
  return gap >= c_line && gap + x_line <= pitch;
}

// What a first call sets up (the status block, the pool, kernel attributes) would invalidate a capture that this thread is
// recording in the usual mode; none of it is work on the captured stream.
struct RelaxedCapture {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  const bool on = cudaThreadExchangeStreamCaptureMode(&mode) == cudaSuccess;
  ~RelaxedCapture() {
    if (on) (void)cudaThreadExchangeStreamCaptureMode(&mode);
  }
};

template <class F>
int guarded(F&& f) {
  try {
    RelaxedCapture relaxed;
    return f();
  } catch (...) {
    return kUnexpectedError;
  }
}

int finish(cudaStream_t s, int async, cudaError_t err, const char* name) {
  note_launch(name, err);
  if (err != cudaSuccess) cudaGetLastError();
  return end_call(s, async, err);
}

// The two operands of a layout-bearing call in kernel orientation.
struct Operands {
  size_t m, n;  // features, vectors
  const void *a, *b;
  size_t lda, ldb;
  int a_mn, b_mn;
};
Operands orient(int layout, int ta, int tb, size_t m, size_t n, const void* a, size_t a_ld, const void* b, size_t b_ld) {
  if (layout == kRowMajor) return {n, m, b, a, b_ld, a_ld, tb == kNo, ta != kNo};
  return {m, n, a, b, a_ld, b_ld, ta == kNo, tb != kNo};
}

// Single precision: the product on the library's SGEMM kernels, then one pass over it. `job` comes with everything but
// P; C takes the product itself where nothing that the pass reads lies there.
cudaError_t single_epilogue(int layout, int ta, int tb, size_t m, size_t n, size_t k, double alpha, const void* a,
                            size_t a_ld, const void* b, size_t b_ld, PointwiseJob job, void* bias_grad,
                            cudaStream_t s, const char** name) {
  const double al[2] = {alpha, 0.0}, zero[2] = {0.0, 0.0};
  const Operands o = orient(layout, ta, tb, m, n, a, a_ld, b, b_ld);
  const bool split = single_fits(job.m, job.n, static_cast<long long>(k));
  SingleJob one = {};
  one.m = job.m; one.n = job.n; one.k = static_cast<long long>(k); one.alpha = static_cast<float>(alpha);
  one.a = static_cast<const float*>(o.a); one.lda = static_cast<long long>(o.lda); one.a_mn = o.a_mn;
  one.b = static_cast<const float*>(o.b); one.ldb = static_cast<long long>(o.ldb); one.b_mn = o.b_mn;
  one.act = kActIdentityCode;
  if (bias_grad == nullptr && job.n <= kFewRows && !o.a_mn && !o.b_mn && (reinterpret_cast<uintptr_t>(o.a) & 15) == 0 && o.lda % 4 == 0) {
    FewRowsJob rows = {};
    rows.type = rows.c_type = 32;
    rows.m = static_cast<int>(job.m); rows.n = static_cast<int>(job.n); rows.k = static_cast<int>(k);
    rows.w = o.a; rows.ldw = one.lda; rows.x = o.b; rows.ldx = one.ldb;
    rows.alpha = one.alpha; rows.beta = job.beta; rows.bias = job.bias; rows.act = job.act; rows.grad = job.grad;
    rows.d = job.d; rows.ldd = job.ldd; rows.z = job.z; rows.ldz = job.ldz; rows.c = job.c; rows.ldc = job.ldc;
    *name = "single_few_rows";
    return launch_few_rows(rows, s);
  }
  if (bias_grad == nullptr && split) {
    one.bias = static_cast<const float*>(job.bias); one.act = job.act; one.grad = job.grad;
    one.d = static_cast<const float*>(job.d); one.ldd = job.ldd; one.beta = job.beta;
    one.z = static_cast<float*>(job.z); one.ldz = job.ldz;
    one.c = static_cast<float*>(job.c); one.ldc = job.ldc;
    *name = "single_split";
    return launch_single(one, s);
  }
  const Span c = span_of(job.c, job.m, job.n, job.ldc, 4);
  PoolScratch product, partial;
  void* p = job.c;
  size_t ldp = static_cast<size_t>(job.ldc);
  // a pass over the product must find its own D and Z whole
  const bool reads_c = overlap(c, span_of(job.d, job.m, job.n, job.ldd, 4)) ||
                       (job.grad && overlap(c, span_of(job.z, job.m, job.n, job.ldz, 4)));
  if (reads_c) {
    ldp = (static_cast<size_t>(job.m) + 3) / 4 * 4;
    const cudaError_t e = product.get(ldp * job.n * 4, s);
    if (e != cudaSuccess) return e;
    p = product.ptr();
  }
  if (split) {
    one.c = static_cast<float*>(p); one.ldc = static_cast<long long>(ldp);
    *name = "single_split_pointwise";
    const cudaError_t e = launch_single(one, s);
    if (e != cudaSuccess) return e;
  } else {
    const int st = gemm_enqueue(32, layout, ta, tb, m, n, k, al, a, 0, a_ld, b, 0, b_ld, zero, p, 0, ldp, s);
    if (st != kSuccess) return st > 0 ? static_cast<cudaError_t>(st) : cudaErrorInvalidValue;
    *name = "single_product_pointwise";
  }
  const bool plain = job.bias == nullptr && job.d == nullptr && job.z == nullptr && job.act == kActIdentityCode;
  if (plain && bias_grad == nullptr && p == job.c) return cudaSuccess;
  job.p = p;
  job.ldp = static_cast<long long>(ldp);
  if (bias_grad != nullptr) {
    const cudaError_t e = partial.get(static_cast<size_t>(pointwise_chunks(job)) * job.m * 4, s);
    if (e != cudaSuccess) return e;
    job.partial = reinterpret_cast<float*>(partial.ptr());
  }
  cudaError_t e = launch_pointwise(job, s);
  if (e == cudaSuccess && bias_grad != nullptr) {
    SumJob sum = {};
    sum.partial = job.partial; sum.m = job.m; sum.type = job.type; sum.out = bias_grad; sum.groups = 1;
    sum.per_tile = kPointwiseChunk; sum.lines_per_tile = 1; sum.tiles = pointwise_chunks(job);
    e = launch_sum_partials(sum, s);
  }
  return e;
}

bool extents_ok(size_t a, size_t b, size_t c) { return a <= kMaxExtent && b <= kMaxExtent && c <= kMaxExtent; }

int check_offsets(const long long* offsets, size_t groups) {
  const int st = check(groups + 1, 1, 1, offsets, 0, groups + 1, 0, 8, kInvalidBatchCount, kInvalidBatchCount, kInvalidBatchCount);
  return st;
}
// Every CTA reads the offsets when it starts, at a time when others may be storing results already: were they written, the
// CTAs of one tile could take different tiles.
Span offsets_span(const long long* offsets, size_t groups) { return span_of(offsets, groups + 1, 1, groups + 1, 8); }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200blas_gemm_epilogue(int dtype, int c_dtype, int layout, int ta, int tb, size_t m, size_t n, size_t k,
                                      double alpha, const void* a, size_t a_offset, size_t a_ld, const void* b,
                                      size_t b_offset, size_t b_ld, const void* bias, size_t bias_offset, int activation,
                                      void* z, size_t z_offset, size_t z_ld, double beta, const void* d, size_t d_offset,
                                      size_t d_ld, void* c, size_t c_offset, size_t c_ld, void* stream, int async) {
  return guarded([&]() -> int {
    int st = check_types(dtype, c_dtype, true);
    if (st != kSuccess) return st;
    if (!valid_enums(layout, ta, tb) || !valid_activation(activation)) return kUnexpectedError;
    if (m == 0 || n == 0 || k == 0 || !extents_ok(m, n, k)) return kInvalidDimension;
    const int elem = elem_of(dtype), c_elem = elem_of(c_dtype);
    const Extents e = extents(layout, ta, tb, m, n, k);
    if ((st = check_a(e.a_one, e.a_two, 1, a, a_offset, a_ld, 0, elem))) return st;
    if ((st = check_b(e.b_one, e.b_two, 1, b, b_offset, b_ld, 0, elem))) return st;
    if (bias && (st = check(e.c_one, 1, 1, bias, bias_offset, e.c_one, 0, elem, kInvalidVectorX, kInsufficientMemoryX, kInvalidVectorX))) return st;
    if (z && (st = check_c(e.c_one, e.c_two, 1, z, z_offset, z_ld, 0, elem))) return st;
    const bool has_d = beta != 0.0;
    if (has_d && (st = check_c(e.c_one, e.c_two, 1, d, d_offset, d_ld, 0, c_elem))) return st;
    if ((st = check_c(e.c_one, e.c_two, 1, c, c_offset, c_ld, 0, c_elem))) return st;
    a = at(a, a_offset, elem); b = at(b, b_offset, elem); bias = at(bias, bias_offset, elem);
    z = at(z, z_offset, elem); d = has_d ? at(d, d_offset, c_elem) : nullptr; c = at(c, c_offset, c_elem);
    const Area at_c = {c, e.c_one, e.c_two, c_ld, c_elem}, at_d = {d, e.c_one, e.c_two, d_ld, c_elem};
    const Area at_z = {z, e.c_one, e.c_two, z_ld, elem}, at_a = {a, e.a_one, e.a_two, a_ld, elem};
    const Area at_b = {b, e.b_one, e.b_two, b_ld, elem}, at_bias = {bias, e.c_one, 1, e.c_one, elem};
    for (const Area& out : {at_c, at_z})
      if (!beside(at_a, out, false) || !beside(at_b, out, false) || !beside(at_bias, out, false)) return kInvalidMatrixC;
    if (!beside(at_z, at_c, false) || !beside(at_d, at_c, true) || !beside(at_d, at_z, false)) return kInvalidMatrixC;
    cudaStream_t s;
    const int r = begin_call(stream, async, &s);
    if (r != 0) return r;
    const Operands o = orient(layout, ta, tb, m, n, a, a_ld, b, b_ld);
    const char* name = "none";
    if (dtype == 32) {
      PointwiseJob job = {};
      job.type = 32; job.act = activation; job.m = static_cast<long long>(o.m); job.n = static_cast<long long>(o.n);
      job.bias = bias; job.d = d; job.ldd = static_cast<long long>(d_ld); job.beta = static_cast<float>(beta);
      job.z = z; job.ldz = static_cast<long long>(z_ld); job.c = c; job.ldc = static_cast<long long>(c_ld);
      job.groups = 1;
      const cudaError_t err = single_epilogue(layout, ta, tb, m, n, k, alpha, a, a_ld, b, b_ld, job, nullptr, s, &name);
      return finish(s, async, err, name);
    }
    FusedDesc f = {};
    f.type = dtype; f.c_type = f.d_type = c_dtype; f.kind = kFusedPlain; f.problems = 1;
    f.m = static_cast<long long>(o.m); f.n = static_cast<long long>(o.n); f.k = static_cast<long long>(k);
    f.a = o.a; f.lda = static_cast<long long>(o.lda); f.a_mn = o.a_mn;
    f.b = o.b; f.ldb = static_cast<long long>(o.ldb); f.b_mn = o.b_mn;
    f.alpha = alpha; f.beta = beta; f.bias = bias; f.act = activation;
    f.d = d; f.ldd = static_cast<long long>(d_ld); f.z = z; f.ldz = static_cast<long long>(z_ld);
    f.c = c; f.ldc = static_cast<long long>(c_ld);
    const cudaError_t err = launch_fused(f, s, &name);
    return finish(s, async, err, name);
  });
}

extern "C" int b200blas_gemm_epilogue_grad(int dtype, int layout, int ta, int tb, size_t m, size_t n, size_t k,
                                           double alpha, const void* a, size_t a_offset, size_t a_ld, const void* b,
                                           size_t b_offset, size_t b_ld, double beta, const void* d, size_t d_offset,
                                           size_t d_ld, int activation, const void* z, size_t z_offset, size_t z_ld,
                                           void* c, size_t c_offset, size_t c_ld, void* bias_grad,
                                           size_t bias_grad_offset, void* stream, int async) {
  return guarded([&]() -> int {
    int st = check_types(dtype, dtype, true);
    if (st != kSuccess) return st;
    if (!valid_enums(layout, ta, tb) || !valid_activation(activation)) return kUnexpectedError;
    if (m == 0 || n == 0 || k == 0 || !extents_ok(m, n, k)) return kInvalidDimension;
    const int elem = elem_of(dtype);
    const Extents e = extents(layout, ta, tb, m, n, k);
    if ((st = check_a(e.a_one, e.a_two, 1, a, a_offset, a_ld, 0, elem))) return st;
    if ((st = check_b(e.b_one, e.b_two, 1, b, b_offset, b_ld, 0, elem))) return st;
    const bool has_d = beta != 0.0, has_z = activation != kActIdentityCode;
    if (has_d && (st = check_c(e.c_one, e.c_two, 1, d, d_offset, d_ld, 0, elem))) return st;
    if (has_z && (st = check_c(e.c_one, e.c_two, 1, z, z_offset, z_ld, 0, elem))) return st;
    if ((st = check_c(e.c_one, e.c_two, 1, c, c_offset, c_ld, 0, elem))) return st;
    if (bias_grad && (st = check(e.c_one, 1, 1, bias_grad, bias_grad_offset, e.c_one, 0, elem, kInvalidVectorY, kInsufficientMemoryY, kInvalidVectorY))) return st;
    a = at(a, a_offset, elem); b = at(b, b_offset, elem);
    d = has_d ? at(d, d_offset, elem) : nullptr; z = has_z ? at(z, z_offset, elem) : nullptr;
    c = at(c, c_offset, elem); bias_grad = at(bias_grad, bias_grad_offset, elem);
    const Area at_c = {c, e.c_one, e.c_two, c_ld, elem}, at_d = {d, e.c_one, e.c_two, d_ld, elem};
    const Area at_z = {z, e.c_one, e.c_two, z_ld, elem}, at_a = {a, e.a_one, e.a_two, a_ld, elem};
    const Area at_b = {b, e.b_one, e.b_two, b_ld, elem}, at_sum = {bias_grad, e.c_one, 1, e.c_one, elem};
    if (!beside(at_a, at_c, false) || !beside(at_b, at_c, false) || !beside(at_z, at_c, true) || !beside(at_d, at_c, true))
      return kInvalidMatrixC;
    for (const Area& in : {at_a, at_b, at_c, at_d, at_z})
      if (overlap(in.span(), at_sum.span())) return kInvalidVectorY;
    cudaStream_t s;
    const int r = begin_call(stream, async, &s);
    if (r != 0) return r;
    const Operands o = orient(layout, ta, tb, m, n, a, a_ld, b, b_ld);
    const char* name = "none";
    if (dtype == 32) {
      PointwiseJob job = {};
      job.type = 32; job.act = activation; job.grad = 1; job.m = static_cast<long long>(o.m); job.n = static_cast<long long>(o.n);
      job.d = d; job.ldd = static_cast<long long>(d_ld); job.beta = static_cast<float>(beta);
      job.z = const_cast<void*>(z); job.ldz = static_cast<long long>(z_ld); job.c = c; job.ldc = static_cast<long long>(c_ld);
      job.groups = 1;
      const cudaError_t err = single_epilogue(layout, ta, tb, m, n, k, alpha, a, a_ld, b, b_ld, job, bias_grad, s, &name);
      return finish(s, async, err, name);
    }
    FusedDesc f = {};
    f.type = f.c_type = f.d_type = dtype; f.kind = kFusedPlain; f.problems = 1; f.grad = 1;
    f.m = static_cast<long long>(o.m); f.n = static_cast<long long>(o.n); f.k = static_cast<long long>(k);
    f.a = o.a; f.lda = static_cast<long long>(o.lda); f.a_mn = o.a_mn;
    f.b = o.b; f.ldb = static_cast<long long>(o.ldb); f.b_mn = o.b_mn;
    f.alpha = alpha; f.beta = beta; f.act = activation;
    f.d = d; f.ldd = static_cast<long long>(d_ld); f.z = const_cast<void*>(z); f.ldz = static_cast<long long>(z_ld);
    f.c = c; f.ldc = static_cast<long long>(c_ld); f.bias_grad = bias_grad;
    const cudaError_t err = launch_fused(f, s, &name);
    return finish(s, async, err, name);
  });
}

extern "C" int b200blas_activation_grad(int dtype, size_t rows, size_t n, int activation, const void* dy,
                                        size_t dy_offset, size_t dy_ld, const void* z, size_t z_offset, size_t z_ld,
                                        void* dz, size_t dz_offset, size_t dz_ld, void* bias_grad,
                                        size_t bias_grad_offset, size_t groups, const long long* group_offsets,
                                        size_t bias_grad_ld, void* stream, int async) {
  return guarded([&]() -> int {
    int st = check_types(dtype, dtype, true);
    if (st != kSuccess) return st;
    if (!valid_activation(activation)) return kUnexpectedError;
    if (groups > static_cast<size_t>(kFusedMaxGroups) || (groups == 0) != (group_offsets == nullptr)) return kInvalidBatchCount;
    if (rows == 0 || n == 0 || !extents_ok(rows, n, 0)) return kInvalidDimension;
    if (groups && (rows + kPointwiseChunk - 1) / kPointwiseChunk + groups > 65535) return kInvalidDimension;
    if (!dz && !bias_grad) return kInvalidMatrixC;
    const int elem = elem_of(dtype);
    const bool has_z = activation != kActIdentityCode;
    if ((st = check_a(n, rows, 1, dy, dy_offset, dy_ld, 0, elem))) return st;
    if (has_z && (st = check_b(n, rows, 1, z, z_offset, z_ld, 0, elem))) return st;
    if (dz && (st = check_c(n, rows, 1, dz, dz_offset, dz_ld, 0, elem))) return st;
    const size_t lines = groups ? groups : 1, line_ld = groups ? bias_grad_ld : n;
    if (bias_grad && (st = check(n, lines, 1, bias_grad, bias_grad_offset, line_ld, 0, elem, kInvalidVectorY, kInsufficientMemoryY, kInvalidVectorY))) return st;
    if (groups && (st = check_offsets(group_offsets, groups))) return st;
    dy = at(dy, dy_offset, elem); z = has_z ? at(z, z_offset, elem) : nullptr;
    dz = at(dz, dz_offset, elem); bias_grad = at(bias_grad, bias_grad_offset, elem);
    const Area at_dy = {dy, n, rows, dy_ld, elem}, at_z = {z, n, rows, z_ld, elem}, at_dz = {dz, n, rows, dz_ld, elem};
    if (!beside(at_dy, at_dz, true) || !beside(at_z, at_dz, true)) return kInvalidMatrixC;
    const Span sums = span_of(bias_grad, n, lines, line_ld, elem), offsets = offsets_span(group_offsets, groups);
    if (overlap(offsets, at_dz.span())) return kInvalidMatrixC;
    for (const Area& in : {at_dy, at_z, at_dz})
      if (overlap(in.span(), sums)) return kInvalidVectorY;
    if (overlap(offsets, sums)) return kInvalidVectorY;
    cudaStream_t s;
    const int r = begin_call(stream, async, &s);
    if (r != 0) return r;
    PointwiseJob job = {};
    job.type = dtype; job.act = activation; job.grad = 1;
    job.m = static_cast<long long>(n); job.n = static_cast<long long>(rows);
    job.p = dy; job.ldp = static_cast<long long>(dy_ld);
    job.z = const_cast<void*>(z); job.ldz = static_cast<long long>(z_ld);
    job.c = dz; job.ldc = static_cast<long long>(dz_ld);
    job.offsets = group_offsets; job.groups = groups ? static_cast<int>(groups) : 1;
    PoolScratch partial;
    cudaError_t e = cudaSuccess;
    if (bias_grad) {
      e = partial.get(static_cast<size_t>(pointwise_chunks(job)) * n * 4, s);
      job.partial = reinterpret_cast<float*>(partial.ptr());
    }
    if (e == cudaSuccess) e = launch_pointwise(job, s);
    if (e == cudaSuccess && bias_grad) {
      SumJob sum = {};
      sum.partial = job.partial; sum.m = job.m; sum.type = dtype; sum.out = bias_grad;
      sum.out_stride = static_cast<long long>(line_ld); sum.offsets = group_offsets; sum.groups = job.groups;
      sum.bound = job.n; sum.per_tile = kPointwiseChunk; sum.lines_per_tile = 1; sum.tiles = pointwise_chunks(job);
      e = launch_sum_partials(sum, s);
    }
    return finish(s, async, e, "activation_grad");
  });
}

namespace {

// Extents of W_g as stored.
size_t w_one(int w_transpose, size_t n, size_t k) { return w_transpose == kNo ? n : k; }
size_t w_two(int w_transpose, size_t n, size_t k) { return w_transpose == kNo ? k : n; }

// The grouped products share everything but the epilogue.
struct GroupedCall {
  int dtype, c_dtype, w_transpose;
  size_t groups, rows, n, k;
  double alpha;
  const void* x; size_t x_offset, x_ld;
  const void* w; size_t w_offset, w_ld, w_stride;
  const long long* offsets;
};

int check_grouped(const GroupedCall& g) {
  if (g.groups < 1 || g.groups > static_cast<size_t>(kFusedMaxGroups)) return kInvalidBatchCount;
  if (g.rows == 0 || g.n == 0 || g.k == 0 || !extents_ok(g.rows, g.n, g.k)) return kInvalidDimension;
  const int elem = elem_of(g.dtype);
  int st = check_a(g.k, g.rows, 1, g.x, g.x_offset, g.x_ld, 0, elem);
  if (st) return st;
  // W_g: k x n (kNo) or n x k, rows contiguous
  return check_b(w_one(g.w_transpose, g.n, g.k), w_two(g.w_transpose, g.n, g.k), g.groups, g.w, g.w_offset, g.w_ld, g.w_stride, elem);
}

// The weights of all groups as one stretch of memory.
Span weights_span(const GroupedCall& g) {
  const int elem = elem_of(g.dtype);
  const size_t one = w_one(g.w_transpose, g.n, g.k), two = w_two(g.w_transpose, g.n, g.k);
  Span s = span_of(at(g.w, g.w_offset, elem), one, two, g.w_ld, elem);
  s.last += (g.groups - 1) * g.w_stride * elem;
  return s;
}

FusedDesc grouped_desc(const GroupedCall& g) {
  const int elem = elem_of(g.dtype);
  FusedDesc f = {};
  f.type = g.dtype; f.c_type = f.d_type = g.c_dtype; f.kind = kFusedRaggedCols;
  f.problems = static_cast<long long>(g.groups); f.offsets = g.offsets;
  f.m = static_cast<long long>(g.n); f.n = static_cast<long long>(g.rows); f.k = static_cast<long long>(g.k);
  f.a = at(g.w, g.w_offset, elem); f.lda = static_cast<long long>(g.w_ld); f.a_stride = static_cast<long long>(g.w_stride);
  f.a_mn = g.w_transpose == kNo;
  f.b = at(g.x, g.x_offset, elem); f.ldb = static_cast<long long>(g.x_ld); f.b_mn = 0;
  f.alpha = g.alpha;
  return f;
}

}  // namespace

extern "C" int b200blas_gemm_grouped(int dtype, int c_dtype, int w_transpose, size_t groups, size_t rows, size_t n,
                                     size_t k, double alpha, const void* x, size_t x_offset, size_t x_ld, const void* w,
                                     size_t w_offset, size_t w_ld, size_t w_stride, const long long* group_offsets,
                                     const void* bias, size_t bias_offset, size_t bias_ld, int activation, void* z,
                                     size_t z_offset, size_t z_ld, double beta, const void* d, size_t d_offset,
                                     size_t d_ld, void* c, size_t c_offset, size_t c_ld, void* stream, int async) {
  return guarded([&]() -> int {
    int st = check_types(dtype, c_dtype, false);
    if (st != kSuccess) return st;
    if (!valid_transpose(w_transpose) || !valid_activation(activation)) return kUnexpectedError;
    const GroupedCall g = {dtype, c_dtype, w_transpose, groups, rows, n, k, alpha, x, x_offset, x_ld, w, w_offset, w_ld, w_stride, group_offsets};
    if ((st = check_grouped(g))) return st;
    const int elem = elem_of(dtype), c_elem = elem_of(c_dtype);
    if (bias && (st = check(n, groups, 1, bias, bias_offset, bias_ld, 0, elem, kInvalidVectorX, kInsufficientMemoryX, kInvalidVectorX))) return st;
    const bool has_d = beta != 0.0;
    if (z && (st = check_c(n, rows, 1, z, z_offset, z_ld, 0, elem))) return st;
    if (has_d && (st = check_c(n, rows, 1, d, d_offset, d_ld, 0, c_elem))) return st;
    if ((st = check_c(n, rows, 1, c, c_offset, c_ld, 0, c_elem))) return st;
    if ((st = check_offsets(group_offsets, groups))) return st;
    FusedDesc f = grouped_desc(g);
    f.beta = beta; f.act = activation;
    f.bias = at(bias, bias_offset, elem); f.bias_stride = static_cast<long long>(bias_ld);
    f.z = at(z, z_offset, elem); f.ldz = static_cast<long long>(z_ld);
    f.d = has_d ? at(d, d_offset, c_elem) : nullptr; f.ldd = static_cast<long long>(d_ld);
    f.c = at(c, c_offset, c_elem); f.ldc = static_cast<long long>(c_ld);
    const Area at_c = {f.c, n, rows, c_ld, c_elem}, at_d = {f.d, n, rows, d_ld, c_elem}, at_z = {f.z, n, rows, z_ld, elem};
    const Area at_x = {f.b, k, rows, x_ld, elem};
    for (const Area& out : {at_c, at_z})
      if (!beside(at_x, out, false) || overlap(weights_span(g), out.span()) ||
          overlap(span_of(f.bias, n, groups, bias_ld, elem), out.span()) || overlap(offsets_span(group_offsets, groups), out.span()))
        return kInvalidMatrixC;
    if (!beside(at_z, at_c, false) || !beside(at_d, at_c, true) || !beside(at_d, at_z, false)) return kInvalidMatrixC;
    cudaStream_t s;
    const int r = begin_call(stream, async, &s);
    if (r != 0) return r;
    const char* name = "none";
    const cudaError_t e = launch_fused(f, s, &name);
    return finish(s, async, e, name);
  });
}

extern "C" int b200blas_gemm_grouped_grad(int dtype, int w_transpose, size_t groups, size_t rows, size_t n, size_t k,
                                          double alpha, const void* x, size_t x_offset, size_t x_ld, const void* w,
                                          size_t w_offset, size_t w_ld, size_t w_stride, const long long* group_offsets,
                                          double beta, const void* d, size_t d_offset, size_t d_ld, int activation,
                                          const void* z, size_t z_offset, size_t z_ld, void* c, size_t c_offset,
                                          size_t c_ld, void* bias_grad, size_t bias_grad_offset, size_t bias_grad_ld,
                                          void* stream, int async) {
  return guarded([&]() -> int {
    int st = check_types(dtype, dtype, false);
    if (st != kSuccess) return st;
    if (!valid_transpose(w_transpose) || !valid_activation(activation)) return kUnexpectedError;
    const GroupedCall g = {dtype, dtype, w_transpose, groups, rows, n, k, alpha, x, x_offset, x_ld, w, w_offset, w_ld, w_stride, group_offsets};
    if ((st = check_grouped(g))) return st;
    const int elem = elem_of(dtype);
    const bool has_d = beta != 0.0, has_z = activation != kActIdentityCode;
    if (has_d && (st = check_c(n, rows, 1, d, d_offset, d_ld, 0, elem))) return st;
    if (has_z && (st = check_c(n, rows, 1, z, z_offset, z_ld, 0, elem))) return st;
    if ((st = check_c(n, rows, 1, c, c_offset, c_ld, 0, elem))) return st;
    if (bias_grad && (st = check(n, groups, 1, bias_grad, bias_grad_offset, bias_grad_ld, 0, elem, kInvalidVectorY, kInsufficientMemoryY, kInvalidVectorY))) return st;
    if ((st = check_offsets(group_offsets, groups))) return st;
    FusedDesc f = grouped_desc(g);
    f.grad = 1; f.beta = beta; f.act = activation;
    f.z = has_z ? const_cast<void*>(at(z, z_offset, elem)) : nullptr; f.ldz = static_cast<long long>(z_ld);
    f.d = has_d ? at(d, d_offset, elem) : nullptr; f.ldd = static_cast<long long>(d_ld);
    f.c = at(c, c_offset, elem); f.ldc = static_cast<long long>(c_ld);
    f.bias_grad = at(bias_grad, bias_grad_offset, elem); f.bias_grad_stride = static_cast<long long>(bias_grad_ld);
    const Area at_c = {f.c, n, rows, c_ld, elem}, at_d = {f.d, n, rows, d_ld, elem}, at_z = {f.z, n, rows, z_ld, elem};
    const Area at_x = {f.b, k, rows, x_ld, elem};
    const Span offsets = offsets_span(group_offsets, groups);
    if (!beside(at_x, at_c, false) || overlap(weights_span(g), at_c.span()) || !beside(at_z, at_c, true) || !beside(at_d, at_c, true) ||
        overlap(offsets, at_c.span()))
      return kInvalidMatrixC;
    const Span sums = span_of(f.bias_grad, n, groups, bias_grad_ld, elem);
    for (const Area& in : {at_x, at_c, at_d, at_z})
      if (overlap(in.span(), sums)) return kInvalidVectorY;
    if (overlap(weights_span(g), sums) || overlap(offsets, sums)) return kInvalidVectorY;
    cudaStream_t s;
    const int r = begin_call(stream, async, &s);
    if (r != 0) return r;
    const char* name = "none";
    const cudaError_t e = launch_fused(f, s, &name);
    return finish(s, async, e, name);
  });
}

extern "C" int b200blas_gemm_grouped_weight(int dtype, int c_dtype, size_t groups, size_t rows, size_t m, size_t n,
                                            double alpha, const void* x, size_t x_offset, size_t x_ld, const void* y,
                                            size_t y_offset, size_t y_ld, const long long* group_offsets, double beta,
                                            void* c, size_t c_offset, size_t c_ld, size_t c_stride, void* stream,
                                            int async) {
  return guarded([&]() -> int {
    int st = check_types(dtype, c_dtype, false);
    if (st != kSuccess) return st;
    if (groups < 1 || groups > static_cast<size_t>(kFusedMaxGroups)) return kInvalidBatchCount;
    if (rows == 0 || m == 0 || n == 0 || !extents_ok(rows, m, n)) return kInvalidDimension;
    const int elem = elem_of(dtype), c_elem = elem_of(c_dtype);
    if ((st = check_a(m, rows, 1, x, x_offset, x_ld, 0, elem))) return st;
    if ((st = check_b(n, rows, 1, y, y_offset, y_ld, 0, elem))) return st;
    if ((st = check_c(n, m, groups, c, c_offset, c_ld, c_stride, c_elem))) return st;
    // the groups' results must not meet
    if (groups > 1 && c_stride < c_ld * (m - 1) + n) return kInvalidDimension;
    if ((st = check_offsets(group_offsets, groups))) return st;
    Span all = span_of(at(c, c_offset, c_elem), n, m, c_ld, c_elem);
    all.last += (groups - 1) * c_stride * c_elem;
    if (overlap(span_of(at(x, x_offset, elem), m, rows, x_ld, elem), all) || overlap(span_of(at(y, y_offset, elem), n, rows, y_ld, elem), all) ||
        overlap(offsets_span(group_offsets, groups), all))
      return kInvalidMatrixC;
    cudaStream_t s;
    const int r = begin_call(stream, async, &s);
    if (r != 0) return r;
    FusedDesc f = {};
    f.type = dtype; f.c_type = f.d_type = c_dtype; f.kind = kFusedRaggedInner;
    f.problems = static_cast<long long>(groups); f.offsets = group_offsets;
    f.m = static_cast<long long>(n); f.n = static_cast<long long>(m); f.k = static_cast<long long>(rows);
    f.a = at(y, y_offset, elem); f.lda = static_cast<long long>(y_ld); f.a_mn = 1;
    f.b = at(x, x_offset, elem); f.ldb = static_cast<long long>(x_ld); f.b_mn = 1;
    f.alpha = alpha; f.beta = beta; f.act = kActIdentityCode;
    f.c = at(c, c_offset, c_elem); f.ldc = static_cast<long long>(c_ld); f.c_stride = static_cast<long long>(c_stride);
    f.d = f.c; f.ldd = f.ldc; f.d_stride = f.c_stride;
    const char* name = "none";
    const cudaError_t e = launch_fused(f, s, &name);
    return finish(s, async, e, name);
  });
}

namespace {

// Largest singular value of a normalised matrix, with a margin for rounding.
constexpr double kNormalisedBound = 1.02;
// Largest singular value that a step can leave, given the largest before it: |a x + b x^3 + c x^5| on [0, s] is largest at s
// or where the slope a + 3 b t + 5 c t^2, t = x^2, is zero. With a margin for rounding.
double step_bound(double s, const double* q) {
  const auto size = [&](double t) { return std::fabs(std::sqrt(t) * (q[0] + t * (q[1] + t * q[2]))); };
  double most = size(s * s);
  const auto candidate = [&](double t) {
    if (t > 0.0 && t < s * s) most = std::fmax(most, size(t));
  };
  const double disc = 9.0 * q[1] * q[1] - 20.0 * q[0] * q[2];
  if (disc >= 0.0) {
    // both roots without cancellation
    const double h = -0.5 * (3.0 * q[1] + std::copysign(std::sqrt(disc), q[1]));
    if (q[2] != 0.0) candidate(h / (5.0 * q[2]));
    if (h != 0.0) candidate(q[0] / h);
  }
  return 1.02 * most;
}
// The power of two that brings a matrix with entries up to `bound` under 2^15, half of half precision's largest number.
double parts_scale(double bound) {
  if (!(bound > 0.0) || !std::isfinite(bound)) return 1.0;
  int e = 0;
  std::frexp(bound, &e);  // bound < 2^e
  e = 15 - e;
  return std::ldexp(1.0, e > 13 ? 13 : e);
}

// Whether halves hold the iteration whatever its matrix: beyond these bounds scales that keep the largest possible values
// finite would push those of most matrices into half's subnormal range.
bool bounded(const double* coefficients, bool per_step, int steps) {
  double bound = kNormalisedBound;
  for (int i = 0; i < steps; ++i) {
    const double* const q = coefficients + (per_step ? 3 * i : 0);
    const double bracket = std::fabs(q[1]) * bound * bound + std::fabs(q[2]) * bound * bound * bound * bound;
    bound = step_bound(bound, q);
    if (!(bracket < 4096.0) || !(bound < 64.0)) return false;
  }
  return true;
}

// X <- a X + (b A + c A A) X with A = X X^T (or X^T X on the shorter side) on 16-bit tensor cores. X, A and the bracket
// are kept in half precision between products whatever the caller's 16-bit type: their entries are bounded by what the
// polynomial makes of the singular values, so half's 11 bits apply (bfloat16 has 8), each matrix scaled by a power of two
// that brings the bound under 2^15 and keeps the entries of large matrices out of half's subnormal range. Sums run in
// fp32 throughout.
cudaError_t newton_schulz_half(long long one, long long two, double alpha, const void* a, long long a_ld, long long a_stride,
                               void* b, long long b_ld, long long b_stride, long long batch, int steps,
                               const double* coefficients, bool per_step, double eps, cudaStream_t s, int dtype,
                               const char** name) {
  const bool gram_of_lines = one > two;  // the shorter side is the number of lines
  // extents inside are multiples of 8, the rest zero: the symmetric products store 16 bytes at a time
  const long long pitch = (one + 7) / 8 * 8, lines = (two + 7) / 8 * 8;
  const long long side = gram_of_lines ? lines : pitch, gram_pitch = side;
  const auto round = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t x_bytes = round(static_cast<size_t>(batch) * lines * pitch * 2);
  const size_t g_bytes = round(static_cast<size_t>(batch) * side * gram_pitch * 2);
  const size_t s_bytes = round(static_cast<size_t>(batch) * kNormBlocks * sizeof(double));
  PoolScratch scratch;
  cudaError_t e = scratch.get(2 * x_bytes + 2 * g_bytes + s_bytes, s);
  if (e != cudaSuccess) return e;
  unsigned char* const base = scratch.ptr();
  void* x[2] = {base, base + x_bytes};
  void* const gram = base + 2 * x_bytes;
  void* const poly = base + 2 * x_bytes + g_bytes;
  double bound = kNormalisedBound, x_scale = parts_scale(bound);
  NormaliseJob norm = {};
  norm.type = dtype; norm.x_type = 16; norm.g = a; norm.one = one; norm.two = two; norm.ld = a_ld; norm.stride = a_stride;
  norm.batch = batch; norm.x = x[0]; norm.pitch = pitch; norm.lines = lines; norm.eps = eps; norm.scale = x_scale;
  norm.sums = reinterpret_cast<double*>(base + 2 * x_bytes + 2 * g_bytes);
  e = launch_normalise(norm, s);
  for (int i = 0; i < steps && e == cudaSuccess; ++i) {
    const double* const q = coefficients + (per_step ? 3 * i : 0);
    const double bracket = std::fabs(q[1]) * bound * bound + std::fabs(q[2]) * bound * bound * bound * bound;
    const double g_scale = parts_scale(bound * bound), p_scale = parts_scale(bracket);
    bound = step_bound(bound, q);
    const bool last = i == steps - 1;
    const void* const from = x[i & 1];
    FusedDesc f = {};
    f.type = f.c_type = f.d_type = 16;
    f.kind = kFusedPlain; f.problems = batch; f.act = kActIdentityCode; f.chained = 1;
    // A = X X^T
    f.m = f.n = side; f.k = gram_of_lines ? pitch : lines;
    f.a = f.b = from; f.lda = f.ldb = pitch; f.a_stride = f.b_stride = lines * pitch;
    f.a_mn = f.b_mn = gram_of_lines ? 0 : 1;
    f.alpha = g_scale / (x_scale * x_scale); f.tri = 1;
    f.c = gram; f.ldc = gram_pitch; f.c_stride = side * gram_pitch;
    e = launch_fused(f, s, name);
    if (e != cudaSuccess) break;
    // b A + c A A
    f.k = side;
    f.a = f.b = gram; f.lda = f.ldb = gram_pitch; f.a_stride = f.b_stride = side * gram_pitch;
    f.a_mn = f.b_mn = 0;
    f.alpha = p_scale * q[2] / (g_scale * g_scale); f.beta = p_scale * q[1] / g_scale; f.d = gram; f.ldd = gram_pitch; f.d_stride = side * gram_pitch;
    f.c = poly;
    e = launch_fused(f, s, name);
    if (e != cudaSuccess) break;
    // a X + (.) X, on the last step straight into the caller's matrix
    const double out = last ? alpha : parts_scale(bound);
    f.tri = 0;
    f.m = last ? one : pitch; f.n = last ? two : lines; f.k = side;
    if (gram_of_lines) {
      f.a = from; f.lda = pitch; f.a_stride = lines * pitch; f.a_mn = 1;
      f.b = poly; f.ldb = gram_pitch; f.b_stride = side * gram_pitch; f.b_mn = 0;
    } else {
      f.a = poly; f.lda = gram_pitch; f.a_stride = side * gram_pitch; f.a_mn = 0;
      f.b = from; f.ldb = pitch; f.b_stride = lines * pitch; f.b_mn = 0;
    }
    f.alpha = out / (p_scale * x_scale); f.beta = out * q[0] / x_scale; f.d = from; f.ldd = pitch; f.d_stride = lines * pitch;
    if (last) {
      f.c_type = dtype; f.c = b; f.ldc = b_ld; f.c_stride = b_stride;
    } else {
      f.c = x[(i + 1) & 1]; f.ldc = pitch; f.c_stride = lines * pitch;
    }
    e = launch_fused(f, s, name);
    x_scale = out;
  }
  return e;
}

// The same iteration in single precision: every matrix is kept as a sum of two halves, hi + lo, about 22 bits, scaled by
// powers of two so that neither part leaves half's range, and a product takes three terms on the 16-bit tensor cores
// (three times their time, where the single-precision kernels take six). Sums run in fp32 as for every result in single
// precision. Returns cudaErrorNotSupported when the coefficients let the iteration grow beyond the scales' reach.
cudaError_t newton_schulz_parts(long long one, long long two, double alpha, const void* a, long long a_ld, long long a_stride,
                                void* b, long long b_ld, long long b_stride, long long batch, int steps,
                                const double* coefficients, bool per_step, double eps, cudaStream_t s) {
  const bool gram_of_lines = one > two;
  const long long pitch = (one + 7) / 8 * 8, lines = (two + 7) / 8 * 8;
  const long long side = gram_of_lines ? lines : pitch;
  const long long x_plane = lines * pitch, g_plane = side * side;
  const auto round = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t x_bytes = round(static_cast<size_t>(batch) * x_plane * 4), g_bytes = round(static_cast<size_t>(batch) * g_plane * 4);
  const size_t s_bytes = round(static_cast<size_t>(batch) * kNormBlocks * sizeof(double));
  PoolScratch scratch;
  cudaError_t e = scratch.get(2 * x_bytes + 2 * g_bytes + s_bytes, s);
  if (e != cudaSuccess) return e;
  unsigned char* const base = scratch.ptr();
  void* x[2] = {base, base + x_bytes};
  void* const gram = base + 2 * x_bytes;
  void* const poly = base + 2 * x_bytes + g_bytes;
  double bound = kNormalisedBound, x_scale = parts_scale(bound);
  NormaliseJob norm = {};
  norm.type = 32; norm.x_type = kParts; norm.g = a; norm.one = one; norm.two = two; norm.ld = a_ld; norm.stride = a_stride;
  norm.batch = batch; norm.x = x[0]; norm.pitch = pitch; norm.lines = lines; norm.eps = eps; norm.scale = x_scale;
  norm.sums = reinterpret_cast<double*>(base + 2 * x_bytes + 2 * g_bytes);
  e = launch_normalise(norm, s);
  const char* name = "none";
  for (int i = 0; i < steps && e == cudaSuccess; ++i) {
    const double* const q = coefficients + (per_step ? 3 * i : 0);
    const double g_scale = parts_scale(bound * bound);
    const double p_scale = parts_scale(std::fabs(q[1]) * bound * bound + std::fabs(q[2]) * bound * bound * bound * bound);
    bound = step_bound(bound, q);
    const double next_scale = parts_scale(bound);
    const void* const from = x[i & 1];
    FusedDesc f = {};
    f.type = f.c_type = f.d_type = 16;
    f.kind = kFusedPlain; f.problems = batch; f.act = kActIdentityCode; f.parts = 1; f.chained = 1;
    // G = X X^T
    f.m = f.n = side; f.k = gram_of_lines ? pitch : lines;
    f.a = f.b = from; f.lda = f.ldb = pitch; f.a_stride = f.b_stride = x_plane;
    f.a_mn = f.b_mn = gram_of_lines ? 0 : 1;
    f.alpha = g_scale / (x_scale * x_scale); f.tri = 1;
    f.c = gram; f.ldc = side; f.c_stride = g_plane;
    e = launch_fused(f, s, &name);
    if (e != cudaSuccess) break;
    // b G + c G G
    f.k = side;
    f.a = f.b = gram; f.lda = f.ldb = side; f.a_stride = f.b_stride = g_plane;
    f.a_mn = f.b_mn = 0;
    f.alpha = p_scale * q[2] / (g_scale * g_scale);
    f.beta = p_scale * q[1] / g_scale; f.d = gram; f.ldd = side; f.d_stride = g_plane;
    f.c = poly;
    e = launch_fused(f, s, &name);
    if (e != cudaSuccess) break;
    // a X + (.) X
    f.tri = 0;
    f.m = pitch; f.n = lines; f.k = side;
    if (gram_of_lines) {
      f.a = from; f.lda = pitch; f.a_stride = x_plane; f.a_mn = 1;
      f.b = poly; f.ldb = side; f.b_stride = g_plane; f.b_mn = 0;
    } else {
      f.a = poly; f.lda = side; f.a_stride = g_plane; f.a_mn = 0;
      f.b = from; f.ldb = pitch; f.b_stride = x_plane; f.b_mn = 0;
    }
    f.alpha = next_scale / (p_scale * x_scale);
    f.beta = next_scale * q[0] / x_scale; f.d = from; f.ldd = pitch; f.d_stride = x_plane;
    f.c = x[(i + 1) & 1]; f.ldc = pitch; f.c_stride = x_plane;
    e = launch_fused(f, s, &name);
    x_scale = next_scale;
  }
  if (e != cudaSuccess) return e;
  JoinJob join = {};
  join.type = 32; join.x_type = kParts; join.x = x[steps & 1]; join.lines = lines; join.pitch = pitch;
  join.b = b; join.one = one; join.two = two; join.ld = b_ld; join.stride = b_stride; join.batch = batch;
  join.scale = static_cast<float>(alpha / x_scale);
  return launch_join(join, s);
}

// The same on the SGEMM kernels, for coefficients whose values halves might not hold; a product that adds to another
// matrix adds to a copy of it.
cudaError_t newton_schulz_single(long long one, long long two, double alpha, const void* a, long long a_ld,
                                 long long a_stride, void* b, long long b_ld, long long b_stride, long long batch, int steps,
                                 const double* coefficients, bool per_step, double eps, cudaStream_t s, int dtype) {
  const bool gram_of_lines = one > two;
  const long long side = gram_of_lines ? two : one;
  const long long pitch = (one + 3) / 4 * 4, gram_pitch = (side + 3) / 4 * 4;
  const auto round = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t x_bytes = round(static_cast<size_t>(batch) * two * pitch * 4);
  const size_t g_bytes = round(static_cast<size_t>(batch) * side * gram_pitch * 4);
  const size_t s_bytes = round(static_cast<size_t>(batch) * kNormBlocks * sizeof(double));
  PoolScratch scratch;
  cudaError_t e = scratch.get(2 * x_bytes + 2 * g_bytes + s_bytes, s);
  if (e != cudaSuccess) return e;
  unsigned char* const base = scratch.ptr();
  void* x[2] = {base, base + x_bytes};
  void* const gram = base + 2 * x_bytes;
  void* const poly = base + 2 * x_bytes + g_bytes;
  NormaliseJob norm = {};
  norm.type = dtype; norm.x_type = 32; norm.g = a; norm.one = one; norm.two = two; norm.ld = a_ld; norm.stride = a_stride;
  norm.batch = batch; norm.x = x[0]; norm.pitch = pitch; norm.lines = two; norm.eps = eps; norm.scale = 1.0;
  norm.sums = reinterpret_cast<double*>(base + 2 * x_bytes + 2 * g_bytes);
  e = launch_normalise(norm, s);
  for (int i = 0; i < steps && e == cudaSuccess; ++i) {
    const double* const q = coefficients + (per_step ? 3 * i : 0);
    void* const from = x[i & 1];
    GemmDesc g = {};
    g.dtype = 32; g.batch = batch;
    g.m = g.n = side; g.k = gram_of_lines ? one : two;
    g.a = g.b = from; g.lda = g.ldb = pitch; g.a_stride = g.b_stride = two * pitch;
    g.a_kcontig = g.b_kcontig = gram_of_lines ? 1 : 0;
    g.alpha[0] = 1.0;
    g.c = gram; g.ldc = gram_pitch; g.c_stride = side * gram_pitch;
    e = dispatch(g, s);
    if (e == cudaSuccess) e = cudaMemcpyAsync(poly, gram, static_cast<size_t>(batch) * side * gram_pitch * 4, cudaMemcpyDeviceToDevice, s);
    if (e != cudaSuccess) break;
    g.k = side;
    g.a = g.b = gram; g.lda = g.ldb = gram_pitch; g.a_stride = g.b_stride = side * gram_pitch;
    g.a_kcontig = g.b_kcontig = 1;
    g.alpha[0] = q[2]; g.beta[0] = q[1];
    g.c = poly;
    e = dispatch(g, s);
    if (e != cudaSuccess) break;
    g.m = one; g.n = two; g.k = side;
    if (gram_of_lines) {
      g.a = from; g.lda = pitch; g.a_stride = two * pitch; g.a_kcontig = 0;
      g.b = poly; g.ldb = gram_pitch; g.b_stride = side * gram_pitch; g.b_kcontig = 1;
    } else {
      g.a = poly; g.lda = gram_pitch; g.a_stride = side * gram_pitch; g.a_kcontig = 1;
      g.b = from; g.ldb = pitch; g.b_stride = two * pitch; g.b_kcontig = 1;
    }
    g.alpha[0] = 1.0; g.beta[0] = q[0];
    g.c = x[(i + 1) & 1]; g.ldc = pitch; g.c_stride = two * pitch;
    e = cudaMemcpyAsync(g.c, from, static_cast<size_t>(batch) * two * pitch * 4, cudaMemcpyDeviceToDevice, s);
    if (e == cudaSuccess) e = dispatch(g, s);
  }
  if (e != cudaSuccess) return e;
  JoinJob join = {};
  join.type = dtype; join.x_type = 32; join.x = x[steps & 1]; join.lines = two; join.pitch = pitch;
  join.b = b; join.one = one; join.two = two; join.ld = b_ld; join.stride = b_stride; join.batch = batch;
  join.scale = static_cast<float>(alpha);
  return launch_join(join, s);
}

}  // namespace

extern "C" int b200blas_newton_schulz(int dtype, int layout, size_t m, size_t n, double alpha, const void* a,
                                      size_t a_offset, size_t a_ld, size_t a_stride, void* b, size_t b_offset, size_t b_ld,
                                      size_t b_stride, size_t batch_count, size_t steps, const double* coefficients,
                                      size_t coefficient_count, double epsilon, void* stream, int async) {
  return guarded([&]() -> int {
    int st = check_types(dtype, dtype, true);
    if (st != kSuccess) return st;
    if ((layout != kRowMajor && layout != kColMajor) || !coefficients) return kUnexpectedError;
    if (batch_count < 1 || batch_count > 65535) return kInvalidBatchCount;
    if (m == 0 || n == 0 || !extents_ok(m, n, 0)) return kInvalidDimension;
    if (steps < 1 || steps > 1000 || (coefficient_count != 1 && coefficient_count < steps) || !(epsilon >= 0.0)) return kInvalidDimension;
    const bool per_step = coefficient_count > 1;
    const bool halves = bounded(coefficients, per_step, static_cast<int>(steps));
    const int elem = elem_of(dtype);
    const size_t one = layout == kRowMajor ? n : m, two = layout == kRowMajor ? m : n;
    if ((st = check_a(one, two, batch_count, a, a_offset, a_ld, a_stride, elem))) return st;
    if ((st = check_b(one, two, batch_count, b, b_offset, b_ld, b_stride, elem))) return st;
    if (batch_count > 1 && b_stride < b_ld * (two - 1) + one) return kInvalidDimension;
    cudaStream_t s;
    const int r = begin_call(stream, async, &s);
    if (r != 0) return r;
    const char* name = halves ? (dtype == 32 ? "newton_schulz_parts" : "none") : "newton_schulz_single";
    const auto run = [&](auto* f, auto... more) {
      return f(static_cast<long long>(one), static_cast<long long>(two), alpha, at(a, a_offset, elem), static_cast<long long>(a_ld),
               static_cast<long long>(a_stride), at(b, b_offset, elem), static_cast<long long>(b_ld),
               static_cast<long long>(b_stride), static_cast<long long>(batch_count), static_cast<int>(steps), coefficients, per_step,
               epsilon, s, more...);
    };
    const cudaError_t e = !halves       ? run(&newton_schulz_single, dtype)
                          : dtype == 32 ? run(&newton_schulz_parts)
                                        : run(&newton_schulz_half, dtype, &name);
    return finish(s, async, e, name);
  });
}

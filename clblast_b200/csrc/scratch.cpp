#include "scratch.h"

#include <mutex>

#include "runtime_state.h"

namespace b200 {

namespace {

std::mutex g_mutex;
cudaMemPool_t g_pools[kMaxDevices] = {};

cudaError_t pool_of_device(cudaMemPool_t* out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(g_mutex);
  if (g_pools[dev] == nullptr) {
    cudaMemPoolProps props = {};
    props.allocType = cudaMemAllocationTypePinned;
    props.handleTypes = cudaMemHandleTypeNone;
    props.location.type = cudaMemLocationTypeDevice;
    props.location.id = dev;
    cudaMemPool_t pool = nullptr;
    e = cudaMemPoolCreate(&pool, &props);
    if (e != cudaSuccess) return e;
    unsigned long long kept = kScratchKept;
    e = cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &kept);
    if (e != cudaSuccess) {
      cudaMemPoolDestroy(pool);
      return e;
    }
    g_pools[dev] = pool;
  }
  *out = g_pools[dev];
  return cudaSuccess;
}

}  // namespace

cudaError_t PoolScratch::get(size_t bytes, cudaStream_t stream) {
  cudaMemPool_t pool = nullptr;
  const cudaError_t e = pool_of_device(&pool);
  if (e != cudaSuccess) return e;
  stream_ = stream;
  return cudaMallocFromPoolAsync(&ptr_, bytes, pool, stream);
}

PoolScratch::~PoolScratch() {
  if (ptr_) cudaFreeAsync(ptr_, stream_);
}

void scratch_trim() {
  std::lock_guard<std::mutex> lock(g_mutex);
  for (cudaMemPool_t pool : g_pools)
    if (pool) cudaMemPoolTrimTo(pool, 0);
}

}  // namespace b200

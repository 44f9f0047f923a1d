// Stream-ordered scratch of the fused routines, from a memory pool of the library's own.
#pragma once

#include <cuda_runtime_api.h>

#include <cstddef>

namespace b200 {

// Scratch that is released, in stream order, when the scope ends. The default pool gives its memory back at every
// synchronisation, after which an allocation costs more than a small product; this one keeps up to kScratchKept bytes
// per device until ClearCache. A captured call gets allocation nodes of its graph instead, so graphs share nothing.
constexpr unsigned long long kScratchKept = 1ull << 30;

class PoolScratch {
 public:
  PoolScratch() = default;
  PoolScratch(const PoolScratch&) = delete;
  PoolScratch& operator=(const PoolScratch&) = delete;
  ~PoolScratch();
  cudaError_t get(size_t bytes, cudaStream_t stream);
  unsigned char* ptr() const { return static_cast<unsigned char*>(ptr_); }

 private:
  void* ptr_ = nullptr;
  cudaStream_t stream_ = nullptr;
};

// Gives the kept memory of all devices back (what is in use stays).
void scratch_trim();

}  // namespace b200

// csrc/runtime_state.cpp over a runtime that keeps one kernel's shared-memory attribute, for two threads whose first calls
// meet. Prints the attribute after each part.
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>

#include "driver_api.h"
#include "runtime_state.h"

namespace {

std::atomic<int> g_attribute{0};  // what the kernel may have at its launches
std::atomic<int> g_inside{0};     // calls that have reached the runtime
std::atomic<bool> g_meet{false};

CUresult current(CUcontext* c) { *c = reinterpret_cast<CUcontext>(16); return CUDA_SUCCESS; }
CUresult context_id(CUcontext, unsigned long long* id) { *id = 1; return CUDA_SUCCESS; }

}  // namespace

namespace b200 {
const DriverApi& driver_api() {
  static DriverApi api = {};
  api.CtxGetCurrent = current;
  api.CtxGetId = context_id;
  api.ok = true;
  return api;
}
}  // namespace b200

extern "C" {
cudaError_t CUDARTAPI cudaFuncSetAttribute(const void*, cudaFuncAttribute, int value) {
  ++g_inside;
  if (g_meet) {
    // the smaller request is the last to arrive where both can be under way
    const auto end = std::chrono::steady_clock::now() + std::chrono::milliseconds(300);
    while (g_inside < 2 && std::chrono::steady_clock::now() < end) std::this_thread::yield();
    if (value < 200000) std::this_thread::sleep_for(std::chrono::milliseconds(100));
  }
  g_attribute = value;
  return cudaSuccess;
}
cudaError_t CUDARTAPI cudaFuncGetAttributes(cudaFuncAttributes* a, const void*) { *a = {}; a->numRegs = 77; return cudaSuccess; }
cudaError_t CUDARTAPI cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t CUDARTAPI cudaSetDevice(int) { return cudaSuccess; }
cudaError_t CUDARTAPI cudaGetLastError(void) { return cudaSuccess; }
cudaError_t CUDARTAPI cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { *v = 148; return cudaSuccess; }
cudaError_t CUDARTAPI cudaHostRegister(void*, size_t, unsigned) { return cudaSuccess; }
cudaError_t CUDARTAPI cudaHostGetDevicePointer(void** d, void* h, unsigned) { *d = h; return cudaSuccess; }
}

int main() {
  static const char first = 0, second = 0;
  int regs = 0;
  // two first calls at once; then one with the larger size, which the table may answer
  g_meet = true;
  std::thread large([] { b200::kernel_ready(&first, 230000); });
  std::thread small([] { b200::kernel_ready(&first, 100000); });
  large.join();
  small.join();
  g_meet = false;
  b200::kernel_ready(&first, 230000);
  std::printf("%d\n", g_attribute.load());
  // a smaller size that also asks for the registers, which no call before has
  g_attribute = 0;
  b200::kernel_ready(&second, 230000);
  b200::kernel_ready(&second, 100000, &regs);
  b200::kernel_ready(&second, 230000);
  std::printf("%d %d\n", g_attribute.load(), regs);
  return 0;
}

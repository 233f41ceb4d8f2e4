// ody_host.h -- what the C entry points share: error reporting, the checks
// of pointers, and the staging of host buffers by the stateless operations.
// Not part of the public C ABI (include/odyssey_mp.h).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>
#include <vector>

#include "../../include/odyssey_mp.h"
#include "ody_internal.h"

namespace ody {

inline int fail(int code, const std::string& msg) {
  record_error(msg);
  return code;
}

#define ODY_CUDA(call)                                                              \
  do {                                                                              \
    cudaError_t e_ = (call);                                                        \
    if (e_ != cudaSuccess)                                                          \
      return fail(ODY_ERR_CUDA, std::string(#call) + ": " + cudaGetErrorString(e_)); \
  } while (0)

inline size_t dtype_size(int gdt) { return gdt == DT_F32 ? 4 : 2; }

inline int check_dtype(int dt) {
  if (dt < DT_F32 || dt > DT_BF16) return fail(ODY_ERR_DTYPE, "unsupported dtype " + std::to_string(dt));
  return ODY_OK;
}

// Device memory usable by this call's kernels: managed memory, or device
// memory of the calling thread's current GPU.  Another GPU's memory is not
// (without peer access a kernel reading it faults): device_elsewhere() names
// that case so the caller can refuse it before any launch.
inline int device_of(const void* p) {
  if (!p) return -1;
  cudaPointerAttributes a;
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  if (a.type == cudaMemoryTypeManaged) return INT32_MAX;  // reachable from every GPU
  return a.type == cudaMemoryTypeDevice ? a.device : -1;
}

inline bool is_device_ptr(const void* p) {
  const int d = device_of(p);
  if (d < 0) return false;
  if (d == INT32_MAX) return true;
  int cur = 0;
  cudaGetDevice(&cur);
  return d == cur;
}

inline bool device_elsewhere(const void* p) {
  const int d = device_of(p);
  return d >= 0 && d != INT32_MAX && !is_device_ptr(p);
}

struct Staged {
  void* user = nullptr;
  void* dev = nullptr;
  size_t bytes = 0;
  bool owned = false;
};

struct Scope {
  cudaStream_t st = cudaStreamPerThread;
  std::vector<Staged> bufs;
  ~Scope() {
    for (auto& b : bufs)
      if (b.owned && b.dev) cudaFreeAsync(b.dev, st);
  }
  // in: copy host data to device; out-only: allocate
  cudaError_t stage(const void* user, size_t bytes, bool copy_in, void** dev) {
    if (!user) {
      *dev = nullptr;
      return cudaSuccess;
    }
    if (device_elsewhere(user)) return cudaErrorInvalidDevice;
    if (is_device_ptr(user)) {
      *dev = const_cast<void*>(user);
      bufs.push_back({const_cast<void*>(user), *dev, bytes, false});
      return cudaSuccess;
    }
    void* d = nullptr;
    cudaError_t e = cudaMallocAsync(&d, bytes < 16 ? 16 : bytes, st);
    if (e != cudaSuccess) return e;
    if (copy_in) {
      e = cudaMemcpyAsync(d, user, bytes, cudaMemcpyHostToDevice, st);
      if (e != cudaSuccess) return e;
    }
    bufs.push_back({const_cast<void*>(user), d, bytes, true});
    *dev = d;
    return cudaSuccess;
  }
  // Results are staged behind the operands, so of two entries of one address
  // (an operand that is the result too) the later one holds the result.
  cudaError_t copy_out(void* user) {
    for (auto b = bufs.rbegin(); b != bufs.rend(); ++b)
      if (b->user == user && b->owned) return cudaMemcpyAsync(user, b->dev, b->bytes, cudaMemcpyDeviceToHost, st);
    return cudaSuccess;
  }
};

#define ODY_STAGE(S, ptr, bytes, in, dev)                                             \
  do {                                                                                \
    cudaError_t se_ = (S).stage((ptr), (bytes), (in), (void**)(dev));                 \
    if (se_ == cudaErrorInvalidDevice)                                                \
      return fail(ODY_ERR_ARG, "a buffer is device memory of another GPU than the current one"); \
    if (se_ != cudaSuccess)                                                           \
      return fail(ODY_ERR_CUDA, std::string("staging a buffer: ") + cudaGetErrorString(se_)); \
  } while (0)

}  // namespace ody

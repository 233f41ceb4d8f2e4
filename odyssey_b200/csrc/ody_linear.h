// ody_linear.h -- the quantised linear layer's kernels, as the host side sees
// them: products with 4-bit weights, 8-bit activations, the weight gradient.
// Not part of the public C ABI (include/odyssey_mp.h).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace ody {

// Lets a kernel take `bytes` of dynamic shared memory on the current device;
// `set` is the kernel's own.  `bytes` is the most that any launch of it takes:
// with one number per kernel two threads may set it in any order.
constexpr int kMaxDevices = 64;
using PerDevice = std::atomic<bool>[kMaxDevices];
inline cudaError_t allow_shared(PerDevice& set, const void* kernel, int bytes) {
  int dev = 0;
  cudaGetDevice(&dev);
  const bool known = dev >= 0 && dev < kMaxDevices;
  if (known && set[dev].load(std::memory_order_acquire)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && known) set[dev].store(true, std::memory_order_release);
  return e;
}

// C[m, n] = alpha * *tscale * sum_r A(m, r) B(n, r) (+ add[m, n]), rounded
// once to the output's type.
struct LinearOut {
  void* c;
  int dtype;
  int64_t ld;
  float alpha;
  const float* tscale;  // device, or NULL
  const void* add;      // device, of the output's type and row pitch, or NULL; may be c
};

// One product: the 16- or 32-bit operand a (activations or gradients) and the
// quantised one.
enum : int { LIN_FORWARD = 0, LIN_DGRAD = 1, LIN_WGRAD = 2 };
struct LinearArgs {
  int op;
  int64_t rows, out, in;  // tokens, out_features, in_features
  const void* a;          // x [rows, in], or dy [rows, out]
  int a_dtype;
  int64_t lda;
  int kind;               // 4-bit kind of the weight (forward, dgrad) or 8-bit format (wgrad)
  const uint8_t* q;       // the weight's bytes, or the activation's codes
  const uint8_t* scales;  // wgrad: one byte per 32 columns
  LinearOut o;
};

enum : int { A8_E4M3 = 0, A8_E5M2 = 1 };
constexpr int kA8Group = 32;

// bytes of workspace launch_linear uses for these shapes, types and kind,
// whatever the pointers' alignment and the strides
int64_t linear_workspace(const LinearArgs& a);
cudaError_t launch_linear(const LinearArgs& a, void* ws, cudaStream_t st);
cudaError_t launch_act8_save(int fmt, const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, uint8_t* codes,
                             uint8_t* scales, cudaStream_t st);
cudaError_t launch_act8_load(int fmt, const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, void* out,
                             int dtype, int64_t ldo, cudaStream_t st);

}  // namespace ody

// ody_linear_gemm.h -- the tensor-core path of the quantised linear layer
// (ody_linear_gemm.cu).
#pragma once
#include <algorithm>

#include "ody_linear.h"

namespace ody {
int64_t gemm_workspace(const LinearArgs& a, int sms);
cudaError_t launch_gemm(const LinearArgs& a, void* ws, int sms, cudaStream_t st);
// whether a bounded wait of the current device's kernels ran out since the
// last call; waits for the device's work on `st`
cudaError_t gemm_wait_error(cudaStream_t st, bool* ran_out);
cudaError_t launch_wait_selftest(long long cycles, cudaStream_t st);
}  // namespace ody

// ody_linear_rows.h -- the few-row path of the quantised linear layer
// (ody_linear_rows.cu).
#pragma once
#include "ody_linear.h"

namespace ody {
bool few_rows(const LinearArgs& a);
// shared memory that one row's backward kernel (MXFP4, bfloat16) may take on the current device
cudaError_t rows_shared_limit(int* bytes);
cudaError_t launch_few_rows(const LinearArgs& a, int sms, cudaStream_t st);
}  // namespace ody

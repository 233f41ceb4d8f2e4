// ody_linear_rows.h -- the few-row path of the quantised linear layer
// (ody_linear_rows.cu).
#pragma once
#include "ody_linear.h"

namespace ody {
bool few_rows(const LinearArgs& a);
cudaError_t launch_few_rows(const LinearArgs& a, int sms, cudaStream_t st);
}  // namespace ody

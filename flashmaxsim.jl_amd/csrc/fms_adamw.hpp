// fms_adamw.hpp -- host launchers of the AdamW step (fms_adamw.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/flashmaxsim_hip.h"

namespace fms {

struct AdamWStep {
  float beta1, rest1;  // and 1 - beta1
  float beta2, rest2;
  float eps;
  float decay;    // 1 - lr * weight_decay
  float lr;       // lr / (1 - beta1^t)
  float inv_bc2;  // 1 / sqrt(1 - beta2^t)
  float grad_scale;
};

hipError_t adamw_step(int64_t count, const fms_adamw_tensor* tensors, const AdamWStep& s,
                      hipStream_t stream);
hipError_t moment_values(int64_t count, const fms_moment8* moments, hipStream_t stream);

}  // namespace fms

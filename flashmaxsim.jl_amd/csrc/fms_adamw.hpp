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

// A plan: this header, `count` entries, and for each workgroup of a step over all tensors the
// tensor it belongs to.  The same bytes on the host and on the device.
struct AdamWPlan {
  int64_t count, blocks;
};
struct AdamWEntry {
  fms_adamw_tensor t;
  int64_t first;  // workgroup of its first element
};
int64_t adamw_blocks(const fms_adamw_tensor& t);
hipError_t adamw_step(const AdamWPlan* plan, const void* device_plan, const void* const* grads,
                      const int32_t* g_dtypes, const AdamWStep& s, hipStream_t stream);
hipError_t moment_values(int64_t count, const fms_moment8* moments, hipStream_t stream);

}  // namespace fms

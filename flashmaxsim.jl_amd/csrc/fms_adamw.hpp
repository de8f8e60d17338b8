// fms_adamw.hpp -- host launchers of the AdamW step (fms_adamw.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/flashmaxsim_hip.h"

namespace fms {

// A step's numbers.  t, a tensor's own steps with this one, is steps[i], or `step` for all of
// them where steps is null.
struct AdamWRates {
  double lr, beta1, beta2, eps, weight_decay, grad_scale;
  int64_t step;
  const int64_t* steps;
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
                      const int32_t* g_dtypes, const AdamWRates& r, hipStream_t stream);
hipError_t moment_values(int64_t count, const fms_moment8* moments, hipStream_t stream);

}  // namespace fms

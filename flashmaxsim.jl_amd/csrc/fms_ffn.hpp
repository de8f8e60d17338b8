// fms_ffn.hpp -- host launchers of the gated feed-forward block (fms_ffn.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fms {

struct FfnArgs {
  int32_t dtype;  // FMS_F32, FMS_F16, FMS_BF16
  int32_t act;    // FMS_ACT_*
  int64_t tokens, dim, hidden;
  const void* x;   // (tokens, dim)
  const void* wg;  // (hidden, dim)
  const void* wu;
};

// Whether the sizes fit the kernels' 32-bit offsets and grids.
bool ffn_supported(const FfnArgs& a);

// h (tokens, hidden) = act(x wg^T) * (x wu^T).
hipError_t ffn_forward(const FfnArgs& a, void* h, hipStream_t stream);

// dx (null: not wanted), dwg and dwu (both or neither null) for the cotangent dh.
hipError_t ffn_pullback(const FfnArgs& a, void* dx, void* dwg, void* dwu, const void* dh,
                        hipStream_t stream);

}  // namespace fms

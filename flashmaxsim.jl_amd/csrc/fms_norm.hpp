// fms_norm.hpp -- host launchers of the block norms (fms_norm.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fms {

struct NormArgs {
  int32_t dtype;  // FMS_F32, FMS_F16, FMS_BF16
  int32_t kind;   // FMS_NORM_*
  float scale, eps;
  int64_t rows, dim;
  int64_t gate_rows;  // rows that share a gate vector (rows of the call: one for all)
  const void* x;      // (rows, dim)
  const void* f;      // (rows, dim) or null: r = x
  const void* gate;   // (rows / gate_rows, dim) or null: 1
  const void* wpost;  // (dim,) or null: the branch as it is
  const void* wpre;   // (dim,) or null: no n
};

constexpr int64_t kNormMaxDim = 16384;

// r (null without f) and n (null without wpre).
hipError_t norm_forward(const NormArgs& a, void* r, void* n, hipStream_t stream);

struct NormGrads {
  const void *dr, *dn;  // cotangents; either null: zero
  void *dx, *df, *dgate, *dwpost, *dwpre;
};
hipError_t norm_pullback(const NormArgs& a, const NormGrads& g, hipStream_t stream);

}  // namespace fms

// fms_embed.hpp -- host launchers of the token lookup (fms_embed.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fms {

struct EmbedArgs {
  int32_t dtype;  // FMS_F32, FMS_F16, FMS_BF16
  int32_t id_bytes;
  const void* ids;  // (n,) 1-based, int32 or int64
  float scale;
  int64_t n, vocabulary, dim;
};

// e (n, dim) = scale * weight[ids - 1]; an id outside 1 .. vocabulary gives zeros.
hipError_t embed_forward(const EmbedArgs& a, void* e, const void* weight, hipStream_t stream);
// dweight (vocabulary, dim) = scale * sums of de's rows by id.
hipError_t embed_pullback(const EmbedArgs& a, void* dweight, const void* de, hipStream_t stream);

}  // namespace fms

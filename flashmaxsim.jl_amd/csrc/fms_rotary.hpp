// fms_rotary.hpp -- host launchers of the norm and rotation of heads (fms_rotary.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fms {

struct RotaryArgs {
  int32_t dtype;    // FMS_F32, FMS_F16, FMS_BF16
  int32_t kind;     // FMS_NORM_*
  int32_t pairing;  // FMS_PAIR_*
  int32_t dim, turned;
  float eps;
  int64_t seqs, tokens;
  int32_t heads, kv_heads;
  const void *q, *k;
  int64_t qs[3], ks[3];  // elements between sequences, tokens, heads
  const float* table;    // (table_rows, turned): cosines, then sines, of turned / 2 pairs
  int64_t table_rows;
  const void* positions;  // 1-based rows of the table, or null: token t takes row t
  int32_t position_bytes;
  int64_t position_seqs;  // sequences that have positions of their own: 1 or seqs
  const void *wq, *wk;    // (dim,) or null: no norm
};

constexpr int64_t kRotaryMaxDim = 512;

hipError_t rotary_forward(const RotaryArgs& a, void* q_out, void* k_out, hipStream_t stream);

struct RotaryGrads {
  const void *dq_out, *dk_out;  // dense cotangents
  void *dq, *dk, *dwq, *dwk;    // dense
};
hipError_t rotary_pullback(const RotaryArgs& a, const RotaryGrads& g, hipStream_t stream);

}  // namespace fms

// fms_gemm.hpp -- device building blocks of the products behind the gated
// feed-forward block (fms_ffn.hip): out[m][n] = sum_k M(m, k) * N(n, k).
//
// A workgroup owns a kBM x kBN tile of the output and walks k in steps of
// 128 bytes per row.  Each step's slices of both operands go HBM/L2 -> LDS
// directly (buffer loads with an LDS destination, no registers), into the
// half of a double buffer that the step before left free; the MFMAs of a step
// run while the next step's slices are in flight.
//
// An operand's matrix lies in memory either with k contiguous (a row per m or
// n: "rows") or with m / n contiguous (a row per k: "columns").  Both land in
// LDS as they lie, in 16-byte units:
//   rows:    kSpan rows of 128 bytes; the unit u of row r is at r*8 + (u ^ (r & 7)).
//   columns: 128 / kEsz rows (k) of kSpan elements; unit u of row r is at
//            r*kUpr + (u ^ (4 * (r & 3))).
// The exclusive-or spreads the rows that one read touches over the banks.  An
// LDS load's destination is linear in the lane, so it is the lane's global
// address that is permuted.  16-bit columns are read with the transposing LDS
// read (four k of one column per lane from a 4 x 16 block that sixteen lanes
// hold), 32-bit columns need none.
//
// Every load is bounds-checked by its buffer resource: rows past the matrix'
// end read as zero, and units past a row's end are sent out of bounds.
#pragma once

#include "fms_device.hpp"

namespace fms {

typedef __attribute__((address_space(3))) void* lds_void_ptr;
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kStepBytes = 128;            // k bytes of a row per step
constexpr int kOutOfBounds = (int)0x80000000u;  // an offset past every resource

// A matrix as a product's operand: `rows` rows of `rowbytes` used bytes (a
// multiple of 16), `pitch` bytes apart, base and pitch multiples of 16.
struct Matrix {
  const char* base;
  int64_t rows;
  int64_t pitch;
  int64_t rowbytes;
};

// The part of a matrix from byte `at` on, as a buffer resource.
__device__ __forceinline__ rsrc_t matrix_from(const Matrix& m, int64_t at) {
  int64_t left = (m.rows - 1) * m.pitch + m.rowbytes - at;
  left = left < 0 ? 0 : (left > 0x7fffffff ? 0x7fffffff : left);
  return make_rsrc_u(m.base + at, (uint32_t)left);
}

// One operand's staging and fragment reads.  kRows: k contiguous.  kParts: the
// span is made of 1 or 2 equal parts, each from a matrix of its own (gate and up
// projections side by side).
template <class Op, bool kRows, int kSpan, int kThreads, int kParts>
struct Stage {
  static constexpr int kBytes = kSpan * kStepBytes;
  static constexpr int kUnits = kBytes / 16;
  static constexpr int kLoads = kUnits / kThreads;         // per thread and step
  static constexpr int kStepK = kStepBytes / Op::kEsz;     // k values per step
  static constexpr int kUpr = kRows ? 8 : kSpan * Op::kEsz / 16;  // units per LDS row
  static_assert(kUnits % (kThreads * kParts) == 0, "whole loads per part");
  static_assert(kRows || kParts == 1, "two parts only of rows");
  static_assert(kRows || kUpr >= 16, "the swizzle spans 16 units");

  int voff[kLoads];   // this lane's offsets into the resource
  int unit[kLoads];   // rows: the byte of the row's step its unit starts at

  __device__ __forceinline__ void init(int tid, int64_t pitch) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int u = i * kThreads + tid;
      const int row = u / kUpr, phys = u % kUpr;
      const int log = kRows ? phys ^ (row & 7) : phys ^ (4 * (row & 3));
      unit[i] = log * 16;
      const int part_row = kRows ? row % (kSpan / kParts) : row;
      voff[i] = (int)((int64_t)part_row * pitch) + log * 16;
    }
  }

  // Requests step `step` of the tile at m/n = first into `lds`.
  __device__ __forceinline__ void load(const Matrix (&mat)[kParts], int64_t first, int step,
                                       char* lds, int wave) const {
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      const Matrix& m = mat[p];
      int64_t at;
      int tail = kStepBytes;  // rows: used bytes of this step
      if constexpr (kRows) {
        at = first * m.pitch + (int64_t)step * kStepBytes;
        const int64_t left = m.rowbytes - (int64_t)step * kStepBytes;
        tail = left < kStepBytes ? (int)left : kStepBytes;
      } else {
        at = (int64_t)step * kStepK * m.pitch + first * Op::kEsz;
      }
      const rsrc_t r = matrix_from(m, at);
#pragma unroll
      for (int i = p * kLoads / kParts; i < (p + 1) * kLoads / kParts; ++i) {
        const int off = (kRows && unit[i] >= tail) ? kOutOfBounds : voff[i];
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            r, (lds_void_ptr)(lds + (i * kThreads + wave * 64) * 16), 16, off, 0, 0, 0);
      }
    }
  }

  // The 16-byte fragment of 32 rows / columns from `at` on, k group ks (0..3) of the
  // step: 16-bit, eight k from 16 ks + 8 h; 32-bit, four k from 8 ks + 4 h (h = lane / 32).
  __device__ static __forceinline__ u32x4 frag(const char* lds, int at, int ks, int lane) {
    const int h = lane >> 5;
    if constexpr (kRows) {
      const int row = at + (lane & 31);
      return *reinterpret_cast<const u32x4*>(lds + row * 128 + (((2 * ks + h) ^ (row & 7)) * 16));
    } else if constexpr (Op::kEsz == 2) {
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const int i = lane & 15;
      const int r3 = (i >> 2) & 3;  // row & 3: the other parts of the row are multiples of 4
      const int unit = (at >> 3) + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
      const char* p = lds + (16 * ks + 8 * h + r3) * (kUpr * 16) + ((unit ^ (4 * r3)) * 16) + (i & 1) * 8;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * kUpr * 16));
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
      const u32x2 l = __builtin_bit_cast(u32x2, lo), u = __builtin_bit_cast(u32x2, hi);
      return u32x4{l[0], l[1], u[0], u[1]};
    } else {
      const int col = at + (lane & 31);
      u32x4 f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 8 * ks + 4 * h + e;
        f[e] = *reinterpret_cast<const uint32_t*>(lds + row * (kUpr * 16) +
                                                  (((col >> 2) ^ (4 * e)) * 16) + (col & 3) * 4);
      }
      return f;
    }
  }
};

// acc += the products of one fragment pair.  The accumulator's columns (lanes) are
// the second fragment's rows, its rows (registers, acc_row) the first's.
template <class Op>
__device__ __forceinline__ typename Op::Acc mma_frag(u32x4 a, u32x4 b, typename Op::Acc acc) {
  if constexpr (Op::kEsz == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = Op::mma(a[e], b[e], acc);
    return acc;
  } else {
    return Op::mma(a, b, acc);
  }
}

// The tile's shape: kWM x kWN waves, each 32 kMF rows by 64 columns.
template <class Op_, bool kMRows_, bool kNRows_, int kParts_, int kWM_, int kWN_, int kMF_>
struct Product {
  typedef Op_ Op;
  static constexpr int kParts = kParts_, kWM = kWM_, kWN = kWN_, kMF = kMF_, kNF = 2;
  static constexpr int kThreads = 64 * kWM * kWN;
  static constexpr int kBM = kWM * kMF * 32, kBN = kWN * 64;
  typedef Stage<Op, kMRows_, kBM, kThreads, 1> StageM;
  typedef Stage<Op, kNRows_, kBN, kThreads, kParts> StageN;
  static constexpr int kHalf = StageM::kBytes + StageN::kBytes;  // one of the two buffers
  static constexpr int kLds = 2 * kHalf;
  static constexpr int kStepK = StageM::kStepK;
  typedef typename Op::Acc Acc;

  // Column of the tile that fragment nf of wave column wn starts at.  With two parts, a
  // wave holds 32 columns of each, so that gate and up of one hidden unit share a lane.
  __device__ static __forceinline__ int col(int wn, int nf) {
    return kParts == 2 ? nf * (kBN / 2) + wn * 32 : wn * 64 + nf * 32;
  }

  // acc[nf][mf] += over steps [s0, s1) of the tile at (m0, n0); n0 counts within a part.
  // All threads of the workgroup call it; it ends with the LDS free for other use.
  __device__ static __forceinline__ void run(Acc (&acc)[kNF][kMF], const Matrix (&M)[1],
                                             const Matrix (&N)[kParts], int64_t m0, int64_t n0,
                                             int s0, int s1, char* lds) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / kWN, wn = wave % kWN;
    StageM sm;
    StageN sn;
    sm.init(tid, M[0].pitch);
    sn.init(tid, N[0].pitch);
    if (s0 < s1) {
      sm.load(M, m0, s0, lds, wave);
      sn.load(N, n0, s0, lds + StageM::kBytes, wave);
    }
    for (int s = s0; s < s1; ++s) {
      char* cur = lds + ((s - s0) & 1) * kHalf;
      char* nxt = lds + (((s - s0) & 1) ^ 1) * kHalf;
      // this step's slices have landed, and every wave is done with the other buffer
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (s + 1 < s1) {
        sm.load(M, m0, s + 1, nxt, wave);
        sn.load(N, n0, s + 1, nxt + StageM::kBytes, wave);
      }
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        u32x4 fn[kNF], fm[kMF];
#pragma unroll
        for (int i = 0; i < kNF; ++i)
          fn[i] = StageN::frag(cur + StageM::kBytes, col(wn, i), ks, lane);
#pragma unroll
        for (int i = 0; i < kMF; ++i) fm[i] = StageM::frag(cur, (wm * kMF + i) * 32, ks, lane);
#pragma unroll
        for (int j = 0; j < kMF; ++j)
#pragma unroll
          for (int i = 0; i < kNF; ++i) acc[i][j] = mma_frag<Op>(fn[i], fm[j], acc[i][j]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
};

}  // namespace fms

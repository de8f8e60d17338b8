// fms_gemm.hpp -- device building blocks of the products behind the gated
// feed-forward block (fms_ffn.hip): out[m][n] = sum_k M(m, k) * N(n, k).
//
// A workgroup owns a kBM x kBN tile of the output at a time and walks k in steps of
// kStepBytes per row.  A step's slices of both operands go HBM/L2 -> LDS directly
// (buffer loads with an LDS destination, no registers) into one of 256 / kStepBytes
// buffers while the steps before are multiplied.  Two schedules:
//   four waves: small tiles, two workgroups to a CU; one's MFMAs run while the
//     other waits at its barrier or is in its epilogue.
//   eight waves, two to a SIMD: the first four and the last four take turns.  While
//     one half multiplies two k groups, the other reads the fragments of its next
//     two, and a barrier swaps them: the matrix cores see one wave after the
//     other without a gap, and no wave waits for LDS in between.
// Tiles of 256 x 256 multiply 8192-long random bf16 rows at 1.38 PFLOP/s (the card's
// power bounds that: zeros run at 1.95), 128 x 128 at 1.1.  Sums of 768 to 1024 terms run at 1.0
// to 1.1 with the matrix cores busy for 55 to 60 % of the cycles: the halves of the eight waves
// work on one tile, a turn apart, and its epilogue meets no more than one turn of products.
//
// An operand's matrix lies in memory either with k contiguous (a row per m or
// n: "rows") or with m / n contiguous (a row per k: "columns").  Both land in
// LDS as they lie, in 16-byte units:
//   rows:    kSpan rows of kStepBytes; the unit u of row r is at r*8 + (u ^ ((r >> 1) & 7))
//            (128 bytes) or r*4 + (u ^ ((r >> 2) & 3)) (64).
//   columns: kStepBytes / kEsz rows (k) of kSpan elements; unit u of row r is at
//            r*kUpr + (u ^ (4 * (r & 3))), or u ^ (4 * ((r >> 1) & 1)) in rows of 8 units.
// The exclusive-or spreads the rows that sixteen lanes read together over all
// 64 banks.  An LDS load's destination is linear in the lane, so it is the
// lane's global address that is permuted.  16-bit columns are read with the
// transposing LDS read (four k of one column per lane from a 4 x 16 block that
// sixteen lanes hold), 32-bit columns need none.
//
// Every load is bounds-checked by its buffer resource: rows past the matrix'
// end read as zero, and units past a row's end are sent out of bounds.
#pragma once

#include "fms_device.hpp"

namespace fms {

typedef __attribute__((address_space(3))) void* lds_void_ptr;
typedef short s16x4 __attribute__((ext_vector_type(4)));

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
template <class Op, bool kRows, int kSpan, int kThreads, int kParts, int kStepBytes>
struct Stage {
  static constexpr int kBytes = kSpan * kStepBytes;
  static constexpr int kUnits = kBytes / 16;
  static constexpr int kLoads = kUnits / kThreads;         // per thread and step
  static constexpr int kStepK = kStepBytes / Op::kEsz;     // k values per step
  static constexpr int kUpr = kRows ? kStepBytes / 16 : kSpan * Op::kEsz / 16;  // units per LDS row
  static_assert(kUnits % (kThreads * kParts) == 0, "whole loads per part");
  static_assert(kRows || kParts == 1, "two parts only of rows");
  static_assert(kRows || kUpr == 8 || kUpr >= 16, "the swizzle's span");

  // What unit indices of LDS row r are exclusive-or'ed with.
  __device__ static __forceinline__ int mix(int r) {
    if (kRows) return kUpr == 8 ? (r >> 1) & 7 : (r >> 2) & 3;
    return kUpr == 8 ? 4 * ((r >> 1) & 1) : 4 * (r & 3);
  }

  int voff[kLoads];  // this lane's offsets into the resource
  // the next step's slice: where it starts and what is left of the matrix from there
  const char* base[kParts];
  int64_t left[kParts];
  int64_t stride;  // bytes from a step's start to the next one's
  int rest;        // rows: bytes of a row from the next step on

  __device__ __forceinline__ void init(int tid, const Matrix (&mat)[kParts], int64_t first, int step) {
    stride = kRows ? kStepBytes : (int64_t)kStepK * mat[0].pitch;
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      const Matrix& m = mat[p];
      const int64_t at = step * stride + first * (kRows ? m.pitch : (int64_t)Op::kEsz);
      base[p] = reinterpret_cast<const char*>(rfl64(reinterpret_cast<uint64_t>(m.base + at)));
      left[p] = (int64_t)rfl64((uint64_t)((m.rows - 1) * m.pitch + m.rowbytes - at));
    }
    const int64_t r = mat[0].rowbytes - step * stride;
    rest = !kRows || r > 0x7fffffff ? 0x7fffffff : (int)r;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int u = i * kThreads + tid;
      const int row = u / kUpr, log = (u % kUpr) ^ mix(row);
      voff[i] = (int)((kRows ? row % (kSpan / kParts) : row) * mat[0].pitch) + log * 16;
    }
  }

  // Sends the units past a row's end out of bounds, before a request of its last, shorter step.
  __device__ __forceinline__ void trim(int tid) {
    if constexpr (kRows) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int u = i * kThreads + tid;
        if (((u % kUpr) ^ mix(u / kUpr)) * 16 >= rest) voff[i] = kOutOfBounds;
      }
    }
  }
  __device__ __forceinline__ bool last() const { return kRows && rest < kStepBytes; }

  // Requests load i of the next step's slice into `lds`.
  __device__ __forceinline__ void load(int i, const rsrc_t (&from)[kParts], char* lds, int wave) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        from[i / (kLoads / kParts)], (lds_void_ptr)(lds + (i * kThreads + wave * 64) * 16), 16, voff[i],
        0, 0, 0);
  }
  __device__ __forceinline__ void resources(rsrc_t (&r)[kParts]) const {
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      const int64_t n = left[p] < 0 ? 0 : (left[p] > 0x7fffffff ? 0x7fffffff : left[p]);
      r[p] = make_rsrc(base[p], (uint32_t)n);
    }
  }
  __device__ __forceinline__ void advance() {
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      base[p] += stride;
      left[p] -= stride;
    }
    rest -= kRows ? kStepBytes : 0;
  }

  // The 16-byte fragment of 32 rows / columns from `at` on, k group ks of the
  // step: 16-bit, eight k from 16 ks + 8 h; 32-bit, four k from 8 ks + 4 h (h = lane / 32).
  __device__ static __forceinline__ u32x4 frag(const char* lds, int at, int ks, int lane) {
    const int h = lane >> 5;
    if constexpr (kRows) {
      const int row = at + (lane & 31);
      return *reinterpret_cast<const u32x4*>(lds + row * kStepBytes + (((2 * ks + h) ^ mix(row)) * 16));
    } else if constexpr (Op::kEsz == 2) {
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const int i = lane & 15;
      const int r3 = (i >> 2) & 3;  // row & 3: the other parts of the row are multiples of 4
      const int unit = (at >> 3) + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
      const char* p = lds + (16 * ks + 8 * h + r3) * (kUpr * 16) + ((unit ^ mix(r3)) * 16) + (i & 1) * 8;
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
                                                  (((col >> 2) ^ mix(e)) * 16) + (col & 3) * 4);
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

// A stretch of k of one tile: steps [first, first + steps) of the products of M's and N's
// rows / columns from m0 and n0 on (n0 counts within a part).  The last leg of a tile ends it.
template <int kParts>
struct Leg {
  Matrix m[1], n[kParts];
  int64_t m0, n0;
  int first, steps;
  bool ends;
};

// The tile's shape: kWM x kWN waves, each 32 kMF rows by 64 columns; kStepBytes of k a step.
template <class Op_, bool kMRows_, bool kNRows_, int kParts_, int kWM_, int kWN_, int kMF_,
          int kStepBytes_ = 128>
struct Product {
  typedef Op_ Op;
  static constexpr int kParts = kParts_, kWM = kWM_, kWN = kWN_, kMF = kMF_, kNF = 2;
  static constexpr int kThreads = 64 * kWM * kWN;
  static constexpr int kStepBytes = kStepBytes_;
  static constexpr int kGroups = kStepBytes / 32;  // fragments of k per step
  static constexpr int kBuffers = 256 / kStepBytes;
  static constexpr int kBM = kWM * kMF * 32, kBN = kWN * 64;
  typedef Stage<Op, kMRows_, kBM, kThreads, 1, kStepBytes> StageM;
  typedef Stage<Op, kNRows_, kBN, kThreads, kParts, kStepBytes> StageN;
  static constexpr int kBuffer = StageM::kBytes + StageN::kBytes;
  static constexpr int kLds = kBuffers * kBuffer;
  static constexpr bool kTurns = kWM * kWN == 8;
  static constexpr int kStepK = StageM::kStepK;
  typedef typename Op::Acc Acc;
  typedef Leg<kParts> Legs;

  // Column of the tile that fragment nf of wave column wn starts at.  With two parts, a
  // wave holds 32 columns of each, so that gate and up of one hidden unit share a lane.
  __device__ static __forceinline__ int col(int wn, int nf) {
    return kParts == 2 ? nf * (kBN / 2) + wn * 32 : wn * 64 + nf * 32;
  }

  // Walks the workgroup's legs 0 .. legs - 1 (all of at least one step), which leg(j) gives,
  // as one run of steps: a tile's first slices are on their way before the tile before is
  // through.  after(j, acc) takes a tile's sums when its last leg j is done, without touching
  // the LDS.  All threads of the workgroup call it.
  template <class LegOf, class After>
  __device__ static __forceinline__ void run(int legs, LegOf&& leg, After&& after, char* lds) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / kWN, wn = wave % kWN;
    // where the requests are: leg `ahead` with `left` of its steps to come
    StageM sm;
    StageN sn;
    int ahead = 0, left = 0;
    const auto enter = [&] {
      const Legs l = leg(ahead);
      sm.init(tid, l.m, l.m0, l.first);
      sn.init(tid, l.n, l.n0, l.first);
      left = l.steps;
    };
    // (past the last leg it asks for more of that one, which no one uses)
    const auto advance = [&] {
      sm.advance();
      sn.advance();
      if (--left == 0 && ++ahead < legs) enter();
    };
    // Load i of both operands' next slices into a buffer, from the resources made before.
    rsrc_t rm[1], rn[kParts];
    const auto aim = [&] {
      if (sm.last()) sm.trim(tid);
      if (sn.last()) sn.trim(tid);
      sm.resources(rm);
      sn.resources(rn);
    };
    const auto load = [&](int i, char* to) {
      if (i < StageM::kLoads)
        sm.load(i, rm, to, wave);
      else
        sn.load(i - StageM::kLoads, rn, to + StageM::kBytes, wave);
    };
    constexpr int kLoads = StageM::kLoads + StageN::kLoads;
    const auto request = [&](char* to) {
      aim();
#pragma unroll
      for (int i = 0; i < kLoads; ++i) load(i, to);
      advance();
    };
    // Fragments of k group g of the step in `cur`, and their products.
    Acc acc[kNF][kMF];
    u32x4 fn[2][kNF], fm[2][kMF];
    const auto read = [&](const char* cur, int g, int i) {
#pragma unroll
      for (int f = 0; f < kNF; ++f) fn[i][f] = StageN::frag(cur + StageM::kBytes, col(wn, f), g, lane);
#pragma unroll
      for (int f = 0; f < kMF; ++f) fm[i][f] = StageM::frag(cur, (wm * kMF + f) * 32, g, lane);
    };
    const auto multiply = [&](int i, int b) {
#pragma unroll
      for (int a = 0; a < kNF; ++a) acc[a][b] = mma_frag<Op>(fn[i][a], fm[i][b], acc[a][b]);
    };
    const auto multiply_all = [&](int i) {
#pragma unroll
      for (int b = 0; b < kMF; ++b) multiply(i, b);
    };
    const auto clear = [&] {
#pragma unroll
      for (int a = 0; a < kNF; ++a)
#pragma unroll
        for (int b = 0; b < kMF; ++b) acc[a][b] = Acc{};
    };
    enter();
    clear();
    // the buffers in turn: step i is in buffer i % kBuffers
    int at = 0;
    const auto buffer = [&](int i) {  // of the i-th step from the current one
      i += at;
      return lds + (i >= kBuffers ? i - kBuffers : i) * kBuffer;
    };
    const auto next = [&] { at = at + 1 == kBuffers ? 0 : at + 1; };
    request(buffer(0));
    if constexpr (!kTurns) {
      static_assert(kBuffers == 2 && kGroups == 4, "two buffers, four groups");
      for (int j = 0; j < legs; ++j) {
        const Legs l = leg(j);
        for (int s = 0; s < l.steps; ++s) {
          // this step's slices have landed; every wave has its last fragments of the step before
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
          turn();
          const char* const cur = buffer(0);
          read(cur, 0, 0);
          if (ahead < legs) request(buffer(1));
          if (s > 0) multiply_all(1);
          read(cur, 1, 1);
          multiply_all(0);
          read(cur, 2, 0);
          multiply_all(1);
          read(cur, 3, 1);
          multiply_all(0);
          next();
        }
        multiply_all(1);
        if (l.ends) {
          after(j, acc);
          clear();
        }
      }
    } else {
      // Two k groups are read in one turn and multiplied in the next: the first half of the
      // waves reads at even turns, the second half at odd ones.  With H = kGroups / 2, step i is
      // read in turns 2H i .. 2H i + 2H - 1, and its buffer is free from turn 2H (i + 1) on.  A
      // wave requests in the one multiplying turn of each step that comes right after a buffer
      // became free, a load after every two MFMAs: the first half step i + kBuffers - 1 in turn
      // 2H i + 1, the second half step i + kBuffers in turn 2H (i + 1).  Each wave waits for its
      // requests of step i + 1, leaving the later ones in flight, before the barrier that ends
      // turn 2H i + 2H - 1.
      constexpr int kHalves = kGroups / 2, kInFlight = (kBuffers - 2) * kLoads;
      const bool second = wave >= 4;
      const auto landed = [] { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kInFlight) : "memory"); };
#pragma unroll
      for (int i = 1; i < kBuffers - 1; ++i) request(buffer(i));
      if (second) request(buffer(kBuffers - 1));
      landed();
      turn();
      if (second) turn();
      for (int j = 0; j < legs; ++j) {
        const Legs l = leg(j);
        for (int s = 0; s < l.steps; ++s) {
          const bool end = j + 1 == legs && s + 1 == l.steps;
          const char* const cur = buffer(0);
          char* const to = buffer(second ? 0 : kBuffers - 1);
#pragma unroll
          for (int half = 0; half < kHalves; ++half) {
            read(cur, 2 * half, 0);
            read(cur, 2 * half + 1, 1);
            if (half == 0) aim();
            if (half == kHalves - 1 && second) landed();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            turn();
            const bool now = kHalves == 1 || (half == 1) == second;
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int i = 0; i < 2 * kMF; ++i) {
              multiply(i / kMF, i % kMF);
              if (now && i < kLoads) load(i, to);
            }
            static_assert(kLoads <= 2 * kMF, "a load for every two MFMAs");
            __builtin_amdgcn_s_setprio(0);
            if (half == kHalves - 1 && !second) landed();
            // (at the very end no load is left in flight)
            if (half == kHalves - 1 && end) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            turn();
          }
          advance();
          next();
        }
        if (j + 1 == legs && !second) turn();
        if (l.ends) {
          after(j, acc);
          clear();
        }
      }
    }
  }

  // The barrier between turns: nothing moves across it.
  __device__ static __forceinline__ void turn() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
  }
};

}  // namespace fms

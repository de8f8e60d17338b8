// fms_attn.hpp -- attention over heads: host launchers and the device building blocks that its
// kernels share (fms_attn.hip, fms_attn_back.hip).
//
// A key head serves `group` query heads.  Its query rows are numbered token by token, the
// group's heads within a token: row = token * group + head, so that heads that share keys
// share the tiles they are read into, whatever the group.  One unit of work is a (sequence,
// key head); its rows go in tiles of 32, one to a wave.
//
// Products put what a lane owns into the accumulator's columns: S^T = K Q^T gives a lane one
// query row and 16 of each 32 keys, so maxima, sums and rescaling are a lane's own business
// (one exchange with lane ^ 32 a tile), and the probabilities are already the second
// operand of the product that follows: its k slots may be in any order that both operands
// share, and the transposing LDS read fetches the other operand in the accumulators' order.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fms_device.hpp"

namespace fms {

struct AttnArgs {
  int32_t dtype;  // FMS_F32, FMS_F16, FMS_BF16
  int32_t dim;    // values of a head
  int32_t units;  // 16-byte units of a head's row as the kernels read and write it (dim, made whole units)
  int32_t heads, kv_heads, group;
  uint32_t group_inv;  // ceil(2^32 / group), 0 for a group of one
  int32_t causal;
  int32_t window;  // < 0: none
  float scale;
  int64_t seqs;
  uint32_t unit0;      // first (sequence, key head) of a launch
  int32_t tq, tk;      // tokens of a sequence, or of the longest one
  int64_t nq, nk;      // token rows in all
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];  // elements between sequences, tokens, heads
  const uint8_t *qmask, *kmask;  // (seqs, tq), (seqs, tk) or null
  const int32_t *cu_q, *cu_k;    // (seqs + 1), 1-based: ragged; null: padded
};

constexpr int64_t kAttnMaxDim = 128;

// o (token rows, heads, whole units of dim, 16-byte aligned); top (seqs, kv_heads, tq * group) or ragged (kv_heads, nq * group),
// the rows' largest products q_i k_j (of the other sign under a negative scale; -inf where no key counts), and rest,
// what o's rounding left (16-bit types): both null where no pullback follows.
struct AttnOut {
  void* o;
  float* top;
  void* rest;
  void* parts;  // attn_forward_bytes of workspace
};
int64_t attn_forward_bytes(const AttnArgs& a);
hipError_t attn_forward(const AttnArgs& a, const AttnOut& out, hipStream_t stream);

struct AttnGrads {
  const void *dout, *o, *rest;  // as o: token rows of heads * dim
  const float* top;
  void *dq, *dk, *dv;  // dense
  float* delta;        // as top: sum_j p_ij dp_ij, from the first kernel to the second
  float* level;        // as top: what the rows' sums are brought to one by, likewise
  float* peaks;        // (units, kPeakParts, 2): largest squared norms of v and dout rows (fp16)
  void* parts;         // attn_pullback_bytes of workspace
};
int64_t attn_pullback_bytes(const AttnArgs& a);
constexpr int kAttnPeakParts = 16;
// All workspace is the caller's, who has it before anything is launched: a captured call that is lent too little
// adds nothing.  Rows of o, rest and dout are whole units apart.
hipError_t attn_pullback(const AttnArgs& a, const AttnGrads& g, hipStream_t stream);

// ---- host helpers of both ----------------------------------------------------------------

// rows x heads x dim -> dense rows x heads x packed_dim, zeros behind dim
hipError_t attn_pack(int32_t dtype, void* to, const void* from, const int64_t* strides, int64_t seqs,
                     int64_t tokens, int64_t heads, int32_t dim, int32_t packed_dim, hipStream_t stream);
// Zeros for the token rows of some results that no sequence covers.
struct AttnGaps {
  struct Result {
    void* out;
    const int32_t* cu;
    int64_t rows, most, width;  // token rows, the longest sequence, values of a row
  } of[3];
  int n;
  int64_t seqs;
};
hipError_t attn_zero_gaps(int32_t dtype, const AttnGaps& gaps, hipStream_t stream);

// ---- device --------------------------------------------------------------------------------

namespace attn {

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
// A score's factor, to base 2.  (Not zero, so that a masked score's -inf stays that: the smallest normal number, which
// makes at most 4 of a score; a NaN stays one.)
__device__ __forceinline__ float factor(const AttnArgs& A) {
  const float c = fabsf(A.scale) * kLog2e;
  return c < 1.17549435e-38f ? 1.17549435e-38f : c;
}
constexpr int kFar = (int)0x80000000u;  // a byte offset past every resource: reads as zero
constexpr int kRows = 64;               // rows of a tile in LDS
inline int instance_dim(const AttnArgs& a) { return a.dim <= 32 ? 32 : a.dim <= 64 ? 64 : 128; }
constexpr int kMaskSpan = 16384;        // rows whose mask bits are held at a time

// A sequence's place: first token rows and lengths.
struct Span {
  int64_t q0, k0;
  int nq, nk;
};
__device__ __forceinline__ void clamp_cu(const int32_t* cu, int64_t b, int64_t n, int most,
                                         int64_t& first, int& len) {
  int64_t a = (int64_t)cu[b] - 1, e = (int64_t)cu[b + 1] - 1;
  a = a < 0 ? 0 : (a > n ? n : a);
  e = e < a ? a : (e > n ? n : e);
  first = a;
  len = e - a > most ? most : (int)(e - a);
}
__device__ __forceinline__ Span span_of(const AttnArgs& A, int64_t b) {
  Span s;
  if (A.cu_q) {
    clamp_cu(A.cu_q, b, A.nq, A.tq, s.q0, s.nq);
    clamp_cu(A.cu_k, b, A.nk, A.tk, s.k0, s.nk);
  } else {
    s.q0 = b * A.tq;
    s.k0 = b * A.tk;
    s.nq = A.tq;
    s.nk = A.tk;
  }
  return s;
}
// Elements from an array's start to a sequence's first token, head 0.
__device__ __forceinline__ int64_t seq_at(const int64_t (&st)[3], bool ragged, int64_t b, int64_t first) {
  return ragged ? first * st[1] : b * st[0];
}
// Where a unit's rows start in top and the like.
__device__ __forceinline__ int64_t rows_at(const AttnArgs& A, int64_t b, int hk, int64_t q0) {
  return A.cu_q ? ((int64_t)hk * A.nq + q0) * A.group : (b * A.kv_heads + hk) * ((int64_t)A.tq * A.group);
}

__device__ __forceinline__ int token_of(int row, const AttnArgs& A) {
  return A.group_inv ? (int)__umulhi((uint32_t)row, A.group_inv) : row;
}

// The workgroup's place in `work` pieces: each XCD takes a contiguous run of them, so that
// what neighbouring pieces share is in one L2.
// (below 2^31 of them, so that the divisions behind it are short ones)
__device__ __forceinline__ uint32_t piece_of(uint32_t work) {
  return (blockIdx.x & 7) * ((work + 7) / 8) + (blockIdx.x >> 3);
}
inline unsigned piece_blocks(int64_t work) { return (unsigned)((work + 7) / 8 * 8); }
// launch(args, units) for all units, so many at a time that a launch's threads, up to 256 for each of a unit's `pieces`,
// can be counted in 32 bits.  (A unit has at most 2^30 rows, 2^23 pieces.)
constexpr int64_t kMostPieces = (int64_t)1 << 23;
template <class F>
hipError_t by_units(AttnArgs a, int64_t pieces, F&& launch) {
  const int64_t units = a.seqs * a.kv_heads, most = pieces < kMostPieces ? kMostPieces / (pieces > 0 ? pieces : 1) : 1;
  for (int64_t u = 0; u < units; u += most) {
    a.unit0 = (uint32_t)u;
    launch(a, units - u < most ? units - u : most);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// The keys that count by position for a query token, or the tokens that count for a key: [lo, hi).
struct Reach {
  int lo, hi;
};
__device__ __forceinline__ Reach keys_of(int token, const Span& s, const AttnArgs& A) {
  const int pos = token + s.nk - s.nq;
  Reach r = {0, s.nk};
  if (A.window >= 0) {
    if (pos - A.window > 0) r.lo = pos - A.window;
    if (r.hi - 1 - A.window > pos) r.hi = pos + A.window + 1;
  }
  if (A.causal && r.hi > pos + 1) r.hi = pos + 1;
  if (r.hi < r.lo) r.hi = r.lo;
  return r;
}
__device__ __forceinline__ Reach tokens_of(int key, const Span& s, const AttnArgs& A) {
  const int pos = key - (s.nk - s.nq);  // the token beside the key
  Reach r = {0, s.nq};
  if (A.window >= 0) {
    if (pos - A.window > 0) r.lo = pos - A.window;
    if (r.hi - 1 - A.window > pos) r.hi = pos + A.window + 1;
  }
  if (A.causal && r.lo < pos) r.lo = pos;
  if (r.lo > s.nq) r.lo = s.nq;  // (rows are counted in 32 bits)
  if (r.hi < r.lo) r.hi = r.lo;
  return r;
}
// Reaches grow with the token (or key), so those of a wave's 32 follow from its first and last: what all have in
// common, and what any has.  (A masked row or key counts too: it was read as zeros, and its
// result is made zero at the end.)
struct Reaches {
  Reach all, any;
};
__device__ __forceinline__ Reaches reaches(const Reach& first, const Reach& last, bool some) {
  return {{last.lo, first.hi}, {some ? first.lo : 0, some ? last.hi : 0}};
}

// ---- tiles in LDS --------------------------------------------------------------------------
// kRows rows of kD values, in 16-byte units; unit u of row r lies at u ^ mix(r): sixteen rows
// read together at one unit, and four rows read together at two, are in different banks.
template <class Op_, int kD_>
struct Tile {
  typedef Op_ Op;
  static constexpr int kD = kD_;
  static constexpr int kRowBytes = kD * Op::kEsz, kUnits = kRowBytes / 16;
  static constexpr int kBytes = kRows * kRowBytes;
  static constexpr int kK = kUnits / 2;  // k groups of a row: two units, one for each wave half
  static constexpr int kBlocks = kD / 32;

  __device__ static __forceinline__ constexpr int mix(int r) {
    return kUnits == 4 ? (r >> 2) & 3
                       : kUnits == 8 ? 4 * ((r >> 1) & 1) + ((r >> 2) & 3)
                                     : ((r & 3) << 2) | ((r >> 2) & 3);
  }
  static constexpr int loads(int threads) { return kBytes / 16 / threads; }

  // Rows as they lie: key / value tokens `stride` bytes apart from `base` on; those not in `bits` are zeros.
  template <int kThreads>
  __device__ static __forceinline__ void request(char* lds, const char* base, int stride, int units,
                                                 uint64_t bits) {
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const rsrc_t from = make_rsrc_u(base, 0x7fffffffu);
#pragma unroll
    for (int i = 0; i < loads(kThreads); ++i) {
      const int u = i * kThreads + tid, row = u / kUnits, unit = (u % kUnits) ^ mix(row);
      const int at = unit < units && (bits >> row & 1) ? row * stride + unit * 16 : kFar;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_ptr)(lds + (i * kThreads + wave * 64) * 16), 16,
                                               at, 0, 0, 0);
    }
  }
  // Query rows row0 .. row0 + kRows - 1 of a unit; base is the unit's token 0, its tokens `token`
  // and heads `head_step` elements apart.
  template <int kThreads>
  __device__ static __forceinline__ void request_rows(char* lds, const char* base, int64_t token, int64_t head_step,
                                                      int units, int row0, const AttnArgs& A, uint64_t bits) {
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int t0 = token_of(row0, A);
    const rsrc_t from = make_rsrc_u(base + (int64_t)t0 * token * Op::kEsz, 0x7fffffffu);
    const int ts = (int)token * Op::kEsz, hs = (int)head_step * Op::kEsz;
#pragma unroll
    for (int i = 0; i < loads(kThreads); ++i) {
      const int u = i * kThreads + tid, row = u / kUnits, unit = (u % kUnits) ^ mix(row);
      const int t = token_of(row0 + row, A), head = row0 + row - t * A.group;
      const int at = unit < units && (bits >> row & 1) ? (t - t0) * ts + head * hs + unit * 16 : kFar;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_ptr)(lds + (i * kThreads + wave * 64) * 16), 16,
                                               at, 0, 0, 0);
    }
  }

  // First operand, rows at .. at + 31 by values: lane's row, unit 2 kb + half.
  __device__ static __forceinline__ u32x4 rows(const char* lds, int at, int kb, int lane) {
    const int r = lane & 31, h = lane >> 5;
    return *reinterpret_cast<const u32x4*>(lds + (at + r) * kRowBytes + (((2 * kb + h) ^ mix(r)) * 16));
  }
  // First operand, values 32 block .. + 31 by rows: for the product over the rows at .. at + 15
  // (16-bit) or at .. at + 7 (32-bit) in the order in which the accumulator's registers hold
  // them: half h has at + 4 h + {0..3}, then (16-bit) at + 8 + 4 h + {0..3}.
  __device__ static __forceinline__ u32x4 columns(const char* lds, int at, int block, int lane) {
    const int h = lane >> 5;
    if constexpr (Op::kEsz == 2) {
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const int i = lane & 15, r = 4 * h + (i >> 2);
      const int unit = block * 4 + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
      const char* p = lds + (at + r) * kRowBytes + (i & 1) * 8;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + ((unit ^ mix(r)) * 16)));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4*)(p + 8 * kRowBytes + ((unit ^ mix(r + 8)) * 16)));
      const u32x2 l = __builtin_bit_cast(u32x2, lo), u = __builtin_bit_cast(u32x2, hi);
      return u32x4{l[0], l[1], u[0], u[1]};
    } else {
      const int col = block * 32 + (lane & 31);
      u32x4 f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * h + e;
        f[e] = *reinterpret_cast<const uint32_t*>(lds + (at + r) * kRowBytes +
                                                  (((col >> 2) ^ mix(at % 16 + r)) * 16) + (col & 3) * 4);
      }
      return f;
    }
  }
};

// Waves of a SIMD that the forward's registers should leave room for: as many as the LDS does.  (256 documents of up
// to 180 tokens, 12 heads of 64 in bf16: 66 us with four, 72 with three, though four spill a few registers.)
template <class Op, int kD, int kWaves>
constexpr int kSimdWaves = kWaves < 4 ? 1 : kD * Op::kEsz <= 128 ? 4 : kD * Op::kEsz <= 256 ? 2 : 1;

template <class Op>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 acc) {
  if constexpr (Op::kEsz == 4) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], acc, 0, 0, 0);
    return acc;
  } else {
    return Op::mma(a, b, acc);
  }
}

// What was asked for above stays above: reads are under way before the work that hides them.  (Left to itself the
// compiler puts each fragment's read right before its product, which waits for it.)
__device__ __forceinline__ void asked() { __builtin_amdgcn_sched_barrier(0); }

template <class Op>
struct Elem {
  typedef float T;
};
template <>
struct Elem<OpF16> {
  typedef _Float16 T;
};
template <>
struct Elem<OpBF16> {
  typedef __bf16 T;
};

// What o's rounding leaves is held this much larger: in fp16 it would be among the subnormal numbers.
template <class Op>
constexpr float kRestScale = std::is_same<Op, OpF16>::value ? 2048.0f : 1.0f;

// Registers 8 j .. 8 j + 7 (16-bit; 4 j .. 4 j + 3 in 32 bits) of a lane's values as the second
// operand of the product that `columns` feeds.  16-bit: two values for each, a rounding and what it left, so that a
// product's terms have twice the feature type's bits: with the rounding alone the sums would be 1.4 times as far
// off as their own rounding takes them, and more where a few terms make them up.
template <class Op>
struct Operand {
  u32x4 hi, lo;
};
template <class Op>
__device__ __forceinline__ Operand<Op> operand(const float (&v)[16], int j) {
  Operand<Op> x;
  if constexpr (Op::kEsz == 4) {
    x.hi = __builtin_bit_cast(u32x4, f32x4{v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]});
  } else {
    typedef typename Elem<Op>::T T;
    typedef T V __attribute__((ext_vector_type(8)));
    V hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) hi[e] = (T)v[8 * j + e];
    x.hi = __builtin_bit_cast(u32x4, hi);
    asm volatile("" : "+v"(x.hi));  // (settled: what it left is of these bits, however they were rounded)
    hi = __builtin_bit_cast(V, x.hi);
#pragma unroll
    for (int e = 0; e < 8; ++e) lo[e] = (T)(v[8 * j + e] - (float)hi[e]);
    x.lo = __builtin_bit_cast(u32x4, lo);
  }
  return x;
}
template <class Op>
__device__ __forceinline__ f32x16 mma(u32x4 a, const Operand<Op>& b, f32x16 acc) {
  acc = mma<Op>(a, b.hi, acc);
  if constexpr (Op::kEsz == 2) acc = mma<Op>(a, b.lo, acc);
  return acc;
}
template <class Op>
constexpr int kGroups = Op::kEsz == 4 ? 4 : 2;  // operands of 32 rows

// Lane's own row as a second operand for `rows`: units 2 kb + half of it, straight from memory, `at` bytes
// into the resource (kFar: zeros).  (Loads behind a branch would wait for one another.)
template <class T>
__device__ __forceinline__ void own_row(u32x4 (&f)[T::kK], rsrc_t from, int at, int units, int h) {
  asm volatile("" : "+v"(at), "+v"(h));  // (offsets are computed here, not kept in registers around a loop)
#pragma unroll
  for (int kb = 0; kb < T::kK; ++kb) f[kb] = buf_load16(from, 2 * kb + h < units ? at + (2 * kb + h) * 16 : kFar);
}

// A negative scale: the same scores from the other sign.
template <class T>
__device__ __forceinline__ void negate(u32x4 (&f)[T::kK]) {
#pragma unroll
  for (int kb = 0; kb < T::kK; ++kb) f[kb] ^= T::Op::kEsz == 4 ? 0x80000000u : 0x80008000u;
}

// Bits lo .. hi - 1 of 32 (bounds anywhere).
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {
  lo = lo < 0 ? 0 : (lo > 32 ? 32 : lo);
  hi = hi < 0 ? 0 : (hi > 32 ? 32 : hi);
  return (uint32_t)((1ull << hi) - 1) & ~(uint32_t)((1ull << lo) - 1);
}

// v where register r's row is in `keep` (shifted to the lane's half), else what: two instructions, and
// no compare whose result a select would wait for.
__device__ __forceinline__ float masked(float v, uint32_t keep, int r, float what) {
  const int bit = 8 * (r >> 2) + (r & 3);
  const uint32_t all = (uint32_t)((int32_t)(keep << (31 - bit)) >> 31);
  return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, v) & all) | (__builtin_bit_cast(uint32_t, what) & ~all));
}

// Which rows (keys, or query rows) of a stretch are there: `to` ends them, a mask leaves some out.  Masks
// are held as bits in LDS, kMaskSpan rows at a time, 64 to a word: a tile's.
static_assert(kRows == 64, "a word of mask bits is a tile");
struct Rows {
  uint64_t* words;
  bool given;  // a mask (without one there is one span)
  int span0, to;

  // Sets `to`: the rows end at `last`, or with the span.
  __device__ __forceinline__ void end(int last) { to = given && last - span0 > kMaskSpan ? span0 + kMaskSpan : last; }
  // The mask bits of rows from span0 on, below n; keep(row): its mask has it.  All threads call it.
  template <int kThreads, class Keep>
  __device__ __forceinline__ void gather(int n, Keep&& keep) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int left = n - span0, most = left < kMaskSpan ? left : kMaskSpan;
    for (int r = wave * 64; r < most; r += kThreads) {
      const uint64_t bits = __ballot(r + lane < most && keep(span0 + r + lane));
      if (lane == 0) words[r / 64] = bits;
    }
  }
  // The first tile from r0 on that has any rows (`to` or past it: none), and which.
  __device__ __forceinline__ int next(int r0, uint64_t& bits) const {
    bits = 0;
    for (; r0 < to; r0 += kRows) {
      bits = r0 + kRows <= to ? ~0ull : (1ull << (to - r0)) - 1;
      if (given) bits &= rfl64(words[(r0 - span0) / 64]);
      if (bits) break;
    }
    return r0;
  }
};

// All that this wave has asked for has landed, and so has every other wave's.
__device__ __forceinline__ void landed() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// A lane's accumulators (values 32 b + 8 (r / 4) + 4 h + r % 4 of its row) times `by` to its row of `units` 16-byte
// units, `at` bytes into the resource (kFar: nowhere).  All lanes of the wave call it.
template <class Op, int kBlocks>
__device__ __forceinline__ void store_row(rsrc_t to, int at, const f32x16 (&acc)[kBlocks], float by, int units, int h) {
  typedef typename Elem<Op>::T T;
  typedef T V4 __attribute__((ext_vector_type(4)));
  asm volatile("" : "+v"(at), "+v"(h));  // (as own_row)
#pragma unroll
  for (int b = 0; b < kBlocks; ++b)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      V4 x[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] = (T)(acc[b][4 * (g + i) + e] * by);
      if constexpr (Op::kEsz == 2) {
        // the halves of the wave trade: half 0 has all of group g's eight values, half 1 all of g + 1's
        const u32x2 lo = __builtin_bit_cast(u32x2, x[0]), hi = __builtin_bit_cast(u32x2, x[1]);
        const auto s0 = __builtin_amdgcn_permlane32_swap(lo[0], hi[0], false, false);
        const auto s1 = __builtin_amdgcn_permlane32_swap(lo[1], hi[1], false, false);
        const int u = 4 * b + g + h;
        __builtin_amdgcn_raw_buffer_store_b128(u32x4{s0[0], s1[0], s0[1], s1[1]}, to, u < units ? at + u * 16 : kFar, 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int u = 8 * b + 2 * (g + i) + h;
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x[i]), to, u < units ? at + u * 16 : kFar, 0, 0);
        }
      }
    }
}

// The rows of a wave, 32 from row `first` on, in an array of tokens `token` and heads `head` elements apart:
// the resource starts at the first row's token, `start` elements into the array being the
// unit's token 0 and its first head.
template <class Op>
__device__ __forceinline__ rsrc_t wave_rows(const void* p, int64_t start, int first_token, int64_t token) {
  return make_rsrc_u(static_cast<const char*>(p) + (start + first_token * token) * Op::kEsz, 0x7fffffffu);
}
// Where a row lies in it.
template <class Op>
__device__ __forceinline__ int row_at(int tokens, int64_t token, int heads, int64_t head) {
  return (tokens * (int)token + heads * (int)head) * Op::kEsz;
}

}  // namespace attn
}  // namespace fms

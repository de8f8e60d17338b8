// fms_attn_back.hip -- the pullback of attention over heads.
//
// With p_ij as in the forward, computed again from q, k and the kept maxima of its rows:
//   dv_j = sum_i p_ij do_i                     dp_ij = do_i v_j
//   ds_ij = p_ij (dp_ij - delta_i)             delta_i = sum_j p_ij dp_ij = do_i o_i
//   dq_i = scale sum_j ds_ij k_j               dk_j = scale sum_i ds_ij q_i
//
// Two kernels, one with a wave's rows in registers and the keys passing by (dq), one with its keys
// there and the rows passing by (dk, dv): seven products where one kernel would need five, but
// each sum stays in registers, in fp32, in a fixed order, with no atomics and no partial sums in
// memory; the heads that share a key head are rows of one run, so their sums are one too.
//
// The maximum goes before the scale, as in the forward, so that p is as exact for large scores as for small ones (a
// kept logarithm of the sum would be off by its own last bit: p by 8e-5 at scores of 1000).  The sums are made again by
// the first kernel, which divides by them at its end and leaves them to the second.
//
// delta takes o with what its rounding left (the forward keeps that): where one key has nearly all
// the weight, dp - delta is a small difference of nearly equal terms.  In 16-bit types p and ds go into their
// products as two values each, a rounding and what it left, and in fp16 both are scaled by powers of
// two: p by 2^15, dp - delta by a bound of its size from the norms of do and v, so that neither small
// probabilities nor small cotangents lose their bits.
//
// What bounds it, as measured (matrix cores busy, vector instructions issued, of the cycles; a card that has run for a
// while, the first passes take a tenth more):
//   128 documents of up to 180 tokens, masked, 16 heads of 64, bf16: dq 62 us (13 %, 39 %), dk and dv 82 (12 %,
//     37 %).  One to three tiles a workgroup: its loads at the start and its stores at the end, which three
//     and two waves a SIMD (accumulators and operands) hide in part.  (dq with four: 83, twenty registers spill.)
//   48 ragged documents of up to 1999 tokens, window 64, 12 heads of 64, fp16: norms 28, dq 137 (19 %, 50 %), dk and dv
//     179 (20 %, 45 %); tiles on the window's edge are half empty.
//   8192 causal tokens, 16 heads on 4 of 128, bf16: dq 587 (61 %, 53 %; four products' work, 0.94 PFLOP/s), dk and
//     dv 1220 and 23 for the join (40 %, 39 %; six, 0.68 PFLOP/s), with one wave a SIMD, whose exponentials nothing else
//     hides.  With p and ds rounded once both took a sixth less; gradients were then 1.4 to 1.5 times as far off as
//     their own rounding takes them.
//   16 sequences of up to 237 queries and 301 keys, 6 heads of 48, fp32: 41 (45 %) and 44 (43 %): the path of the
//     longest sequence's workgroups, one wave a SIMD; fp32 products run at about an eighth of the rate.
#include "fms_attn.hpp"

#include "../../include/flashmaxsim_hip.h"

namespace fms {
namespace attn {
namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// p in fp16 is held 2^15 times as large.
template <class Op>
constexpr float kShift = std::is_same<Op, OpF16>::value ? 15.0f : 0.0f;
template <class Op>
constexpr float kUnshift = std::is_same<Op, OpF16>::value ? 1.0f / 32768.0f : 1.0f;

// A power of two that brings what is at most 2 sqrt(a) sqrt(b) below one (1 where that says nothing).
__device__ __forceinline__ float scale_below_one(float a, float b) {
  const float bound = 2.0f * sqrtf(a) * sqrtf(b);
  if (!(bound > 1e-30f && bound < 1e30f)) return 1.0f;
  int e;
  frexpf(bound, &e);
  return ldexpf(1.0f, -e);
}

// The values of a fragment as floats.  (fp32: the whole fragment is bit-cast before an element is
// taken; element by element, this compiler shrinks the load behind it to its first word.)
template <class Op>
__device__ __forceinline__ float value(const u32x4& f, int e) {
  if constexpr (Op::kEsz == 4) {
    return __builtin_bit_cast(f32x4, f)[e];
  } else {
    typedef typename Elem<Op>::T T;
    typedef T V __attribute__((ext_vector_type(8)));
    return (float)__builtin_bit_cast(V, f)[e];
  }
}

// x[i][i] for i = lane % 32, in both halves of the wave.
__device__ __forceinline__ float diagonal(const f32x16& x, int lane) {
  const int i = lane & 31, r = 4 * (i >> 3) + (i & 3);
  float v = x[0];
#pragma unroll
  for (int j = 1; j < 16; ++j) v = r == j ? x[j] : v;
  return __shfl(v, i + 32 * ((i >> 2) & 1));
}

// Largest squared norms of a unit's v and do rows, in kAttnPeakParts parts.
__global__ void __launch_bounds__(256) attn_peaks_kernel(AttnArgs A, AttnGrads G) {
  __shared__ float lds[4][2];
  const int64_t unit = A.unit0 + blockIdx.x / kAttnPeakParts;
  const int part = blockIdx.x % kAttnPeakParts;
  const int64_t b = unit / A.kv_heads;
  const int hk = (int)(unit % A.kv_heads);
  const Span S = span_of(A, b);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int sub = lane >> 3, in = lane & 7;  // eight lanes a row
  float top[2] = {0.0f, 0.0f};
  const int width = A.units * 8;
  const auto norm = [&](const _Float16* p) {
    float s = 0.0f;
    typedef _Float16 V __attribute__((ext_vector_type(8)));
    for (int d = in * 8; d < width; d += 64) {
      const V v = *reinterpret_cast<const V*>(p + d);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += (float)v[e] * (float)v[e];
    }
    s += __shfl_xor(s, 1);
    s += __shfl_xor(s, 2);
    s += __shfl_xor(s, 4);
    return s < INFINITY ? s : 0.0f;  // (a row that is not finite has no say in the scale of the others)
  };
  const int step = kAttnPeakParts * 32, at = part * 32 + wave * 8 + sub;
  const _Float16* v = static_cast<const _Float16*>(A.v) + seq_at(A.vs, A.cu_k, b, S.k0) + hk * A.vs[2];
  for (int j = at; j < S.nk; j += step)
    if (!A.kmask || A.kmask[b * A.tk + j]) top[0] = fmaxf(top[0], norm(v + j * A.vs[1]));
  const _Float16* d = static_cast<const _Float16*>(G.dout) + S.q0 * A.heads * width;
  for (int r = at; r < S.nq * A.group; r += step) {
    const int t = token_of(r, A), head = hk * A.group + r - t * A.group;
    if (!A.qmask || A.qmask[b * A.tq + t]) top[1] = fmaxf(top[1], norm(d + ((int64_t)t * A.heads + head) * width));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    for (int o = 8; o < 64; o <<= 1) top[i] = fmaxf(top[i], __shfl_xor(top[i], o));
    if (lane == 0) lds[wave][i] = top[i];
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    const int i = threadIdx.x;
    G.peaks[(unit * kAttnPeakParts + part) * 2 + i] = fmaxf(fmaxf(lds[0][i], lds[1][i]), fmaxf(lds[2][i], lds[3][i]));
  }
}
__device__ __forceinline__ float peak(const float* peaks, int64_t unit, int which) {
  float x = peaks[(unit * kAttnPeakParts + (threadIdx.x & (kAttnPeakParts - 1))) * 2 + which];
#pragma unroll
  for (int o = 1; o < kAttnPeakParts; o <<= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}

template <class Op, int kD, int kWaves>
__global__ void __launch_bounds__(kWaves * 64) attn_dq_kernel(AttnArgs A, AttnGrads G, uint32_t tiles, uint32_t work) {
  typedef Tile<Op, kD> T;
  constexpr int kThreads = kWaves * 64;
  __shared__ __attribute__((aligned(1024))) char lds[4 * T::kBytes + kMaskSpan / 8];  // (one array: as forward)
  uint64_t* const words = reinterpret_cast<uint64_t*>(lds + 4 * T::kBytes);
  const uint32_t piece = piece_of(work);
  if (piece >= work) return;
  const uint32_t nth = piece / tiles, unit = A.unit0 + nth;
  const int tile = (int)(A.causal ? tiles - 1 - (piece - nth * tiles) : piece - nth * tiles);
  const int64_t b = unit / (uint32_t)A.kv_heads;
  const int hk = (int)(unit % (uint32_t)A.kv_heads);
  const Span S = span_of(A, b);
  const int nrows = S.nq * A.group;
  const int row0 = tile * (32 * kWaves);
  if (row0 >= nrows) return;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int h = lane >> 5;
  const int row = row0 + wave * 32 + (lane & 31);
  const int t = token_of(row, A), head = row - t * A.group;  // (of the key head's)
  const int wt = token_of(row0 + wave * 32, A);              // the wave's first token
  const int64_t at = rows_at(A, b, hk, S.q0) + row;
  const float top = row < nrows ? G.top[at] : 0.0f, base = top == -INFINITY ? 0.0f : top;
  const bool there = row < nrows && (!A.qmask || A.qmask[b * A.tq + t]);
  u32x4 q[T::kK], d[T::kK], o[T::kK], rest[T::kK];
  own_row<T>(q, wave_rows<Op>(A.q, seq_at(A.qs, A.cu_q, b, S.q0) + (int64_t)hk * A.group * A.qs[2], wt, A.qs[1]),
             there ? row_at<Op>(t - wt, A.qs[1], head, A.qs[2]) : kFar, A.units, h);
  const int64_t dim = A.units * (16 / Op::kEsz), width = A.heads * dim;
  const int64_t start = S.q0 * width + hk * A.group * dim;
  const int place = row < nrows ? row_at<Op>(t - wt, width, head, dim) : kFar;
  const int from = there ? place : kFar;  // (rows behind a mask are not read: zeros, as their results are)
  own_row<T>(d, wave_rows<Op>(G.dout, start, wt, width), from, A.units, h);
  own_row<T>(o, wave_rows<Op>(G.o, start, wt, width), from, A.units, h);
  if constexpr (Op::kEsz == 2) own_row<T>(rest, wave_rows<Op>(G.rest, start, wt, width), from, A.units, h);
  const Reach mine = keys_of(t, S, A);
  const auto reach = [&](int r) { return keys_of(token_of(r < nrows ? r : nrows - 1, A), S, A); };
  const int first = reach(row0).lo / kRows * kRows;
  const int last = reach(row0 + 32 * kWaves - 1).hi;
  Rows keys = {words, A.kmask != nullptr, first / kMaskSpan * kMaskSpan, 0};
  const auto gather = [&] {
    const uint8_t* km = A.kmask + b * A.tk;
    keys.gather<kThreads>(S.nk, [&](int j) { return km[j] != 0; });
  };
  if (keys.given && first < last) gather();
  f32x16 acc[T::kBlocks];
#pragma unroll
  for (int i = 0; i < T::kBlocks; ++i) acc[i] = f32x16{};
  if (!__syncthreads_or(there)) {  // padding: zeros, and no keys are read
    store_row<Op, T::kBlocks>(wave_rows<Op>(G.dq, start, wt, width), place, acc, 0.0f, A.units, h);
    if (h == 0 && row < nrows) G.delta[at] = G.level[at] = 0.0f;
    return;
  }
  const Reaches wide = reaches(reach(row0 + wave * 32), reach(row0 + wave * 32 + 31), __any(there));
  float delta = 0.0f, norm = 0.0f;
  {
    // by the same products as dp below, of which the diagonal is wanted: a row that sees one key has
    // o = v, and dp - delta is then zero and not a rounding
    f32x16 x = f32x16{};
#pragma unroll
    for (int kb = 0; kb < T::kK; ++kb) x = mma<Op>(o[kb], d[kb], x);
    delta = diagonal(x, lane);
    if constexpr (Op::kEsz == 2) {
      x = f32x16{};
#pragma unroll
      for (int kb = 0; kb < T::kK; ++kb) x = mma<Op>(rest[kb], d[kb], x);
      delta += diagonal(x, lane) * (1.0f / kRestScale<Op>);
    }
    if constexpr (kShift<Op> != 0.0f) {
#pragma unroll
      for (int kb = 0; kb < T::kK; ++kb)
#pragma unroll
        for (int e = 0; e < 8; ++e) norm = __builtin_fmaf(value<Op>(d[kb], e), value<Op>(d[kb], e), norm);
      norm += __builtin_bit_cast(float, lane_xor32(__builtin_bit_cast(uint32_t, norm), h));
    }
  }
  if (h == 0 && row < nrows) G.delta[at] = delta;
  float by = 1.0f;
  if constexpr (kShift<Op> != 0.0f) by = scale_below_one(norm, peak(G.peaks, unit, 0));
  const float c = factor(A);
  float l = 0.0f;  // of this half's keys
  if (A.scale < 0) negate<T>(q);

  const char* kbase = static_cast<const char*>(A.k) + (seq_at(A.ks, A.cu_k, b, S.k0) + (int64_t)hk * A.ks[2]) * Op::kEsz;
  const char* vbase = static_cast<const char*>(A.v) + (seq_at(A.vs, A.cu_k, b, S.k0) + (int64_t)hk * A.vs[2]) * Op::kEsz;
  const int64_t kstep = A.ks[1] * Op::kEsz, vstep = A.vs[1] * Op::kEsz;

  for (bool more = false; keys.span0 < last; keys.span0 += kMaskSpan, more = true) {
    const int from = first > keys.span0 ? first : keys.span0;
    const int to = last < keys.span0 + kMaskSpan ? last : keys.span0 + kMaskSpan;
    keys.to = to;
    if (more) {  // (every wave is through with the words, and with the buffers)
      landed();
      if (keys.given) gather();
      landed();
    }
    const auto request = [&](int j0, uint64_t bits, int buffer) {
      T::template request<kThreads>(lds + buffer * 2 * T::kBytes, kbase + j0 * kstep, (int)kstep, A.units, bits);
      T::template request<kThreads>(lds + (buffer * 2 + 1) * T::kBytes, vbase + j0 * vstep, (int)vstep, A.units, bits);
    };
    uint64_t bits, bits1;  // of this tile, and of the next
    int j0 = keys.next(from, bits);
    int buffer = 0;
    if (j0 < to) request(j0, bits, 0);
    while (j0 < to) {
      landed();
      const int j1 = keys.next(j0 + kRows, bits1);
      if (j1 < to) request(j1, bits1, buffer ^ 1);
      const char* const K = lds + buffer * 2 * T::kBytes;
      const char* const V = K + T::kBytes;
      const bool none = j0 >= wide.any.hi || j0 + kRows <= wide.any.lo;
      const int now = j0;
      const uint32_t w[2] = {(uint32_t)bits, (uint32_t)(bits >> 32)};
      j0 = j1;
      bits = bits1;
      buffer ^= 1;
      if (none) continue;  // (none of this wave's rows reaches here)
      const bool whole_tile = (w[0] & w[1]) == 0xffffffffu && now >= wide.all.lo && now + kRows <= wide.all.hi;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        f32x16 x = f32x16{}, y = f32x16{};
#pragma unroll
        for (int kb = 0; kb < T::kK; ++kb) {
          x = mma<Op>(T::rows(K, 32 * half, kb, lane), q[kb], x);
          y = mma<Op>(T::rows(V, 32 * half, kb, lane), d[kb], y);
        }
        if (!whole_tile) {
          const int j = now + 32 * half;
          const uint32_t keep = (w[half] & bits_between(mine.lo - j, mine.hi - j)) >> (4 * h);
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = masked(x[r], keep, r, -INFINITY);
        }
        float s[16], sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r] - base, c, kShift<Op>));
          sum += s[r];
          s[r] *= (y[r] - delta) * by;
          // (four at a time: all sixteen at once take as many registers more, and a wave of each SIMD with them: 8192
          // causal tokens, 16 heads on 4 of 128 in bf16, 917 us for 654, on a card that has just begun.  Not in fp32: a
          // second wave only shares the matrix cores, 8 sequences of 700 causal tokens, 8 heads on 4 of 64, 139 us for
          // 101)
          if (Op::kEsz == 2 && r % 4 == 3) asm volatile("" : "+v"(sum), "+v"(s[r]));
        }
        l += sum;
        constexpr int kPer = 32 / kGroups<Op>;
#pragma unroll
        for (int g = 0; g < kGroups<Op>; ++g) {
          const Operand<Op> ds = operand<Op>(s, g);
#pragma unroll
          for (int i = 0; i < T::kBlocks; ++i)
            acc[i] = mma(T::columns(K, 32 * half + kPer * g, i, lane), ds, acc[i]);
        }
      }
    }
  }
  l += __builtin_bit_cast(float, lane_xor32(__builtin_bit_cast(uint32_t, l), h));
  if (A.qmask && !there) {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) acc[i] = f32x16{};
    l = 0.0f;
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;  // (no key counts: the sums are zeros)
  store_row<Op, T::kBlocks>(wave_rows<Op>(G.dq, start, wt, width), place, acc, A.scale / by * inv, A.units, h);
  // (what the second kernel's exponents take, or in fp32, where that would cost bits, its exponentials are multiplied by)
  if (h == 0 && row < nrows)
    G.level[at] = Op::kEsz == 4 ? inv : inv > 0.0f ? 2.0f * kShift<Op> - __builtin_amdgcn_logf(l) : inv;
}

// `splits` workgroups share the rows of a tile of keys; with more than one their sums go to `parts`:
// (split, dk or dv, unit, key, value).
template <class Op, int kD, int kWaves>
__global__ void __launch_bounds__(kWaves * 64, 1)
    attn_dkv_kernel(AttnArgs A, AttnGrads G, float* parts, uint32_t splits, uint32_t tiles, uint32_t work) {
  typedef Tile<Op, kD> T;
  constexpr int kThreads = kWaves * 64;
  constexpr int kBuffer = 2 * T::kBytes + 3 * kRows * 4;  // q, do, top, delta, level
  __shared__ __attribute__((aligned(1024))) char lds[2 * kBuffer + kMaskSpan / 8];
  uint64_t* const words = reinterpret_cast<uint64_t*>(lds + 2 * kBuffer);
  const uint32_t piece = piece_of(work);
  if (piece >= work) return;
  const uint32_t shared = piece / splits, split = piece - shared * splits;
  const uint32_t nth = shared / tiles, unit = A.unit0 + nth;
  const int tile = (int)(shared - nth * tiles);  // (under a causal mask the first tiles have the most rows)
  const int64_t b = unit / (uint32_t)A.kv_heads;
  const int hk = (int)(unit % (uint32_t)A.kv_heads);
  const Span S = span_of(A, b);
  const int key0 = tile * (32 * kWaves);
  if (key0 >= S.nk) return;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int h = lane >> 5;
  const int key = key0 + wave * 32 + (lane & 31);
  const int wkey = key0 + wave * 32;  // the wave's first
  const bool there = key < S.nk && (!A.kmask || A.kmask[b * A.tk + key]);
  u32x4 k[T::kK], v[T::kK];  // (keys behind a mask are not read: zeros, as their results are)
  own_row<T>(k, wave_rows<Op>(A.k, seq_at(A.ks, A.cu_k, b, S.k0) + (int64_t)hk * A.ks[2], wkey, A.ks[1]),
             there ? row_at<Op>(key - wkey, A.ks[1], 0, 0) : kFar, A.units, h);
  own_row<T>(v, wave_rows<Op>(A.v, seq_at(A.vs, A.cu_k, b, S.k0) + (int64_t)hk * A.vs[2], wkey, A.vs[1]),
             there ? row_at<Op>(key - wkey, A.vs[1], 0, 0) : kFar, A.units, h);
  const auto reach = [&](int j) {  // in rows
    Reach r = tokens_of(j < S.nk ? j : S.nk - 1, S, A);
    r.lo *= A.group;
    r.hi *= A.group;
    return r;
  };
  const Reach mine = reach(key);
  int first = reach(key0).lo / kRows * kRows;
  int last = reach(key0 + 32 * kWaves - 1).hi;
  if (splits > 1) {  // an equal share of the row tiles that this tile of keys reaches
    const int64_t n = last > first ? (last - first + kRows - 1) / kRows : 0;
    const int end = first + (int)(n * (split + 1) / splits) * kRows;
    first += (int)(n * split / splits) * kRows;
    last = end < last ? end : last;
  }
  Rows rows = {words, A.qmask != nullptr, first / kMaskSpan * kMaskSpan, 0};
  const auto gather = [&] {
    const uint8_t* qm = A.qmask + b * A.tq;
    rows.gather<kThreads>(S.nq * A.group, [&](int r) { return qm[token_of(r, A)] != 0; });
  };
  if (rows.given && first < last) gather();
  const int64_t width = A.units * (16 / Op::kEsz);
  const int64_t wide_row = A.kv_heads * width, start = S.k0 * wide_row + hk * width;
  const int at = key < S.nk ? row_at<Op>(key - wkey, wide_row, 0, 0) : kFar;
  f32x16 dk[T::kBlocks], dv[T::kBlocks];
#pragma unroll
  for (int i = 0; i < T::kBlocks; ++i) dk[i] = dv[i] = f32x16{};
  if (!__syncthreads_or(there)) last = first;  // (padding: zeros, and no rows are read)
  const Reaches wide = reaches(reach(key0 + wave * 32), reach(key0 + wave * 32 + 31), __any(there));
  const float c = factor(A);
  if (A.scale < 0) negate<T>(k);
  float by = 1.0f;
  if constexpr (kShift<Op> != 0.0f) by = scale_below_one(peak(G.peaks, unit, 1), peak(G.peaks, unit, 0));

  const char* qbase = static_cast<const char*>(A.q) +
                      (seq_at(A.qs, A.cu_q, b, S.q0) + (int64_t)hk * A.group * A.qs[2]) * Op::kEsz;
  const char* dbase = static_cast<const char*>(G.dout) + (S.q0 * A.heads + hk * A.group) * width * Op::kEsz;
  const int64_t stat = rows_at(A, b, hk, S.q0);

  for (bool more = false; rows.span0 < last; rows.span0 += kMaskSpan, more = true) {
    const int from = first > rows.span0 ? first : rows.span0;
    const int to = last < rows.span0 + kMaskSpan ? last : rows.span0 + kMaskSpan;
    rows.to = to;
    if (more) {  // (every wave is through with the words, and with the buffers)
      landed();
      if (rows.given) gather();
      landed();
    }
    const auto request = [&](int r0, uint64_t bits, int buffer) {
      char* const base = lds + buffer * kBuffer;
      T::template request_rows<kThreads>(base, qbase, A.qs[1], A.qs[2], A.units, r0, A, bits);
      T::template request_rows<kThreads>(base + T::kBytes, dbase, A.heads * width, width, A.units, r0, A, bits);
      static_assert(kWaves >= 3, "a wave for each of a row's numbers");
      if (wave < 3) {
        const float* const of = wave == 0 ? G.top : wave == 1 ? G.delta : G.level;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(make_rsrc_u(of + stat + r0, 0x7fffffffu),
                                                 (lds_ptr)(base + 2 * T::kBytes + wave * kRows * 4), 4,
                                                 r0 + lane < to ? lane * 4 : kFar, 0, 0, 0);
      }
    };
    uint64_t bits, bits1;  // of this tile, and of the next
    int r0 = rows.next(from, bits);
    int buffer = 0;
    if (r0 < to) request(r0, bits, 0);
    while (r0 < to) {
      landed();
      const int r1 = rows.next(r0 + kRows, bits1);
      if (r1 < to) request(r1, bits1, buffer ^ 1);
      const char* const Q = lds + buffer * kBuffer;
      const char* const D = Q + T::kBytes;
      const float* const top = reinterpret_cast<const float*>(D + T::kBytes);
      const bool none = r0 >= wide.any.hi || r0 + kRows <= wide.any.lo;
      const int now = r0;
      const uint32_t w[2] = {(uint32_t)bits, (uint32_t)(bits >> 32)};
      r0 = r1;
      bits = bits1;
      buffer ^= 1;
      if (none) continue;  // (no row here reaches this wave's keys)
      const bool whole_tile = (w[0] & w[1]) == 0xffffffffu && now >= wide.all.lo && now + kRows <= wide.all.hi;
      // fragments: of the rows by values, and (two groups in turn) of the values by rows
      // (wide 16-bit heads only, whose registers leave room for one wave of a SIMD: 1317 -> 1077 us for 8192 causal
      // tokens, 16 heads on 4 of 128 in bf16; narrow ones have other waves to hide a read behind, 165 -> 180
      // us for 48 ragged documents, 12 heads of 64 in fp16, and 32-bit ones no registers left)
      constexpr bool kAhead = Op::kEsz == 2 && kD > 64;
      u32x4 fq[T::kK], fd[T::kK], cq[2][T::kBlocks], cd[2][T::kBlocks];
      const auto read_rows = [&](int half) {
#pragma unroll
        for (int kb = 0; kb < T::kK; ++kb) {
          fq[kb] = T::rows(Q, 32 * half, kb, lane);
          fd[kb] = T::rows(D, 32 * half, kb, lane);
        }
      };
      constexpr int kPer = 32 / kGroups<Op>;
      const auto read_columns = [&](int half, int g) {
#pragma unroll
        for (int i = 0; i < T::kBlocks; ++i) {
          cd[g & 1][i] = T::columns(D, 32 * half + kPer * g, i, lane);
          cq[g & 1][i] = T::columns(Q, 32 * half + kPer * g, i, lane);
        }
      };
      if (kAhead) read_rows(0);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (kAhead) asked();
        f32x16 x = f32x16{}, y = f32x16{};
#pragma unroll
        for (int kb = 0; kb < T::kK; ++kb) {
          x = mma<Op>(kAhead ? fq[kb] : T::rows(Q, 32 * half, kb, lane), k[kb], x);
          y = mma<Op>(kAhead ? fd[kb] : T::rows(D, 32 * half, kb, lane), v[kb], y);
        }
        if (kAhead) read_columns(half, 0);
        float p[16], ds[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float* const of = top + 32 * half + 8 * g + 4 * h;
          const f32x4 t4 = *reinterpret_cast<const f32x4*>(of);
          const f32x4 d4 = *reinterpret_cast<const f32x4*>(of + kRows);
          const f32x4 l4 = *reinterpret_cast<const f32x4*>(of + 2 * kRows);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * g + e;
            if constexpr (Op::kEsz == 4)
              p[r] = __builtin_amdgcn_exp2f((x[r] - t4[e]) * c) * l4[e];
            else
              p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r] - t4[e], c, l4[e]));
            ds[r] = p[r] * ((y[r] - d4[e]) * by);
          }
        }
        if (!whole_tile) {
          const int r0h = now + 32 * half;
          const uint32_t keep = ((half ? w[1] : w[0]) & bits_between(mine.lo - r0h, mine.hi - r0h)) >> (4 * h);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            p[r] = masked(p[r], keep, r, 0.0f);
            ds[r] = masked(ds[r], keep, r, 0.0f);
          }
        }
        if (kAhead && half == 0) read_rows(1);
#pragma unroll
        for (int g = 0; g < kGroups<Op>; ++g) {
          if (kAhead && g + 1 < kGroups<Op>) read_columns(half, g + 1);
          if (kAhead) asked();
          const Operand<Op> po = operand<Op>(p, g), so = operand<Op>(ds, g);
#pragma unroll
          for (int i = 0; i < T::kBlocks; ++i) {
            dv[i] = mma(kAhead ? cd[g & 1][i] : T::columns(D, 32 * half + kPer * g, i, lane), po, dv[i]);
            dk[i] = mma(kAhead ? cq[g & 1][i] : T::columns(Q, 32 * half + kPer * g, i, lane), so, dk[i]);
          }
        }
      }
    }
  }
  if (A.kmask && !there)
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) dk[i] = dv[i] = f32x16{};
  const float by_k = A.scale * kUnshift<Op> / by;
  if (splits > 1) {
    if (key >= S.nk) return;
    const int64_t units = A.seqs * A.kv_heads;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float* const to = parts + (((int64_t)(split * 2 + which) * units + unit) * A.tk + key) * kD;
      const float scale = which ? kUnshift<Op> : by_k;
#pragma unroll
      for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = (which ? dv[i][4 * g + e] : dk[i][4 * g + e]) * scale;
          *reinterpret_cast<f32x4*>(to + 32 * i + 8 * g + 4 * h) = x;
        }
    }
    return;
  }
  store_row<Op, T::kBlocks>(wave_rows<Op>(G.dk, start, wkey, wide_row), at, dk, by_k, A.units, h);
  store_row<Op, T::kBlocks>(wave_rows<Op>(G.dv, start, wkey, wide_row), at, dv, kUnshift<Op>, A.units, h);
}

// The splits' sums of dk (blockIdx.y 0) and dv (1), four values a thread.
template <class Op, int kD>
__global__ void __launch_bounds__(256) attn_dkv_join_kernel(AttnArgs A, AttnGrads G, const float* parts, int splits) {
  typedef typename Elem<Op>::T E;
  typedef E V4 __attribute__((ext_vector_type(4)));
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, row = i / (kD / 4);  // (unit, key)
  const int d = (int)(i % (kD / 4)) * 4, width = A.units * (16 / Op::kEsz);
  const int64_t rows = A.seqs * A.kv_heads * A.tk;
  const uint32_t unit = row / (uint32_t)A.tk, key = row - unit * (uint32_t)A.tk;
  if (row >= rows || d >= width) return;
  const int64_t b = unit / (uint32_t)A.kv_heads;
  const int hk = (int)(unit % (uint32_t)A.kv_heads);
  const Span S = span_of(A, b);
  if ((int)key >= S.nk) return;
  f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int j = 0; j < splits; ++j) s += *reinterpret_cast<const f32x4*>(parts + ((j * 2 + blockIdx.y) * rows + row) * kD + d);
  V4 x;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = (E)s[e];
  *reinterpret_cast<V4*>(static_cast<E*>(blockIdx.y ? G.dv : G.dk) + ((S.k0 + key) * A.kv_heads + hk) * width + d) = x;
}

// (Four waves a workgroup: two, where four leave CUs idle, gain nothing -- 16 sequences of 237 queries and 301 keys, 6
// heads of 48 in fp32, dq 38 us with four and 41 with two, dk and dv 42 and 45.)
constexpr int kWaves = 4;

template <class Op, int kD>
hipError_t launch_dq(const AttnArgs& a, const AttnGrads& g, hipStream_t stream) {
  const int64_t tiles = cdiv((int64_t)a.tq * a.group, 32 * kWaves);
  if (!tiles) return hipSuccess;
  return by_units(a, tiles, [&](const AttnArgs& part, int64_t n) {
    hipLaunchKernelGGL((attn_dq_kernel<Op, kD, kWaves>), dim3(piece_blocks(n * tiles)), dim3(kWaves * 64), 0, stream,
                       part, g, (uint32_t)tiles, (uint32_t)(n * tiles));
  });
}

// Few workgroups of many rows each: the rows of a tile of keys are shared out, eight tiles of them to a
// workgroup at least, until there are four workgroups to a CU.  (Their sums cost 2 * 4 bytes a value and
// split, written and read; 8192 causal tokens, 16 heads on 4 of 128 in bf16, fragments read where they are
// used: 1583 us unsplit, 1290 + 23 for the join in four.)
int64_t dkv_splits(const AttnArgs& a) {
  const int64_t work = a.seqs * a.kv_heads * cdiv(a.tk, 32 * kWaves);
  const int64_t most = cdiv((int64_t)a.tq * a.group, kRows) / 8, wanted = work ? 1024 / work : 1;
  const int64_t n = wanted < most ? wanted : most;
  return n < 1 ? 1 : n > 8 ? 8 : n;
}

template <class Op, int kD>
hipError_t launch_dkv(const AttnArgs& a, const AttnGrads& g, float* parts, int64_t splits, hipStream_t stream) {
  const int64_t units = a.seqs * a.kv_heads, tiles = cdiv(a.tk, 32 * kWaves);
  if (!tiles) return hipSuccess;
  const hipError_t e = by_units(a, tiles * splits, [&](const AttnArgs& part, int64_t n) {
    const int64_t work = n * tiles * splits;
    hipLaunchKernelGGL((attn_dkv_kernel<Op, kD, kWaves>), dim3(piece_blocks(work)), dim3(kWaves * 64), 0, stream, part,
                       g, parts, (uint32_t)splits, (uint32_t)tiles, (uint32_t)work);
  });
  if (e != hipSuccess) return e;
  if (splits > 1)
    hipLaunchKernelGGL((attn_dkv_join_kernel<Op, kD>), dim3((unsigned)cdiv(units * a.tk * (kD / 4), 256), 2), dim3(256),
                       0, stream, a, g, static_cast<const float*>(parts), (int)splits);
  return hipGetLastError();
}

template <class Op, int kD>
hipError_t pullback_dim(const AttnArgs& a, const AttnGrads& g, hipStream_t stream) {
  hipError_t e = hipSuccess;
  if (std::is_same<Op, OpF16>::value)
    e = by_units(a, kAttnPeakParts, [&](const AttnArgs& part, int64_t n) {
      hipLaunchKernelGGL(attn_peaks_kernel, dim3((unsigned)(n * kAttnPeakParts)), dim3(256), 0, stream, part, g);
    });
  if (e == hipSuccess) e = launch_dq<Op, kD>(a, g, stream);
  if (e == hipSuccess) e = launch_dkv<Op, kD>(a, g, static_cast<float*>(g.parts), dkv_splits(a), stream);
  return e;
}
template <class Op>
hipError_t pullback_op(const AttnArgs& a, const AttnGrads& g, hipStream_t stream) {
  switch (instance_dim(a)) {
    case 32: return pullback_dim<Op, 32>(a, g, stream);
    case 64: return pullback_dim<Op, 64>(a, g, stream);
    default: return pullback_dim<Op, 128>(a, g, stream);
  }
}

}  // namespace
}  // namespace attn

int64_t attn_pullback_bytes(const AttnArgs& a) {
  const int64_t splits = attn::dkv_splits(a);
  return splits > 1 ? splits * 2 * a.seqs * a.kv_heads * a.tk * attn::instance_dim(a) * 4 : 0;
}

hipError_t attn_pullback(const AttnArgs& a, const AttnGrads& g, hipStream_t stream) {
  switch (a.dtype) {
    case FMS_F16: return attn::pullback_op<OpF16>(a, g, stream);
    case FMS_BF16: return attn::pullback_op<OpBF16>(a, g, stream);
    default: return attn::pullback_op<OpF32>(a, g, stream);
  }
}

}  // namespace fms

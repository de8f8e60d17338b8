// fms_attn.hip -- attention over heads, forward.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i k_j) / sum_j exp(scale q_i k_j)
// over the keys j that count for row i (masks, causal, window); 0 where none does.
//
// One pass over the keys: a running maximum m and sum l per row, and what was summed so far
// rescaled where m grows.  Scores, m, l and the sums of values are fp32; p is rounded once to
// the feature type for its product with v, which costs about what rounding o costs, and l is the
// sum of the p as rounded: o is then a mean of the values with weights that are a little off, and the
// pullback's delta, do . o, is off by no more than those weights' share of ds.  (p is at most 1
// and exactly 1 at the maximum, so a row that attends to one key is exact.)
#include <cmath>

#include "fms_attn.hpp"

#include "../../include/flashmaxsim_hip.h"
#include "fms_group.hpp"

namespace fms {
namespace attn {
namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// What the splits of a row leave for their join: sums of values, maximum and sum.
struct Parts {
  float* acc;   // (piece, value, row) pieces of 32 rows
  float* stat;  // (piece, 2, row)
  int splits;
  int keys;  // of a split
};

template <class Op, int kD, int kWaves, bool kSplit>
__global__ void __launch_bounds__(kWaves * 64) attn_forward_kernel(AttnArgs A, AttnOut out, Parts P,
                                                                   int tiles, int64_t work) {
  typedef Tile<Op, kD> T;
  typedef typename Elem<Op>::T E;
  constexpr int kThreads = kWaves * 64;
  // p in fp16 is held 2^10 times as large, so that small ones keep their bits
  constexpr float kShift = std::is_same<Op, OpF16>::value ? 10.0f : 0.0f;
  __shared__ __attribute__((aligned(1024))) char lds[4 * T::kBytes];
  __shared__ uint32_t words[kMaskSpan / 32];
  const int64_t piece = piece_of(work);
  if (piece >= work) return;
  const int split = kSplit ? (int)(piece % P.splits) : 0;
  const int64_t whole = kSplit ? piece / P.splits : piece;
  const int64_t unit = whole / tiles;
  // (under a causal mask the last tiles have the most keys: they start first)
  const int tile = A.causal ? tiles - 1 - (int)(whole % tiles) : (int)(whole % tiles);
  const int64_t b = unit / A.kv_heads;
  const int hk = (int)(unit % A.kv_heads);
  const Span S = span_of(A, b);
  const int nrows = S.nq * A.group;
  const int row0 = tile * (32 * kWaves);
  if (row0 >= nrows) return;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int h = lane >> 5;
  const int row = row0 + wave * 32 + (lane & 31);
  const int t = token_of(row, A), head = hk * A.group + row - t * A.group;
  const bool there = row < nrows && (!A.qmask || A.qmask[b * A.tq + t]);
  Reach mine = there ? keys_of(t, S, A) : Reach{0, 0};
  // of the whole workgroup (reaches grow with the token), and of all of this wave's rows
  const int rlast = row0 + 32 * kWaves < nrows ? row0 + 32 * kWaves - 1 : nrows - 1;
  int first = keys_of(token_of(row0, A), S, A).lo / kRows * kRows;
  int last = keys_of(token_of(rlast, A), S, A).hi;
  if constexpr (kSplit) {
    const int from = split * P.keys;
    first = first > from ? first : from;
    last = last < from + P.keys ? last : from + P.keys;
  }
  const Reach inner = common(mine);

  const char* qrow = static_cast<const char*>(A.q) +
                     (seq_at(A.qs, A.cu_q, b, S.q0) + (int64_t)t * A.qs[1] + (int64_t)head * A.qs[2]) * Op::kEsz;
  u32x4 q[T::kK];
  own_row<T>(q, qrow, there, A.units, h);
  const float c = fabsf(A.scale) * kLog2e;
  if (A.scale < 0) negate<T>(q);
  const char* kbase = static_cast<const char*>(A.k) + (seq_at(A.ks, A.cu_k, b, S.k0) + (int64_t)hk * A.ks[2]) * Op::kEsz;
  const char* vbase = static_cast<const char*>(A.v) + (seq_at(A.vs, A.cu_k, b, S.k0) + (int64_t)hk * A.vs[2]) * Op::kEsz;
  const int64_t kstep = A.ks[1] * Op::kEsz, vstep = A.vs[1] * Op::kEsz;

  f32x16 acc[T::kBlocks];
#pragma unroll
  for (int i = 0; i < T::kBlocks; ++i) acc[i] = f32x16{};
  float m = -INFINITY, l = 0.0f;

  for (int span0 = first / kMaskSpan * kMaskSpan; span0 < last; span0 += kMaskSpan) {
    const int from = first > span0 ? first : span0;
    const int to = last < span0 + kMaskSpan ? last : span0 + kMaskSpan;
    if (A.kmask) {
      landed();
      const uint8_t* km = A.kmask + b * A.tk;
      mask_words<kThreads>(words, span0, S.nk, [&](int j) { return km[j] != 0; });
      landed();
    }
    const auto bits_of = [&](int j0) -> uint32_t {  // of keys j0 .. j0 + 31, which may end the keys
      const uint32_t there = bits_between(0, to - j0);
      return A.kmask && there ? rfl32(words[(j0 - span0) / 32]) & there : there;
    };
    const auto next = [&](int j0) {  // the first tile from j0 on that has keys
      while (j0 < to && !(bits_of(j0) | bits_of(j0 + 32))) j0 += kRows;
      return j0;
    };
    const auto request = [&](int j0, int buffer) {
      const uint32_t w0 = bits_of(j0), w1 = bits_of(j0 + 32);
      const auto ok = [&](int r) { return ((r < 32 ? w0 : w1) >> (r & 31) & 1u) != 0; };
      T::template request<kThreads>(lds + buffer * 2 * T::kBytes, kbase + j0 * kstep, (int)kstep, A.units, ok);
      T::template request<kThreads>(lds + (buffer * 2 + 1) * T::kBytes, vbase + j0 * vstep, (int)vstep, A.units, ok);
    };
    int j0 = next(from);
    int buffer = 0;
    if (j0 < to) request(j0, 0);
    while (j0 < to) {
      landed();
      const int j1 = next(j0 + kRows);
      if (j1 < to) request(j1, buffer ^ 1);
      const char* const K = lds + buffer * 2 * T::kBytes;
      const char* const V = K + T::kBytes;
      float s[2][16];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        f32x16 x = f32x16{};
#pragma unroll
        for (int kb = 0; kb < T::kK; ++kb) x = mma<Op>(T::rows(K, 32 * half, kb, lane), q[kb], x);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[half][r] = x[r];
      }
      const uint32_t w0 = bits_of(j0), w1 = bits_of(j0 + 32);
      const bool whole_tile = (w0 & w1) == 0xffffffffu && j0 >= inner.lo && j0 + kRows <= inner.hi;
      uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
      if (!whole_tile) {
        keep[0] = (w0 & bits_between(mine.lo - j0, mine.hi - j0)) >> (4 * h);
        keep[1] = (w1 & bits_between(mine.lo - j0 - 32, mine.hi - j0 - 32)) >> (4 * h);
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[half][r] = (keep[half] >> (8 * (r >> 2) + (r & 3))) & 1u ? s[half][r] : -INFINITY;
      }
      // (NaN scores are ignored here and make p, and with it the row, NaN)
      float top = m;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int r = 0; r < 16; r += 2) top = max3_ieee(s[half][r], s[half][r + 1], top);
      top = merge_halves_max(top);
      if (__any(top > m)) {
        const float by = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - top) * c);
        l *= by;
#pragma unroll
        for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][r] *= by;
        m = top;
      }
      const float off = m == -INFINITY ? 0.0f : kShift - m * c;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[half][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[half][r], c, off));
      if (!whole_tile) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[half][r] = (keep[half] >> (8 * (r >> 2) + (r & 3))) & 1u ? s[half][r] : 0.0f;
      }
      float sum[2] = {0.0f, 0.0f};
      constexpr int kPer = 32 / kGroups<Op>;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int g = 0; g < kGroups<Op>; ++g) {
          const u32x4 p = operand<Op>(s[half], g);
          sum[half] = add_operand<Op>(p, sum[half]);
#pragma unroll
          for (int i = 0; i < T::kBlocks; ++i)
            acc[i] = mma<Op>(T::columns(V, 32 * half + kPer * g, i, lane), p, acc[i]);
        }
      l += sum[0] + sum[1];
      j0 = j1;
      buffer ^= 1;
    }
  }
  // both halves of the wave summed other keys of the same row
  l += __builtin_bit_cast(float, lane_xor32(__builtin_bit_cast(uint32_t, l), h));
  if constexpr (kSplit) {
    float* to = P.acc + (piece * (kWaves * 32 * kD) + wave * 32 * kD);
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) to[(32 * i + acc_row(r, h)) * 32 + (lane & 31)] = acc[i][r];
    float* st = P.stat + (piece * kWaves + wave) * 64;
    st[lane] = h ? l : m;
    return;
  }
  if (row >= nrows) return;
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  const bool vec = A.dim % 4 == 0 && aligned(out.o) && aligned(out.rest);
  const int64_t at = ((S.q0 + t) * A.heads + head) * (int64_t)A.dim;
  store_row<Op, T::kBlocks>(static_cast<E*>(out.o) + at, acc, inv, A.dim, vec, h);
  if (out.lse && h == 0)
    out.lse[rows_at(A, b, hk, S.q0) + row] = l > 0.0f || l != l ? m * c + __builtin_amdgcn_logf(l) - kShift : -INFINITY;
  if (Op::kEsz == 2 && out.rest) {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float o = acc[i][r] * inv;
        acc[i][r] = (o - (float)(E)o) * kRestScale<Op>;
      }
    store_row<Op, T::kBlocks>(static_cast<E*>(out.rest) + at, acc, 1.0f, A.dim, vec, h);
  }
}

template <class E>
__global__ void __launch_bounds__(256) attn_pack_kernel(E* to, const E* from, int64_t s0, int64_t s1, int64_t s2,
                                                        int64_t tokens, int64_t heads, int dim, int packed,
                                                        int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int d = (int)(i % packed);
    const int64_t r = i / packed, hd = r % heads, t = r / heads;
    to[i] = d < dim ? from[t / tokens * s0 + t % tokens * s1 + hd * s2 + d] : (E)0;
  }
}

// One wave a token row.
template <class E>
__global__ void __launch_bounds__(256) attn_gap_kernel(E* out, const int32_t* cu, int64_t seqs, int64_t rows,
                                                       int64_t most, int64_t width) {
  const int64_t stride = (int64_t)gridDim.x * 4;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += stride) {
    // the last sequence that starts at r or before
    int64_t a = 0, e = seqs;  // cu[a] - 1 <= r < cu[e] - 1, as if cu[seqs] were past all
    const bool before = seqs == 0 || r < (int64_t)cu[0] - 1;
    while (!before && e - a > 1) {
      const int64_t mid = (a + e) / 2;
      if ((int64_t)cu[mid] - 1 <= r) a = mid;
      else e = mid;
    }
    if (!before && r < (int64_t)cu[a + 1] - 1 && r - ((int64_t)cu[a] - 1) < most) continue;
    for (int64_t i = threadIdx.x & 63; i < width; i += 64) out[r * width + i] = (E)0;
  }
}

template <class F>
hipError_t by_type(int32_t dtype, F&& f) {
  switch (dtype) {
    case FMS_F16: return f(OpF16());
    case FMS_BF16: return f(OpBF16());
    default: return f(OpF32());
  }
}

template <class Op, int kD, int kWaves>
hipError_t forward_waves(const AttnArgs& a, const AttnOut& out, hipStream_t stream) {
  const int64_t tiles = cdiv((int64_t)a.tq * a.group, 32 * kWaves), units = a.seqs * a.kv_heads;
  const int64_t work = units * tiles;
  hipLaunchKernelGGL((attn_forward_kernel<Op, kD, kWaves, false>), dim3(piece_blocks(work)), dim3(kWaves * 64), 0,
                     stream, a, out, Parts{}, (int)tiles, work);
  return hipGetLastError();
}

template <class Op, int kD>
hipError_t forward_dim(const AttnArgs& a, const AttnOut& out, hipStream_t stream) {
  if ((int64_t)a.tq * a.group <= 32) return forward_waves<Op, kD, 1>(a, out, stream);
  return forward_waves<Op, kD, 4>(a, out, stream);
}

template <class Op>
hipError_t forward_op(const AttnArgs& a, const AttnOut& out, hipStream_t stream) {
  if (a.dim <= 32) return forward_dim<Op, 32>(a, out, stream);
  if (a.dim <= 64) return forward_dim<Op, 64>(a, out, stream);
  return forward_dim<Op, 128>(a, out, stream);
}

}  // namespace
}  // namespace attn

hipError_t attn_pack(int32_t dtype, void* to, const void* from, const int64_t* st, int64_t seqs, int64_t tokens,
                     int64_t heads, int32_t dim, int32_t packed_dim, hipStream_t stream) {
  const int64_t n = seqs * tokens * heads * packed_dim;
  if (n == 0) return hipSuccess;
  const int64_t blocks = attn::cdiv(n, 256) < 8192 ? attn::cdiv(n, 256) : 8192;
  if (dtype == FMS_F32)
    hipLaunchKernelGGL((attn::attn_pack_kernel<uint32_t>), dim3((unsigned)blocks), dim3(256), 0, stream,
                       static_cast<uint32_t*>(to), static_cast<const uint32_t*>(from), st[0], st[1], st[2], tokens,
                       heads, (int)dim, (int)packed_dim, n);
  else
    hipLaunchKernelGGL((attn::attn_pack_kernel<uint16_t>), dim3((unsigned)blocks), dim3(256), 0, stream,
                       static_cast<uint16_t*>(to), static_cast<const uint16_t*>(from), st[0], st[1], st[2], tokens,
                       heads, (int)dim, (int)packed_dim, n);
  return hipGetLastError();
}

hipError_t attn_zero_gaps(int32_t dtype, void* out, const int32_t* cu, int64_t seqs, int64_t rows, int64_t most,
                          int64_t width, hipStream_t stream) {
  if (rows == 0 || width == 0) return hipSuccess;
  const int64_t blocks = attn::cdiv(rows, 4) < 8192 ? attn::cdiv(rows, 4) : 8192;
  if (dtype == FMS_F32)
    hipLaunchKernelGGL((attn::attn_gap_kernel<uint32_t>), dim3((unsigned)blocks), dim3(256), 0, stream,
                       static_cast<uint32_t*>(out), cu, seqs, rows, most, width);
  else
    hipLaunchKernelGGL((attn::attn_gap_kernel<uint16_t>), dim3((unsigned)blocks), dim3(256), 0, stream,
                       static_cast<uint16_t*>(out), cu, seqs, rows, most, width);
  return hipGetLastError();
}

hipError_t attn_forward(const AttnArgs& a, const AttnOut& out, hipStream_t stream) {
  return attn::by_type(a.dtype, [&](auto op) { return attn::forward_op<decltype(op)>(a, out, stream); });
}

}  // namespace fms

// fms_attn.hip -- attention over heads, forward.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i k_j) / sum_j exp(scale q_i k_j)
// over the keys j that count for row i (masks, causal, window); 0 where none does.
//
// One pass over the keys: a running maximum m and sum l per row, and what was summed so far
// rescaled where m grows.  Scores, p, m, l and the sums of values are fp32; in 16-bit types p goes
// into its product with v as two values, a rounding and what it left.
//
// The rows of a key head's group of query heads are one run, row = token * group + head, 32 to a wave: a
// tile of 64 keys in LDS serves all of them.  The scores are formed transposed, K Q^T, so that a lane
// has half the keys of one row: maximum and sum are a lane's own but for one exchange, and p lies as
// the product with v wants it.  v is read by columns through the transposing LDS read.  While a tile is
// worked on the next is on its way into LDS.  Masked rows and keys are not loaded, tiles in which no
// key counts are skipped.
//
// What bounds it, as measured (a card that has run for a while; the first passes take a tenth more):
//   256 documents of up to 180 tokens, masked, 12 heads of 64, bf16: 66 us.  Vector
//     instructions (about 9 a score, one of them at a quarter of the rate) are issued in 53 % of the cycles, the
//     matrix cores busy in 11 %: a workgroup has one to three tiles, whose first loads and last stores
//     other workgroups of the CU hide in part.
//   8192 causal tokens, 16 heads on 4 of 128, bf16: 507 us, three products' work (p in two values), 0.81
//     PFLOP/s of it, matrix cores busy in 53 % of the cycles, vector units in 60; one rounding of p took a fifth
//     less, and results were 1.4 times as far off.
//   one token on 32768 keys, 16 heads on 4 of 128, bf16: 20 us and 5 for the join, 67 MB at 3.4 TB/s:
//     512 workgroups of a wave have four tiles each, and wait for the first.
#include <algorithm>
#include <cmath>

#include "fms_attn.hpp"

#include "../../include/flashmaxsim_hip.h"

namespace fms {
namespace attn {
namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Where a row's keys are split among workgroups: what each leaves for the join.
struct Parts {
  float* acc;   // (piece, row of the tile, value): sums of values
  float* stat;  // (piece, row of the tile, 2): maximum and sum
  int splits;
  int keys;  // of a split, a multiple of kRows
};

// Few workgroups of many keys each leave most of the card idle: their keys are split, 256 to a
// workgroup at least, until there are two to a CU (16 heads on 4 of 128 values in bf16, one token, 32768
// keys: 1414 us in 4 workgroups, 20 and 5 for the join in 512).  Above 128 workgroups none are: single tokens of 16
// sequences on 8192 keys each, 32 heads on 8 of 128 in bf16, take 111 us in 128 times four, those of 17 sequences 337
// in 136.
struct SplitPlan {
  int64_t tiles, pieces, keys, splits, slots;
};
int waves_of(const AttnArgs& a) { return (int64_t)a.tq * a.group <= 32 ? 1 : 4; }
SplitPlan split_plan(const AttnArgs& a) {
  SplitPlan p;
  const int rows = 32 * waves_of(a);
  p.tiles = cdiv((int64_t)a.tq * a.group, rows);
  p.pieces = a.seqs * a.kv_heads * p.tiles;
  const int64_t wanted = p.pieces <= 128 ? 512 / p.pieces : 1;
  p.keys = (cdiv(a.tk, wanted) + 255) / 256 * 256;
  p.splits = a.tk > p.keys ? cdiv(a.tk, p.keys) : 1;
  p.slots = p.splits > 1 ? p.pieces * p.splits * rows : 0;
  return p;
}

// p in fp16 is held 2^10 times as large, so that small ones keep their bits.
template <class Op>
constexpr float kShift = std::is_same<Op, OpF16>::value ? 10.0f : 0.0f;

template <class Op, int kD, int kWaves, bool kSplit>
__global__ void __launch_bounds__(kWaves * 64, (kSimdWaves<Op, kD, kWaves>))
    attn_forward_kernel(AttnArgs A, AttnOut out, Parts P, uint32_t tiles, uint32_t work) {
  typedef Tile<Op, kD> T;
  typedef typename Elem<Op>::T E;
  constexpr int kThreads = kWaves * 64;
  // (one array: beside a second one the compiler waits for all loads into LDS before it reads there)
  __shared__ __attribute__((aligned(1024))) char lds[4 * T::kBytes + kMaskSpan / 8];
  uint64_t* const words = reinterpret_cast<uint64_t*>(lds + 4 * T::kBytes);
  const uint32_t piece = piece_of(work);
  if (piece >= work) return;
  const uint32_t whole = kSplit ? piece / (uint32_t)P.splits : piece;
  const int split = (int)(piece - whole * (kSplit ? (uint32_t)P.splits : 1u));
  const uint32_t nth = whole / tiles, unit = A.unit0 + nth;
  // (under a causal mask the last tiles have the most keys: they start first)
  const int tile = (int)(A.causal ? tiles - 1 - (whole - nth * tiles) : whole - nth * tiles);
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
  const bool there = row < nrows && (!A.qmask || A.qmask[b * A.tq + t]);
  // (rows behind a mask are not read: zeros, as their results are)
  u32x4 q[T::kK];
  const int64_t qstart = seq_at(A.qs, A.cu_q, b, S.q0) + (int64_t)hk * A.group * A.qs[2];
  const int qat = there ? row_at<Op>(t - wt, A.qs[1], head, A.qs[2]) : kFar;
  own_row<T>(q, wave_rows<Op>(A.q, qstart, wt, A.qs[1]), qat, A.units, h);
  if (A.scale < 0) negate<T>(q);
  // the keys that count for this row by position, and for the workgroup (reaches grow with the token)
  const Reach mine = keys_of(t, S, A);
  const auto reach = [&](int r) { return keys_of(token_of(r < nrows ? r : nrows - 1, A), S, A); };
  int first = reach(row0).lo / kRows * kRows, last = reach(row0 + 32 * kWaves - 1).hi;
  if constexpr (kSplit) {
    const int from = split * P.keys;
    first = first > from ? first : from;
    last = last < from + P.keys ? last : from + P.keys;
  }
  Rows keys = {words, A.kmask != nullptr, first / kMaskSpan * kMaskSpan, 0};
  const auto gather = [&] {
    const uint8_t* km = A.kmask + b * A.tk;
    keys.gather<kThreads>(S.nk, [&](int j) { return km[j] != 0; });
  };
  if (keys.given && first < last) gather();
  if (!__syncthreads_or(there)) last = first;  // (padding: zeros, and no keys are read)

  const int64_t dim = A.units * (16 / Op::kEsz), width = A.heads * dim;
  const int64_t start = S.q0 * width + hk * A.group * dim;
  const int at = row < nrows ? row_at<Op>(t - wt, width, head, dim) : kFar;
  const float c = factor(A);
  f32x16 acc[T::kBlocks];
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < T::kBlocks; ++i) acc[i] = f32x16{};
  const Reaches wide = reaches(reach(row0 + wave * 32), reach(row0 + wave * 32 + 31), __any(there));
  const char* const kbase =
      static_cast<const char*>(A.k) + (seq_at(A.ks, A.cu_k, b, S.k0) + (int64_t)hk * A.ks[2]) * Op::kEsz;
  const char* const vbase =
      static_cast<const char*>(A.v) + (seq_at(A.vs, A.cu_k, b, S.k0) + (int64_t)hk * A.vs[2]) * Op::kEsz;
  const auto request = [&](int j0, uint64_t bits, int buffer) {
    T::template request<kThreads>(lds + buffer * 2 * T::kBytes, kbase + j0 * A.ks[1] * Op::kEsz,
                                  (int)A.ks[1] * Op::kEsz, A.units, bits);
    T::template request<kThreads>(lds + (buffer * 2 + 1) * T::kBytes, vbase + j0 * A.vs[1] * Op::kEsz,
                                  (int)A.vs[1] * Op::kEsz, A.units, bits);
  };
  // (While a tile is worked on the next is on its way.)
  uint64_t bits;
  keys.end(last);
  int j0 = keys.next(first, bits), buffer = 0;
  if (j0 < keys.to) request(j0, bits, 0);
  for (;;) {
    while (j0 < keys.to) {
      landed();
      uint64_t bits1;
      const int j1 = keys.next(j0 + kRows, bits1);
      if (j1 < keys.to) request(j1, bits1, buffer ^ 1);
      const char* const K = lds + buffer * 2 * T::kBytes;
      const char* const V = K + T::kBytes;
      const int now = j0;
      const uint64_t in = bits;
      j0 = j1;
      bits = bits1;
      buffer ^= 1;
      if (now >= wide.any.hi || now + kRows <= wide.any.lo) continue;  // (none of this wave's rows reaches here)
      float s[2][16];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        f32x16 x = f32x16{};
#pragma unroll
        for (int kb = 0; kb < T::kK; ++kb) x = mma<Op>(T::rows(K, 32 * half, kb, lane), q[kb], x);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[half][r] = x[r];
      }
      const bool whole_tile = in == ~0ull && now >= wide.all.lo && now + kRows <= wide.all.hi;
      uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
      if (!whole_tile) {
        keep[0] = ((uint32_t)in & bits_between(mine.lo - now, mine.hi - now)) >> (4 * h);
        keep[1] = ((uint32_t)(in >> 32) & bits_between(mine.lo - now - 32, mine.hi - now - 32)) >> (4 * h);
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[half][r] = masked(s[half][r], keep[half], r, -INFINITY);
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
      const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          // (The maximum goes before the factor: p is exactly 1 there, so a row that sees one key has that key's
          // value, and of large scores too the difference is what counts.)
          s[half][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[half][r] - base, c, kShift<Op>));
      float sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[half] += s[half][r];
      l += sum[0] + sum[1];
      constexpr int kPer = 32 / kGroups<Op>;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int g = 0; g < kGroups<Op>; ++g) {
          const Operand<Op> p = operand<Op>(s[half], g);
#pragma unroll
          for (int i = 0; i < T::kBlocks; ++i)
            acc[i] = mma(T::columns(V, 32 * half + kPer * g, i, lane), p, acc[i]);
        }
    }
    if (keys.to >= last) break;
    landed();  // (every wave is through with the words, and with the buffers)
    keys.span0 += kMaskSpan;
    keys.end(last);
    gather();
    landed();
    j0 = keys.next(keys.span0, bits);
    if (j0 < keys.to) request(j0, bits, buffer);
  }
  if (A.qmask && !there) {
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) acc[i] = f32x16{};
    m = -INFINITY;
    l = 0.0f;
  }
  // both halves of the wave summed other keys of the same row
  l += __builtin_bit_cast(float, lane_xor32(__builtin_bit_cast(uint32_t, l), h));
  if constexpr (kSplit) {
    if (row >= nrows) return;
    const int64_t slot = (int64_t)piece * (32 * kWaves) + wave * 32 + (lane & 31);
    float* to = P.acc + slot * kD;
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(to + 32 * i + 8 * g + 4 * h) =
            f32x4{acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]};
    P.stat[slot * 2 + h] = h ? l : m;
  } else {
    const bool any = l > 0.0f || l != l;
    const float inv = any ? 1.0f / l : 0.0f;
    // (the quotient is settled before it is rounded: fp16's rounding could be of the product in full, and what it left
    // of the product in 32 bits, which near a tie is a step away)
#pragma unroll
    for (int i = 0; i < T::kBlocks; ++i) {
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] *= inv;
      asm volatile("" : "+v"(acc[i]));
    }
    store_row<Op, T::kBlocks>(wave_rows<Op>(out.o, start, wt, width), at, acc, 1.0f, A.units, h);
    if (out.top && h == 0 && row < nrows) out.top[rows_at(A, b, hk, S.q0) + row] = m;
    if (Op::kEsz == 2 && out.rest) {
#pragma unroll
      for (int i = 0; i < T::kBlocks; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = (acc[i][r] - (float)(E)acc[i][r]) * kRestScale<Op>;
      store_row<Op, T::kBlocks>(wave_rows<Op>(out.rest, start, wt, width), at, acc, 1.0f, A.units, h);
    }
  }
}

// The splits of row blockIdx.x (of units * most rows), joined by the four waves of a workgroup.
template <class Op, int kD, int kWaves>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs A, AttnOut out, Parts P, int tiles, int most) {
  typedef typename Elem<Op>::T E;
  constexpr int kPer = (kD + 63) / 64;
  __shared__ float lds[4][kD + 1];
  const int64_t unit = blockIdx.x / most;
  const int row = (int)(blockIdx.x % most);
  const int64_t b = unit / A.kv_heads;
  const int hk = (int)(unit % A.kv_heads);
  const Span S = span_of(A, b);
  if (row >= S.nq * A.group) return;
  const int tile = row / (32 * kWaves), r = row % (32 * kWaves);
  const int64_t whole = unit * tiles + (A.causal ? tiles - 1 - tile : tile);
  const auto slot = [&](int s) { return (whole * P.splits + s) * (32 * kWaves) + r; };
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  float m = -INFINITY;
  for (int s = lane; s < P.splits; s += 64) m = fmaxf(m, P.stat[slot(s) * 2]);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
  const float c = factor(A), base = m == -INFINITY ? 0.0f : m;
  float l = 0.0f, acc[kPer] = {};
#pragma unroll 4
  for (int s = wave; s < P.splits; s += 4) {
    const float* st = P.stat + slot(s) * 2;
    const float by = __builtin_amdgcn_exp2f((st[0] - base) * c);
    l += by * st[1];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane + 64 * i < kD) acc[i] += by * P.acc[slot(s) * kD + lane + 64 * i];
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (lane + 64 * i < kD) lds[wave][lane + 64 * i] = acc[i];
  if (lane == 0) lds[wave][kD] = l;
  __syncthreads();
  l = (lds[0][kD] + lds[1][kD]) + (lds[2][kD] + lds[3][kD]);
  const bool any = l > 0.0f || l != l;
  const float inv = any ? 1.0f / l : 0.0f;
  const int t = token_of(row, A), head = hk * A.group + row - t * A.group;
  const int dim = A.units * (16 / Op::kEsz);
  const int64_t at = ((S.q0 + t) * A.heads + head) * (int64_t)dim;
  for (int d = threadIdx.x; d < dim; d += 256) {
    float o = ((lds[0][d] + lds[1][d]) + (lds[2][d] + lds[3][d])) * inv;
    asm volatile("" : "+v"(o));  // (settled, as in the kernel above)
    static_cast<E*>(out.o)[at + d] = (E)o;
    if (Op::kEsz == 2 && out.rest) static_cast<E*>(out.rest)[at + d] = (E)((o - (float)(E)o) * kRestScale<Op>);
  }
  if (out.top && threadIdx.x == 0) out.top[rows_at(A, b, hk, S.q0) + row] = m;
}

// A thread a value.  What heads of no whole 16 bytes cost: with 16 heads of 60 in bf16 instead of 64, 128 x 180 tokens
// forward and back take 1099 us instead of 202, 14 copies of 65 us each (forward alone 301 instead of 46).
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

// A thread a token row finds whether a sequence covers it; the wave clears those of its 64 that none does.  All
// results of a call in one launch (blockIdx.y): one is 4 us, nearly all of it latency.
template <class E>
__global__ void __launch_bounds__(256) attn_gap_kernel(AttnGaps gaps) {
  const AttnGaps::Result& x = gaps.of[blockIdx.y];
  const int64_t r0 = (int64_t)blockIdx.x * 256 + (threadIdx.x & ~63u), r = r0 + (threadIdx.x & 63);
  bool gap = r < x.rows;
  if (gap && gaps.seqs > 0 && r >= (int64_t)x.cu[0] - 1) {
    int64_t a = 0, e = gaps.seqs;  // the last sequence that starts at r or before is in [a, e)
    while (e - a > 1) {
      const int64_t mid = (a + e) / 2;
      if ((int64_t)x.cu[mid] - 1 <= r) a = mid;
      else e = mid;
    }
    gap = !(r < (int64_t)x.cu[a + 1] - 1 && r - ((int64_t)x.cu[a] - 1) < x.most);
  }
  for (uint64_t left = __ballot(gap); left; left &= left - 1) {
    E* const row = static_cast<E*>(x.out) + (r0 + __builtin_ctzll(left)) * x.width;
    for (int64_t i = threadIdx.x & 63; i < x.width; i += 64) row[i] = (E)0;
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
  const SplitPlan plan = split_plan(a);
  const int64_t tiles = plan.tiles, units = a.seqs * a.kv_heads;
  if (plan.splits > 1) {
    Parts p;
    p.splits = (int)plan.splits;
    p.keys = (int)plan.keys;
    p.acc = static_cast<float*>(out.parts);
    p.stat = p.acc + plan.slots * kD;
    const int64_t work = plan.pieces * plan.splits;
    hipLaunchKernelGGL((attn_forward_kernel<Op, kD, kWaves, true>), dim3(piece_blocks(work)), dim3(kWaves * 64), 0,
                       stream, a, out, p, (uint32_t)tiles, (uint32_t)work);
    const int most = a.tq * a.group;
    hipLaunchKernelGGL((attn_join_kernel<Op, kD, kWaves>), dim3((unsigned)(units * most)), dim3(256), 0, stream, a,
                       out, p, (int)tiles, most);
    return hipGetLastError();
  }
  return by_units(a, tiles, [&](const AttnArgs& part, int64_t n) {
    hipLaunchKernelGGL((attn_forward_kernel<Op, kD, kWaves, false>), dim3(piece_blocks(n * tiles)), dim3(kWaves * 64), 0,
                       stream, part, out, Parts{}, (uint32_t)tiles, (uint32_t)(n * tiles));
  });
}

template <class Op, int kD>
hipError_t forward_dim(const AttnArgs& a, const AttnOut& out, hipStream_t stream) {
  return waves_of(a) == 1 ? forward_waves<Op, kD, 1>(a, out, stream) : forward_waves<Op, kD, 4>(a, out, stream);
}

template <class Op>
hipError_t forward_op(const AttnArgs& a, const AttnOut& out, hipStream_t stream) {
  switch (instance_dim(a)) {
    case 32: return forward_dim<Op, 32>(a, out, stream);
    case 64: return forward_dim<Op, 64>(a, out, stream);
    default: return forward_dim<Op, 128>(a, out, stream);
  }
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

hipError_t attn_zero_gaps(int32_t dtype, const AttnGaps& gaps, hipStream_t stream) {
  int64_t rows = 0;
  for (int i = 0; i < gaps.n; ++i) rows = std::max(rows, gaps.of[i].width ? gaps.of[i].rows : 0);
  if (rows == 0) return hipSuccess;
  const dim3 blocks((unsigned)attn::cdiv(rows, 256), (unsigned)gaps.n);
  if (dtype == FMS_F32)
    hipLaunchKernelGGL((attn::attn_gap_kernel<uint32_t>), blocks, dim3(256), 0, stream, gaps);
  else
    hipLaunchKernelGGL((attn::attn_gap_kernel<uint16_t>), blocks, dim3(256), 0, stream, gaps);
  return hipGetLastError();
}

int64_t attn_forward_bytes(const AttnArgs& a) { return attn::split_plan(a).slots * (attn::instance_dim(a) + 2) * 4; }

hipError_t attn_forward(const AttnArgs& a, const AttnOut& out, hipStream_t stream) {
  return attn::by_type(a.dtype, [&](auto op) { return attn::forward_op<decltype(op)>(a, out, stream); });
}

}  // namespace fms

// fms_ffn.hip -- gated feed-forward block: both projections, the activation and
// the product in one kernel, and its pullback.
//
//   g = x wg^T,  u = x wu^T,  h = act(g) * u                     (per token and hidden unit)
//   dg = dh * u * act'(g),  du = dh * act(g)
//   dx = dg wg + du wu,  dwg = dg^T x,  dwu = du^T x
//
// Products run on the matrix cores (fms_gemm.hpp) and accumulate in fp32.  g and
// u never leave the registers: forward writes h alone and keeps nothing, and the
// pullback computes them again in the kernel that makes dg and du for the three
// products after it.  (Keeping g and u from the forward in 16 bits would round them,
// and in fp32 would move 16 bytes a hidden unit, against 4 dim operations to compute them.)
//
// The matrix cores take dg and du in the feature type, and one rounding to 16 bits there
// costs as much as the outputs' own: 1.41 times the error of the result, and in fp16 their
// range, since each is a product of three values.  So in 16 bits they are held as two values
// each, the rounding and what it left (two planes), and the products sum both: 16 significant
// bits in bf16, 22 in fp16, for twice the products' work (a pullback of 23040 x 1024 x 4096 in
// bf16: 2040 us, about 1130 with one plane; 2100 in fp16).  In fp16 they are multiplied with a
// power of two, from a bound of the largest of them (ffn_bound_kernel, 50 us there), and the
// products' results with its reciprocal: the bound comes to 2^14 .. 2^15, so nothing overflows
// and what falls off the second plane is less than 2^-39 of the bound.
//
// act(g) = g s with s = sigmoid(y(g)) for silu (y = g) and gelu_tanh
// (y = 2 sqrt(2/pi) (g + 0.044715 g^3), since (1 + tanh z) / 2 = sigmoid(2z));
// act'(g) = s + g s (1 - s) y'(g).  gelu is g Phi(g), act' = Phi + g phi.
#include "fms_ffn.hpp"

#include <math.h>

#include "../../include/flashmaxsim_hip.h"
#include "fms_gemm.hpp"
#include "fms_group.hpp"

namespace fms {
namespace {

struct OutF16 {
  typedef _Float16 T;
};
struct OutBF16 {
  typedef __bf16 T;
};
struct OutF32 {
  typedef float T;
};
template <class Op>
struct OutOf;
template <>
struct OutOf<OpF16> : OutF16 {};
template <>
struct OutOf<OpBF16> : OutBF16 {};
template <>
struct OutOf<OpF32> : OutF32 {};

// act(g) in a, act'(g) in da.  With the hardware's exponential and reciprocal s is within about
// 2 + |y| / 2 units of its last place; g's own rounding to fp32 moves an exponential of it by |g| / 2.
template <int kAct>
__device__ __forceinline__ void activate(float g, float& a, float& da) {
  float s, dy;
  if constexpr (kAct == FMS_ACT_GELU) {
    s = 0.5f * erfcf(g * -0.70710678118654752f);
    const float pdf = 0.39894228040143268f * __expf(-0.5f * g * g);
    a = g * s;
    da = pdf > 0.0f ? s + g * pdf : s;
    return;
  }
  float y = g;
  dy = 1.0f;
  if constexpr (kAct == FMS_ACT_GELU_TANH) {
    const float g2 = g * g;
    y = 1.5957691216057308f * (g + 0.044715f * g * g2);
    dy = 1.5957691216057308f * (1.0f + 0.134145f * g2);
  }
  s = __builtin_amdgcn_rcpf(1.0f + __expf(-y));
  const float d = s * (1.0f - s);
  a = g * s;
  da = d > 0.0f ? s + g * d * dy : s;  // (past the last step of s, y' may be infinite)
}

// A lane holds, of one row, columns 8 q + 4 h + 0..3 of 32 in quad q (h = lane / 32).  Its
// part of the quads 2p and 2p + 1 goes to and from memory without LDS: in 16 bits the halves
// trade a quad, so that each has eight neighbouring columns (from 16 p + 8 h on), 16 bytes; in
// 32 bits a quad is 16 bytes already.
template <class Op>
struct Quads {
  typedef typename OutOf<Op>::T T;
  static constexpr bool kTrade = Op::kEsz == 2;
  static constexpr int kPer = 16 / Op::kEsz;  // neighbouring columns
  typedef T V __attribute__((ext_vector_type(kPer)));
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

  // First column of this lane's 16 bytes i of the pair p.
  __device__ static __forceinline__ int col(int p, int i, int h) {
    return kTrade ? 16 * p + 8 * h : 16 * p + 8 * i + 4 * h;
  }
  static constexpr int kWords = kTrade ? 1 : 2;  // 16 bytes per pair and lane

  // 16 bytes at byte `at` of a resource, with `left` columns of the row from there (none or
  // all of them are inside).
  __device__ static __forceinline__ void put(V v, rsrc_t to, int at, int left) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), to,
                                           left > 0 ? at : kOutOfBounds, 0, 0);
  }
  __device__ static __forceinline__ V get(rsrc_t from, int at, int left) {
    return __builtin_bit_cast(V, buf_load16(from, left > 0 ? at : kOutOfBounds));
  }
  // Stores the pair a, b at byte `at` of the row's first column (of `cols` from there).
  __device__ static __forceinline__ void store(const float (&a)[4], const float (&b)[4], rsrc_t to,
                                               int at, int p, int h, int cols) {
    typedef T V4 __attribute__((ext_vector_type(4)));
    const V4 qa = {(T)a[0], (T)a[1], (T)a[2], (T)a[3]}, qb = {(T)b[0], (T)b[1], (T)b[2], (T)b[3]};
    const int c0 = col(p, 0, h);
    if constexpr (kTrade) {
      const u32x2 wa = __builtin_bit_cast(u32x2, qa), wb = __builtin_bit_cast(u32x2, qb);
      const auto r0 = __builtin_amdgcn_permlane32_swap(wa[0], wb[0], false, false);
      const auto r1 = __builtin_amdgcn_permlane32_swap(wa[1], wb[1], false, false);
      const u32x4 w = {(uint32_t)r0[0], (uint32_t)r1[0], (uint32_t)r0[1], (uint32_t)r1[1]};
      put(__builtin_bit_cast(V, w), to, at + c0 * Op::kEsz, cols - c0);
    } else {
      const int c1 = col(p, 1, h);
      put(qa, to, at + c0 * Op::kEsz, cols - c0);
      put(qb, to, at + c1 * Op::kEsz, cols - c1);
    }
  }
  // To be called before a is rounded in two places: a as it is in a register.  (The compiler
  // fuses a product with its conversion to fp16, which rounds once where product and conversion
  // round twice: near a tie the two places would have had different roundings.)
  __device__ static __forceinline__ void settle(float (&a)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) asm volatile("" : "+v"(a[e]));
  }
  // What a's rounding to the type leaves, in a; nothing where that is not finite.
  __device__ static __forceinline__ void rest(float (&a)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float r = a[e] - (float)(T)a[e];
      a[e] = fabsf(r) < INFINITY ? r : 0.0f;
    }
  }
  // Reads such a pair.
  __device__ static __forceinline__ void fetch(V (&w)[kWords], rsrc_t from, int at, int p, int h,
                                               int cols) {
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      w[i] = get(from, at + col(p, i, h) * Op::kEsz, cols - col(p, i, h));
  }
  __device__ static __forceinline__ void split(const V (&w)[kWords], float (&a)[4], float (&b)[4]) {
    typedef T V4 __attribute__((ext_vector_type(4)));
    V4 qa, qb;
    if constexpr (kTrade) {
      const u32x4 x = __builtin_bit_cast(u32x4, w[0]);
      const auto r0 = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false);
      const auto r1 = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
      qa = __builtin_bit_cast(V4, u32x2{(uint32_t)r0[0], (uint32_t)r1[0]});
      qb = __builtin_bit_cast(V4, u32x2{(uint32_t)r0[1], (uint32_t)r1[1]});
    } else {
      qa = w[0];
      qb = w[1];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] = (float)qa[e];
      b[e] = (float)qb[e];
    }
  }

  // Rows that are no whole 16-byte units: 32 x 32 values pass through `box`, the wave's own
  // LDS, and go to or come from memory element by element, two rows at a time.
  static constexpr int kBox = 32 * 32 * Op::kEsz;
  __device__ static __forceinline__ void box_in(char* box, int lane, int q, const float (&a)[4]) {
    typedef T V4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<V4*>(box + ((lane & 31) * 32 + 8 * q + 4 * (lane >> 5)) * Op::kEsz) =
        V4{(T)a[0], (T)a[1], (T)a[2], (T)a[3]};
  }
  __device__ static __forceinline__ void box_out(const char* box, int lane, int q, float (&a)[4]) {
    typedef T V4 __attribute__((ext_vector_type(4)));
    const V4 v = *reinterpret_cast<const V4*>(box + ((lane & 31) * 32 + 8 * q + 4 * (lane >> 5)) * Op::kEsz);
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = (float)v[e];
  }
  // `at`: byte of the box's first value, `pitch` bytes a row, `cols` columns left there.
  __device__ static __forceinline__ void box_store(const char* box, int lane, rsrc_t to, int at, int pitch,
                                                   int cols) {
    box_wait();
    const int c = lane & 31;
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
      const int r = 2 * i + (lane >> 5), to_at = c < cols ? at + r * pitch + c * Op::kEsz : kOutOfBounds;
      const T v = reinterpret_cast<const T*>(box)[r * 32 + c];
      if constexpr (kTrade)
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, v), to, to_at, 0, 0);
      else
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), to, to_at, 0, 0);
    }
    box_wait();
  }
  __device__ static __forceinline__ void box_load(char* box, int lane, rsrc_t from, int at, int pitch,
                                                  int cols) {
    const int c = lane & 31;
#pragma unroll 1
    for (int i0 = 0; i0 < 16; i0 += 8) {
      T v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int off = c < cols ? at + (2 * (i0 + i) + (lane >> 5)) * pitch + c * Op::kEsz : kOutOfBounds;
        if constexpr (kTrade)
          v[i] = __builtin_bit_cast(T, (uint16_t)buf_load2(from, off));
        else
          v[i] = __builtin_bit_cast(T, buf_load4(from, off));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(box)[(2 * (i0 + i) + (lane >> 5)) * 32 + c] = v[i];
    }
    box_wait();
  }
  // A wave's LDS accesses are done, for all its lanes.
  __device__ static __forceinline__ void box_wait() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
};

// A tile of a row-major matrix as a resource: rows past its end are out of bounds.
template <class T>
__device__ __forceinline__ rsrc_t tile_at(const void* p, int64_t rows, int64_t pitch, int64_t m0,
                                          int64_t n0) {
  const int64_t at = m0 * pitch + n0, left = (rows * pitch - at) * (int64_t)sizeof(T);
  return make_rsrc_u(static_cast<const T*>(p) + at,
                     (uint32_t)(left < 0 ? 0 : (left > 0x7fffffff ? 0x7fffffff : left)));
}
// x, as if it were not known before: what an epilogue derives from it is computed there, not
// held in registers all through the products.
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
__device__ __forceinline__ int columns_left(int64_t cols, int64_t n0) {
  return cols - n0 > 0x7fffffff ? 0x7fffffff : (int)(cols - n0);
}

// Workgroup -> tile.  Workgroup ids go round robin over the 8 XCDs, each with an L2 of
// its own: every XCD takes a contiguous run of tiles, and a run walks kGroupM row tiles
// per column tile, so that the tiles in flight on an XCD share their operands.  (In the
// pullback's products a unit's number has its workgroup's residue only where the tiles, and the
// units of the product before, are multiples of 8; otherwise neighbours part.)
constexpr int kXcds = 8;
constexpr int kGroupM = 8;
__device__ __forceinline__ void tile_of(int id, int tm, int tn, int& im, int& in) {
  const int total = tm * tn;
  const int q = total / kXcds, r = total % kXcds, x = id % kXcds;
  const int t = x * q + (x < r ? x : r) + id / kXcds;
  const int per = kGroupM * tn, g = t / per;
  const int rows = tm - g * kGroupM < kGroupM ? tm - g * kGroupM : kGroupM;
  im = g * kGroupM + (t % per) % rows;
  in = (t % per) / rows;
}

struct GateArgs {
  Matrix x, wg, wu;
  int32_t act, tm, tn, steps;
  int64_t tokens, hidden;
  // forward: out0 = h; pullback: in = dh, out0 = dg, out1 = du, each kPlanes planes
  void *out0, *out1;
  const void* in;
  int64_t out_cols, out_pitch, in_pitch;  // values
  int64_t plane;  // bytes from a plane of dg or du to its second one
  int32_t vec;    // whole 16-byte units of outputs and input
  // fp16 pullback: the parts of the bound, and where the reciprocal of its power of two goes
  int32_t nbounds;
  const float2* bounds;
  float* unscale;
};

// How many values hold one of dg or du, and whether they are scaled.
template <class Op>
constexpr int kPlanes = Op::kEsz == 2 ? 2 : 1;
template <class Op>
constexpr bool kScaled = std::is_same_v<Op, OpF16>;

// |act(g)| <= |g| and |act'(g)| < 1.13, so with Cauchy and Schwarz no dg or du is larger than
//   1.13 max over tokens (max |dh| of its row, |x|_2) * max over hidden units (|wg|_2, |wu|_2).
// A workgroup's part of the two maxima, over rows that are finite (others' products are not
// finite whatever they are scaled by).  One read of the inputs, a wave a row.
constexpr int kMostBounds = 256, kBoundWaves = 16;
struct BoundArgs {
  Matrix x, wg, wu;  // fp16, whole 16-byte units, zero beyond dim
  const _Float16* dh;
  int64_t tokens, hidden;
  int32_t vec;  // whole 16-byte units of dh
  float2* bounds;
};
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
// A lane's part of |row|_2^2.
__device__ __forceinline__ float squares(const Matrix& m, int64_t row, int lane) {
  const char* const p = m.base + row * m.pitch;
  float s = 0.0f;
#pragma unroll 4
  for (int64_t at = lane * 16; at < m.rowbytes; at += 64 * 16) {
    const f16x8 v = *reinterpret_cast<const f16x8*>(p + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += (float)v[e] * (float)v[e];
  }
  return s;
}
// The length that the lanes' parts make, 0 where it is not finite.
__device__ __forceinline__ float length(float part) {
  const float s = wave_sum(part);
  return s < INFINITY ? sqrtf(s) : 0.0f;
}
__global__ void __launch_bounds__(64 * kBoundWaves) ffn_bound_kernel(BoundArgs A) {
  __shared__ float2 lds[kBoundWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float token = 0.0f, unit = 0.0f;
  for (int64_t i = (int64_t)blockIdx.x * kBoundWaves + wave; i < A.tokens + 2 * A.hidden;
       i += (int64_t)gridDim.x * kBoundWaves) {
    if (i >= A.tokens) {
      const int64_t j = i - A.tokens;
      unit = fmaxf(unit, length(j < A.hidden ? squares(A.wg, j, lane) : squares(A.wu, j - A.hidden, lane)));
      continue;
    }
    const float part = squares(A.x, i, lane);
    const _Float16* const row = A.dh + i * A.hidden;
    float top = 0.0f;
    const auto see = [&](_Float16 h) {
      const float v = fabsf((float)h);
      top = v < INFINITY && v > top ? v : top;
    };
    if (A.vec) {
#pragma unroll 4
      for (int64_t k = lane * 8; k < A.hidden; k += 64 * 8) {
        const f16x8 v = *reinterpret_cast<const f16x8*>(row + k);
#pragma unroll
        for (int e = 0; e < 8; ++e) see(v[e]);
      }
    } else {
#pragma unroll 4
      for (int64_t k = lane; k < A.hidden; k += 64) see(row[k]);
    }
    token = fmaxf(token, wave_max(top) * length(part));
  }
  if (lane == 0) lds[wave] = make_float2(token, unit);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 0; w < kBoundWaves; ++w) {
      token = fmaxf(token, lds[w].x);
      unit = fmaxf(unit, lds[w].y);
    }
    A.bounds[blockIdx.x] = make_float2(token, unit);
  }
}
// The power of two that takes the bound (without its 1.13) to 2^14 .. 2^15, as an exponent; a
// wave's lanes all take part.
__device__ __forceinline__ int scale_exponent(const GateArgs& A) {
  float token = 0.0f, unit = 0.0f;
#pragma unroll
  for (int j = 0; j < kMostBounds; j += 64) {
    const int i = j + (threadIdx.x & 63);
    if (i >= A.nbounds) break;
    token = fmaxf(token, A.bounds[i].x);
    unit = fmaxf(unit, A.bounds[i].y);
  }
  const float bound = wave_max(token) * wave_max(unit);  // (2^-72 .. 2^70, or 0)
  const int e = bound > 0.0f ? 14 - ilogbf(bound) : 0;
  return __builtin_amdgcn_readfirstlane(e);
}

// LDS behind the products' buffers, a box for each wave.
template <class P>
constexpr int kBoxes = P::kThreads / 64 * Quads<typename P::Op>::kBox;

// A tile's sums -> h, or dg and du.  kVec: rows of whole 16-byte units; else through `box`.
template <class P, bool kPull, int kAct, bool kVec>
__device__ __forceinline__ void gate_store(const GateArgs& A, const typename P::Acc (&acc)[2][P::kMF],
                                           int64_t m0, int64_t n0, char* box, float scale) {
  typedef Quads<typename P::Op> Q;
  typedef typename Q::T T;
  constexpr int kSize = (int)sizeof(T);
  constexpr bool kTwo = kPull && kPlanes<typename P::Op> == 2;
  const int lane = here(threadIdx.x & 63), wave = threadIdx.x >> 6;
  const int wm = wave / P::kWN, wn = wave % P::kWN, h = lane >> 5;
  const rsrc_t to0 = tile_at<T>(A.out0, A.tokens, A.out_pitch, m0, n0);
  const rsrc_t to1 = tile_at<T>(A.out1, kPull ? A.tokens : 0, A.out_pitch, m0, n0);
  const rsrc_t rest0 = tile_at<T>(static_cast<char*>(A.out0) + A.plane, kTwo ? A.tokens : 0, A.out_pitch, m0, n0);
  const rsrc_t rest1 = tile_at<T>(static_cast<char*>(A.out1) + A.plane, kTwo ? A.tokens : 0, A.out_pitch, m0, n0);
  const rsrc_t from = tile_at<T>(A.in, kPull ? A.tokens : 0, A.in_pitch, m0, n0);
  // of the wave's first row
  const int out_pitch = (int)A.out_pitch * kSize, in_pitch = (int)A.in_pitch * kSize;
  const int out = wm * P::kMF * 32 * out_pitch + wn * 32 * kSize;
  const int in = wm * P::kMF * 32 * in_pitch + wn * 32 * kSize;
  const int out_left = columns_left(A.out_cols, n0) - wn * 32, in_left = columns_left(A.hidden, n0) - wn * 32;
  // the cotangent's part of a row fragment, read one ahead
  typename Q::V dh[2][2][Q::kWords];
  const auto fetch = [&](int mf) {
#pragma unroll
    for (int p = 0; p < 2; ++p)
      Q::fetch(dh[mf & 1][p], from, in + (mf * 32 + (lane & 31)) * in_pitch, p, h, in_left);
  };
  if constexpr (kPull && kVec) fetch(0);
#pragma unroll
  for (int mf = 0; mf < P::kMF; ++mf) {
    if constexpr (kPull && kVec)
      if (mf + 1 < P::kMF) fetch(mf + 1);
    const int at = out + (mf * 32 + (lane & 31)) * out_pitch;
    float y[4][4], z[4][4];
    if constexpr (kPull && !kVec) {
      Q::box_load(box, lane, from, in + mf * 32 * in_pitch, in_pitch, in_left);
#pragma unroll
      for (int q = 0; q < 4; ++q) Q::box_out(box, lane, q, y[q]);
      Q::box_wait();
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if constexpr (kPull && kVec) Q::split(dh[mf & 1][p], y[2 * p], y[2 * p + 1]);
#pragma unroll
      for (int q = 2 * p; q < 2 * p + 2; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float g = acc[0][mf][4 * q + e], u = acc[1][mf][4 * q + e];
          float a, da;
          activate<kAct>(g, a, da);
          if constexpr (kPull) {
            if constexpr (kScaled<typename P::Op>) y[q][e] *= scale;
            z[q][e] = y[q][e] * a;
            y[q][e] = y[q][e] * u * da;
          } else {
            y[q][e] = a * u;
          }
        }
      if constexpr (kVec) {
        const auto put = [&](float (&a)[4][4], rsrc_t to, rsrc_t rest) {
          if constexpr (kTwo) {
            Q::settle(a[2 * p]);
            Q::settle(a[2 * p + 1]);
          }
          Q::store(a[2 * p], a[2 * p + 1], to, at, p, h, out_left);
          if constexpr (kTwo) {
            Q::rest(a[2 * p]);
            Q::rest(a[2 * p + 1]);
            Q::store(a[2 * p], a[2 * p + 1], rest, at, p, h, out_left);
          }
        };
        put(y, to0, rest0);
        __builtin_amdgcn_sched_barrier(0);  // (few values at a time)
        if constexpr (kPull) {
          put(z, to1, rest1);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    if constexpr (!kVec) {
      const auto put = [&](const float (&a)[4][4], rsrc_t to) {
#pragma unroll
        for (int q = 0; q < 4; ++q) Q::box_in(box, lane, q, a[q]);
        Q::box_store(box, lane, to, out + mf * 32 * out_pitch, out_pitch, out_left);
      };
      const auto put_all = [&](float (&a)[4][4], rsrc_t to, rsrc_t rest) {
        if constexpr (kTwo) {
#pragma unroll
          for (int q = 0; q < 4; ++q) Q::settle(a[q]);
        }
        put(a, to);
        if constexpr (kTwo) {
#pragma unroll
          for (int q = 0; q < 4; ++q) Q::rest(a[q]);
          put(a, rest);
        }
      };
      put_all(y, to0, rest0);
      if constexpr (kPull) put_all(z, to1, rest1);
    }
  }
}

template <class P, bool kPull, bool kVec>
__device__ __forceinline__ void by_act(const GateArgs& A, const typename P::Acc (&acc)[2][P::kMF],
                                       int64_t m0, int64_t n0, char* box, float scale) {
  if (A.act == FMS_ACT_SILU)
    gate_store<P, kPull, FMS_ACT_SILU, kVec>(A, acc, m0, n0, box, scale);
  else if (A.act == FMS_ACT_GELU)
    gate_store<P, kPull, FMS_ACT_GELU, kVec>(A, acc, m0, n0, box, scale);
  else
    gate_store<P, kPull, FMS_ACT_GELU_TANH, kVec>(A, acc, m0, n0, box, scale);
}

// Forward (kPull false): h.  Pullback: dg and du, their rows filled up with zeros to out_cols.
// Workgroup b takes tiles b, b + gridDim.x, ...
template <class P, bool kPull>
__global__ void __launch_bounds__(P::kThreads, 2) ffn_gate_kernel(GateArgs A) {
  constexpr int kCols = P::kBN / 2;
  __shared__ __attribute__((aligned(16))) char lds[P::kLds + kBoxes<P>];
  char* const box = lds + P::kLds + (threadIdx.x >> 6) * Quads<typename P::Op>::kBox;
  const int tiles = A.tm * A.tn, mine = (tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  float scale = 1.0f;
  if constexpr (kPull && kScaled<typename P::Op>) {
    const int e = scale_exponent(A);
    scale = ldexpf(1.0f, e);
    if (blockIdx.x == 0 && threadIdx.x == 0) *A.unscale = ldexpf(1.0f, -e);
  }
  const auto place = [&](int j, int64_t& m0, int64_t& n0) {
    int im, in;
    tile_of(blockIdx.x + j * gridDim.x, A.tm, A.tn, im, in);
    m0 = (int64_t)im * P::kBM;
    n0 = (int64_t)in * kCols;
  };
  const auto leg = [&](int j) {
    typename P::Legs l;
    l.m[0] = A.x;
    l.n[0] = A.wg;
    l.n[1] = A.wu;
    place(j, l.m0, l.n0);
    l.first = 0;
    l.steps = A.steps;
    l.ends = true;
    return l;
  };
  const auto after = [&](int j, const typename P::Acc(&acc)[2][P::kMF]) {
    int64_t m0, n0;
    place(j, m0, n0);
    if (!A.vec)
      by_act<P, kPull, false>(A, acc, m0, n0, box, scale);
    else
      by_act<P, kPull, true>(A, acc, m0, n0, box, scale);
  };
  P::run(mine, leg, after, lds);
}

// ---- few tokens ----------------------------------------------------------------------------
// Bound by the weights' bytes, and for one query by latency: no LDS staging and no barrier on
// the way.  A workgroup takes kHidden units (their rows of wg and of wu) and 16 kNT
// tokens; its eight waves share k, 128 bytes of every row at a time, each loading its operands
// straight into the 16 x 16 MFMAs' registers with everything of a round in flight, and join
// their sums through LDS.
template <class Op>
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 acc) {
  if constexpr (std::is_same_v<Op, OpF16>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
  } else if constexpr (std::is_same_v<Op, OpBF16>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  } else {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], acc, 0, 0, 0);
    return acc;
  }
}

constexpr int kFewWaves = 8;

template <class Op, int kNT, int kHidden>
__global__ void __launch_bounds__(64 * kFewWaves) ffn_few_kernel(GateArgs A) {
  typedef typename OutOf<Op>::T T;
  // lane: row (hidden unit, token) lane % 16 of a fragment, bytes 16 (lane / 16) of 64
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * kHidden, m0 = (int64_t)blockIdx.y * 16 * kNT;
  const int pitch = (int)A.x.pitch, bytes = (int)A.x.rowbytes, in = 16 * (lane >> 4);
  const rsrc_t rx = matrix_from(A.x, m0 * A.x.pitch);
  const int row = (lane & 15) * pitch + in;
  // 16 hidden units: a fragment of each projection; 8: one, its rows 0..7 of wg and 8..15 of wu
  constexpr int kFrags = kHidden / 8;
  const int64_t unit = n0 + (lane & (kHidden - 1));
  const int wbytes = unit < A.hidden ? bytes - in : 0;  // of this lane's row, from its first on
  const char* w[kFrags];
#pragma unroll
  for (int f = 0; f < kFrags; ++f)
    w[f] = ((kFrags == 2 ? f == 1 : (lane & 8) != 0) ? A.wu.base : A.wg.base) + unit * A.wg.pitch + in;
  f32x4 acc[kFrags][kNT] = {};
  struct Round {
    u32x4 w[2][kFrags], x[2][kNT];
  };
  const auto load = [&](Round& r, int at) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int off = at + 64 * i + in < bytes ? row + at + 64 * i : kOutOfBounds;
#pragma unroll
      for (int f = 0; f < kFrags; ++f) {
        r.w[i][f] = u32x4{0u, 0u, 0u, 0u};
        if (at + 64 * i < wbytes) r.w[i][f] = *reinterpret_cast<const u32x4*>(w[f] + at + 64 * i);
      }
#pragma unroll
      for (int t = 0; t < kNT; ++t)
        r.x[i][t] = buf_load16(rx, off == kOutOfBounds ? off : off + t * 16 * pitch);
    }
  };
  const auto multiply = [&](const Round& r) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int t = 0; t < kNT; ++t)
#pragma unroll
        for (int f = 0; f < kFrags; ++f) acc[f][t] = mma16<Op>(r.w[i][f], r.x[i][t], acc[f][t]);
  };
  constexpr int kRound = kFewWaves * 128;  // bytes of k between a wave's rounds
  Round a, b;
  int at = wave * 128;
  load(a, at);
  load(b, at + kRound);
  for (; at < bytes; at += 2 * kRound) {  // (rounds past the end read zeros)
    multiply(a);
    load(a, at + 2 * kRound);
    multiply(b);
    load(b, at + 3 * kRound);
  }
  // sums of the waves: lane holds rows 4 (lane / 16) + e of token lane % 16, gate and then up
  __shared__ __attribute__((aligned(16))) f32x4 sums[kFewWaves][kFrags][kNT][64];
#pragma unroll
  for (int f = 0; f < kFrags; ++f)
#pragma unroll
    for (int t = 0; t < kNT; ++t) sums[wave][f][t][lane] = acc[f][t];
  __syncthreads();
  constexpr int kLanes = 4 * kHidden;  // that hold gates
  for (int o = tid; o < kLanes * kNT; o += 64 * kFewWaves) {
    const int t = o / kLanes, l = o % kLanes;
    f32x4 g = {}, u = {};
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {  // (in order)
      g += sums[w][0][t][l];
      u += kFrags == 2 ? sums[w][kFrags - 1][t][l] : sums[w][0][t][l + 32];
    }
    const int64_t m = m0 + t * 16 + (l & 15), n = n0 + 4 * (l >> 4);
    if (m >= A.tokens) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float y, dy;
      if (A.act == FMS_ACT_SILU)
        activate<FMS_ACT_SILU>(g[e], y, dy);
      else if (A.act == FMS_ACT_GELU)
        activate<FMS_ACT_GELU>(g[e], y, dy);
      else
        activate<FMS_ACT_GELU_TANH>(g[e], y, dy);
      if (n + e < A.hidden) static_cast<T*>(A.out0)[m * A.out_pitch + n + e] = (T)(y * u[e]);
    }
  }
}

// A product of the pullback.  Unit u of its tiles * splits * outputs: out[z] or, with splits,
// a part of it over k, in fp32.  With dg's planes first and du's after them, output z is the sum of planes
// z segments .. (z + 1) segments - 1 times n[0] (dg's) or n[1] (du's).
struct ProductArgs {
  Matrix m;       // the first plane
  int64_t plane;  // bytes to the next one
  Matrix n[2];
  const float* unscale;  // fp16: what the sums are multiplied with, or null
  int32_t segments;
  int32_t outputs;
  int64_t bytes;                  // of a segment's k
  int32_t tm, tn, steps, splits;  // steps of all segments
  int64_t rows, cols;
  void* out[2];
  int32_t vec;
  float* parts;  // splits > 1: (splits, outputs, rows, part_pitch)
  int64_t part_pitch;
};

// A tile's sums -> rows of `cols` values, `pitch` apart.  kVec: rows of whole 16-byte units.
template <class P, class Q, bool kVec>
__device__ __forceinline__ void product_store(const typename P::Acc (&acc)[2][P::kMF], void* out,
                                              int64_t rows, int64_t cols, int64_t pitch_, int64_t m0,
                                              int64_t n0, char* box, float unscale) {
  typedef typename Q::T T;
  const int lane = here(threadIdx.x & 63), wave = threadIdx.x >> 6, h = lane >> 5;
  const rsrc_t to = tile_at<T>(out, rows, pitch_, m0, n0);
  const int pitch = (int)pitch_ * (int)sizeof(T), left = columns_left(cols, n0);
#pragma unroll
  for (int mf = 0; mf < P::kMF; ++mf)
#pragma unroll
    for (int nf = 0; nf < 2; ++nf) {
      const int n = P::col(wave % P::kWN, nf);
      const int at = (wave / P::kWN * P::kMF + mf) * 32 * pitch + n * (int)sizeof(T);
      const auto& c = acc[nf][mf];
      const auto quad = [&](int q, float (&a)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = kScaled<typename P::Op> ? c[4 * q + e] * unscale : c[4 * q + e];
      };
      float a[4], b[4];
      if constexpr (kVec) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          quad(2 * p, a);
          quad(2 * p + 1, b);
          Q::store(a, b, to, at + (lane & 31) * pitch, p, h, left - n);
        }
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          quad(q, a);
          Q::box_in(box, lane, q, a);
        }
        Q::box_store(box, lane, to, at, pitch, left - n);
      }
    }
}

template <class P>
__device__ __forceinline__ void product_unit(const ProductArgs& A, int unit, char* lds) {
  char* const box = lds + P::kLds + (threadIdx.x >> 6) * Quads<typename P::Op>::kBox;
  const int tiles = A.tm * A.tn, z = unit / (tiles * A.splits), split = unit / tiles % A.splits;
  int im, in;
  tile_of(unit % tiles, A.tm, A.tn, im, in);
  const int64_t m0 = (int64_t)im * P::kBM, n0 = (int64_t)in * P::kBN;
  // the split's steps, counted over the segments: a leg in each that it reaches into
  const int s0 = (int)((int64_t)A.steps * split / A.splits);
  const int s1 = (int)((int64_t)A.steps * (split + 1) / A.splits);
  const int each = A.steps / A.segments;
  const int lo = each > 0 ? s0 / each : 0, hi = each > 0 ? (s1 - 1) / each : 0;
  float unscale = 1.0f;
  if constexpr (kScaled<typename P::Op>)
    if (A.unscale) unscale = *A.unscale;
  const auto leg = [&](int j) {
    const int s = lo + j, from = s0 - s * each, to = s1 - s * each, plane = z * A.segments + s;
    typename P::Legs l;
    l.m[0] = A.m;
    l.m[0].base += plane * A.plane;
    l.n[0] = plane < kPlanes<typename P::Op> ? A.n[0] : A.n[1];
    l.m0 = m0;
    l.n0 = n0;
    l.first = from > 0 ? from : 0;
    l.steps = (to < each ? to : each) - l.first;
    l.ends = s == hi;
    return l;
  };
  const auto after = [&](int, const typename P::Acc(&acc)[2][P::kMF]) {
    if (A.splits > 1)
      product_store<P, Quads<OpF32>, true>(
          acc, A.parts + ((int64_t)split * A.outputs + z) * A.rows * A.part_pitch, A.rows, A.part_pitch,
          A.part_pitch, m0, n0, box, unscale);
    else if (A.vec)
      product_store<P, Quads<typename P::Op>, true>(acc, z == 0 ? A.out[0] : A.out[1], A.rows, A.cols,
                                                    A.cols, m0, n0, box, unscale);
    else
      product_store<P, Quads<typename P::Op>, false>(acc, z == 0 ? A.out[0] : A.out[1], A.rows, A.cols,
                                                     A.cols, m0, n0, box, unscale);
  };
  if (s0 < s1) {
    P::run(hi - lo + 1, leg, after, lds);
  } else {  // a sum of nothing
    const typename P::Acc zero[2][P::kMF] = {};
    after(0, zero);
  }
}

// Both products in one launch: the first `weights` workgroups take units of dwg and dwu, the
// others units of dx.
template <class PW, class PX>
__global__ void __launch_bounds__(PW::kThreads, 2) ffn_products_kernel(ProductArgs W, ProductArgs X,
                                                                       int weights) {
  static_assert(PW::kThreads == PX::kThreads && PW::kLds == PX::kLds, "one shape");
  __shared__ __attribute__((aligned(16))) char lds[PW::kLds + kBoxes<PW>];
  if ((int)blockIdx.x < weights)
    product_unit<PW>(W, blockIdx.x, lds);
  else
    product_unit<PX>(X, blockIdx.x - weights, lds);
}

// out[z][r][c] = sum over splits of parts[s][z][r][c], in the order of s, of up to two products.
struct JoinArgs {
  void* out[2];
  const float* parts;
  int32_t splits, outputs;  // splits 0: nothing to join
  int64_t rows, cols, pitch;
};
template <class Op>
__device__ __forceinline__ void join(const JoinArgs& A, int64_t i) {
  typedef typename OutOf<Op>::T T;
  const int64_t quads = A.pitch / 4, each = A.rows * quads;
  const int64_t z = i / each, r = i % each / quads, c = i % each % quads * 4;
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int s = 0; s < A.splits; ++s) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(
        A.parts + (((int64_t)s * A.outputs + z) * A.rows + r) * A.pitch + c);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += v[e];
  }
  T* const p = static_cast<T*>(z ? A.out[1] : A.out[0]) + r * A.cols + c;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < A.cols) p[e] = (T)sum[e];
}
template <class Op>
__global__ void __launch_bounds__(256) ffn_join_kernel(JoinArgs W, JoinArgs X, int64_t nw, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    if (i < nw)
      join<Op>(W, i);
    else
      join<Op>(X, i - nw);
  }
}

// Up to three matrices' rows of `cols` values copied to rows of `pitch`, the rest zero.
struct PadArgs {
  void* out[3];
  const void* in[3];
  int64_t rows[3];
  int64_t cols, pitch;
};
template <class T>
__global__ void __launch_bounds__(256) ffn_pad_kernel(PadArgs A) {
  const int y = blockIdx.y;
  T* const out = static_cast<T*>(y == 0 ? A.out[0] : y == 1 ? A.out[1] : A.out[2]);
  const T* const in = static_cast<const T*>(y == 0 ? A.in[0] : y == 1 ? A.in[1] : A.in[2]);
  const int64_t n = (y == 0 ? A.rows[0] : y == 1 ? A.rows[1] : A.rows[2]) * A.pitch;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / A.pitch, c = i % A.pitch;
    out[i] = c < A.cols ? in[r * A.cols + c] : (T)0;
  }
}

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t a, int64_t b) { return cdiv(a, b) * b; }
bool whole_units(const void* p, int64_t rowbytes) {
  return rowbytes % 16 == 0 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}
unsigned grid_for(int64_t items) {
  const int64_t b = cdiv(items, 256);
  return (unsigned)(b < 1 ? 1 : (b > 65536 ? 65536 : b));
}
int esz_of(int32_t dtype) { return dtype == FMS_F32 ? 4 : 2; }

// Stream-ordered workspace, handed back when it goes out of scope.
struct Workspace {
  char* p = nullptr;
  hipStream_t st;
  explicit Workspace(hipStream_t s) : st(s) {}
  hipError_t take(int64_t bytes) {
    return bytes > 0 ? workspace_alloc(reinterpret_cast<void**>(&p), (size_t)bytes, st, true)
                     : hipSuccess;
  }
  ~Workspace() {
    if (p) (void)workspace_free(p, st);
  }
};

// The inputs as operands: as they are when their rows are whole 16-byte units, else copied
// into workspace rows that are.
struct Inputs {
  bool copy;
  int64_t pitch;  // bytes
  int64_t bytes;  // of workspace
};
Inputs inputs_of(const FfnArgs& a) {
  const int64_t row = a.dim * esz_of(a.dtype);
  Inputs in;
  in.copy = !(whole_units(a.x, row) && whole_units(a.wg, row) && whole_units(a.wu, row));
  in.pitch = round_up(row, 16);
  in.bytes = in.copy ? round_up((a.tokens + 2 * a.hidden) * in.pitch, 256) : 0;
  return in;
}
hipError_t launch_pad(int esz, const PadArgs& p, hipStream_t st) {
  int64_t most = p.rows[0] > p.rows[1] ? p.rows[0] : p.rows[1];
  most = (most > p.rows[2] ? most : p.rows[2]) * p.pitch;
  const dim3 grid(grid_for(most), 3);
  if (esz == 4)
    hipLaunchKernelGGL(ffn_pad_kernel<uint32_t>, grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL(ffn_pad_kernel<uint16_t>, grid, dim3(256), 0, st, p);
  return hipGetLastError();
}
hipError_t place_inputs(const FfnArgs& a, const Inputs& in, char* ws, Matrix (&m)[3],
                        hipStream_t st) {
  const int esz = esz_of(a.dtype);
  PadArgs p = {{nullptr, nullptr, nullptr}, {a.x, a.wg, a.wu}, {a.tokens, a.hidden, a.hidden},
               a.dim, in.pitch / esz};
  for (int i = 0; i < 3; ++i) {
    p.out[i] = ws;
    m[i] = Matrix{in.copy ? ws : static_cast<const char*>(p.in[i]), p.rows[i], in.pitch, in.pitch};
    ws += in.copy ? p.rows[i] * in.pitch : 0;
  }
  return in.copy && in.bytes > 0 ? launch_pad(esz, p, st) : hipSuccess;
}

// The tile shapes by element size: wave grid and 32-row fragments per wave.
template <class Op, bool kMRows, bool kNRows, int kParts>
struct Shapes {
  // 256 x 256, 8 waves (the one that makes dg and du spills 7 registers).  The pullback's products read dg and du from HBM and keep three
  // shorter steps in flight (23040 x 1024 x 4096, with dg and du in one plane each: 1490 us a
  // training step, 1512 with one step of 128 bytes); the projections' operands come from the
  // caches (290 us for 46080 x 768 x 2048, 315 with shorter steps).
  typedef Product<Op, kMRows, kNRows, kParts, 2, 4, 4, kParts == 2 ? 128 : 64> Big;
  typedef Product<Op, kMRows, kNRows, kParts, 2, 2, 2> Small;  // 128 x 128, 4 waves
  typedef Product<Op, kMRows, kNRows, kParts, 2, 2, 1> Tiny;   // 64 x 128, 4 waves
};

template <class P, bool kPull>
hipError_t launch_gate(GateArgs g, hipStream_t st) {
  g.tm = (int32_t)cdiv(g.tokens, P::kBM);
  g.tn = (int32_t)cdiv(g.out_cols, P::kBN / 2);
  g.steps = (int32_t)cdiv(g.x.rowbytes, P::kStepBytes);
  const int tiles = g.tm * g.tn, most = P::kThreads == 512 ? 256 : 512;  // a round of workgroups
  hipLaunchKernelGGL((ffn_gate_kernel<P, kPull>), dim3((unsigned)(tiles < most ? tiles : most)),
                     dim3(P::kThreads), 0, st, g);
  return hipGetLastError();
}

// 256 x 256 tiles run one workgroup to a CU; below one round of them 128 x 128 fills more
// CUs, and where those leave every CU at most one, 64 x 128 does (2048 tokens of 768 x 2048 in
// bf16: 16 us with 128 rows a tile, 21 with 64; 512 tokens: 11 and 9; in fp32 98 and 106, 54 and 32).
enum class Shape { kTiny, kSmall, kBig };
Shape gate_shape(int64_t rows, int64_t cols, int esz) {
  if (esz == 2 && cdiv(rows, 256) * cdiv(cols, 256) >= 192) return Shape::kBig;
  return cdiv(rows, 128) * cdiv(cols, 128) > 256 ? Shape::kSmall : Shape::kTiny;
}

// Eight hidden units a workgroup where sixteen would leave half the CUs without one (us in
// replayed graphs, 0.4 to 0.8 less than in a kernel trace, at dim 1024, one and 32 tokens: hidden
// 2048, 128 workgroups of sixteen, bf16 3.8 and 5.6 against 4.6 and 6.3, fp32 5.1 and 8.3 against
// 7.6 and 11.5; hidden 2560 bf16 5.0 and 8.6 against 4.6 and 6.4).
template <class Op, int kNT>
hipError_t launch_few(const GateArgs& g, hipStream_t st) {
  const int64_t ny = cdiv(g.tokens, 16 * kNT);
  const auto launch = [&](auto kernel, int hidden) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)cdiv(g.hidden, hidden), (unsigned)ny), dim3(64 * kFewWaves), 0, st,
                       g);
    return hipGetLastError();
  };
  if (cdiv(g.hidden, 16) * ny <= 128) return launch(ffn_few_kernel<Op, kNT, 8>, 8);
  return launch(ffn_few_kernel<Op, kNT, 16>, 16);
}

// Few tokens: against the 64-row tiles, whose time does not fall with the tokens (us in replayed
// graphs at 768 x 2048 / 1024 x 4096):
//   16 bits: 1 token 3.7 / 4.7, 32 tokens 5.1 / 6.5, 64 tokens 6.9 / 8.9 (tiles 7.8 / 9.6;
//   at dim 512 6.0 / 6.7 and 6.1 / 6.2, at dim 256 4.6 / 4.9 and 4.5 / 4.5);
//   32 bits: 1 token 4.9 / 7.7, 128 tokens 16 / 34 (tiles 31 / 42), 256 tokens 31 / 67 (32 / 42).
bool few_tokens(const GateArgs& g, int esz) {
  if (esz == 2) return g.tokens <= (g.x.rowbytes > 1024 ? 64 : 32);
  return g.tokens <= 256 && cdiv(g.hidden, 16) * cdiv(g.tokens, 64) <= 512;
}

template <class Op, bool kPull>
hipError_t run_gate(const GateArgs& g, hipStream_t st) {
  if (g.tokens == 0 || g.out_cols == 0) return hipSuccess;
  if (g.x.rowbytes == 0) {  // sums of nothing: h is zero (and no one asks for the gradients)
    return kPull ? hipErrorInvalidValue
                 : launch_pad(Op::kEsz, PadArgs{{g.out0, nullptr, nullptr}, {}, {g.tokens, 0, 0}, 0, g.out_pitch}, st);
  }
  if constexpr (!kPull)
    if (few_tokens(g, Op::kEsz)) {
      if (g.tokens <= 16) return launch_few<Op, 1>(g, st);
      if (g.tokens > 32) return launch_few<Op, 4>(g, st);
      return launch_few<Op, 2>(g, st);
    }
  typedef Shapes<Op, true, true, 2> S;
  const Shape shape = gate_shape(g.tokens, 2 * g.out_cols, Op::kEsz);
  if constexpr (Op::kEsz == 2)
    if (shape == Shape::kBig) return launch_gate<typename S::Big, kPull>(g, st);
  return shape == Shape::kSmall ? launch_gate<typename S::Small, kPull>(g, st)
                                : launch_gate<typename S::Tiny, kPull>(g, st);
}

// ---- how the pullback's products are cut --------------------------------------------------
// dwg and dwu have few tiles of many steps (a step is 64 tokens), dx has many tiles of few.
// One launch takes both, the longer units first, so that the shorter ones fill what the
// longer leave idle; a product whose units would outlast the others is cut along k into parts
// that a second kernel adds.  The choice is the least estimate over tile shapes and numbers of
// parts, with the times measured on this card: of 23040 x 1024 x 4096 in bf16 and one plane of dg
// and du the two products take 750 us in one launch and 850 one after the other (two planes, in
// one launch: 1430-1520).
struct Cut {
  Shape shape;
  int w, x;  // splits of the weights' products and of dx
};

// When `slots` workgroups at a time are through with nw units of uw us and then nx of ux.
double makespan(int64_t nw, double uw, int64_t nx, double ux, int64_t slots) {
  if (nw + nx > 16 * slots) return ((double)nw * uw + (double)nx * ux) / (double)slots;
  struct Group {
    int64_t slots;
    double free;
  } g[2] = {{slots - nw % slots, (double)(nw / slots) * uw}, {nw % slots, (double)(nw / slots + 1) * uw}};
  double end = g[1].slots > 0 ? g[1].free : g[0].free;
  while (nx > 0) {
    Group& first = g[1].slots > 0 && g[1].free < g[0].free ? g[1] : g[0];
    nx -= first.slots;  // (the last round's idle slots do not matter)
    first.free += ux;
    end = first.free > end ? first.free : end;
  }
  return end;
}
// us of a step (128 bytes of k) of a tile's unit that has a CU to itself, and of one of two on a CU.
struct Costs {
  int64_t rows, cols;  // of the tile
  double alone, shared;
};
constexpr Costs kCosts16[3] = {{64, 128, 0.45, 0.70}, {128, 128, 0.58, 1.00}, {256, 256, 1.55, 0.0}};
constexpr Costs kCosts32[2] = {{64, 128, 1.15, 2.20}, {128, 128, 2.10, 4.00}};

Cut choose_cut(const ProductArgs* w, const ProductArgs* x, int esz) {
  Cut best = {Shape::kSmall, 1, 1};
  double least = 1e300;
  for (int shape = 0; shape < (esz == 2 ? 3 : 2); ++shape) {
    const Costs& c = esz == 2 ? kCosts16[shape] : kCosts32[shape];
    const auto tiles = [&](const ProductArgs* p) {
      return p ? cdiv(p->rows, c.rows) * cdiv(p->cols, c.cols) * p->outputs : 0;
    };
    const int64_t tw = tiles(w), tx = tiles(x);
    for (int sw = 1; sw <= (w ? 64 : 1); sw *= 2)
      for (int sx = 1; sx <= (x ? 16 : 1); sx *= 2) {
        const bool alone = shape == (int)Shape::kBig || tw * sw + tx * sx <= 256;
        // (besides its steps a unit takes about 3 us to begin and to end, and a second kernel 3
        // us and the parts' way to memory and back)
        double joins = 0.0;
        const auto unit = [&](const ProductArgs* p, int splits) {
          if (p == nullptr) return 0.0;
          if (splits > 1)
            joins += 3.0 + 0.4 * splits * (double)(p->outputs * p->rows * p->cols) * 4 / (1 << 20);
          return 3.0 + (alone ? c.alone : c.shared) * (double)cdiv(p->segments * cdiv(p->bytes, 128), splits);
        };
        const double uw = unit(w, sw), ux = unit(x, sx);
        const double t = makespan(tw * sw, uw, tx * sx, ux, alone ? 256 : 512) + joins;
        if (t < least) {
          least = t;
          best = Cut{(Shape)shape, sw, sx};
        }
      }
  }
  return best;
}

template <class Op, class PW, class PX>
hipError_t launch_products(ProductArgs w, ProductArgs x, const Cut& cut, hipStream_t st) {
  const auto shape = [](ProductArgs& p, int64_t bm, int64_t bn, int splits) {
    p.tm = (int32_t)cdiv(p.rows, bm);
    p.tn = (int32_t)cdiv(p.cols, bn);
    p.steps = p.segments * (int32_t)cdiv(p.bytes, PW::kStepBytes);
    p.splits = splits < p.steps ? splits : (p.steps > 0 ? p.steps : 1);
    p.part_pitch = round_up(p.cols, 4);
    return p.splits > 1 ? round_up((int64_t)p.splits * p.outputs * p.rows * p.part_pitch * 4, 256) : 0;
  };
  const int64_t wb = shape(w, PW::kBM, PW::kBN, cut.w), xb = shape(x, PX::kBM, PX::kBN, cut.x);
  Workspace ws(st);
  hipError_t e = ws.take(wb + xb);
  if (e != hipSuccess) return e;
  w.parts = reinterpret_cast<float*>(ws.p);
  x.parts = reinterpret_cast<float*>(ws.p + wb);
  const int64_t nw = (int64_t)w.tm * w.tn * w.splits * w.outputs;
  const int64_t nx = (int64_t)x.tm * x.tn * x.splits * x.outputs;
  if (nw + nx == 0) return hipSuccess;
  hipLaunchKernelGGL((ffn_products_kernel<PW, PX>), dim3((unsigned)(nw + nx)), dim3(PW::kThreads), 0, st,
                     w, x, (int)nw);
  e = hipGetLastError();
  const auto joined = [](const ProductArgs& p) {
    return JoinArgs{{p.out[0], p.out[1]}, p.parts, p.splits > 1 ? p.splits : 0, p.outputs, p.rows, p.cols,
                    p.part_pitch};
  };
  const auto quads = [](const ProductArgs& p) {
    return p.splits > 1 ? p.outputs * p.rows * p.part_pitch / 4 : 0;
  };
  const int64_t jw = quads(w), jx = quads(x);
  if (e != hipSuccess || jw + jx == 0) return e;
  hipLaunchKernelGGL((ffn_join_kernel<Op>), dim3(grid_for(jw + jx)), dim3(256), 0, st, joined(w), joined(x),
                     jw, jw + jx);
  return hipGetLastError();
}

// w: dwg and dwu (or null), x: dx (or null).
template <class Op>
hipError_t run_products(const ProductArgs* w, const ProductArgs* x, hipStream_t st) {
  typedef Shapes<Op, false, false, 1> W;
  typedef Shapes<Op, true, false, 1> X;
  const Cut cut = choose_cut(w, x, Op::kEsz);
  const ProductArgs none = {};
  const ProductArgs &pw = w ? *w : none, &px = x ? *x : none;
  if constexpr (Op::kEsz == 2)
    if (cut.shape == Shape::kBig)
      return launch_products<Op, typename W::Big, typename X::Big>(pw, px, cut, st);
  if (cut.shape == Shape::kSmall)
    return launch_products<Op, typename W::Small, typename X::Small>(pw, px, cut, st);
  return launch_products<Op, typename W::Tiny, typename X::Tiny>(pw, px, cut, st);
}

GateArgs gate_args(const FfnArgs& a, const Matrix (&m)[3]) {
  GateArgs g = {};
  g.x = m[0];
  g.wg = m[1];
  g.wu = m[2];
  g.act = a.act;
  g.tokens = a.tokens;
  g.hidden = a.hidden;
  return g;
}

template <class Op>
hipError_t forward(const FfnArgs& a, void* h, hipStream_t st) {
  const Inputs in = inputs_of(a);
  Workspace ws(st);
  hipError_t e = ws.take(in.bytes);
  if (e != hipSuccess) return e;
  Matrix m[3];
  e = place_inputs(a, in, ws.p, m, st);
  if (e != hipSuccess) return e;
  GateArgs g = gate_args(a, m);
  g.out0 = h;
  g.out_cols = g.out_pitch = a.hidden;
  g.vec = whole_units(h, a.hidden * Op::kEsz);
  return run_gate<Op, false>(g, st);
}

template <class Op>
hipError_t pullback(const FfnArgs& a, void* dx, void* dwg, void* dwu, const void* dh,
                    hipStream_t st) {
  const Inputs in = inputs_of(a);
  const int64_t pitch = round_up(a.hidden * Op::kEsz, 16);  // of dg and du
  const int64_t each = round_up(a.tokens * pitch, 256);     // a plane of them
  constexpr int kDg = kPlanes<Op>;
  const bool any = a.tokens > 0 && a.hidden > 0, scaled = kScaled<Op> && any;
  // behind the planes the reciprocal of the power of two, and 256 bytes on the bound's parts
  Workspace ws(st);
  hipError_t e = ws.take(in.bytes + 2 * kDg * each + (scaled ? 256 + kMostBounds * (int64_t)sizeof(float2) : 0));
  if (e != hipSuccess) return e;
  Matrix m[3];
  e = place_inputs(a, in, ws.p, m, st);
  if (e != hipSuccess) return e;
  char* const dg = ws.p + in.bytes;
  GateArgs g = gate_args(a, m);
  g.in = dh;
  g.in_pitch = a.hidden;
  g.vec = whole_units(dh, a.hidden * Op::kEsz);
  g.out0 = dg;
  g.out1 = dg + kDg * each;
  g.plane = each;
  g.out_cols = g.out_pitch = pitch / Op::kEsz;
  if constexpr (kScaled<Op>)
    if (scaled) {
      g.unscale = reinterpret_cast<float*>(dg + 2 * kDg * each);
      float2* const bounds = reinterpret_cast<float2*>(dg + 2 * kDg * each + 256);
      g.bounds = bounds;
      const int64_t want = cdiv(a.tokens + 2 * a.hidden, kBoundWaves);
      g.nbounds = (int32_t)(want < kMostBounds ? want : kMostBounds);
      const BoundArgs b = {m[0], m[1], m[2], static_cast<const _Float16*>(dh), a.tokens, a.hidden, g.vec, bounds};
      hipLaunchKernelGGL(ffn_bound_kernel, dim3((unsigned)g.nbounds), dim3(64 * kBoundWaves), 0, st,
                         b);
      e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
  e = run_gate<Op, true>(g, st);
  if (e != hipSuccess) return e;
  ProductArgs w = {}, x = {};
  w.m = x.m = Matrix{dg, a.tokens, pitch, pitch};
  w.plane = x.plane = each;
  w.unscale = x.unscale = g.unscale;
  w.n[0] = w.n[1] = m[0];
  w.segments = kDg;
  w.outputs = 2;
  w.bytes = a.tokens * Op::kEsz;
  w.rows = a.hidden;
  w.cols = a.dim;
  w.out[0] = dwg;
  w.out[1] = dwu;
  w.vec = whole_units(dwg, a.dim * Op::kEsz) && whole_units(dwu, a.dim * Op::kEsz);
  x.n[0] = m[1];
  x.n[1] = m[2];
  x.segments = 2 * kDg;
  x.outputs = 1;
  x.bytes = pitch;
  x.rows = a.tokens;
  x.cols = a.dim;
  x.out[0] = dx;
  x.vec = whole_units(dx, a.dim * Op::kEsz);
  return run_products<Op>(dwg ? &w : nullptr, dx ? &x : nullptr, st);
}

}  // namespace

bool ffn_supported(const FfnArgs& a) {
  // a tile's 256 rows and a step's rows stay below 2^31 bytes from their first, and a
  // launch below 2^32 work-items of 128 x 128 tiles (of 64 hidden units)
  const int64_t most = ((int64_t)1 << 31) / 256 / 4 - 64;
  if (a.dim > most || a.hidden > most || a.tokens >= (int64_t)1 << 31) return false;
  const int64_t tm = cdiv(a.tokens, 128);
  return tm * cdiv(a.hidden + 8, 64) < (int64_t)1 << 24 && tm * cdiv(a.dim, 128) < (int64_t)1 << 24 &&
         cdiv(a.hidden, 128) * cdiv(a.dim, 128) * 2 < (int64_t)1 << 24;
}

hipError_t ffn_forward(const FfnArgs& a, void* h, hipStream_t stream) {
  switch (a.dtype) {
    case FMS_F16: return forward<OpF16>(a, h, stream);
    case FMS_BF16: return forward<OpBF16>(a, h, stream);
    default: return forward<OpF32>(a, h, stream);
  }
}

hipError_t ffn_pullback(const FfnArgs& a, void* dx, void* dwg, void* dwu, const void* dh,
                        hipStream_t stream) {
  switch (a.dtype) {
    case FMS_F16: return pullback<OpF16>(a, dx, dwg, dwu, dh, stream);
    case FMS_BF16: return pullback<OpBF16>(a, dx, dwg, dwu, dh, stream);
    default: return pullback<OpF32>(a, dx, dwg, dwu, dh, stream);
  }
}

}  // namespace fms

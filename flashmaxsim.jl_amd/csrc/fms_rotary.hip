// fms_rotary.hip -- the norm of each head of queries and keys and their rotation, in one pass.
//
//   n = norm(x) * w        (x itself without w), over the values of a head
//   y_a = n_a cos - n_b sin,  y_b = n_b cos + n_a sin     for the pairs (a, b) of the first `turned`
// values; the others are n.  The pullback turns the cotangent back, d = R^T dy, and then
//   dw = sum d * x^,  dx = i (d w - [mean(d w)] - x^ mean(d w x^))
// with x^ = norm(x) and i = 1 / sqrt(..) computed again from x.
//
// Bound by memory: forward moves 2 values an element, the pullback 3 (128 x 180 tokens of 16 and 16 heads
// of 64 in bf16: 41 us at 4.6 TB/s, 66 at 4.3, and 4 for the join).  A wave takes a token: its
// cosines and sines stay in registers while the token's heads, queries' and keys' alike, pass by,
// as many at a time as fit (a head of 64 16-bit values takes four lanes).  A lane holds both
// values of its pairs, so that the rotation needs no exchange, and the norm's sums run over the
// head's few lanes.  The weights' gradients stay in registers over a wave's tokens and are joined in a
// fixed order: lanes, waves through LDS, workgroups by a second kernel.
#include "fms_rotary.hpp"

#include <initializer_list>

#include "../../include/flashmaxsim_hip.h"
#include "fms_device.hpp"
#include "fms_group.hpp"

namespace fms {
namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A lane's share of a head: kN units of kU neighbouring pairs, units `lanes` apart.
template <class T_, int kU_, int kN_>
struct Share {
  typedef T_ T;
  static constexpr int kU = kU_, kN = kN_, kPairs = kU * kN;
  typedef T V __attribute__((ext_vector_type(kU)));

  struct Pairs {
    float a[kPairs], b[kPairs];
  };
  // Where unit u's a values and b values start in a head.
  struct Place {
    int a, b;
  };
  __device__ static __forceinline__ Place place(int u, int turned, int pairing) {
    const int p = u * kU, half = turned >> 1;
    if (pairing == FMS_PAIR_HALVES && p < half) return {p, half + p};
    return {2 * p, 2 * p + kU};  // (neighbours, and what is not turned: `half` pairs are behind it)
  }
  __device__ static __forceinline__ bool neighbours(int u, int turned, int pairing) {
    return pairing != FMS_PAIR_HALVES && u * kU < (turned >> 1);
  }
  __device__ static __forceinline__ void load(Pairs& x, const T* head, int first, int lanes, int pairs, int turned,
                                              int pairing) {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int u = first + n * lanes;
      V va = {}, vb = {};
      if (u * kU < pairs) {
        const Place at = place(u, turned, pairing);
        va = *reinterpret_cast<const V*>(head + at.a);
        vb = *reinterpret_cast<const V*>(head + at.b);
      }
      const bool mixed = neighbours(u, turned, pairing);
#pragma unroll
      for (int e = 0; e < kU; ++e) {
        // the 2 kU neighbouring values, or the pairs' first and second ones
        const float s = (float)va[e], t = (float)vb[e];
        const int i = 2 * e, j = 2 * e + 1;
        const float m = i < kU ? (float)va[i % kU] : (float)vb[i % kU];
        const float o = j < kU ? (float)va[j % kU] : (float)vb[j % kU];
        x.a[n * kU + e] = mixed ? m : s;
        x.b[n * kU + e] = mixed ? o : t;
      }
    }
  }
  __device__ static __forceinline__ void store(const Pairs& x, T* head, int first, int lanes, int pairs, int turned,
                                               int pairing) {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int u = first + n * lanes;
      if (u * kU >= pairs) continue;
      const Place at = place(u, turned, pairing);
      const bool mixed = neighbours(u, turned, pairing);
      V va, vb;
#pragma unroll
      for (int e = 0; e < kU; ++e) {
        const int i = e, j = kU + e;  // of the 2 kU neighbouring values
        const float m = i % 2 == 0 ? x.a[n * kU + i / 2] : x.b[n * kU + i / 2];
        const float o = j % 2 == 0 ? x.a[n * kU + j / 2] : x.b[n * kU + j / 2];
        va[e] = (T)(mixed ? m : x.a[n * kU + e]);
        vb[e] = (T)(mixed ? o : x.b[n * kU + e]);
      }
      *reinterpret_cast<V*>(head + at.a) = va;
      *reinterpret_cast<V*>(head + at.b) = vb;
    }
  }
};

// The sum over a head's lanes (a power of two of them).
__device__ __forceinline__ float head_sum(float v, int lanes) {
  for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

template <class S>
struct Turn {
  float cos[S::kPairs], sin[S::kPairs];
  __device__ __forceinline__ void load(const float* row, int first, int lanes, int turned) {
    const int half = turned >> 1;
#pragma unroll
    for (int n = 0; n < S::kN; ++n)
#pragma unroll
      for (int e = 0; e < S::kU; ++e) {
        const int p = (first + n * lanes) * S::kU + e;
        cos[n * S::kU + e] = p < half ? row[p] : 1.0f;
        sin[n * S::kU + e] = p < half ? row[half + p] : 0.0f;
      }
  }
  // by: 1, or -1 to turn back
  __device__ __forceinline__ void apply(typename S::Pairs& x, float by) const {
#pragma unroll
    for (int i = 0; i < S::kPairs; ++i) {
      const float a = x.a[i], b = x.b[i], s = by * sin[i];
      x.a[i] = a * cos[i] - b * s;
      x.b[i] = b * cos[i] + a * s;
    }
  }
};

// x -> norm(x) over a head's lanes; returns 1 / sqrt(..).  What is past the head is zero and stays it.
template <class S>
__device__ __forceinline__ float standardise(typename S::Pairs& x, int kind, int first, int lanes, int pairs,
                                             float inv_dim, float eps) {
  float s = 0.0f;
  if (kind == FMS_NORM_LAYER) {
#pragma unroll
    for (int i = 0; i < S::kPairs; ++i) s += x.a[i] + x.b[i];
    const float mean = head_sum(s, lanes) * inv_dim;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < S::kPairs; ++i) {
      const bool in = (first + i / S::kU * lanes) * S::kU < pairs;
      x.a[i] = in ? x.a[i] - mean : 0.0f;
      x.b[i] = in ? x.b[i] - mean : 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < S::kPairs; ++i) s += x.a[i] * x.a[i] + x.b[i] * x.b[i];
  const float inv = 1.0f / sqrtf(head_sum(s, lanes) * inv_dim + eps);
#pragma unroll
  for (int i = 0; i < S::kPairs; ++i) {
    x.a[i] *= inv;
    x.b[i] *= inv;
  }
  return inv;
}

// The table row of token (b, t), or -1 where its position is none of the table's.
__device__ __forceinline__ int64_t table_row(const RotaryArgs& A, int64_t b, int64_t t) {
  int64_t row = t;
  if (A.positions) {
    const int64_t at = A.position_seqs == 1 ? t : b * A.tokens + t;
    row = A.position_bytes == 8 ? static_cast<const int64_t*>(A.positions)[at] - 1
                                : (int64_t) static_cast<const int32_t*>(A.positions)[at] - 1;
  }
  return row >= 0 && row < A.table_rows ? row : -1;
}

template <class S>
__global__ void __launch_bounds__(256) rotary_forward_kernel(RotaryArgs A, typename S::T* q_out, typename S::T* k_out,
                                                             int lanes) {
  typedef typename S::T T;
  const int lane = threadIdx.x & 63, first = lane & (lanes - 1), sub = lane / lanes;
  const int pairs = A.dim >> 1, all = A.heads + A.kv_heads, at_once = 64 / lanes;
  const float inv_dim = 1.0f / (float)A.dim;
  typename S::Pairs wq, wk;
  if (A.wq) S::load(wq, static_cast<const T*>(A.wq), first, lanes, pairs, A.turned, A.pairing);
  if (A.wk) S::load(wk, static_cast<const T*>(A.wk), first, lanes, pairs, A.turned, A.pairing);
  const int64_t n = A.seqs * A.tokens;
  for (int64_t token = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); token < n; token += (int64_t)gridDim.x * 4) {
    const int64_t b = A.seqs == 1 ? 0 : token / A.tokens, t = token - b * A.tokens;
    const int64_t row = table_row(A, b, t);
    Turn<S> turn;
    if (row >= 0) turn.load(A.table + row * A.turned, first, lanes, A.turned);
    // (a head is all or nothing of its lanes: the sums see whole heads)
    for (int h = sub; h < all; h += at_once) {
      const bool key = h >= A.heads;
      const T* from = key ? static_cast<const T*>(A.k) + b * A.ks[0] + t * A.ks[1] + (h - A.heads) * A.ks[2]
                          : static_cast<const T*>(A.q) + b * A.qs[0] + t * A.qs[1] + h * A.qs[2];
      T* to = key ? k_out + (token * A.kv_heads + h - A.heads) * A.dim : q_out + (token * A.heads + h) * A.dim;
      typename S::Pairs x = {};
      if (row >= 0) {
        S::load(x, from, first, lanes, pairs, A.turned, A.pairing);
        if (key ? A.wk : A.wq) {
          standardise<S>(x, A.kind, first, lanes, pairs, inv_dim, A.eps);
#pragma unroll
          for (int i = 0; i < S::kPairs; ++i) {
            x.a[i] *= key ? wk.a[i] : wq.a[i];
            x.b[i] *= key ? wk.b[i] : wq.b[i];
          }
        }
        turn.apply(x, 1.0f);
      }
      S::store(x, to, first, lanes, pairs, A.turned, A.pairing);
    }
  }
}

// parts[block][0] dwq, [1] dwk: dim floats each.
template <class S>
__global__ void __launch_bounds__(256) rotary_pullback_kernel(RotaryArgs A, RotaryGrads G, int lanes, float* parts) {
  typedef typename S::T T;
  __shared__ float lds[4][2 * kRotaryMaxDim];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = lane & (lanes - 1), sub = lane / lanes;
  const int pairs = A.dim >> 1, all = A.heads + A.kv_heads, at_once = 64 / lanes;
  const float inv_dim = 1.0f / (float)A.dim;
  typename S::Pairs wq, wk, sum[2] = {};
  if (A.wq) S::load(wq, static_cast<const T*>(A.wq), first, lanes, pairs, A.turned, A.pairing);
  if (A.wk) S::load(wk, static_cast<const T*>(A.wk), first, lanes, pairs, A.turned, A.pairing);
  const int64_t n = A.seqs * A.tokens;
  for (int64_t token = (int64_t)blockIdx.x * 4 + wave; token < n; token += (int64_t)gridDim.x * 4) {
    const int64_t b = A.seqs == 1 ? 0 : token / A.tokens, t = token - b * A.tokens;
    const int64_t row = table_row(A, b, t);
    Turn<S> turn;
    if (row >= 0) turn.load(A.table + row * A.turned, first, lanes, A.turned);
    for (int h = sub; h < all; h += at_once) {
      const bool key = h >= A.heads;
      const T* from = key ? static_cast<const T*>(A.k) + b * A.ks[0] + t * A.ks[1] + (h - A.heads) * A.ks[2]
                          : static_cast<const T*>(A.q) + b * A.qs[0] + t * A.qs[1] + h * A.qs[2];
      const int64_t at = key ? (token * A.kv_heads + h - A.heads) * A.dim : (token * A.heads + h) * A.dim;
      typename S::Pairs d = {};
      if (row >= 0) {
        S::load(d, static_cast<const T*>(key ? G.dk_out : G.dq_out) + at, first, lanes, pairs, A.turned, A.pairing);
        const bool norm = key ? A.wk : A.wq;
        typename S::Pairs x;
        if (norm) S::load(x, from, first, lanes, pairs, A.turned, A.pairing);
        turn.apply(d, -1.0f);
        if (norm) {
          const float inv = standardise<S>(x, A.kind, first, lanes, pairs, inv_dim, A.eps);
          float dot = 0.0f, mean = 0.0f;
#pragma unroll
          for (int i = 0; i < S::kPairs; ++i) {
            const float da = d.a[i] * x.a[i], db = d.b[i] * x.b[i];
            sum[0].a[i] += key ? 0.0f : da;
            sum[0].b[i] += key ? 0.0f : db;
            sum[1].a[i] += key ? da : 0.0f;
            sum[1].b[i] += key ? db : 0.0f;
            d.a[i] *= key ? wk.a[i] : wq.a[i];
            d.b[i] *= key ? wk.b[i] : wq.b[i];
            dot += d.a[i] * x.a[i] + d.b[i] * x.b[i];
            mean += d.a[i] + d.b[i];
          }
          dot = head_sum(dot, lanes) * inv_dim;
          mean = A.kind == FMS_NORM_LAYER ? head_sum(mean, lanes) * inv_dim : 0.0f;
#pragma unroll
          for (int i = 0; i < S::kPairs; ++i) {
            d.a[i] = (d.a[i] - mean - x.a[i] * dot) * inv;
            d.b[i] = (d.b[i] - mean - x.b[i] * dot) * inv;
          }
        }
      }
      S::store(d, static_cast<T*>(key ? G.dk : G.dq) + at, first, lanes, pairs, A.turned, A.pairing);
    }
  }
  if (!parts) return;
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int i = 0; i < S::kPairs; ++i) {
      float a = sum[w].a[i], b = sum[w].b[i];
      for (int o = lanes; o < 64; o <<= 1) {
        a += __shfl_xor(a, o);
        b += __shfl_xor(b, o);
      }
      const int u = first + i / S::kU * lanes;
      if (sub == 0 && u * S::kU < pairs) {
        // (where the values lie in a head: a pair's own, or its place among neighbours)
        const typename S::Place at = S::place(u, A.turned, A.pairing);
        const int e = i % S::kU;
        const bool mixed = S::neighbours(u, A.turned, A.pairing);
        lds[wave][w * kRotaryMaxDim + (mixed ? at.a + 2 * e : at.a + e)] = a;
        lds[wave][w * kRotaryMaxDim + (mixed ? at.a + 2 * e + 1 : at.b + e)] = b;
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * A.dim; i += 256) {
    const int w = i / A.dim, k = i - w * A.dim, at = w * kRotaryMaxDim + k;
    parts[(int64_t)blockIdx.x * 2 * A.dim + i] = (lds[0][at] + lds[1][at]) + (lds[2][at] + lds[3][at]);
  }
}

// The workgroups' partial sums -> dwq (blockIdx.y 0) and dwk (1): 64 columns a workgroup.
template <class T>
__global__ void __launch_bounds__(1024) rotary_join_kernel(T* dwq, T* dwk, const float* parts, int64_t blocks, int dim) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = blockIdx.x * 64 + lane;
  T* out = blockIdx.y ? dwk : dwq;
  if (out == nullptr) return;  // (the whole workgroup)
  float s = 0.0f;
  if (k < dim)
#pragma unroll 8
    for (int64_t b = wave; b < blocks; b += 16) s += parts[(b * 2 + blockIdx.y) * dim + k];
  lds[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && k < dim) {
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += lds[w][lane];
    out[k] = (T)s;
  }
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Units of 16 bytes: every part of a head, and every head, is whole ones.  (Other widths take a value at a time: 128 x
// 180 tokens of 16 and 16 heads in bf16, forward and back, 558 us with heads of 72 and 169 with heads of 80.)
bool whole_units(const RotaryArgs& a, std::initializer_list<const void*> ptrs) {
  const int64_t esz = a.dtype == FMS_F32 ? 4 : 2;
  if (a.dim * esz % 32 != 0 || a.turned * esz % 32 != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (a.qs[i] * esz % 16 != 0 || a.ks[i] * esz % 16 != 0) return false;
  for (const void* p : ptrs)
    if (!aligned(p)) return false;
  return true;
}

template <class T, class F>
hipError_t by_dim(const RotaryArgs& a, bool vec, F&& f) {
  constexpr int kU = 16 / sizeof(T);
  const auto lanes = [&](int per) {  // of a head, a power of two
    int n = 1;
    while (n * per < a.dim / 2) n <<= 1;
    return n;
  };
  if (vec) return f(Share<T, kU, 1>(), lanes(kU));
  if (a.dim <= 128) return f(Share<T, 1, 1>(), lanes(1));
  return f(Share<T, 1, 4>(), lanes(4));
}
template <class F>
hipError_t by_share(const RotaryArgs& a, bool vec, F&& f) {
  switch (a.dtype) {
    case FMS_F16: return by_dim<_Float16>(a, vec, f);
    case FMS_BF16: return by_dim<__bf16>(a, vec, f);
    default: return by_dim<float>(a, vec, f);
  }
}

}  // namespace

hipError_t rotary_forward(const RotaryArgs& a, void* q_out, void* k_out, hipStream_t stream) {
  const bool vec = whole_units(a, {a.q, a.k, a.wq, a.wk, q_out, k_out});
  return by_share(a, vec, [&](auto share, int lanes) {
    typedef decltype(share) S;
    const int64_t want = cdiv(a.seqs * a.tokens, 4), most = 8192;
    hipLaunchKernelGGL((rotary_forward_kernel<S>), dim3((unsigned)(want < most ? want : most)), dim3(256), 0, stream, a,
                       static_cast<typename S::T*>(q_out), static_cast<typename S::T*>(k_out), lanes);
    return hipGetLastError();
  });
}

hipError_t rotary_pullback(const RotaryArgs& a, const RotaryGrads& g, hipStream_t stream) {
  const bool vec = whole_units(a, {a.q, a.k, a.wq, a.wk, g.dq_out, g.dk_out, g.dq, g.dk});
  return by_share(a, vec, [&](auto share, int lanes) {
    typedef decltype(share) S;
    typedef typename S::T T;
    // (three to a CU, as many as the largest share's registers let in: 66 us for the header's case, 81 with four, whose
    // last quarter runs by itself, 78 with two)
    const int64_t want = cdiv(a.seqs * a.tokens, 4), most = 768;
    const int64_t blocks = want < most ? want : most;
    const bool weights = g.dwq || g.dwk;
    void* parts = nullptr;
    hipError_t e = hipSuccess;
    if (weights && blocks > 0) e = workspace_alloc(&parts, (size_t)(blocks * 2 * a.dim * 4), stream, true);
    if (e != hipSuccess) return e;
    if (blocks > 0)
      hipLaunchKernelGGL((rotary_pullback_kernel<S>), dim3((unsigned)blocks), dim3(256), 0, stream, a, g, lanes,
                         static_cast<float*>(parts));
    if (weights)
      hipLaunchKernelGGL((rotary_join_kernel<T>), dim3((unsigned)cdiv(a.dim, 64), 2), dim3(1024), 0, stream,
                         static_cast<T*>(g.dwq), static_cast<T*>(g.dwk), static_cast<const float*>(parts), blocks,
                         (int)a.dim);
    e = hipGetLastError();
    const hipError_t ef = parts ? workspace_free(parts, stream) : hipSuccess;
    return e != hipSuccess ? e : ef;
  });
}

}  // namespace fms

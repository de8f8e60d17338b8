// fms_norm.hip -- norms before and after a block, fused with its gate and residual.
//
//   z = norm(f) * wpost   (f itself without wpost)
//   r = x + scale * gate * z
//   n = norm(r) * wpre
// with norm(a) = (a - mean a) / sqrt(var a + eps) (layer) or a / sqrt(mean a^2 + eps)
// (rms): the end of one block and the start of the next in one pass.  Given dr and dn, with
// a^ = norm(a), i = 1 / sqrt(..) and D(d, a^, i) = i (d - [mean d] - a^ mean(d a^)):
//   dr' = dr + D(dn wpre, r^, i_r)      dx = dr'
//   dz  = scale gate dr'                df = D(dz wpost, f^, i_f)  (dz without wpost)
//   dgate = sum scale z dr',  dwpost = sum dz f^,  dwpre = sum dn r^
//
// Everything is bound by memory: forward moves 4 values an element, the pullback 6 (it
// computes r, both norms and their statistics again from x and f, so the forward keeps
// nothing and nothing is rounded in between).  A row lives in the registers of one wave
// (up to 1024 elements), of four (4096) or of sixteen; statistics are fp32 sums over the
// registers, the mean first and then the squares around it.  The column sums over rows
// stay in registers over a workgroup's rows and are joined in a fixed order: waves
// through LDS, workgroups by a second kernel.
//
// That does not hold for the pullback of rows over 4096: a workgroup of sixteen waves has 128
// registers a lane, and 235 to 354 of them spill to 532 to 832 bytes of scratch.  Measured
// (with all inputs, one gate): 8192 rows of 4096 in bf16 forward 44 us and pullback 110, 4096 rows of
// 8192 57 and 2785 (fp32: 102 and 1028), 2048 rows of 16384 49 and 1482 (103 and 620).
#include "fms_norm.hpp"

#include "../../include/flashmaxsim_hip.h"
#include "fms_device.hpp"
#include "fms_group.hpp"

namespace fms {
namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A lane's share of a row: kPer elements, in units of kUnit neighbours (16 bytes, or one
// element where rows are no whole 16-byte units).
template <class T_, int kUnit_, int kPer_, int kWaves_>
struct Row {
  typedef T_ T;
  static constexpr int kUnit = kUnit_, kPer = kPer_, kUnits = kPer / kUnit;
  static constexpr int kWaves = kWaves_;                    // waves that share a row
  static constexpr int kThreads = kWaves == 16 ? 1024 : 256;
  static constexpr int kRows = kThreads / 64 / kWaves;      // rows in flight
  typedef T V __attribute__((ext_vector_type(kUnit)));  // (one element: a vector of one)
  // Rows of at most 64 elements, one a lane, are computed in double: a short row's gradient
  // is a difference of nearly equal terms (of two elements, all of it), and one value a
  // lane costs nothing beside the load.
  typedef std::conditional_t<kPer == 1, double, float> F;

  // A share as it lies in memory: what is read before it is needed, and weights.
  struct Packed {
    V v[kUnits];
    __device__ __forceinline__ F operator[](int j) const { return (F)(float)v[j / kUnit][j % kUnit]; }
  };
  __device__ static __forceinline__ void load(Packed& p, const T* row, int dim) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      p.v[i] = V{};
      if (at(i) < dim) p.v[i] = *reinterpret_cast<const V*>(row + at(i));
    }
  }
  __device__ static __forceinline__ void unpack(F (&v)[kPer], const Packed& p) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = p[j];
  }

  // The first element of this thread's unit i.
  __device__ static __forceinline__ int at(int i) {
    const int t = kWaves == 1 ? threadIdx.x & 63 : threadIdx.x;
    return (i * (64 * kWaves) + t) * kUnit;
  }
  __device__ static __forceinline__ void load(F (&v)[kPer], const T* row, int dim) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int k = at(i);
      if constexpr (kUnit == 1) {
        v[i] = k < dim ? (F)row[k] : (F)0;
      } else {
        V u = {};
        if (k < dim) u = *reinterpret_cast<const V*>(row + k);
#pragma unroll
        for (int e = 0; e < kUnit; ++e) v[i * kUnit + e] = (float)u[e];
      }
    }
  }
  __device__ static __forceinline__ void store(const F (&v)[kPer], T* row, int dim) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int k = at(i);
      if (k >= dim) continue;
      if constexpr (kUnit == 1) {
        row[k] = (T)(float)v[i];
      } else {
        V u;
#pragma unroll
        for (int e = 0; e < kUnit; ++e) u[e] = (T)v[i * kUnit + e];
        *reinterpret_cast<V*>(row + k) = u;
      }
    }
  }
  // Whether element j of this thread's share is inside the row.
  __device__ static __forceinline__ bool inside(int j, int dim) {
    return at(j / kUnit) < dim;  // (a row is whole units)
  }
};

// The sum over a row's threads of one value each, the same in all of them.
template <class R>
__device__ __forceinline__ typename R::F row_sum(typename R::F v, float* lds) {
  if constexpr (R::kPer == 1) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  } else {  // rotations within 16 lanes, then the four sixteens (no trip through LDS)
    v = dpp_add<0x121>(v);
    v = dpp_add<0x122>(v);
    v = dpp_add<0x124>(v);
    v = dpp_add<0x128>(v);
    const auto of = [&](int lane) {
      return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    };
    v = (of(0) + of(16)) + (of(32) + of(48));
  }
  if constexpr (R::kWaves > 1) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[wave] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < R::kWaves; ++w) v += lds[w];
  }
  return v;
}

// v -> norm(v); returns 1 / sqrt(..).
template <class R>
__device__ __forceinline__ typename R::F standardise(typename R::F (&v)[R::kPer], int kind, int dim,
                                                     typename R::F inv_dim, float eps, float* lds) {
  typedef typename R::F F;
  F s = 0;
  if (kind == FMS_NORM_LAYER) {
#pragma unroll
    for (int j = 0; j < R::kPer; ++j) s += v[j];
    const F mean = row_sum<R>(s, lds) * inv_dim;
    s = 0;
#pragma unroll
    for (int j = 0; j < R::kPer; ++j) v[j] = R::inside(j, dim) ? v[j] - mean : (F)0;
  }
#pragma unroll
  for (int j = 0; j < R::kPer; ++j) s += v[j] * v[j];
  const F inv = (F)1 / sqrt(row_sum<R>(s, lds) * inv_dim + (F)eps);
#pragma unroll
  for (int j = 0; j < R::kPer; ++j) v[j] *= inv;
  return inv;
}

// d -> D(d, hat, inv).
template <class R>
__device__ __forceinline__ void standardise_back(typename R::F (&d)[R::kPer],
                                                 const typename R::F (&hat)[R::kPer],
                                                 typename R::F inv, int kind, typename R::F inv_dim,
                                                 float* lds) {
  typedef typename R::F F;
  F s = 0, m = 0;
#pragma unroll
  for (int j = 0; j < R::kPer; ++j) s += d[j] * hat[j];
  const F dot = row_sum<R>(s, lds) * inv_dim;
  if (kind == FMS_NORM_LAYER) {
#pragma unroll
    for (int j = 0; j < R::kPer; ++j) m += d[j];
    m = row_sum<R>(m, lds) * inv_dim;
  }
#pragma unroll
  for (int j = 0; j < R::kPer; ++j) d[j] = (d[j] - m - hat[j] * dot) * inv;
}

template <class R>
__global__ void __launch_bounds__(R::kThreads) norm_forward_kernel(NormArgs A, typename R::T* r_out,
                                                                   typename R::T* n_out) {
  typedef typename R::T T;
  typedef typename R::F F;
  __shared__ float lds[16];
  const int dim = (int)A.dim;
  const F inv_dim = (F)1 / (F)dim;
  const int sub = R::kWaves == 1 ? threadIdx.x >> 6 : 0;
  typename R::Packed wpost, wpre, gate;
  if (A.wpost) R::load(wpost, static_cast<const T*>(A.wpost), dim);
  if (A.wpre) R::load(wpre, static_cast<const T*>(A.wpre), dim);
  int64_t group = -1;
  for (int64_t row = (int64_t)blockIdx.x * R::kRows + sub; row < A.rows;
       row += (int64_t)gridDim.x * R::kRows) {
    const int64_t at = row * A.dim;
    F v[R::kPer];
    R::load(v, static_cast<const T*>(A.x) + at, dim);
    if (A.f) {
      F z[R::kPer];
      R::load(z, static_cast<const T*>(A.f) + at, dim);
      if (A.gate && row / A.gate_rows != group) {
        group = row / A.gate_rows;
        R::load(gate, static_cast<const T*>(A.gate) + group * A.dim, dim);
      }
      if (A.wpost) {
        standardise<R>(z, A.kind, dim, inv_dim, A.eps, lds);
#pragma unroll
        for (int j = 0; j < R::kPer; ++j) z[j] *= wpost[j];
      }
#pragma unroll
      for (int j = 0; j < R::kPer; ++j) v[j] += (A.gate ? A.scale * gate[j] : A.scale) * z[j];
      R::store(v, r_out + at, dim);
    }
    if (A.wpre) {
      standardise<R>(v, A.kind, dim, inv_dim, A.eps, lds);
#pragma unroll
      for (int j = 0; j < R::kPer; ++j) v[j] *= wpre[j];
      R::store(v, n_out + at, dim);
    }
  }
}

// What the pullback's column sums are cut into: a workgroup takes `groups` whole groups of
// `group_rows` rows, or one of `parts` equal parts of one group.
struct Spans {
  int64_t group_rows, ngroups;
  int64_t groups;  // per workgroup
  int64_t parts;   // per group
  int64_t blocks;
};

// Sums over the workgroup's rows in flight of each column's value, to out[column].
template <class R, class S>
__device__ __forceinline__ void join_columns(const typename R::F (&v)[R::kPer], float* lds, int dim, S&& put) {
  if constexpr (R::kWaves > 1) {
#pragma unroll
    for (int j = 0; j < R::kPer; ++j) {
      const int k = R::at(j / R::kUnit) + j % R::kUnit;
      if (k < dim) put(k, (float)v[j]);
    }
  } else {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < R::kPer; ++j) {
      const int k = R::at(j / R::kUnit) + j % R::kUnit;
      if (k < dim) lds[wave * (64 * R::kPer) + k] = (float)v[j];
    }
    __syncthreads();
    for (int k = threadIdx.x; k < dim; k += R::kThreads) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < R::kRows; ++w) s += lds[w * (64 * R::kPer) + k];
      put(k, s);
    }
  }
}

// What the pullback reads of a row; what was not given is zero.
template <class R>
struct Inputs {
  typename R::Packed dr, dn, x, f;
  __device__ __forceinline__ void load(const NormArgs& A, const NormGrads& G, int64_t row) {
    typedef typename R::T T;
    const int64_t at = row * A.dim;
    const auto one = [&](typename R::Packed& p, const void* from, bool given) {
      p = typename R::Packed{};
      if (given) R::load(p, static_cast<const T*>(from) + at, (int)A.dim);
    };
    one(dr, G.dr, G.dr != nullptr);
    one(dn, G.dn, G.dn != nullptr);
    one(x, A.x, G.dn != nullptr);
    one(f, A.f, A.f != nullptr);
  }
};

// Partial sums of a workgroup: parts[block][0] dwpost, [1] dwpre, [2] dgate (only where a
// group has several parts), each dim floats.
template <class R>
__global__ void __launch_bounds__(R::kThreads) norm_pullback_kernel(NormArgs A, NormGrads G, Spans S,
                                                                    float* parts) {
  typedef typename R::T T;
  typedef typename R::F F;
  __shared__ float lds[R::kWaves == 1 ? R::kRows * 64 * R::kPer : 16];
  const int dim = (int)A.dim;
  const F inv_dim = (F)1 / (F)dim;
  const int sub = R::kWaves == 1 ? threadIdx.x >> 6 : 0;
  typename R::Packed wpost, wpre, gate;
  F spost[R::kPer] = {}, spre[R::kPer] = {};
  if (A.wpost) R::load(wpost, static_cast<const T*>(A.wpost), dim);
  if (A.wpre) R::load(wpre, static_cast<const T*>(A.wpre), dim);
  const int64_t g0 = blockIdx.x / S.parts * S.groups, part = blockIdx.x % S.parts;
  const bool own_gate = A.gate && A.gate_rows == 1;  // a gate per row: its gradient is one too
  float* mine = parts + (int64_t)blockIdx.x * 3 * A.dim;
  for (int64_t g = g0; g < g0 + S.groups && g < S.ngroups; ++g) {
    const int64_t first = g * S.group_rows + S.group_rows * part / S.parts;
    const int64_t last = g * S.group_rows + S.group_rows * (part + 1) / S.parts;
    F sgate[R::kPer] = {};
    if (A.gate && !own_gate) R::load(gate, static_cast<const T*>(A.gate) + g * A.dim, dim);
    for (int64_t row = first + sub; row < last; row += R::kRows) {
      const int64_t at = row * A.dim;
      Inputs<R> in;
      in.load(A, G, row);
      F d[R::kPer], r[R::kPer], fhat[R::kPer], dn[R::kPer], finv = 0;
      R::unpack(d, in.dr);
      R::unpack(r, in.x);
      R::unpack(fhat, in.f);
      R::unpack(dn, in.dn);
      if (own_gate) R::load(gate, static_cast<const T*>(A.gate) + at, dim);
      if (A.f && A.wpost) finv = standardise<R>(fhat, A.kind, dim, inv_dim, A.eps, lds);
      if (G.dn) {
        if (A.f)
#pragma unroll
          for (int j = 0; j < R::kPer; ++j)
            r[j] += (A.gate ? A.scale * gate[j] : A.scale) * (A.wpost ? fhat[j] * wpost[j] : fhat[j]);
        const F rinv = standardise<R>(r, A.kind, dim, inv_dim, A.eps, lds);
#pragma unroll
        for (int j = 0; j < R::kPer; ++j) {
          spre[j] += dn[j] * r[j];
          dn[j] *= wpre[j];
        }
        standardise_back<R>(dn, r, rinv, A.kind, inv_dim, lds);
#pragma unroll
        for (int j = 0; j < R::kPer; ++j) d[j] += dn[j];
      }
      if (G.dx) R::store(d, static_cast<T*>(G.dx) + at, dim);
      if (!A.f) continue;
      if (A.gate) {
        F dg[R::kPer];
#pragma unroll
        for (int j = 0; j < R::kPer; ++j) {
          dg[j] = A.scale * (A.wpost ? fhat[j] * wpost[j] : fhat[j]) * d[j];
          sgate[j] += dg[j];
        }
        if (own_gate) R::store(dg, static_cast<T*>(G.dgate) + at, dim);
      }
#pragma unroll
      for (int j = 0; j < R::kPer; ++j) d[j] *= A.gate ? A.scale * gate[j] : A.scale;
      if (A.wpost) {
#pragma unroll
        for (int j = 0; j < R::kPer; ++j) {
          spost[j] += d[j] * fhat[j];
          d[j] *= wpost[j];
        }
        standardise_back<R>(d, fhat, finv, A.kind, inv_dim, lds);
      }
      R::store(d, static_cast<T*>(G.df) + at, dim);
    }
    if (A.gate && !own_gate) {
      if (S.parts > 1) {
        join_columns<R>(sgate, lds, dim, [&](int k, float v) { mine[2 * A.dim + k] = v; });
      } else {
        T* out = static_cast<T*>(G.dgate) + g * A.dim;
        join_columns<R>(sgate, lds, dim, [&](int k, float v) { out[k] = (T)v; });
      }
    }
  }
  if (A.wpost) join_columns<R>(spost, lds, dim, [&](int k, float v) { mine[k] = v; });
  if (A.wpre) join_columns<R>(spre, lds, dim, [&](int k, float v) { mine[A.dim + k] = v; });
}

// The workgroups' partial sums -> dwpost (blockIdx.y 0), dwpre (1), dgate of group
// blockIdx.y - 2: 64 columns a workgroup, its 16 waves over the partials.
template <class T>
__global__ void __launch_bounds__(1024) norm_join_kernel(NormGrads G, const float* parts,
                                                         int64_t blocks, int64_t per_group, int dim) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int k = blockIdx.x * 64 + lane;
  const int what = blockIdx.y < 2 ? blockIdx.y : 2;
  T* out = static_cast<T*>(what == 0 ? G.dwpost : what == 1 ? G.dwpre : G.dgate);
  if (out == nullptr) return;  // (the whole workgroup)
  const int64_t first = what < 2 ? 0 : (int64_t)(blockIdx.y - 2) * per_group;
  const int64_t last = what < 2 ? blocks : first + per_group;
  float s = 0.0f;
  if (k < dim)
#pragma unroll 8
    for (int64_t b = first + wave; b < last; b += 16) s += parts[(b * 3 + what) * dim + k];
  lds[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && k < dim) {
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += lds[w][lane];
    out[(what == 2 ? (int64_t)(blockIdx.y - 2) * dim : 0) + k] = (T)s;
  }
}

// Calls f(Row<...>) for the row's shape.
template <class T, int kUnit, class F>
hipError_t by_dim(int64_t dim, F&& f) {
  if (dim <= 64) return f(Row<T, 1, 1, 1>());
  if (dim <= 512) return f(Row<T, kUnit, 8, 1>());
  if (dim <= 1024) return f(Row<T, kUnit, 16, 1>());
  if (dim <= 2048) return f(Row<T, kUnit, 8, 4>());
  if (dim <= 4096) return f(Row<T, kUnit, 16, 4>());
  return f(Row<T, kUnit, 16, 16>());
}
template <class F>
hipError_t by_row(int32_t dtype, bool vec, int64_t dim, F&& f) {
  switch (dtype) {
    case FMS_F16: return vec ? by_dim<_Float16, 8>(dim, f) : by_dim<_Float16, 1>(dim, f);
    case FMS_BF16: return vec ? by_dim<__bf16, 8>(dim, f) : by_dim<__bf16, 1>(dim, f);
    default: return vec ? by_dim<float, 4>(dim, f) : by_dim<float, 1>(dim, f);
  }
}

bool whole_units(int32_t dtype, int64_t dim, std::initializer_list<const void*> ptrs) {
  if (dim * (dtype == FMS_F32 ? 4 : 2) % 16 != 0) return false;
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) & 15u) return false;
  return true;
}

}  // namespace

hipError_t norm_forward(const NormArgs& a, void* r, void* n, hipStream_t stream) {
  const bool vec = whole_units(a.dtype, a.dim, {a.x, a.f, a.gate, a.wpost, a.wpre, r, n});
  return by_row(a.dtype, vec, a.dim, [&](auto row) {
    typedef decltype(row) R;
    typedef typename R::T T;
    const int64_t want = cdiv(a.rows, R::kRows), most = 256 * 2048 / R::kThreads;
    hipLaunchKernelGGL((norm_forward_kernel<R>), dim3((unsigned)(want < most ? want : most)),
                       dim3(R::kThreads), 0, stream, a, static_cast<T*>(r), static_cast<T*>(n));
    return hipGetLastError();
  });
}

hipError_t norm_pullback(const NormArgs& a, const NormGrads& g, hipStream_t stream) {
  const bool vec = whole_units(a.dtype, a.dim, {a.x, a.f, a.gate, a.wpost, a.wpre, g.dr, g.dn,
                                                g.dx, g.df, g.dgate});
  return by_row(a.dtype, vec, a.dim, [&](auto row) {
    typedef decltype(row) R;
    typedef typename R::T T;
    if (a.rows == 0) {  // the weights' gradients are zeros
      hipLaunchKernelGGL((norm_join_kernel<T>), dim3((unsigned)cdiv(a.dim, 64), 2), dim3(1024), 0,
                         stream, g, static_cast<const float*>(nullptr), (int64_t)0, (int64_t)0,
                         (int)a.dim);
      return hipGetLastError();
    }
    Spans s;
    s.group_rows = a.gate && a.gate_rows > 1 ? a.gate_rows : a.rows;
    s.ngroups = a.rows / s.group_rows;
    // about two workgroups of four waves to a CU; with fewer rows one or two rows a wave, so that
    // they are read at once (999 rows of 531 in fp32: 16 us, 24 with four a wave and 21 with one,
    // whose many partial sums take longer to join; 32 rows of 768: 9 with one, 11 with two)
    const int64_t target = 512 * 256 / R::kThreads;
    int64_t span = cdiv(a.rows, target);
    const int64_t least = a.rows <= 64 * R::kRows ? R::kRows : 2 * R::kRows;
    if (span < least) span = least;
    s.parts = s.group_rows > span ? cdiv(s.group_rows, span) : 1;
    s.groups = s.parts == 1 ? span / s.group_rows : 1;
    s.blocks = s.parts == 1 ? cdiv(s.ngroups, s.groups) : s.ngroups * s.parts;
    void* parts = nullptr;
    hipError_t e = workspace_alloc(&parts, (size_t)(s.blocks * 3 * a.dim * 4), stream, true);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((norm_pullback_kernel<R>), dim3((unsigned)s.blocks), dim3(R::kThreads), 0,
                       stream, a, g, s, static_cast<float*>(parts));
    e = hipGetLastError();
    const bool gates = a.gate && a.gate_rows > 1 && s.parts > 1;
    if (e == hipSuccess && (a.wpost || a.wpre || gates)) {
      hipLaunchKernelGGL((norm_join_kernel<T>),
                         dim3((unsigned)cdiv(a.dim, 64), (unsigned)(2 + (gates ? s.ngroups : 0))),
                         dim3(1024), 0, stream, g, static_cast<const float*>(parts), s.blocks,
                         s.parts, (int)a.dim);
      e = hipGetLastError();
    }
    const hipError_t ef = workspace_free(parts, stream);
    return e != hipSuccess ? e : ef;
  });
}

}  // namespace fms

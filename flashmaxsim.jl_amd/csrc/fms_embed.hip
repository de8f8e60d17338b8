// fms_embed.hip -- rows of a table looked up by token, scaled, and the table's gradient.
//
//   e[t] = scale * W[id_t],   dW[v] = scale * sum of de[t] over the tokens t with id_t = v
//
// Bound by memory: the lookup writes every e once (its reads repeat), the gradient reads every de once
// and writes all of dW (128 x 180 tokens, 70 % of them real, 32768 rows
// of 1024 in bf16: lookup 11 us; gradient 31 for the sort, 16 of it for the order inside its buckets and the
// rest short kernels that are latency, 25 for the rows, 14 for the longer runs).  For the gradient the tokens are grouped by id (the candidate scans'
// counting sort, whose atomics stay in LDS); a wave takes a row of dW and adds its tokens' rows in
// fp32 and in the order of the tokens, which it restores first (the sort leaves a group's order
// open), so the sums are the same every time.  Ids of more than 64 tokens (a text's most frequent
// words: one token in fifteen can be of one id) are left to a second kernel, in which a workgroup
// spreads such a row's tokens, as bits of a map that is in order by itself, over 64 quarters of
// waves (16 lanes), and joins their sums in a fixed order.
#include "fms_embed.hpp"

#include "../../include/flashmaxsim_hip.h"
#include "fms_device.hpp"
#include "fms_group.hpp"

namespace fms {
namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int kRun = 64;              // tokens of an id that one wave adds up
constexpr int kMapBits = 1 << 18;     // tokens whose bits are held at a time
constexpr int kHotThreads = 1024, kHotBlocks = 64;  // workgroups (of sixteen units) that share the longer runs

template <class T_, int kU_>
struct Unit {
  typedef T_ T;
  static constexpr int kU = kU_;
  typedef T V __attribute__((ext_vector_type(kU)));
};

__device__ __forceinline__ int64_t id_of(const EmbedArgs& A, int64_t t) {
  return (A.id_bytes == 8 ? static_cast<const int64_t*>(A.ids)[t] : (int64_t) static_cast<const int32_t*>(A.ids)[t]) - 1;
}

// `lanes` (a power of two) lanes a token.
template <class U>
__global__ void __launch_bounds__(256) embed_forward_kernel(EmbedArgs A, typename U::T* e, const typename U::T* weight,
                                                            int lanes, int units) {
  typedef typename U::T T;
  typedef typename U::V V;
  const int per = 256 / lanes, first = threadIdx.x & (lanes - 1);
  for (int64_t t = (int64_t)blockIdx.x * per + threadIdx.x / lanes; t < A.n; t += (int64_t)gridDim.x * per) {
    const int64_t id = id_of(A, t);
    const bool in = id >= 0 && id < A.vocabulary;
    const T* from = weight + (in ? id : 0) * A.dim;
    T* to = e + t * A.dim;
#pragma unroll 2
    for (int u = first; u < units; u += lanes) {
      V v = {};
      if (in) {
        const V w = *reinterpret_cast<const V*>(from + u * U::kU);
#pragma unroll
        for (int i = 0; i < U::kU; ++i) v[i] = (T)((float)w[i] * A.scale);
      }
      *reinterpret_cast<V*>(to + u * U::kU) = v;
    }
  }
}

__global__ void embed_zero_kernel(uint32_t* hots) { *hots = 0u; }

// A wave a row of dW: rows without tokens, and with at most kRun.  The others are listed, in any order: a row's sum
// is its own.
template <class U>
__global__ void __launch_bounds__(256) embed_rows_kernel(EmbedArgs A, typename U::T* dweight, const typename U::T* de,
                                                         const PairRef* order, const uint32_t* ends, int units,
                                                         uint32_t* hots, uint32_t* hot) {
  typedef typename U::T T;
  typedef typename U::V V;
  constexpr int kPer = 2, kAtOnce = 4;  // units a lane holds, tokens whose rows are read at once
  const int lane = threadIdx.x & 63;
  for (int64_t v = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); v < A.vocabulary; v += (int64_t)gridDim.x * 4) {
    const uint32_t s = rfl32(v ? ends[v - 1] : 0u), run = rfl32(ends[v]) - s;
    if (run > (uint32_t)kRun) {
      if (lane == 0) hot[atomicAdd(hots, 1u)] = (uint32_t)v;
      continue;
    }
    int token = 0;
    if (run > 0) token = order ? order[s + ((uint32_t)lane < run ? lane : 0)].p : 0;
    if (run > 1) {
      int rank = 0;
      for (uint32_t i = 0; i < run; ++i) rank += __builtin_amdgcn_readlane(token, i) < token;
      if ((uint32_t)lane >= run) rank = lane;
      token = __builtin_amdgcn_ds_permute(rank * 4, token);
    }
    T* to = dweight + v * A.dim;
    for (int u0 = 0; u0 < units; u0 += 64 * kPer) {
      float acc[kPer][U::kU] = {};
      for (uint32_t i0 = 0; i0 < run; i0 += kAtOnce) {
        V x[kAtOnce][kPer];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          const bool one = i0 + i < run;
          const T* from = de + (int64_t)__builtin_amdgcn_readlane(token, one ? i0 + i : 0) * A.dim;
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const int u = u0 + j * 64 + lane;
            x[i][j] = V{};
            if (one && u < units) x[i][j] = *reinterpret_cast<const V*>(from + u * U::kU);
          }
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
          for (int j = 0; j < kPer; ++j)
#pragma unroll
            for (int k = 0; k < U::kU; ++k) acc[j][k] += (float)x[i][j][k];
      }
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int u = u0 + j * 64 + lane;
        V x;
#pragma unroll
        for (int k = 0; k < U::kU; ++k) x[k] = (T)(acc[j][k] * A.scale);
        if (u < units) *reinterpret_cast<V*>(to + u * U::kU) = x;
      }
    }
  }
}

// The listed rows, sixteen units of them (blockIdx.y).
template <class U>
__global__ void __launch_bounds__(kHotThreads) embed_hot_kernel(EmbedArgs A, typename U::T* dweight,
                                                                const typename U::T* de, const PairRef* order,
                                                                const uint32_t* ends, int units, const uint32_t* hots,
                                                                const uint32_t* hot) {
  typedef typename U::T T;
  typedef typename U::V V;
  __shared__ uint32_t map[kMapBits / 32];
  __shared__ float sums[64][16][U::kU];
  const int tid = threadIdx.x;
  const int group = tid >> 4, lane = tid & 15;
  const int u = blockIdx.y * 16 + lane;
  const bool in = u < units;
  const uint32_t n = *hots;
  for (uint32_t i = blockIdx.x; i < n; i += kHotBlocks) {
    const int64_t v = hot[i];
    const uint32_t s = v ? ends[v - 1] : 0u, e = ends[v];
    float acc[U::kU] = {};
    for (int64_t w0 = 0; w0 < A.n; w0 += kMapBits) {
      const int bits = A.n - w0 < kMapBits ? (int)(A.n - w0) : kMapBits, words = (bits + 31) / 32;
      __syncthreads();  // (the map and the sums before are read)
      for (int w = tid; w < words; w += kHotThreads) map[w] = 0u;
      __syncthreads();
      for (uint32_t k = s + tid; k < e; k += kHotThreads) {
        const int64_t p = order[k].p - w0;
        if (p >= 0 && p < bits) atomicOr(&map[p / 32], 1u << (p & 31));
      }
      __syncthreads();
      // this group's words, eight tokens at a time
      int w = (int)((int64_t)words * group / 64);
      const int end = (int)((int64_t)words * (group + 1) / 64);
      uint32_t left = w < end ? map[w] : 0u;
      while (w < end) {
        int t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          while (left == 0u && w < end) left = ++w < end ? map[w] : 0u;
          t[j] = w < end ? w * 32 + __builtin_ctz(left) : -1;
          left &= left - 1;
        }
        V x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = V{};
          if (t[j] >= 0 && in) x[j] = *reinterpret_cast<const V*>(de + (w0 + t[j]) * A.dim + u * U::kU);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int k = 0; k < U::kU; ++k) acc[k] += (float)x[j][k];
      }
    }
#pragma unroll
    for (int k = 0; k < U::kU; ++k) sums[group][lane][k] = acc[k];
    __syncthreads();
    // sixteen threads a value, four groups each, and then the sixteen
    constexpr int kValues = 16 * U::kU;
    for (int k = tid; k < kValues * 16; k += kHotThreads) {
      const int value = k % kValues, part = k / kValues;
      float* const s0 = &sums[part * 4][0][0] + value;
      *s0 = (s0[0] + s0[kValues]) + (s0[2 * kValues] + s0[3 * kValues]);
    }
    __syncthreads();
    if (tid < kValues) {
      const int unit = blockIdx.y * 16 + tid / U::kU;
      float total = 0.0f;
#pragma unroll
      for (int g = 0; g < 64; g += 4) total += (&sums[g][0][0])[tid];
      if (unit < units) dweight[v * A.dim + unit * U::kU + tid % U::kU] = (T)(total * A.scale);
    }
    __syncthreads();
  }
}

bool whole_units(const EmbedArgs& a, const void* p, const void* q) {
  return a.dim * (a.dtype == FMS_F32 ? 4 : 2) % 16 == 0 && ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) & 15u) == 0;
}
template <class F>
hipError_t by_unit(const EmbedArgs& a, bool vec, F&& f) {
  switch (a.dtype) {
    case FMS_F16: return vec ? f(Unit<_Float16, 8>()) : f(Unit<_Float16, 1>());
    case FMS_BF16: return vec ? f(Unit<__bf16, 8>()) : f(Unit<__bf16, 1>());
    default: return vec ? f(Unit<float, 4>()) : f(Unit<float, 1>());
  }
}

}  // namespace

hipError_t embed_forward(const EmbedArgs& a, void* e, const void* weight, hipStream_t stream) {
  return by_unit(a, whole_units(a, e, weight), [&](auto unit) {
    typedef decltype(unit) U;
    const int64_t units = a.dim / U::kU;
    int lanes = 1;
    while (lanes < 64 && lanes < units) lanes <<= 1;
    const int64_t want = cdiv(a.n, 256 / lanes), most = 16384;
    hipLaunchKernelGGL((embed_forward_kernel<U>), dim3((unsigned)(want < most ? want : most)), dim3(256), 0, stream, a,
                       static_cast<typename U::T*>(e), static_cast<const typename U::T*>(weight), lanes, (int)units);
    return hipGetLastError();
  });
}

hipError_t embed_pullback(const EmbedArgs& a, void* dweight, const void* de, hipStream_t stream) {
  void* mem = nullptr;
  // the sort's workspace, then the count and list of the longer runs
  const size_t sort = (group_workspace_bytes(a.n, a.vocabulary) + 255) / 256 * 256;
  hipError_t e = workspace_alloc(&mem, sort + 256 + (size_t)(a.n / (kRun + 1)) * 4, stream, true);
  if (e != hipSuccess) return e;
  uint32_t* const hots = reinterpret_cast<uint32_t*>(static_cast<char*>(mem) + sort);
  uint32_t* const hot = hots + 64;
  const bool runs = a.n > kRun;
  if (runs) hipLaunchKernelGGL(embed_zero_kernel, dim3(1), dim3(1), 0, stream, hots);
  const PairRef* order = nullptr;
  const uint32_t* ends = nullptr;
  e = group_pairs_by_document(a.ids, a.id_bytes == 8, a.n, a.vocabulary, mem, &order, &ends, stream);
  if (e == hipSuccess)
    e = by_unit(a, whole_units(a, dweight, de), [&](auto unit) {
      typedef decltype(unit) U;
      typedef typename U::T T;
      const int64_t units = a.dim / U::kU, rows = cdiv(a.vocabulary, 4), most = 16384;
      hipLaunchKernelGGL((embed_rows_kernel<U>), dim3((unsigned)(rows < most ? rows : most)), dim3(256), 0, stream, a,
                         static_cast<T*>(dweight), static_cast<const T*>(de), order, ends, (int)units, hots, hot);
      if (runs)
        hipLaunchKernelGGL((embed_hot_kernel<U>), dim3(kHotBlocks, (unsigned)cdiv(units, 16)),
                           dim3(kHotThreads), 0, stream, a, static_cast<T*>(dweight), static_cast<const T*>(de), order,
                           ends, (int)units, static_cast<const uint32_t*>(hots), static_cast<const uint32_t*>(hot));
      return hipGetLastError();
    });
  const hipError_t ef = workspace_free(mem, stream);
  return e != hipSuccess ? e : ef;
}

}  // namespace fms

// fms_adamw.hip -- one AdamW step over many tensors at once, moments in 32 or 8 bits.
//
//   g = grad * grad_scale
//   m = beta1 m + (1 - beta1) g
//   v = beta2 v + (1 - beta2) (g * g)
//   p = p (1 - lr decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
// with t the tensor's own steps, in fp32, every operation rounded by itself (the library is built without contraction), on
// the fp32 master where a tensor has one, else on the parameter.
//
// 8-bit moments: 256 neighbouring elements share an fp32 scale a, the largest magnitude among
// them (0 where that is below the least normal number).
//   m: int8 code  c = sign(m) round(127 sqrt(|m| / a)),   value  sign(c) (c / 127)^2 a
//   v: uint8 code c = round(255 (v / a)^(1/4)),           value  (c / 255)^4 a
// Codes are dense near zero and even in relative terms over four decades; a v above zero keeps
// a code of at least 1, so that sqrt(v) never becomes 0 under an m that did not.  A NaN or
// infinity makes its block's scale NaN and with it the block's values.
//
// Bound by memory: 28 bytes an element in fp32, 22 with 16-bit parameters and gradients, 10
// with 8-bit moments.  A workgroup takes 2048 elements of one tensor, eight a lane, so that
// half a wave holds a block of 8-bit moments.  What stays (parameters, moments, sizes, and which
// tensor a workgroup belongs to) is read from the caller's plan in device memory; the gradients'
// addresses travel as kernel arguments, 480 to a launch, with up to 16 different t.  (With whole tables as arguments, 52 to a
// launch, 148 tensors of 8 million elements took three launches and 68 us,
// now one and 62; 64 million 8-bit elements in 12 tensors take 262 us with their values, 254 then.)
#include "fms_adamw.hpp"

#include <float.h>
#include <math.h>

#include "fms_device.hpp"

namespace fms {
namespace {

constexpr int kPer = 8;                    // elements per lane
constexpr int kChunk = 256 * kPer;         // elements per workgroup
constexpr int kBlock = FMS_MOMENT_BLOCK;   // elements that share a scale
static_assert(kBlock == 32 * kPer, "a half wave holds a block");

// The tensors' pointers come out of memory, where the compiler cannot tell that they are to
// device memory (a flat access instead of a global one: 277 us against 273 for 64 million 8-bit
// elements).
template <class T>
using Global = __attribute__((address_space(1))) T;
template <class T>
__device__ __forceinline__ Global<T>* global(T* p) {
  return (Global<T>*)p;
}

// Eight neighbouring values from element k of n; vec: whole 16-byte units from the base on.
template <class T>
__device__ __forceinline__ void load8(float (&v)[kPer], const T* p, int64_t k, int64_t n, bool vec) {
  typedef T V __attribute__((ext_vector_type(kPer), aligned(16)));
  if (vec && k + kPer <= n) {
    const V u = *(const Global<V>*)(global(p) + k);
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = (float)u[e];
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = k + e < n ? (float)global(p)[k + e] : 0.0f;
  }
}
template <class T>
__device__ __forceinline__ void store8(const float (&v)[kPer], T* p, int64_t k, int64_t n, bool vec) {
  typedef T V __attribute__((ext_vector_type(kPer), aligned(16)));
  if (vec && k + kPer <= n) {
    V u;
#pragma unroll
    for (int e = 0; e < kPer; ++e) u[e] = (T)v[e];
    *(Global<V>*)(global(p) + k) = u;
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (k + e < n) global(p)[k + e] = (T)v[e];
  }
}
__device__ __forceinline__ void load_typed(float (&v)[kPer], const void* p, int dtype, int64_t k,
                                           int64_t n, bool vec) {
  if (dtype == FMS_F32)
    load8(v, static_cast<const float*>(p), k, n, vec);
  else if (dtype == FMS_F16)
    load8(v, static_cast<const _Float16*>(p), k, n, vec);
  else
    load8(v, static_cast<const __bf16*>(p), k, n, vec);
}
__device__ __forceinline__ void store_typed(const float (&v)[kPer], void* p, int dtype, int64_t k,
                                            int64_t n, bool vec) {
  if (dtype == FMS_F32)
    store8(v, static_cast<float*>(p), k, n, vec);
  else if (dtype == FMS_F16)
    store8(v, static_cast<_Float16*>(p), k, n, vec);
  else
    store8(v, static_cast<__bf16*>(p), k, n, vec);
}

// The largest magnitude of a block, in its 32 lanes.  Magnitudes compare as their bits, NaN
// above all: a NaN is never lost.
__device__ __forceinline__ float block_top(const float (&v)[kPer]) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    const uint32_t b = (uint32_t)__shfl_xor((int)top, o);
    top = b > top ? b : top;
  }
  return __builtin_bit_cast(float, top);
}

__device__ __forceinline__ float value_m(int c, float a) {
  const float t = (float)c * (1.0f / 127.0f);
  return t * fabsf(t) * a;
}
__device__ __forceinline__ float value_v(int c, float a) {
  const float t = (float)c * (1.0f / 255.0f);
  const float q = t * t;
  return q * q * a;
}
// A block's scale and the reciprocal its codes are made with.  An infinity is NaN here: no
// code stands for it beside finite values.
__device__ __forceinline__ void scale_of(float top, float& a, float& inv) {
  const bool tiny = top < FLT_MIN;
  a = tiny ? 0.0f : top + (top - top);
  inv = tiny ? 0.0f : 1.0f / top;
}
// round(sqrt(q) * 127) and round(q^(1/4) * 255) for q in 0..1, as IEEE square roots give them,
// the second at least 1 for a q above 0.  The hardware's root is within a unit or two of that:
// only a product within 1e-4 of a tie needs the exact one.  (The step of 64 million 8-bit
// elements is bound by its instructions: 205 us with exact roots, 149.)
__device__ __forceinline__ float code_m(float q) {
  const float t = __builtin_amdgcn_sqrtf(q) * 127.0f;
  float c = __builtin_rintf(t);
  if (__builtin_expect(fabsf(t - c) > 0.4999f, 0)) c = __builtin_rintf(sqrtf(q) * 127.0f);
  return c;
}
__device__ __forceinline__ float code_v(float q) {
  const float t = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(q)) * 255.0f;
  float c = __builtin_rintf(t);
  if (__builtin_expect(fabsf(t - c) > 0.4999f, 0)) c = __builtin_rintf(sqrtf(sqrtf(q)) * 255.0f);
  return fmaxf(c, __builtin_ceilf(q));
}

// Codes of eight neighbouring elements.
struct Codes {
  uint32_t w[2];
  __device__ __forceinline__ int get(int e, bool sign) const {
    const uint32_t b = w[e >> 2] >> (8 * (e & 3));
    return sign ? (int)(int8_t)b : (int)(b & 0xffu);
  }
};
typedef uint32_t CodeWords __attribute__((ext_vector_type(2)));
__device__ __forceinline__ Codes load_codes(const uint8_t* p, int64_t k, int64_t n, bool vec) {
  Codes c = {{0u, 0u}};
  if (vec && k + kPer <= n) {
    const CodeWords w = *(const Global<CodeWords>*)(global(p) + k);
    c.w[0] = w[0];
    c.w[1] = w[1];
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (k + e < n) c.w[e >> 2] |= (uint32_t)global(p)[k + e] << (8 * (e & 3));
  }
  return c;
}
__device__ __forceinline__ void store_codes(const Codes& c, uint8_t* p, int64_t k, int64_t n, bool vec) {
  if (vec && k + kPer <= n) {
    *(Global<CodeWords>*)(global(p) + k) = CodeWords{c.w[0], c.w[1]};
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (k + e < n) global(p)[k + e] = (uint8_t)(c.w[e >> 2] >> (8 * (e & 3)));
  }
}

template <class... P>
__device__ __forceinline__ bool aligned(P... p) {
  return ((reinterpret_cast<uintptr_t>(p) | ...) & 15u) == 0;
}

struct AdamWStep {
  float beta1, rest1;  // and 1 - beta1
  float beta2, rest2;
  float eps;
  float decay;  // 1 - lr * weight_decay
  float grad_scale;
};
struct Correction {  // of a number of steps
  float lr;          // lr / (1 - beta1^t)
  float inv_bc2;     // 1 / sqrt(1 - beta2^t)
};
constexpr int kTensors = 480;     // per launch: the arguments stay within 4 KiB
constexpr int kCorrections = 16;  // likewise
// a gradient's address and, above it, its element type and which correction its tensor takes
constexpr int kTypeShift = 56, kCorrectionShift = 58;
struct Grads {
  uint64_t g[kTensors];  // 0: none
  Correction c[kCorrections];
  int32_t first;  // tensor of the launch
};
static_assert(FMS_BF16 < 1 << (kCorrectionShift - kTypeShift) && kCorrections <= 1 << (64 - kCorrectionShift),
              "room above the address");
static_assert(sizeof(Grads) + sizeof(AdamWStep) + 32 <= 4096, "kernel arguments");

// Eight elements a lane from k on; whole half waves take part past the tensor's end.
__device__ __forceinline__ void adamw_elements(const fms_adamw_tensor& t, const void* grad, int g_dtype,
                                           const AdamWStep& S, const Correction& c, int64_t k, bool vec) {
  const int64_t n = t.n;
  const bool codes = t.m_scale != nullptr;
  float g[kPer], p[kPer], m[kPer], v[kPer];
  load_typed(g, grad, g_dtype, k, n, vec);
  if (t.master)
    load8(p, t.master, k, n, vec);
  else
    load_typed(p, t.p, (int)t.p_dtype, k, n, vec);
  if (codes) {
    const Codes cm = load_codes(static_cast<const uint8_t*>(t.m), k, n, vec);
    const Codes cv = load_codes(static_cast<const uint8_t*>(t.v), k, n, vec);
    const float am = k < n ? global(t.m_scale)[k / kBlock] : 0.0f;
    const float av = k < n ? global(t.v_scale)[k / kBlock] : 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      m[e] = value_m(cm.get(e, true), am);
      v[e] = value_v(cv.get(e, false), av);
    }
  } else {
    load8(m, static_cast<const float*>(t.m), k, n, vec);
    load8(v, static_cast<const float*>(t.v), k, n, vec);
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const float gs = g[e] * S.grad_scale;
    m[e] = m[e] * S.beta1 + gs * S.rest1;
    v[e] = v[e] * S.beta2 + gs * gs * S.rest2;
    const float den = sqrtf(v[e]) * c.inv_bc2 + S.eps;
    p[e] = p[e] * S.decay - m[e] / den * c.lr;
  }
  if (t.master) store8(p, t.master, k, n, vec);
  store_typed(p, t.p, (int)t.p_dtype, k, n, vec);
  if (codes) {
    // (elements past the end are zero and the whole half wave takes part)
    float am, im, av, iv;
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (k + e >= n) m[e] = v[e] = 0.0f;
    scale_of(block_top(m), am, im);
    scale_of(block_top(v), av, iv);
    Codes cm = {{0u, 0u}}, cv = {{0u, 0u}};
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      // (c + 128 as a byte, its top bit turned: c in two's complement)
      const float c = copysignf(code_m(fabsf(m[e]) * im), m[e]) + 128.0f;
      cm.w[e >> 2] = __builtin_amdgcn_cvt_pk_u8_f32(c, e & 3, cm.w[e >> 2]);
      cv.w[e >> 2] = __builtin_amdgcn_cvt_pk_u8_f32(code_v(v[e] * iv), e & 3, cv.w[e >> 2]);
    }
    cm.w[0] ^= 0x80808080u;
    cm.w[1] ^= 0x80808080u;
    store_codes(cm, static_cast<uint8_t*>(t.m), k, n, vec);
    store_codes(cv, static_cast<uint8_t*>(t.v), k, n, vec);
    if ((threadIdx.x & 31) == 0 && k < n) {
      global(t.m_scale)[k / kBlock] = am;
      global(t.v_scale)[k / kBlock] = av;
    }
  } else {
    store8(m, static_cast<float*>(t.m), k, n, vec);
    store8(v, static_cast<float*>(t.v), k, n, vec);
  }
}

// A wave-uniform entry in scalar registers.
__device__ __forceinline__ AdamWEntry uniform(const AdamWEntry& e) {
  uint64_t w[sizeof(AdamWEntry) / 8];
  __builtin_memcpy(w, &e, sizeof(e));
#pragma unroll
  for (uint64_t& x : w) x = rfl64(x);
  AdamWEntry u;
  __builtin_memcpy(&u, w, sizeof(u));
  return u;
}

__global__ void __launch_bounds__(256) adamw_kernel(const AdamWEntry* entries, const int32_t* tensor_of,
                                                    int64_t first_block, Grads G, AdamWStep S) {
  const int64_t block = first_block + blockIdx.x;
  const int at = __builtin_amdgcn_readfirstlane(tensor_of[block]), i = at - G.first;
  const uint64_t g = G.g[i];
  if (g == 0) return;  // (the whole workgroup)
  const void* const grad = reinterpret_cast<const void*>(g & (((uint64_t)1 << kTypeShift) - 1));
  // (copied to scalar registers: what the stores below may alias would be read again after them)
  const AdamWEntry entry = uniform(entries[at]);
  const fms_adamw_tensor& t = entry.t;
  const int type = (int)(g >> kTypeShift) & ((1 << (kCorrectionShift - kTypeShift)) - 1);
  adamw_elements(t, grad, type, S, G.c[g >> kCorrectionShift],
                 (block - entry.first) * kChunk + threadIdx.x * kPer, aligned(t.p, grad, t.m, t.v, t.master));
}

constexpr int kMoments = 92;
struct Moments {
  fms_moment8 t[kMoments];
  int32_t end[kMoments];
  int32_t count;
};
static_assert(sizeof(Moments) <= 4096, "kernel arguments");

__global__ void __launch_bounds__(256) moment_values_kernel(Moments L) {
  // the first whose workgroups end past this one
  int i = 0;
  for (int hi = L.count - 1; i < hi;) {
    const int mid = (i + hi) >> 1;
    if (L.end[mid] > (int)blockIdx.x)
      hi = mid;
    else
      i = mid + 1;
  }
  const fms_moment8& t = L.t[i];
  const int first = i > 0 ? L.end[i - 1] : 0;
  const int64_t k = (int64_t)(blockIdx.x - first) * kChunk + threadIdx.x * kPer, n = t.n;
  if (k >= n) return;
  const bool vec = aligned(t.codes, t.values);
  const Codes c = load_codes(static_cast<const uint8_t*>(t.codes), k, n, vec);
  const float a = t.scales[k / kBlock];
  float v[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e)
    v[e] = t.is_signed ? value_m(c.get(e, true), a) : value_v(c.get(e, false), a);
  store8(v, t.values, k, n, vec);
}

}  // namespace

int64_t adamw_blocks(const fms_adamw_tensor& t) { return (t.n + kChunk - 1) / kChunk; }

hipError_t adamw_step(const AdamWPlan* plan, const void* device_plan, const void* const* grads,
                      const int32_t* g_dtypes, const AdamWRates& r, hipStream_t stream) {
  AdamWStep s;
  s.beta1 = (float)r.beta1;
  s.rest1 = (float)(1.0 - r.beta1);
  s.beta2 = (float)r.beta2;
  s.rest2 = (float)(1.0 - r.beta2);
  s.eps = (float)r.eps;
  s.decay = (float)(1.0 - r.lr * r.weight_decay);
  s.grad_scale = (float)r.grad_scale;
  const auto correction = [&](int64_t t) {
    return Correction{(float)(r.lr / (1.0 - pow(r.beta1, (double)t))),
                      (float)(1.0 / sqrt(1.0 - pow(r.beta2, (double)t)))};
  };
  const AdamWEntry* const entries = reinterpret_cast<const AdamWEntry*>(plan + 1);
  const AdamWEntry* const on_device =
      reinterpret_cast<const AdamWEntry*>(static_cast<const AdamWPlan*>(device_plan) + 1);
  const int32_t* const tensor_of = reinterpret_cast<const int32_t*>(on_device + plan->count);
  constexpr int64_t kGrid = (int64_t)1 << 23;
  for (int64_t i = 0; i < plan->count;) {
    // as many tensors as the arguments and the grid take (a tensor alone fits: fms_adamw_plan)
    Grads g;
    g.first = (int32_t)i;
    const int64_t first = entries[i].first;
    int64_t last = first, counts[kCorrections];
    int n = 0, ncounts = 0, at = 0;
    for (; i < plan->count && n < kTensors; ++i, ++n) {
      const int64_t end = entries[i].first + adamw_blocks(entries[i].t);
      if (n > 0 && end - first > kGrid) break;
      g.g[n] = reinterpret_cast<uint64_t>(grads[i]);
      if (g.g[n] != 0) {
        const int64_t t = r.steps ? r.steps[i] : r.step;
        if (ncounts == 0 || counts[at] != t)
          for (at = 0; at < ncounts && counts[at] != t;) ++at;
        if (at == kCorrections) break;
        if (at == ncounts) {
          counts[ncounts] = t;
          g.c[ncounts++] = correction(t);
        }
        g.g[n] |= (uint64_t)g_dtypes[i] << kTypeShift | (uint64_t)at << kCorrectionShift;
      }
      last = end;
    }
    if (last == first) continue;
    hipLaunchKernelGGL(adamw_kernel, dim3((unsigned)(last - first)), dim3(256), 0, stream, on_device,
                       tensor_of, first, g, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t moment_values(int64_t count, const fms_moment8* moments, hipStream_t stream) {
  // lists of as many as the arguments and the grid take
  Moments list;
  list.count = 0;
  int64_t blocks = 0;
  for (int64_t i = 0; i <= count; ++i) {
    const int64_t need = i < count ? (moments[i].n + kChunk - 1) / kChunk : 0;
    if (list.count > 0 && (i == count || list.count == kMoments || blocks + need > ((int64_t)1 << 23))) {
      hipLaunchKernelGGL(moment_values_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, list);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
      list.count = 0;
      blocks = 0;
    }
    if (need == 0) continue;
    blocks += need;
    list.t[list.count] = moments[i];
    list.end[list.count++] = (int32_t)blocks;
  }
  return hipSuccess;
}

}  // namespace fms

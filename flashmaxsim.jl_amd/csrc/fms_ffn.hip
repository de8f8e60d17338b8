// fms_ffn.hip -- gated feed-forward block: both projections, the activation and
// the product in one kernel, and its pullback.
//
//   g = x wg^T,  u = x wu^T,  h = act(g) * u                     (per token and hidden unit)
//   dg = dh * u * act'(g),  du = dh * act(g)
//   dx = dg wg + du wu,  dwg = dg^T x,  dwu = du^T x
//
// Products run on the matrix cores (fms_gemm.hpp) and accumulate in fp32.  g and
// u never leave the registers: forward writes h alone and keeps nothing, and the
// pullback computes them again in the kernel that makes dg and du, which are
// rounded once to the feature type for the three products after it.  (Keeping g
// and u from the forward in 16 bits would round them once more, and in fp32
// would move 16 bytes a hidden unit, against 4 dim operations to compute them.)
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

// act(g) in a, act'(g) in da.
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

// Four neighbouring values as one LDS word.
template <class Op>
struct Quad {
  typedef typename OutOf<Op>::T T;
  typedef T V __attribute__((ext_vector_type(4)));
  __device__ static __forceinline__ V pack(float a, float b, float c, float d) {
    return V{(T)a, (T)b, (T)c, (T)d};
  }
};

// A kBM x kCols tile of feature values in LDS, rows of 16-byte units permuted over the
// banks by their row, and its way from and to memory.
template <class Op, int kBM, int kCols, int kThreads>
struct LdsTile {
  typedef typename OutOf<Op>::T T;
  typedef typename Quad<Op>::V V;
  static constexpr int kPer = 16 / Op::kEsz;      // values per unit
  static constexpr int kUpr = kCols / kPer;       // units per row
  static constexpr int kBytes = kBM * kCols * Op::kEsz;
  static constexpr int kMix = (kUpr < 16 ? kUpr : 16) - 1;

  __device__ static __forceinline__ V* quad(char* lds, int row, int col) {
    const int unit = (col / kPer) ^ (row & kMix);
    return reinterpret_cast<V*>(lds + (row * kUpr + unit) * 16 + (col % kPer) * Op::kEsz);
  }
  // rows [m0, m0 + kBM) x columns [n0, n0 + kCols) of a (rows, cols) matrix, `pitch`
  // values a row; `vec`: base and pitch are whole 16-byte units.
  __device__ static __forceinline__ void store(const char* lds, T* out, int64_t rows, int64_t cols,
                                               int64_t pitch, int64_t m0, int64_t n0, bool vec) {
#pragma unroll 4
    for (int u = threadIdx.x; u < kBM * kUpr; u += kThreads) {
      const int row = u / kUpr, log = (u % kUpr) ^ (row & kMix);
      const int64_t m = m0 + row, n = n0 + log * kPer;
      if (m >= rows || n >= cols) continue;
      const u32x4 v = *reinterpret_cast<const u32x4*>(lds + u * 16);
      T* p = out + m * pitch + n;
      if (vec && n + kPer <= cols) {
        *reinterpret_cast<u32x4*>(p) = v;
      } else {
        const T* e = reinterpret_cast<const T*>(lds + u * 16);
        for (int k = 0; k < kPer && n + k < cols; ++k) p[k] = e[k];
      }
    }
  }
  __device__ static __forceinline__ void load(char* lds, const T* in, int64_t rows, int64_t cols,
                                              int64_t pitch, int64_t m0, int64_t n0, bool vec) {
#pragma unroll 4
    for (int u = threadIdx.x; u < kBM * kUpr; u += kThreads) {
      const int row = u / kUpr, log = (u % kUpr) ^ (row & kMix);
      const int64_t m = m0 + row, n = n0 + log * kPer;
      u32x4 v{0u, 0u, 0u, 0u};
      if (m < rows && n < cols) {
        const T* p = in + m * pitch + n;
        if (vec && n + kPer <= cols) {
          v = *reinterpret_cast<const u32x4*>(p);
        } else {
          T e[kPer];
          for (int k = 0; k < kPer; ++k) e[k] = n + k < cols ? p[k] : (T)0.0f;
          __builtin_memcpy(&v, e, 16);
        }
      }
      *reinterpret_cast<u32x4*>(lds + u * 16) = v;
    }
  }
};

// Workgroup -> tile.  Workgroup ids go round robin over the 8 XCDs, each with an L2 of
// its own: every XCD takes a contiguous run of tiles, and a run walks kGroupM row tiles
// per column tile, so that the tiles in flight on an XCD share their operands.
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
  // forward: out0 = h; pullback: in = dh, out0 = dg, out1 = du
  void *out0, *out1;
  const void* in;
  int64_t out_cols, out_pitch, in_pitch;  // values
  int32_t out_vec, in_vec;
};

// The accumulators' tile -> LDS: h, or dg over the dh that lies there and du behind it.
template <class P, bool kPull, int kAct>
__device__ __forceinline__ void gate_epilogue(const typename P::Acc (&acc)[2][P::kMF], char* lds) {
  typedef typename P::Op Op;
  typedef LdsTile<Op, P::kBM, P::kBN / 2, P::kThreads> Tile;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / P::kWN, wn = wave % P::kWN, h = lane >> 5;
#pragma unroll
  for (int mf = 0; mf < P::kMF; ++mf) {
    const int row = (wm * P::kMF + mf) * 32 + (lane & 31);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int col = wn * 32 + 8 * q + 4 * h;
      auto* at = Tile::quad(lds, row, col);
      float a[4], da[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) activate<kAct>(acc[0][mf][4 * q + e], a[e], da[e]);
      if constexpr (kPull) {
        const auto d = *at;
        float dg[4], du[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dg[e] = (float)d[e] * acc[1][mf][4 * q + e] * da[e];
          du[e] = (float)d[e] * a[e];
        }
        *at = Quad<Op>::pack(dg[0], dg[1], dg[2], dg[3]);
        *Tile::quad(lds + Tile::kBytes, row, col) = Quad<Op>::pack(du[0], du[1], du[2], du[3]);
      } else {
        const auto& u = acc[1][mf];
        *at = Quad<Op>::pack(a[0] * u[4 * q], a[1] * u[4 * q + 1], a[2] * u[4 * q + 2],
                             a[3] * u[4 * q + 3]);
      }
    }
  }
}

// Forward (kPull false): h.  Pullback: dg and du, their rows filled up with zeros to out_cols.
template <class P, bool kPull>
__global__ void __launch_bounds__(P::kThreads, 2) ffn_gate_kernel(GateArgs A) {
  typedef typename P::Op Op;
  typedef typename OutOf<Op>::T T;
  constexpr int kCols = P::kBN / 2;
  typedef LdsTile<Op, P::kBM, kCols, P::kThreads> Tile;
  static_assert((kPull ? 2 : 1) * Tile::kBytes <= P::kLds, "the output tile reuses the LDS");
  __shared__ __attribute__((aligned(16))) char lds[P::kLds];
  int im, in;
  tile_of(blockIdx.x, A.tm, A.tn, im, in);
  const int64_t m0 = (int64_t)im * P::kBM, n0 = (int64_t)in * kCols;
  typename P::Acc acc[2][P::kMF] = {};
  const Matrix M[1] = {A.x}, N[2] = {A.wg, A.wu};
  P::run(acc, M, N, m0, n0, 0, A.steps, lds);
  if constexpr (kPull) {
    Tile::load(lds, static_cast<const T*>(A.in), A.tokens, A.hidden, A.in_pitch, m0, n0, A.in_vec);
    __syncthreads();
  }
  if (A.act == FMS_ACT_SILU)
    gate_epilogue<P, kPull, FMS_ACT_SILU>(acc, lds);
  else if (A.act == FMS_ACT_GELU)
    gate_epilogue<P, kPull, FMS_ACT_GELU>(acc, lds);
  else
    gate_epilogue<P, kPull, FMS_ACT_GELU_TANH>(acc, lds);
  __syncthreads();
  Tile::store(lds, static_cast<T*>(A.out0), A.tokens, A.out_cols, A.out_pitch, m0, n0, A.out_vec);
  if constexpr (kPull)
    Tile::store(lds + Tile::kBytes, static_cast<T*>(A.out1), A.tokens, A.out_cols, A.out_pitch, m0,
                n0, A.out_vec);
}

// A product of the pullback.  Unit u of its tiles * splits * outputs: out[z] or, with splits,
// a part of it over k, in fp32.
struct ProductArgs {
  Matrix m[2], n[2];
  int32_t segments;  // 2: out[0] = m0 n0 + m1 n1; 1: out[z] = m_z n_z
  int32_t outputs;
  int32_t tm, tn, steps, splits;  // steps of all segments
  int64_t rows, cols;
  void* out[2];
  int32_t vec;
  float* parts;  // splits > 1: (splits, outputs, rows, part_pitch)
  int64_t part_pitch;
};

template <class P, int kLds>
__device__ __forceinline__ void product_unit(const ProductArgs& A, int unit, char (&lds)[kLds]) {
  typedef typename P::Op Op;
  typedef typename OutOf<Op>::T T;
  typedef LdsTile<Op, P::kBM, P::kBN, P::kThreads> Tile;
  static_assert(Tile::kBytes <= kLds && P::kLds <= kLds, "the output tile reuses the LDS");
  const int tiles = A.tm * A.tn, z = unit / (tiles * A.splits), split = unit / tiles % A.splits;
  int im, in;
  tile_of(unit % tiles, A.tm, A.tn, im, in);
  const int64_t m0 = (int64_t)im * P::kBM, n0 = (int64_t)in * P::kBN;
  typename P::Acc acc[2][P::kMF] = {};
  // the split's steps, counted over the segments
  const int s0 = (int)((int64_t)A.steps * split / A.splits);
  const int s1 = (int)((int64_t)A.steps * (split + 1) / A.splits);
  const int each = A.steps / A.segments;
  for (int s = 0; s < A.segments; ++s) {
    const Matrix M[1] = {A.m[z + s]}, N[1] = {A.n[z + s]};
    const int from = s0 - s * each, to = s1 - s * each;
    P::run(acc, M, N, m0, n0, from > 0 ? from : 0, to < each ? to : each, lds);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / P::kWN, wn = wave % P::kWN, h = lane >> 5;
  float* const part = A.splits > 1 ? A.parts + ((int64_t)split * A.outputs + z) * A.rows * A.part_pitch
                                   : nullptr;
#pragma unroll
  for (int mf = 0; mf < P::kMF; ++mf) {
    const int row = (wm * P::kMF + mf) * 32 + (lane & 31);
#pragma unroll
    for (int nf = 0; nf < 2; ++nf)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = P::col(wn, nf) + 8 * q + 4 * h;
        const auto& c = acc[nf][mf];
        if (part != nullptr) {
          if (m0 + row < A.rows && n0 + col < A.part_pitch)
            *reinterpret_cast<f32x4*>(part + (m0 + row) * A.part_pitch + n0 + col) =
                f32x4{c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]};
        } else {
          *Tile::quad(lds, row, col) =
              Quad<Op>::pack(c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]);
        }
      }
  }
  if (part != nullptr) return;
  __syncthreads();
  Tile::store(lds, static_cast<T*>(A.out[z]), A.rows, A.cols, A.cols, m0, n0, A.vec);
}

// Both products in one launch: the first `weights` workgroups take units of dwg and dwu, the
// others units of dx.
template <class PW, class PX>
__global__ void __launch_bounds__(PW::kThreads, 2) ffn_products_kernel(ProductArgs W, ProductArgs X,
                                                                       int weights) {
  typedef LdsTile<typename PW::Op, PW::kBM, PW::kBN, PW::kThreads> Tile;
  static_assert(PW::kBM == PX::kBM && PW::kBN == PX::kBN && PW::kLds == PX::kLds, "one shape");
  __shared__ __attribute__((aligned(16))) char lds[Tile::kBytes > PW::kLds ? Tile::kBytes : PW::kLds];
  if ((int)blockIdx.x < weights)
    product_unit<PW>(W, blockIdx.x, lds);
  else
    product_unit<PX>(X, blockIdx.x - weights, lds);
}

// out[z][r][c] = sum over splits of parts[s][z][r][c], in the order of s.
template <class Op>
__global__ void __launch_bounds__(256) ffn_join_kernel(void* out0, void* out1, const float* parts,
                                                       int splits, int nz, int64_t rows,
                                                       int64_t cols, int64_t pitch) {
  typedef typename OutOf<Op>::T T;
  const int64_t quads = pitch / 4, each = rows * quads;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nz * each;
       i += (int64_t)gridDim.x * 256) {
    const int64_t z = i / each, r = i % each / quads, c = i % each % quads * 4;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < splits; ++s) {
      const f32x4 v =
          *reinterpret_cast<const f32x4*>(parts + (((int64_t)s * nz + z) * rows + r) * pitch + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += v[e];
    }
    T* p = static_cast<T*>(z ? out1 : out0) + r * cols + c;
    for (int e = 0; e < 4 && c + e < cols; ++e) p[e] = (T)sum[e];
  }
}

// Rows of `cols` values copied to rows of `pitch`, the rest zero.
template <class T>
__global__ void __launch_bounds__(256) ffn_pad_kernel(T* out, const T* in, int64_t rows,
                                                      int64_t cols, int64_t pitch) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * pitch;
       i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / pitch, c = i % pitch;
    out[i] = c < cols ? in[r * cols + c] : (T)0;
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
hipError_t place_inputs(const FfnArgs& a, const Inputs& in, char* ws, Matrix (&m)[3],
                        hipStream_t st) {
  const void* src[3] = {a.x, a.wg, a.wu};
  const int64_t rows[3] = {a.tokens, a.hidden, a.hidden};
  const int esz = esz_of(a.dtype);
  for (int i = 0; i < 3; ++i) {
    const void* base = src[i];
    if (in.copy) {
      const int64_t n = rows[i] * in.pitch / esz;
      if (n > 0) {
        if (esz == 4)
          hipLaunchKernelGGL(ffn_pad_kernel<uint32_t>, dim3(grid_for(n)), dim3(256), 0, st,
                             reinterpret_cast<uint32_t*>(ws), static_cast<const uint32_t*>(src[i]),
                             rows[i], a.dim, in.pitch / esz);
        else
          hipLaunchKernelGGL(ffn_pad_kernel<uint16_t>, dim3(grid_for(n)), dim3(256), 0, st,
                             reinterpret_cast<uint16_t*>(ws), static_cast<const uint16_t*>(src[i]),
                             rows[i], a.dim, in.pitch / esz);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
      }
      base = ws;
      ws += rows[i] * in.pitch;
    }
    m[i].base = static_cast<const char*>(base);
    m[i].rows = rows[i];
    m[i].pitch = in.pitch;
    m[i].rowbytes = in.pitch;
  }
  return hipSuccess;
}

// The tile shapes by element size: wave grid and 32-row fragments per wave.
template <class Op, bool kMRows, bool kNRows, int kParts>
struct Shapes {
  typedef Product<Op, kMRows, kNRows, kParts, 2, 4, 4> Big;    // 256 x 256, 8 waves
  typedef Product<Op, kMRows, kNRows, kParts, 2, 2, 2> Small;  // 128 x 128, 4 waves
};

template <class P, bool kPull>
hipError_t launch_gate(GateArgs g, hipStream_t st) {
  g.tm = (int32_t)cdiv(g.tokens, P::kBM);
  g.tn = (int32_t)cdiv(g.out_cols, P::kBN / 2);
  g.steps = (int32_t)cdiv(g.x.rowbytes, kStepBytes);
  hipLaunchKernelGGL((ffn_gate_kernel<P, kPull>), dim3((unsigned)(g.tm * g.tn)), dim3(P::kThreads),
                     0, st, g);
  return hipGetLastError();
}

// 256 x 256 tiles run one workgroup to a CU; below one round of them the smaller tile
// fills more CUs.
bool big_tiles(int64_t rows, int64_t cols) { return cdiv(rows, 256) * cdiv(cols, 256) >= 192; }

template <class Op, bool kPull>
hipError_t run_gate(const GateArgs& g, hipStream_t st) {
  if (g.tokens == 0 || g.out_cols == 0) return hipSuccess;
  typedef Shapes<Op, true, true, 2> S;
  if constexpr (Op::kEsz == 2)
    if (big_tiles(g.tokens, 2 * g.out_cols)) return launch_gate<typename S::Big, kPull>(g, st);
  return launch_gate<typename S::Small, kPull>(g, st);
}

// ---- how the pullback's products are cut --------------------------------------------------
// dwg and dwu have few tiles of many steps (a step is 64 tokens), dx has many tiles of few.
// One launch takes both, the longer units first, so that the shorter ones fill what the
// longer leave idle; a product whose units would outlast the others is cut along k into parts
// that a second kernel adds.  The choice is the least estimate over tile shapes and numbers of
// parts, with the times measured on this card: of 23040 x 1024 x 4096 in bf16 the two
// products take 620 us in one launch and 890 one after the other.
struct Cut {
  bool big;
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
struct Costs {  // us: of a step, of a unit besides, of a MiB of parts written and read again
  double step, unit, part;
  int slots;
};

int64_t units_of(const ProductArgs& p, int64_t span) {
  return cdiv(p.rows, span) * cdiv(p.cols, span) * p.outputs;
}

Cut choose_cut(const ProductArgs* w, const ProductArgs* x, bool wide) {
  Cut best = {false, 1, 1};
  double least = 1e300;
  for (int big = 0; big < (wide ? 2 : 1); ++big) {
    const Costs c = wide ? (big ? Costs{1.55, 4.0, 0.4, 256} : Costs{1.0, 3.0, 0.4, 512})
                         : Costs{4.0, 3.0, 0.4, 512};
    const int64_t span = big ? 256 : 128;
    for (int sw = 1; sw <= (w ? 64 : 1); sw *= 2)
      for (int sx = 1; sx <= (x ? 16 : 1); sx *= 2) {
        double unit[2] = {0.0, 0.0}, joins = 0.0;
        int64_t units[2] = {0, 0};
        const auto add = [&](int i, const ProductArgs* p, int splits) {
          if (p == nullptr) return;
          unit[i] = c.unit + c.step * (double)cdiv(p->steps, splits);
          units[i] = units_of(*p, span) * splits;
          if (splits > 1)
            joins += 4.0 + c.part * splits * (double)(p->outputs * p->rows * p->cols) * 4 / (1 << 20);
        };
        add(0, w, sw);
        add(1, x, sx);
        const double t = makespan(units[0], unit[0], units[1], unit[1], c.slots) + joins;
        if (t < least) {
          least = t;
          best = Cut{big != 0, sw, sx};
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
  for (const ProductArgs* p : {&w, &x}) {
    if (e != hipSuccess || p->splits == 1 || p->rows * p->cols == 0) continue;
    hipLaunchKernelGGL((ffn_join_kernel<Op>), dim3(grid_for(p->outputs * p->rows * p->part_pitch / 4)),
                       dim3(256), 0, st, p->out[0], p->out[1], p->parts, p->splits, p->outputs, p->rows,
                       p->cols, p->part_pitch);
    e = hipGetLastError();
  }
  return e;
}

// w: dwg and dwu (or null), x: dx (or null).
template <class Op>
hipError_t run_products(const ProductArgs* w, const ProductArgs* x, hipStream_t st) {
  typedef Shapes<Op, false, false, 1> W;
  typedef Shapes<Op, true, false, 1> X;
  const Cut cut = choose_cut(w, x, Op::kEsz == 2);
  const ProductArgs none = {};
  if constexpr (Op::kEsz == 2)
    if (cut.big)
      return launch_products<Op, typename W::Big, typename X::Big>(w ? *w : none, x ? *x : none, cut, st);
  return launch_products<Op, typename W::Small, typename X::Small>(w ? *w : none, x ? *x : none, cut, st);
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
  g.out_vec = whole_units(h, a.hidden * Op::kEsz);
  return run_gate<Op, false>(g, st);
}

template <class Op>
hipError_t pullback(const FfnArgs& a, void* dx, void* dwg, void* dwu, const void* dh,
                    hipStream_t st) {
  const Inputs in = inputs_of(a);
  const int64_t pitch = round_up(a.hidden * Op::kEsz, 16);  // of dg and du
  const int64_t each = round_up(a.tokens * pitch, 256);
  Workspace ws(st);
  hipError_t e = ws.take(in.bytes + 2 * each);
  if (e != hipSuccess) return e;
  Matrix m[3];
  e = place_inputs(a, in, ws.p, m, st);
  if (e != hipSuccess) return e;
  char* const dg = ws.p + in.bytes;
  GateArgs g = gate_args(a, m);
  g.in = dh;
  g.in_pitch = a.hidden;
  g.in_vec = whole_units(dh, a.hidden * Op::kEsz);
  g.out0 = dg;
  g.out1 = dg + each;
  g.out_cols = g.out_pitch = pitch / Op::kEsz;
  g.out_vec = 1;
  e = run_gate<Op, true>(g, st);
  if (e != hipSuccess) return e;
  const Matrix d[2] = {{dg, a.tokens, pitch, pitch}, {dg + each, a.tokens, pitch, pitch}};
  ProductArgs w = {}, x = {};
  w.m[0] = d[0];
  w.m[1] = d[1];
  w.n[0] = w.n[1] = m[0];
  w.segments = 1;
  w.outputs = 2;
  w.steps = (int32_t)cdiv(a.tokens * Op::kEsz, kStepBytes);
  w.rows = a.hidden;
  w.cols = a.dim;
  w.out[0] = dwg;
  w.out[1] = dwu;
  w.vec = whole_units(dwg, a.dim * Op::kEsz) && whole_units(dwu, a.dim * Op::kEsz);
  x.m[0] = d[0];
  x.m[1] = d[1];
  x.n[0] = m[1];
  x.n[1] = m[2];
  x.segments = 2;
  x.outputs = 1;
  x.steps = 2 * (int32_t)cdiv(pitch, kStepBytes);
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

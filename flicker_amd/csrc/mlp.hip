// The matrix products of the gated MLP and of its gradients, on bf16 / fp16 MFMA.
//
//   forward   [g | u] = x Win,  h = silu(g) u,  y = h Wout
//   backward  dh = dy Wout^T,  [dg | du] from dh, g, u (swiglu.hip's formulas),
//             dWout = h^T dy,  dWin = x^T [dg | du],  dx = [dg | du] Win^T
//
// Each is D (rows, cols) = A B with float32 sums, computed transposed (D^T = B^T A^T: the MFMA's A
// operand holds 16 columns of D, its B operand 16 rows), so that a lane ends with four neighbouring
// columns of one row.  The gate's product takes g's and u's columns into one tile: a lane that holds
// g of a column holds u of the same column, and h leaves the registers as the only output.

#include "elems.h"

namespace {

using flk::f32x4;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kT = 64, kK = 32;       // tile edge, inner terms a step
constexpr int kPitch = kK + 8;        // an LDS row, padded

enum Epilogue { kPlain, kGate, kGateBackward };

struct Operand {      // rows x inner: element (r, k) at r * stride + k, or with kAcross k * stride + r
  const void* p;
  int64_t stride;
  int rows;
};

struct Product {
  Operand a, b;       // b: the columns of D as rows
  int inner;
  void* d;
  int64_t d_stride;
  float* gu;          // kGate: out, may be NULL; kGateBackward: in
  int hidden;         // kGate, kGateBackward
  int tiles_a, tiles_b;
};

template <typename T>
struct Mfma;
template <>
struct Mfma<__bf16> {
  typedef flk::bf16x8 vec;
  static __device__ __forceinline__ f32x4 run(vec a, vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mfma<_Float16> {
  typedef f16x8 vec;
  static __device__ __forceinline__ f32x4 run(vec a, vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// Row of the operand that tile row r holds: with kPair, 16 rows of the first half, then the same 16 of
// the second (hidden further), for each 32 of the tile; -1 past the end.
template <bool kPair>
__device__ __forceinline__ int source_row(int tile, int r, int rows, int hidden) {
  if constexpr (!kPair) return tile * kT + r < rows ? tile * kT + r : -1;
  const int col = tile * (kT / 2) + r / 32 * 16 + r % 16;
  return col >= hidden ? -1 : r % 32 < 16 ? col : hidden + col;
}

template <typename T, bool kAcross, bool kPair>
__device__ __forceinline__ void stage(T (*lds)[kPitch], const Operand& o, int tile, int k0, int inner, int hidden) {
  typedef typename Mfma<T>::vec vec;
  const T* p = static_cast<const T*>(o.p);
  vec v{};
  if constexpr (!kAcross) {
    const int r = threadIdx.x / 4, k = k0 + threadIdx.x % 4 * 8;
    const int row = source_row<kPair>(tile, r, o.rows, hidden);
    if (row >= 0 && k < inner) v = *reinterpret_cast<const vec*>(p + row * o.stride + k);
    *reinterpret_cast<vec*>(&lds[r][threadIdx.x % 4 * 8]) = v;
  } else {
    const int k = k0 + threadIdx.x / 8, r = threadIdx.x % 8 * 8;
    const int row = source_row<kPair>(tile, r, o.rows, hidden);
    if (row >= 0 && k < inner) v = *reinterpret_cast<const vec*>(p + k * o.stride + row);
#pragma unroll
    for (int i = 0; i < 8; ++i) lds[r + i][threadIdx.x / 8] = v[i];
  }
}

template <typename T, bool kAAcross, bool kBAcross, Epilogue kE>
__global__ __launch_bounds__(kThreads) void mlp_kernel(const Product P) {
  typedef typename Mfma<T>::vec vec;
  __shared__ __attribute__((aligned(16))) T la[kT][kPitch], lb[kT][kPitch];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wb = wave >> 1, wa = wave & 1, l16 = lane & 15, h4 = lane >> 4;
  const int ta = blockIdx.x % P.tiles_a, tb = blockIdx.x / P.tiles_a;
  f32x4 acc[2][2] = {};
  for (int k0 = 0; k0 < P.inner; k0 += kK) {
    stage<T, kAAcross, false>(la, P.a, ta, k0, P.inner, 0);
    stage<T, kBAcross, kE == kGate>(lb, P.b, tb, k0, P.inner, P.hidden);
    __syncthreads();
    vec fa[2], fb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fa[i] = *reinterpret_cast<const vec*>(&la[wa * 32 + i * 16 + l16][h4 * 8]);
      fb[i] = *reinterpret_cast<const vec*>(&lb[wb * 32 + i * 16 + l16][h4 * 8]);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int m = 0; m < 2; ++m) acc[n][m] = Mfma<T>::run(fb[n], fa[m], acc[n][m]);
    __syncthreads();
  }
  T* d = static_cast<T*>(P.d);
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const int64_t row = (int64_t)ta * kT + wa * 32 + m * 16 + l16;
    if (row >= P.a.rows) continue;
    if constexpr (kE == kGate) {
      const int col = tb * (kT / 2) + wb * 16 + h4 * 4;
      if (col >= P.hidden) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float g = acc[0][m][i], u = acc[1][m][i];
        d[row * P.d_stride + col + i] = (T)flk::gate(g, u);
        if (P.gu) {
          P.gu[row * 2 * P.hidden + col + i] = g;
          P.gu[row * 2 * P.hidden + P.hidden + col + i] = u;
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int col = tb * kT + wb * 32 + n * 16 + h4 * 4;
        if (col >= P.b.rows) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = acc[n][m][i];
          if constexpr (kE == kPlain) {
            d[row * P.d_stride + col + i] = (T)x;
          } else {
            const float g = P.gu[row * 2 * P.hidden + col + i], u = P.gu[row * 2 * P.hidden + P.hidden + col + i];
            float dg, du;
            flk::gate_backward(x, g, u, dg, du);
            d[row * P.d_stride + col + i] = (T)dg;
            d[row * P.d_stride + P.hidden + col + i] = (T)du;
          }
        }
      }
    }
  }
}

constexpr int kMaxDim = INT32_MAX - 256;

template <bool kAAcross, bool kBAcross, Epilogue kE>
int launch(Product& p, int dtype, void* stream) {
  p.tiles_a = (p.a.rows + kT - 1) / kT;
  p.tiles_b = kE == kGate ? (p.hidden + kT / 2 - 1) / (kT / 2) : (p.b.rows + kT - 1) / kT;
  const int64_t blocks = (int64_t)p.tiles_a * p.tiles_b;
  if (blocks > (1 << 23)) return FLK_E_INVALID;   // work-items of a launch are counted in 32 bits
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == FLK_BF16)
    mlp_kernel<__bf16, kAAcross, kBAcross, kE><<<dim3((unsigned)blocks), kThreads, 0, s>>>(p);
  else
    mlp_kernel<_Float16, kAAcross, kBAcross, kE><<<dim3((unsigned)blocks), kThreads, 0, s>>>(p);
  return flk_launch_status();
}

bool odd8(int64_t v) { return v % 8 != 0; }

}  // namespace

extern "C" int flk_mlp_plan(int product, int rows, int cols, int inner, int64_t* workspace_bytes) {
  if (product < FLK_MLP_GATE || product > FLK_MLP_MATMUL_AT || rows < 0 || cols < 0 || inner < 0 || !workspace_bytes)
    return FLK_E_INVALID;
  *workspace_bytes = 0;
  return FLK_OK;
}

extern "C" int flk_mlp_gate(const void* x, int64_t x_row_stride, const void* w_in, int64_t w_in_row_stride, int dtype,
                            int m, int width, int hidden, void* h, int64_t h_row_stride, float* gu, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  if (dtype != FLK_BF16 && dtype != FLK_F16) return FLK_E_INVALID;
  if (m < 0 || width < 0 || hidden < 0 || x_row_stride < width || w_in_row_stride < 2LL * hidden ||
      h_row_stride < hidden)
    return FLK_E_INVALID;
  if (m > kMaxDim || width > kMaxDim || hidden > kMaxDim / 2) return FLK_E_INVALID;
  if (m == 0 || hidden == 0) return FLK_OK;
  if (!x || !w_in || !h || width == 0) return FLK_E_INVALID;
  if (odd8(width) || odd8(hidden)) return FLK_E_UNSUPPORTED;
  if (odd8(x_row_stride) || odd8(w_in_row_stride) || odd8(h_row_stride) || !flk_host_aligned(x, 16) ||
      !flk_host_aligned(w_in, 16) || !flk_host_aligned(h, 16) || !flk_host_aligned(gu, 16))
    return FLK_E_ALIGN;
  Product p{};
  p.a = Operand{x, x_row_stride, m};
  p.b = Operand{w_in, w_in_row_stride, 2 * hidden};
  p.inner = width;
  p.d = h;
  p.d_stride = h_row_stride;
  p.gu = gu;
  p.hidden = hidden;
  return launch<false, true, kGate>(p, dtype, stream);
}

extern "C" int flk_mlp_gate_backward(const void* dy, int64_t dy_row_stride, const void* w_out, int64_t w_out_row_stride,
                                     const float* gu, int dtype, int m, int width, int hidden, void* dgu,
                                     int64_t dgu_row_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype != FLK_BF16 && dtype != FLK_F16) return FLK_E_INVALID;
  if (m < 0 || width < 0 || hidden < 0 || dy_row_stride < width || w_out_row_stride < width ||
      dgu_row_stride < 2LL * hidden)
    return FLK_E_INVALID;
  if (m > kMaxDim || width > kMaxDim || hidden > kMaxDim / 2) return FLK_E_INVALID;
  if (m == 0 || hidden == 0) return FLK_OK;
  if (!dy || !w_out || !gu || !dgu || width == 0) return FLK_E_INVALID;
  if (odd8(width) || odd8(hidden)) return FLK_E_UNSUPPORTED;
  if (odd8(dy_row_stride) || odd8(w_out_row_stride) || odd8(dgu_row_stride) || !flk_host_aligned(dy, 16) ||
      !flk_host_aligned(w_out, 16) || !flk_host_aligned(gu, 16) || !flk_host_aligned(dgu, 16))
    return FLK_E_ALIGN;
  Product p{};
  p.a = Operand{dy, dy_row_stride, m};
  p.b = Operand{w_out, w_out_row_stride, hidden};
  p.inner = width;
  p.d = dgu;
  p.d_stride = dgu_row_stride;
  p.gu = const_cast<float*>(gu);
  p.hidden = hidden;
  return launch<false, false, kGateBackward>(p, dtype, stream);
}

extern "C" int flk_mlp_matmul(const void* a, int64_t a_row_stride, int a_transposed, const void* b,
                              int64_t b_row_stride, int b_transposed, int dtype, int rows, int cols, int inner, void* d,
                              int64_t d_row_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype != FLK_BF16 && dtype != FLK_F16) return FLK_E_INVALID;
  if (rows < 0 || cols < 0 || inner < 0 || a_row_stride < (a_transposed ? rows : inner) ||
      b_row_stride < (b_transposed ? inner : cols) || d_row_stride < cols)
    return FLK_E_INVALID;
  if (rows > kMaxDim || cols > kMaxDim || inner > kMaxDim) return FLK_E_INVALID;
  if (a_transposed && b_transposed) return FLK_E_UNSUPPORTED;
  if (rows == 0 || cols == 0) return FLK_OK;
  if (!a || !b || !d || inner == 0) return FLK_E_INVALID;
  if (odd8(cols) || odd8(a_transposed ? rows : inner)) return FLK_E_UNSUPPORTED;
  if (odd8(a_row_stride) || odd8(b_row_stride) || odd8(d_row_stride) || !flk_host_aligned(a, 16) ||
      !flk_host_aligned(b, 16) || !flk_host_aligned(d, 16))
    return FLK_E_ALIGN;
  Product p{};
  p.a = Operand{a, a_row_stride, rows};
  p.b = Operand{b, b_row_stride, cols};
  p.inner = inner;
  p.d = d;
  p.d_stride = d_row_stride;
  if (a_transposed) return launch<true, true, kPlain>(p, dtype, stream);
  if (b_transposed) return launch<false, false, kPlain>(p, dtype, stream);
  return launch<false, true, kPlain>(p, dtype, stream);
}

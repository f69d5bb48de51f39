// The gate of the blocks' MLP on projected halves, and its gradients (elementwise).
//
//   h = silu(g) u,  silu(z) = z s(z),  s(z) = 1 / (1 + exp(-z))
//   dg = dh u s (1 + g (1 - s)),  du = dh g s
//
// float32 arithmetic, each output rounded once.  HBM bounds it: three values move per output
// forwards, five per pair of outputs backwards; a lane takes 8 columns of both halves, so
// every access is 16 bytes (32 for float32) and neighbouring lanes' are adjacent.  16-bit operands and outputs
// pass the caches by (nontemporal): at the blocks' sizes they are as large as the caches.  4608 x 9216
// bf16 from a row of 27648: forward 42 us (6.0 TB/s; 49 through the caches), backward 66 (6.4; 83); a large copy
// reaches 5.2.  Float32 ones do not: 512 x 9216 forward 10.6 us (past the caches 12.5), backward 17.8 (19.7), 1536 rows
// between two neighbours that write gu and read h 78 (84) and 103 (112); 4608 rows 90.6 (92.1; 5.6 TB/s) and 150
// (157; 5.7), within 2% between neighbours.

#include "elems.h"

namespace {

constexpr int kThreads = 256;

struct Rows {
  const void* p;
  int64_t batch_stride, row_stride;
};

struct GateArgs {
  Rows gu, dh, out;
  int length, hidden, chunks;   // chunks of 8 columns a row
  int64_t total;                // rows * chunks
};

template <typename T>
__device__ __forceinline__ T* row_at(const Rows& r, int64_t b, int64_t t) {
  return static_cast<T*>(const_cast<void*>(r.p)) + b * r.batch_stride + t * r.row_stride;
}

template <typename T, bool kBackward>
__global__ __launch_bounds__(kThreads) void swiglu_kernel(const GateArgs A) {
  constexpr bool kStream = sizeof(T) == 2;
  for (int64_t first = (int64_t)blockIdx.x * kThreads; first < A.total; first += (int64_t)gridDim.x * kThreads) {
    // The block's first row is scalar; a lane's own is at most kThreads rows on.
    const int64_t row0 = first / A.chunks;
    const int in_row = (int)(first - row0 * A.chunks) + (int)threadIdx.x;
    const int ahead = in_row / A.chunks;
    const int64_t row = row0 + ahead;
    if (first + threadIdx.x >= A.total) return;
    const int at = (in_row - ahead * A.chunks) * 8, left = A.hidden - at;
    const int64_t b = row / A.length, t = row - b * A.length;
    const T* gu = row_at<T>(A.gu, b, t) + at;
    const flk::Raw8<T> g8 = flk::load8<kStream>(gu, left), u8 = flk::load8<kStream>(gu + A.hidden, left);
    T* out = row_at<T>(A.out, b, t) + at;
    float o0[8], o1[8];
    if constexpr (kBackward) {
      const flk::Raw8<T> d8 = flk::load8<kStream>(row_at<T>(A.dh, b, t) + at, left);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        flk::gate_backward((float)d8.v[i], (float)g8.v[i], (float)u8.v[i], o0[i], o1[i]);
      flk::store8<kStream>(out + A.hidden, left, o1);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) o0[i] = flk::gate((float)g8.v[i], (float)u8.v[i]);
    }
    flk::store8<kStream>(out, left, o0);
  }
}

template <typename T>
int launch(const GateArgs& a, hipStream_t s) {
  const int64_t blocks = (a.total + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)(blocks < (1 << 23) ? blocks : 1 << 23));   // work-items are counted in 32 bits
  if (a.dh.p)
    swiglu_kernel<T, true><<<grid, kThreads, 0, s>>>(a);
  else
    swiglu_kernel<T, false><<<grid, kThreads, 0, s>>>(a);
  return flk_launch_status();
}

int run(GateArgs& a, int dtype, int batch, int length, int hidden, bool backward, void* stream) {
  if (dtype < FLK_BF16 || dtype > FLK_F32 || batch < 0 || length < 0 || hidden <= 0 || hidden > INT32_MAX - 4096)
    return FLK_E_INVALID;
  if (batch == 0 || length == 0) return FLK_OK;
  if (!a.gu.p || !a.out.p || (backward && !a.dh.p)) return FLK_E_INVALID;
  const unsigned bytes = dtype == FLK_F32 ? 4 : 2;
  if (!flk_host_aligned(a.gu.p, bytes) || !flk_host_aligned(a.out.p, bytes) || !flk_host_aligned(a.dh.p, bytes))
    return FLK_E_ALIGN;
  a.length = length;
  a.hidden = hidden;
  a.chunks = (hidden + 7) / 8;
  a.total = (int64_t)batch * length * a.chunks;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == FLK_F32 ? launch<float>(a, s) : dtype == FLK_BF16 ? launch<__bf16>(a, s) : launch<_Float16>(a, s);
}

}  // namespace

extern "C" int flk_swiglu(const void* gu, int64_t gu_batch_stride, int64_t gu_row_stride, int dtype, int batch,
                          int length, int hidden, void* h, int64_t h_batch_stride, int64_t h_row_stride,
                          void* stream) {
  GateArgs a{};
  a.gu = Rows{gu, gu_batch_stride, gu_row_stride};
  a.out = Rows{h, h_batch_stride, h_row_stride};
  return run(a, dtype, batch, length, hidden, false, stream);
}

extern "C" int flk_swiglu_backward(const void* dh, int64_t dh_batch_stride, int64_t dh_row_stride, const void* gu,
                                   int64_t gu_batch_stride, int64_t gu_row_stride, int dtype, int batch, int length,
                                   int hidden, void* dgu, int64_t dgu_batch_stride, int64_t dgu_row_stride,
                                   void* stream) {
  GateArgs a{};
  a.dh = Rows{dh, dh_batch_stride, dh_row_stride};
  a.gu = Rows{gu, gu_batch_stride, gu_row_stride};
  a.out = Rows{dgu, dgu_batch_stride, dgu_row_stride};
  return run(a, dtype, batch, length, hidden, true, stream);
}

// Layer norm with a per-channel factor and offset, and its gradients.
//
// Row r of batch entry b (nn.py:17-21 and modules.py:38-40 of the reference, rounded once):
//   m = mean_j x_j,  v = mean_j (x_j - m)^2,  q = 1 / sqrt(v + eps),  n_j = (x_j - m) q
//   y_j = n_j a_j + c_j
// where a = factor and c = offset, either one row for every batch entry (an affine norm) or one
// row each with a = 1 + factor (the blocks' modulation).  Backward, with t_j = dy_j a_j:
//   dx_j = q (t_j - mean(t) - n_j mean(t n))
//   dfactor_j = sum over the rows that share it of dy_j n_j,  doffset_j = sum of dy_j
//
// All arithmetic is float32 and every output is rounded once.  The variance is summed from the
// centred row (two passes over registers): sums of squares of an uncentred residual stream,
// whose tokens sit off zero, would cancel.
//
// HBM bounds both directions: a row is read once and kept in registers, kW lanes of it at a
// time, kV chunks of 8 elements a lane.  The backward pass recomputes m and q from the row it has
// to read anyway, so the forward pass keeps nothing.  Its column sums stay in the lanes that own
// the columns while a block walks its rows; blocks write them as partial rows, which a second
// kernel adds in a fixed order: the gradients do not depend on timing.

#include <algorithm>

#include "elems.h"

namespace {

constexpr int kThreads = 256;

struct Rows {            // row t of batch entry b at p + b * batch_stride + t * row_stride
  const void* p;
  int64_t batch_stride, row_stride;
};

struct NormArgs {
  Rows x, dy, y;         // y: the output (dx backwards)
  const void* factor;    // NULL: 1
  const void* offset;    // NULL: 0
  int64_t param_stride;  // elements from one batch entry's row to the next (0: one row for all)
  float add;             // a = factor + add
  float eps, inv_width;
  int length, width;
  int64_t rows;          // batch * length
  // backward: blocks of `per_block` rows of one group; partial sums (block, 2, width)
  float* partial;
  int64_t group_rows;
  int per_block, blocks_per_group;
};

template <typename T>
__device__ __forceinline__ const T* row_at(const Rows& r, int64_t b, int64_t t) {
  return static_cast<const T*>(r.p) + b * r.batch_stride + t * r.row_stride;
}

// Sum over 64 lanes; every lane ends with the same value.
__device__ __forceinline__ float wave_sum(float v) {
  v = flk::row16_sum(v);
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Sums of a and b over the kW lanes of a row.  With more than one wave a row, the waves exchange
// their sums through `scratch`; the halves alternate (turn), so one barrier a call is enough.
template <int kW>
__device__ __forceinline__ void row_sums(float& a, float& b, float (*scratch)[2][kW / 64], int& turn) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (kW > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      scratch[turn][0][wave] = a;
      scratch[turn][1][wave] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < kW / 64; ++w) {
      a += scratch[turn][0][w];
      b += scratch[turn][1][w];
    }
    turn ^= 1;
  }
}

// Centres the row in xs (elements past the row's end become 0) and returns 1 / sqrt(v + eps).
template <int kW, int kV>
__device__ __forceinline__ float centre(float (&xs)[kV][8], const int (&left)[kV], const NormArgs& A,
                                        float (*scratch)[2][kW / 64], int& turn) {
  float sum = 0.0f, none = 0.0f;
#pragma unroll
  for (int c = 0; c < kV; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += xs[c][i];
  row_sums<kW>(sum, none, scratch, turn);
  const float mean = sum * A.inv_width;
  float square = 0.0f;
#pragma unroll
  for (int c = 0; c < kV; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      xs[c][i] = i < left[c] ? xs[c][i] - mean : 0.0f;
      square += xs[c][i] * xs[c][i];
    }
  row_sums<kW>(square, none, scratch, turn);
  return 1.0f / sqrtf(square * A.inv_width + A.eps);
}

template <typename T, typename P, int kW, int kV>
__global__ __launch_bounds__(kW > kThreads ? kW : kThreads) void norm_kernel(const NormArgs A) {
  constexpr int kRows = kW > kThreads ? 1 : kThreads / kW;   // rows per block
  __shared__ float scratch[2][2][kW / 64];
  int turn = 0;
  const int lane = threadIdx.x % kW;
  // Rows past kMaxBlocks blocks' are walked in turns, whole waves (one row a block: whole blocks).
  for (int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kW; row < A.rows; row += (int64_t)gridDim.x * kRows) {
    const int64_t b = row / A.length, t = row - b * A.length;
    const T* x = row_at<T>(A.x, b, t);
    T* y = const_cast<T*>(row_at<T>(A.y, b, t));
    int left[kV];
    float xs[kV][8];
  #pragma unroll
    for (int c = 0; c < kV; ++c) {
      const int at = (lane + kW * c) * 8;
      left[c] = A.width - at;
      const flk::Raw8<T> r = flk::load8(x + at, left[c]);
  #pragma unroll
      for (int i = 0; i < 8; ++i) xs[c][i] = (float)r.v[i];
    }
    const float q = centre<kW, kV>(xs, left, A, scratch, turn);
    const P* factor = static_cast<const P*>(A.factor);
    const P* offset = static_cast<const P*>(A.offset);
    if (factor) factor += b * A.param_stride;
    if (offset) offset += b * A.param_stride;
  #pragma unroll
    for (int c = 0; c < kV; ++c) {
      const int at = (lane + kW * c) * 8;
      if (left[c] <= 0) continue;
      float out[8];
  #pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = xs[c][i] * q;
      if (factor) {
        const flk::Raw8<P> f = flk::load8(factor + at, left[c]);
  #pragma unroll
        for (int i = 0; i < 8; ++i) out[i] *= (float)f.v[i] + A.add;
      }
      if (offset) {
        const flk::Raw8<P> f = flk::load8(offset + at, left[c]);
  #pragma unroll
        for (int i = 0; i < 8; ++i) out[i] += (float)f.v[i];
      }
      flk::store8(y + at, left[c], out);
    }
  }
}

template <typename T, typename P, int kW, int kV>
__global__ __launch_bounds__(kW > kThreads ? kW : kThreads) void norm_backward_kernel(const NormArgs A) {
  constexpr int kRows = kW > kThreads ? 1 : kThreads / kW;
  __shared__ float scratch[2][2][kW / 64];
  __shared__ float sums[kRows > 1 ? 2 * kV * 8 * kW : 1];
  int turn = 0;
  const int lane = threadIdx.x % kW, slot = threadIdx.x / kW;
  const int64_t group = blockIdx.x / A.blocks_per_group;
  const int64_t first = (int64_t)(blockIdx.x - group * A.blocks_per_group) * A.per_block;   // of the group's rows
  const int64_t end = min(first + A.per_block, A.group_rows);
  const P* factor = static_cast<const P*>(A.factor);
  if (factor) factor += group * A.param_stride;
  int left[kV];
  flk::Raw8<P> f[kV];
  float da[kV][8], dc[kV][8];
#pragma unroll
  for (int c = 0; c < kV; ++c) {
    const int at = (lane + kW * c) * 8;
    left[c] = A.width - at;
    if (factor) f[c] = flk::load8(factor + at, left[c]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!factor) f[c].v[i] = (P)0.0f;
      da[c][i] = dc[c][i] = 0.0f;
    }
  }
  const float add = factor ? A.add : 1.0f;
  // With several rows a block each slot walks its own rows without barriers; with one, all waves
  // of the block walk the same rows.
  for (int64_t r = first + slot; r < end; r += kRows) {
    const int64_t row = group * A.group_rows + r;
    const int64_t b = row / A.length, t = row - b * A.length;
    const T* x = row_at<T>(A.x, b, t);
    const T* dy = row_at<T>(A.dy, b, t);
    T* dx = const_cast<T*>(row_at<T>(A.y, b, t));
    float xs[kV][8];
    flk::Raw8<T> g[kV];
#pragma unroll
    for (int c = 0; c < kV; ++c) {
      const int at = (lane + kW * c) * 8;
      const flk::Raw8<T> raw = flk::load8(x + at, left[c]);
      g[c] = flk::load8(dy + at, left[c]);
#pragma unroll
      for (int i = 0; i < 8; ++i) xs[c][i] = (float)raw.v[i];
    }
    const float q = centre<kW, kV>(xs, left, A, scratch, turn);
    float st = 0.0f, stn = 0.0f;
#pragma unroll
    for (int c = 0; c < kV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = (float)g[c].v[i], n = xs[c][i] * q;
        const float tt = d * ((float)f[c].v[i] + add);
        xs[c][i] = n;
        da[c][i] += d * n;
        dc[c][i] += d;
        st += tt;
        stn += tt * n;
      }
    row_sums<kW>(st, stn, scratch, turn);
    const float mt = st * A.inv_width, mtn = stn * A.inv_width;
#pragma unroll
    for (int c = 0; c < kV; ++c) {
      if (left[c] <= 0) continue;
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float tt = (float)g[c].v[i] * ((float)f[c].v[i] + add);
        out[i] = q * (tt - mt - xs[c][i] * mtn);
      }
      flk::store8(dx + (lane + kW * c) * 8, left[c], out);
    }
  }
  if (!A.partial) return;
  if constexpr (kRows > 1) {   // slot 0 adds the other slots' sums, one slot at a time
    for (int s = 1; s < kRows; ++s) {
      __syncthreads();
      if (slot == s) {
#pragma unroll
        for (int c = 0; c < kV; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            sums[(c * 8 + i) * kW + lane] = da[c][i];
            sums[(kV * 8 + c * 8 + i) * kW + lane] = dc[c][i];
          }
      }
      __syncthreads();
      if (slot == 0) {
#pragma unroll
        for (int c = 0; c < kV; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            da[c][i] += sums[(c * 8 + i) * kW + lane];
            dc[c][i] += sums[(kV * 8 + c * 8 + i) * kW + lane];
          }
      }
    }
    if (slot) return;
  }
  float* out = A.partial + (int64_t)blockIdx.x * 2 * A.width;
#pragma unroll
  for (int c = 0; c < kV; ++c) {
    const int at = (lane + kW * c) * 8;
    if (left[c] <= 0) continue;
    flk::store8(out + at, left[c], da[c]);
    flk::store8(out + A.width + at, left[c], dc[c]);
  }
}

// Adds a group's partial rows in order: 64 columns a block, four waves take every fourth row each.
template <typename P>
__global__ __launch_bounds__(kThreads) void norm_params_kernel(const float* __restrict__ partial, int blocks, int width,
                                                               int cuts, P* dfactor, P* doffset) {
  __shared__ float part[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t group = blockIdx.x / cuts;
  const int col = (int)(blockIdx.x - group * cuts) * 64 + lane;
  const int which = blockIdx.y;              // 0: factor, 1: offset
  P* out = which ? doffset : dfactor;
  if (!out) return;
  const float* src = partial + group * blocks * 2 * width + (int64_t)which * width + col;
  float sum = 0.0f;
  if (col < width)
    for (int i = wave; i < blocks; i += 4) sum += src[(int64_t)i * 2 * width];
  part[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && col < width) out[group * width + col] = (P)((part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]));
}

constexpr int kMaxWidth = 512 * 8 * 8;
constexpr int kMaxRows = INT32_MAX;
constexpr int64_t kMaxBlocks = 1 << 22;   // a launch's work-items are counted in 32 bits

// Rows each backward block walks: about 512 blocks, so that two share a CU, but no more than 64
// rows a block are needed to make the partial rows cheap.
int backward_rows(int64_t group_rows, int64_t groups) {
  const int64_t blocks = 512 / groups > 0 ? 512 / groups : 1;
  const int64_t per = (group_rows + blocks - 1) / blocks;
  return (int)(per < 4 ? 4 : per);
}

template <typename T, typename P, int kW, int kV>
int launch(const NormArgs& a, int64_t groups, bool backward, hipStream_t s) {
  constexpr int threads = kW > kThreads ? kW : kThreads, rows = threads / kW;
  if (backward)
    norm_backward_kernel<T, P, kW, kV><<<dim3((unsigned)(groups * a.blocks_per_group)), threads, 0, s>>>(a);
  else
    norm_kernel<T, P, kW, kV><<<dim3((unsigned)std::min((a.rows + rows - 1) / rows, kMaxBlocks)), threads, 0, s>>>(a);
  return flk_launch_status();
}

template <typename T, typename P>
int dispatch(const NormArgs& a, int64_t groups, bool backward, hipStream_t s) {
  if (a.width <= 512) return launch<T, P, 64, 1>(a, groups, backward, s);
  if (a.width <= 1024) return launch<T, P, 64, 2>(a, groups, backward, s);
  if (a.width <= 2048) return launch<T, P, 64, 4>(a, groups, backward, s);
  if (a.width <= 3 * 1024) return launch<T, P, 64, 6>(a, groups, backward, s);
  if (a.width <= 4096) return launch<T, P, 256, 2>(a, groups, backward, s);
  if (a.width <= 8192) return launch<T, P, 256, 4>(a, groups, backward, s);
  return launch<T, P, 512, 8>(a, groups, backward, s);
}

int dispatch_types(int dtype, int params, const NormArgs& a, int64_t groups, bool backward, hipStream_t s) {
  if (dtype == FLK_F32) return params == FLK_F32 ? dispatch<float, float>(a, groups, backward, s) : FLK_E_UNSUPPORTED;
  if (dtype == FLK_BF16) {
    if (params == FLK_BF16) return dispatch<__bf16, __bf16>(a, groups, backward, s);
    if (params == FLK_F32) return dispatch<__bf16, float>(a, groups, backward, s);
  }
  if (dtype == FLK_F16) {
    if (params == FLK_F16) return dispatch<_Float16, _Float16>(a, groups, backward, s);
    if (params == FLK_F32) return dispatch<_Float16, float>(a, groups, backward, s);
  }
  return FLK_E_UNSUPPORTED;
}

unsigned elem_bytes(int dtype) { return dtype == FLK_F32 ? 4 : 2; }

int check(int dtype, int params, const void* x, const void* y, const void* factor, const void* offset,
          int64_t param_stride, float eps, int batch, int length, int width) {
  if (dtype < FLK_BF16 || dtype > FLK_F32 || params < FLK_BF16 || params > FLK_F32) return FLK_E_INVALID;
  if (batch < 0 || length < 0 || width <= 0 || !(eps >= 0.0f) || param_stride < 0) return FLK_E_INVALID;
  if (param_stride && param_stride < width) return FLK_E_INVALID;
  if ((int64_t)batch * length > kMaxRows) return FLK_E_INVALID;
  if (width > kMaxWidth) return FLK_E_UNSUPPORTED;
  if (batch == 0 || length == 0) return FLK_OK;
  if (!x || !y) return FLK_E_INVALID;
  if (!flk_host_aligned(x, elem_bytes(dtype)) || !flk_host_aligned(y, elem_bytes(dtype)) ||
      !flk_host_aligned(factor, elem_bytes(params)) || !flk_host_aligned(offset, elem_bytes(params)))
    return FLK_E_ALIGN;
  return FLK_OK;
}

NormArgs common_args(const void* x, int64_t xb, int64_t xr, const void* factor, const void* offset,
                     int64_t param_stride, int add_one, float eps, int batch, int length, int width) {
  NormArgs a{};
  a.x = Rows{x, xb, xr};
  a.factor = factor;
  a.offset = offset;
  a.param_stride = param_stride;
  a.add = add_one ? 1.0f : 0.0f;
  a.eps = eps;
  a.inv_width = 1.0f / (float)width;
  a.length = length;
  a.width = width;
  a.rows = (int64_t)batch * length;
  return a;
}

}  // namespace

extern "C" int flk_layer_norm(const void* x, int64_t x_batch_stride, int64_t x_row_stride, int dtype,
                              const void* factor, const void* offset, int params_dtype, int64_t param_batch_stride,
                              int add_one, float eps, int batch, int length, int width, void* y,
                              int64_t y_batch_stride, int64_t y_row_stride, void* stream) {
  if (const int st = check(dtype, params_dtype, x, y, factor, offset, param_batch_stride, eps, batch, length, width))
    return st;
  if (batch == 0 || length == 0) return FLK_OK;
  NormArgs a = common_args(x, x_batch_stride, x_row_stride, factor, offset, param_batch_stride, add_one, eps, batch,
                           length, width);
  a.y = Rows{y, y_batch_stride, y_row_stride};
  return dispatch_types(dtype, params_dtype, a, 0, false, static_cast<hipStream_t>(stream));
}

extern "C" int flk_layer_norm_backward_plan(int batch, int length, int width, int shared_params,
                                            int64_t* workspace_bytes) {
  if (batch < 0 || length < 0 || width <= 0 || !workspace_bytes) return FLK_E_INVALID;
  if ((int64_t)batch * length > kMaxRows) return FLK_E_INVALID;
  *workspace_bytes = 0;
  if (batch == 0 || length == 0) return FLK_OK;
  const int64_t groups = shared_params ? 1 : batch, group_rows = shared_params ? (int64_t)batch * length : length;
  const int per = backward_rows(group_rows, groups);
  *workspace_bytes = groups * ((group_rows + per - 1) / per) * 2 * width * 4;
  return FLK_OK;
}

extern "C" int flk_layer_norm_backward(const void* dy, int64_t dy_batch_stride, int64_t dy_row_stride, const void* x,
                                       int64_t x_batch_stride, int64_t x_row_stride, int dtype, const void* factor,
                                       int params_dtype, int64_t param_batch_stride, int add_one, float eps, int batch,
                                       int length, int width, void* dx, int64_t dx_batch_stride, int64_t dx_row_stride,
                                       void* dfactor, void* doffset, void* workspace, int64_t workspace_bytes,
                                       void* stream) {
  if (const int st = check(dtype, params_dtype, x, dx, factor, dfactor, param_batch_stride, eps, batch, length, width))
    return st;
  if (batch == 0 || length == 0) return FLK_OK;   // the sums over no rows are the caller's to clear
  if (!dy) return FLK_E_INVALID;
  if (!flk_host_aligned(dy, elem_bytes(dtype)) || !flk_host_aligned(doffset, elem_bytes(params_dtype)))
    return FLK_E_ALIGN;
  NormArgs a = common_args(x, x_batch_stride, x_row_stride, factor, nullptr, param_batch_stride, add_one, eps, batch,
                           length, width);
  a.dy = Rows{dy, dy_batch_stride, dy_row_stride};
  a.y = Rows{dx, dx_batch_stride, dx_row_stride};
  const bool shared = param_batch_stride == 0;
  const int64_t groups = shared ? 1 : batch;
  a.group_rows = shared ? a.rows : length;
  a.per_block = backward_rows(a.group_rows, groups);
  a.blocks_per_group = (int)((a.group_rows + a.per_block - 1) / a.per_block);
  const int cuts = (width + 63) / 64;
  if (groups * a.blocks_per_group > kMaxBlocks || groups * cuts > kMaxBlocks) return FLK_E_INVALID;
  if (dfactor || doffset) {
    const int64_t need = groups * a.blocks_per_group * 2 * width * 4;
    if (!workspace || workspace_bytes < need) return FLK_E_SCRATCH;
    if (!flk_host_aligned(workspace, 16)) return FLK_E_ALIGN;
    a.partial = static_cast<float*>(workspace);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (const int st = dispatch_types(dtype, params_dtype, a, groups, true, s)) return st;
  if (!a.partial) return FLK_OK;
  const dim3 grid((unsigned)(groups * cuts), 2);
  if (params_dtype == FLK_F32)
    norm_params_kernel<float><<<grid, kThreads, 0, s>>>(a.partial, a.blocks_per_group, width, cuts,
                                                        static_cast<float*>(dfactor), static_cast<float*>(doffset));
  else if (params_dtype == FLK_BF16)
    norm_params_kernel<__bf16><<<grid, kThreads, 0, s>>>(a.partial, a.blocks_per_group, width, cuts,
                                                         static_cast<__bf16*>(dfactor), static_cast<__bf16*>(doffset));
  else
    norm_params_kernel<_Float16><<<grid, kThreads, 0, s>>>(a.partial, a.blocks_per_group, width, cuts,
                                                           static_cast<_Float16*>(dfactor),
                                                           static_cast<_Float16*>(doffset));
  return flk_launch_status();
}

// Gradients of qk_prep (qk_prep.hip): of the projection and of both norm scales.
//
// Forward, per (b, t, h) and section, with inv = 1 / sqrt(mean x^2 + 1e-6):
//   n = x inv;  y = n scale;  r[2j] = c y[2j] + s[2j] y[2j+1], r[2j+1] = c y[2j+1] + s[2j+1] y[2j];  out = gain r
// whose roundings to bf16 along the way pass gradients through.  Backward, for the gradient d of out:
//   dr = gain d;  dy[2j] = c[2j] dr[2j] + s[2j+1] dr[2j+1],  dy[2j+1] = c[2j+1] dr[2j+1] + s[2j] dr[2j]
//   dscale = sum over b, t, h of dy n;  dn = dy scale;  dx = inv (dn - n mean(dn n))
// and v's gradient is copied to its section bit for bit.  All arithmetic is float32, each output rounded once.
//
// HBM-bound: per (b, t, h) it reads 5 * 256 bytes (dq, dk, dv, x of q and of k) and writes 3 * 256.  The mapping is
// qk_prep's: 16 lanes a head row, 8 elements a lane, so both means are 16-lane DPP butterflies and each rotated pair
// stays inside a lane; 4 consecutive tokens of a wave read 1 KiB of a head's gradient.  A lane owns the same 8 columns of every row it meets,
// so the scales' gradients gather in 16 registers while a block walks its tokens and heads; blocks write them as
// partial rows, which a second kernel adds in a fixed order.
//
// Measured (24 heads): 2 x 4096 tokens 79.5 us, 5.1 TB/s, a large copy's rate (stored through the caches 85, read through
// them too 87-92; 3 blocks a CU 78.9, 6 84.5, 8 82; of one, three or four heads a group two are fastest); 512 tokens 11 us,
// two launches of 7 and 4.

#include <algorithm>

#include "qk_math.h"

namespace {

constexpr int kD = 128;
constexpr int kThreads = 128;
constexpr int kTokens = kThreads / 16;   // of a block at a time
constexpr int64_t kMaxItems = 1LL << 31;

struct Grad {   // row t of head h of batch entry b
  const uint16_t* p;
  int64_t batch, head, row;
};

struct Args {
  Grad dq, dk, dv;
  const uint16_t* qkv;
  int64_t qkv_batch, qkv_row;
  const float* cos;
  const float* sin;
  int64_t table_row;
  const void* q_scale;
  const void* k_scale;
  float gain;
  int length, heads, token_blocks, items;   // items: token blocks x groups of heads x batch entries
  uint16_t* out;
  int64_t out_batch, out_row;
  float* partial;   // (block, 2, 128)
};

// Operands are read once, and what is written is read next by matrix products, which wait for no memory: both go past the
// caches (nontemporal).
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint4 load16(const uint16_t* p) {
  const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ void store16(uint16_t* p, uint4 v) {
  const u32x4 w = {v.x, v.y, v.z, v.w};
  __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(p));
}

__device__ __forceinline__ void widen(uint4 raw, float (&x)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = flk::bf16_lo(w[i]);
    x[2 * i + 1] = flk::bf16_hi(w[i]);
  }
}

// dx of one row, whose dy n it adds to dscale.
__device__ __forceinline__ uint4 row_gradient(uint4 grad, uint4 raw, const float (&sc)[8], const float (&c)[8],
                                              const float (&s)[8], float gain, float (&dscale)[8]) {
  float d[8], x[8], dn[8];
  widen(grad, d);
  widen(raw, x);
  float ss = 0.0f, dot = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = gain * d[2 * j], b = gain * d[2 * j + 1];
    d[2 * j] = c[2 * j] * a + s[2 * j + 1] * b;
    d[2 * j + 1] = c[2 * j + 1] * b + s[2 * j] * a;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    ss += x[i] * x[i];
    dn[i] = d[i] * sc[i];
    dot += dn[i] * x[i];
  }
  ss = flk::row16_sum(ss);
  dot = flk::row16_sum(dot);
  const float inv = 1.0f / sqrtf(ss * (1.0f / kD) + 1e-6f);
  const float back = dot * inv * (1.0f / kD);   // mean(dn n)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float n = x[i] * inv;
    dscale[i] += d[i] * n;
    dn[i] = inv * (dn[i] - n * back);
  }
  return make_uint4(flk::pack_bf16x2(dn[0], dn[1]), flk::pack_bf16x2(dn[2], dn[3]), flk::pack_bf16x2(dn[4], dn[5]),
                    flk::pack_bf16x2(dn[6], dn[7]));
}

template <bool kScaleF32, int kHeads>
__global__ __launch_bounds__(kThreads) void qk_prep_backward_kernel(const Args A) {
  __shared__ float sums[kTokens][2 * kD];
  const int lane = threadIdx.x & 15, slot = threadIdx.x >> 4;
  const int groups = A.heads / kHeads;
  float qs[8], ks[8], dqs[8] = {}, dks[8] = {};
  flk::load_scale8<kScaleF32>(A.q_scale, lane, qs);
  flk::load_scale8<kScaleF32>(A.k_scale, lane, ks);
  for (int item = blockIdx.x; item < A.items; item += gridDim.x) {
    const int tb = item % A.token_blocks, rest = item / A.token_blocks;
    const int h0 = rest % groups * kHeads, b = rest / groups;
    const int t = tb * kTokens + slot;
    if (t >= A.length) continue;   // whole 16-lane rows together, so DPP rows stay intact
    const uint16_t* x = A.qkv + b * A.qkv_batch + t * A.qkv_row + lane * 8;
    uint16_t* out = A.out + b * A.out_batch + t * A.out_row + lane * 8;
    auto of = [&](const Grad& g, int h) {
      return load16(g.p + b * g.batch + h * g.head + t * g.row + lane * 8);
    };
    uint4 xq[kHeads], xk[kHeads], gq[kHeads], gk[kHeads], gv[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int h = h0 + i;
      xq[i] = load16(x + (int64_t)h * kD);
      xk[i] = load16(x + (int64_t)(A.heads + h) * kD);
      gq[i] = of(A.dq, h);
      gk[i] = of(A.dk, h);
      gv[i] = of(A.dv, h);
    }
    float c[8], s[8];
    flk::load_table8(A.cos + t * A.table_row, lane, c);
    flk::load_table8(A.sin + t * A.table_row, lane, s);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int h = h0 + i;
      store16(out + (int64_t)h * kD, row_gradient(gq[i], xq[i], qs, c, s, A.gain, dqs));
      store16(out + (int64_t)(A.heads + h) * kD, row_gradient(gk[i], xk[i], ks, c, s, 1.0f, dks));
      store16(out + (int64_t)(2 * A.heads + h) * kD, gv[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    sums[slot][lane * 8 + i] = dqs[i];
    sums[slot][kD + lane * 8 + i] = dks[i];
  }
  __syncthreads();
  for (int col = threadIdx.x; col < 2 * kD; col += kThreads) {
    float sum = sums[0][col];
#pragma unroll
    for (int i = 1; i < kTokens; ++i) sum += sums[i][col];
    A.partial[(int64_t)blockIdx.x * 2 * kD + col] = sum;
  }
}

// Adds the partial rows in a fixed order: 16 columns a block, 64 rows at a time, then those 64 sums in order.
constexpr int kJoinThreads = 1024;
template <typename P>
__global__ __launch_bounds__(kJoinThreads) void qk_scales_kernel(const float* __restrict__ partial, int rows, P* dq_scale,
                                                                 P* dk_scale) {
  __shared__ float part[kJoinThreads / 16][17];
  const int col = blockIdx.x * 16 + (threadIdx.x & 15), first = threadIdx.x >> 4;
  float sum = 0.0f;
#pragma unroll 8
  for (int r = first; r < rows; r += kJoinThreads / 16) sum += partial[(int64_t)r * 2 * kD + col];
  part[first][threadIdx.x & 15] = sum;
  __syncthreads();
  if (first) return;
#pragma unroll 8
  for (int i = 1; i < kJoinThreads / 16; ++i) sum += part[i][threadIdx.x];
  (col < kD ? dq_scale : dk_scale)[col % kD] = (P)sum;
}

int heads_of(int heads) { return heads % 2 == 0 ? 2 : 1; }   // heads a 16-lane group takes at a time

constexpr int kMaxBlocks = 256 * 4;
int64_t items_of(int batch, int length, int heads) {
  return ((int64_t)length + kTokens - 1) / kTokens * (heads / heads_of(heads)) * batch;
}
int blocks_of(int64_t items) { return (int)std::min<int64_t>(items, kMaxBlocks); }

bool sizes_ok(int batch, int length, int heads) {
  if (batch < 0 || length < 0 || heads <= 0 || length > INT32_MAX - 256 || heads > 1 << 20) return false;
  const int64_t of_one = items_of(1, length, heads);
  return batch == 0 || of_one <= (INT32_MAX - kMaxBlocks) / batch;
}

int check_grad(const void* p, const int64_t* strides) {
  if (!p || !strides) return FLK_E_INVALID;
  if (!flk_host_aligned(p, 16) || strides[0] % 8 || strides[1] % 8 || strides[2] % 8) return FLK_E_ALIGN;
  return FLK_OK;
}
Grad grad(const void* p, const int64_t* s) { return Grad{static_cast<const uint16_t*>(p), s[0], s[1], s[2]}; }

template <bool kScaleF32, int kHeads>
void launch(const Args& a, int blocks, hipStream_t s) {
  qk_prep_backward_kernel<kScaleF32, kHeads><<<blocks, kThreads, 0, s>>>(a);
}

}  // namespace

extern "C" int flk_qk_prep_backward_plan(int batch, int length, int num_heads, int64_t* workspace_bytes) {
  if (!workspace_bytes || !sizes_ok(batch, length, num_heads)) return FLK_E_INVALID;
  *workspace_bytes = (int64_t)blocks_of(items_of(batch, length, num_heads)) * 2 * kD * 4;
  return FLK_OK;
}

extern "C" int flk_qk_prep_backward(const void* dq, const int64_t* dq_strides, const void* dk, const int64_t* dk_strides,
                                    const void* dv, const int64_t* dv_strides, const void* qkv, int64_t qkv_batch_stride,
                                    int64_t qkv_row_stride, const float* cos, const float* sin, int64_t table_row_stride,
                                    const void* q_scale, const void* k_scale, int scale_is_f32, float q_gain, int batch,
                                    int length, int num_heads, int head_dim, void* dqkv, int64_t dqkv_batch_stride,
                                    int64_t dqkv_row_stride, void* dq_scale, void* dk_scale, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  if (head_dim != kD) return FLK_E_UNSUPPORTED;
  if (!sizes_ok(batch, length, num_heads)) return FLK_E_INVALID;
  if (batch == 0 || length == 0) return FLK_OK;   // the sums over no rows are the caller's to clear
  if (const int st = check_grad(dq, dq_strides)) return st;
  if (const int st = check_grad(dk, dk_strides)) return st;
  if (const int st = check_grad(dv, dv_strides)) return st;
  if (!qkv || !cos || !sin || !q_scale || !k_scale || !dqkv || !dq_scale || !dk_scale) return FLK_E_INVALID;
  if (table_row_stride < kD) return FLK_E_INVALID;
  for (const void* p : {qkv, static_cast<const void*>(cos), static_cast<const void*>(sin), q_scale, k_scale,
                        static_cast<const void*>(dqkv)})
    if (!flk_host_aligned(p, 16)) return FLK_E_ALIGN;
  if (qkv_batch_stride % 8 || qkv_row_stride % 8 || dqkv_batch_stride % 8 || dqkv_row_stride % 8 || table_row_stride % 4)
    return FLK_E_ALIGN;
  if (!flk_host_aligned(dq_scale, scale_is_f32 ? 4 : 2) || !flk_host_aligned(dk_scale, scale_is_f32 ? 4 : 2))
    return FLK_E_ALIGN;
  Args a{};
  a.dq = grad(dq, dq_strides);
  a.dk = grad(dk, dk_strides);
  a.dv = grad(dv, dv_strides);
  a.qkv = static_cast<const uint16_t*>(qkv);
  a.qkv_batch = qkv_batch_stride;
  a.qkv_row = qkv_row_stride;
  a.cos = cos;
  a.sin = sin;
  a.table_row = table_row_stride;
  a.q_scale = q_scale;
  a.k_scale = k_scale;
  a.gain = q_gain;
  a.length = length;
  a.heads = num_heads;
  a.token_blocks = (length + kTokens - 1) / kTokens;
  a.items = (int)items_of(batch, length, num_heads);
  a.out = static_cast<uint16_t*>(dqkv);
  a.out_batch = dqkv_batch_stride;
  a.out_row = dqkv_row_stride;
  a.partial = static_cast<float*>(workspace);
  const int blocks = blocks_of(a.items);
  if (!workspace || workspace_bytes < (int64_t)blocks * 2 * kD * 4) return FLK_E_SCRATCH;
  if (!flk_host_aligned(workspace, 16)) return FLK_E_ALIGN;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (heads_of(num_heads) == 2) scale_is_f32 ? launch<true, 2>(a, blocks, s) : launch<false, 2>(a, blocks, s);
  else scale_is_f32 ? launch<true, 1>(a, blocks, s) : launch<false, 1>(a, blocks, s);
  if (const int st = flk_launch_status()) return st;
  if (scale_is_f32)
    qk_scales_kernel<float><<<2 * kD / 16, kJoinThreads, 0, s>>>(a.partial, blocks, static_cast<float*>(dq_scale),
                                                                 static_cast<float*>(dk_scale));
  else
    qk_scales_kernel<__bf16><<<2 * kD / 16, kJoinThreads, 0, s>>>(a.partial, blocks, static_cast<__bf16*>(dq_scale),
                                                                  static_cast<__bf16*>(dk_scale));
  return flk_launch_status();
}

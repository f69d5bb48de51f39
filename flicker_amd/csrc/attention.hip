// attention: softmax(q k^T) v of any lengths, with the keys that a mask keeps, and its gradients.
//
// Per (b, h) and query i, over the kept keys j of key head h / (heads / kv_heads); q comes scaled:
//   S_ij = q_i . k_j,  lse_i = log sum_j exp S_ij,  P_ij = exp(S_ij - lse_i),  o_i = sum_j P_ij v_j
// and backwards, for the gradient g_i of o_i,
//   delta_i = g_i . o_i,  dP_ij = g_i . v_j,  dS_ij = P_ij (dP_ij - delta_i)
//   dq_i = sum_j dS_ij k_j,  dk_j = sum_i dS_ij q_i,  dv_j = sum_i P_ij g_i
// (dk and dv also over the query heads that share the key head).  A query that keeps no key has o = 0, lse = -inf and
// no gradient.

#include <algorithm>

#include "common.h"

namespace {

constexpr int kD = 128;
constexpr int kRowBytes = kD * 2;
constexpr int kTile = 64;              // rows of a staged tile, keys of a mask word
constexpr int kUnit = 32;              // rows of a unit: the contraction length of one MFMA
constexpr int kUnitBytes = kUnit * kRowBytes;
constexpr int kTileBytes = kTile * kRowBytes;
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kBlock = 32 * kWaves;    // queries (or keys) of a block, 32 a wave
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int64_t kMaxItems = 1LL << 31;

using flk::f32x4;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Vec;
template <>
struct Vec<__bf16> {
  typedef flk::bf16x2 two;
  typedef flk::bf16x8 eight;
};
template <>
struct Vec<_Float16> {
  typedef f16x2 two;
  typedef f16x8 eight;
};
template <typename T>
using vec8 = typename Vec<T>::eight;

__device__ __forceinline__ f32x4 mfma(const flk::bf16x8& a, const flk::bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(const f16x8& a, const f16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const typename Vec<T>::two p = {(T)lo, (T)hi};
  return __builtin_bit_cast(uint32_t, p);
}

struct Tensor {   // element d of row t of head h of batch entry b at p + b * batch + h * head + t * row + d
  void* p;
  int64_t batch, head, row;
  template <typename T>
  __device__ __forceinline__ T* at(int b, int h) const {
    return static_cast<T*>(p) + b * batch + h * head;
  }
};

// What the mask's bytes come to: of batch entry b the words words[b * tiles + t], bit i of word t set where key 64 t + i
// is kept, the tiles live[b * tiles + n], n < counts[b], whose words are not zero, in order.  NULL words: all are kept.
struct Mask {
  const uint64_t* words;
  const int* live;
  const int* counts;
};

struct Args {
  Tensor q, k, v, o, dO, dq, dk, dv;
  void* low;        // (batch, queries, heads, 128): what o's rounding left, in the same type
  float* lse;       // (batch, heads, queries)
  float* stats;     // (batch, heads, units, 2, 32): a unit's log2(e) lse and -delta; rows past the end inf and 0
  Mask mask;
  int batch, heads, kv_heads, group, queries, keys, tiles, units;
};

// Which bits of tile t are kept.
__device__ __forceinline__ uint64_t kept(const Args& A, int b, int t) {
  if (A.mask.words) return A.mask.words[(int64_t)b * A.tiles + t];
  const int left = A.keys - t * kTile;
  return left >= 64 ? ~0ull : (1ull << left) - 1;
}
__device__ __forceinline__ int live_tiles(const Args& A, int b) { return A.mask.words ? A.mask.counts[b] : A.tiles; }
__device__ __forceinline__ int live_tile(const Args& A, int b, int n) {
  return A.mask.words ? A.mask.live[(int64_t)b * A.tiles + n] : n;
}

__device__ __forceinline__ int swz(int row) { return ((row & 7) << 1) | ((row >> 3) & 1); }

// Operands of a staged tile, whose 16-byte chunk c of row r sits in place c ^ swz(r).
struct Places {
  int row[4];   // 16 rows x 32 d as they are: row lane % 16, d step st
  int col[8];   // 16 d x 32 rows transposed: d tile dt
};
__device__ __forceinline__ Places places() {
  Places at;
  const int lane = threadIdx.x & 63, h = lane >> 4, col = lane & 15;
  const int hperm = ((h & 1) << 1) | (h >> 1);
#pragma unroll
  for (int st = 0; st < 4; ++st) at.row[st] = col * kRowBytes + ((((st << 2) | hperm) ^ swz(col)) << 4);
  const int r = h * 4 + (col >> 2);
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) at.col[dt] = r * kRowBytes + (((2 * dt + ((col & 3) >> 1)) ^ swz(r)) << 4) + (col & 1) * 8;
  return at;
}
template <typename T>
__device__ __forceinline__ vec8<T> row_operand(const uint8_t* unit, const Places& at, int st, int kt) {
  return *reinterpret_cast<const vec8<T>*>(unit + at.row[st] + kt * 16 * kRowBytes);
}
template <typename T>
__device__ __forceinline__ vec8<T> col_operand(const uint8_t* unit, const Places& at, int dt) {
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(unit + at.col[dt]));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(unit + at.col[dt] + 16 * kRowBytes));
  return __builtin_bit_cast(vec8<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Stages 64 rows from `first`, those that `bits` leaves out as zeros.
__device__ __forceinline__ void stage(uint8_t* dst, const uint16_t* src, int64_t stride, int first, uint64_t bits) {
  for (int i = threadIdx.x; i < kTile * 16; i += kThreads) {
    const int r = i >> 4, c = i & 15;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (bits >> r & 1) x = *reinterpret_cast<const uint4*>(src + (int64_t)(first + r) * stride + c * 8);
    *reinterpret_cast<uint4*>(dst + r * kRowBytes + ((c ^ swz(r)) << 4)) = x;
  }
}

// The wave's two groups of 16 rows from row0 as the right operand: row lane % 16 of group g, d step st; zeros past `end`.
template <typename T>
__device__ __forceinline__ void load_rows(vec8<T> (&x)[4][2], const T* src, int64_t stride, int row0, int end) {
  const int lane = threadIdx.x & 63, h = lane >> 4, hperm = ((h & 1) << 1) | (h >> 1);
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int r = row0 + g * 16 + (lane & 15);
#pragma unroll
    for (int st = 0; st < 4; ++st)
      x[st][g] = r < end ? *reinterpret_cast<const vec8<T>*>(src + (int64_t)r * stride + st * 32 + hperm * 8) : vec8<T>{};
  }
}

// acc (d tile, group) of the wave's rows, times scale[g], as rows of 128: 4 d values a store.
template <typename T>
__device__ __forceinline__ void store_rows(const f32x4 (&acc)[8][2], const float (&scale)[2], T* dst, int64_t stride,
                                           int row0, int end, T* low = nullptr, int64_t low_stride = 0) {
  const int lane = threadIdx.x & 63, h = lane >> 4;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int r = row0 + g * 16 + (lane & 15);
    if (r >= end) continue;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = acc[dt][g][i] * scale[g];
      uint2 w = make_uint2(pack<T>(x[0], x[1]), pack<T>(x[2], x[3]));
      *reinterpret_cast<uint2*>(dst + (int64_t)r * stride + dt * 16 + h * 4) = w;
      if (low) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] -= (float)(T)x[i];
        w = make_uint2(pack<T>(x[0], x[1]), pack<T>(x[2], x[3]));
        *reinterpret_cast<uint2*>(low + (int64_t)r * low_stride + dt * 16 + h * 4) = w;
      }
    }
  }
}

__device__ __forceinline__ float across(float x) {   // the four lane groups' sum
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void attention_kernel(const Args A) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * kTileBytes];
  const int lane = threadIdx.x & 63, h4 = lane >> 4;
  const int blocks = (A.queries + kBlock - 1) / kBlock;
  const int bh = blockIdx.x / blocks, b = bh / A.heads, h = bh - b * A.heads;
  const int q0 = (blockIdx.x - bh * blocks) * kBlock + (threadIdx.x >> 6) * 32;
  vec8<T> q[4][2];
  load_rows<T>(q, A.q.at<T>(b, h), A.q.row, q0, A.queries);
  const Places at = places();
  f32x4 acc[8][2] = {};
  float m[2] = {-1e30f, -1e30f}, l[2] = {}, l_exact[2] = {};   // sums of the rounded and of the unrounded P
  const int n = live_tiles(A, b);
  for (int i = 0; i < n; ++i) {
    const int t = live_tile(A, b, i);
    const uint64_t bits = kept(A, b, t);
    __syncthreads();
    stage(smem, A.k.at<uint16_t>(b, h / A.group), A.k.row, t * kTile, bits);
    stage(smem + kTileBytes, A.v.at<uint16_t>(b, h / A.group), A.v.row, t * kTile, bits);
    __syncthreads();
    for (int u = 0; u < 2; ++u) {
      f32x4 s[2][2] = {};
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          const vec8<T> a = row_operand<T>(smem + u * kUnitBytes, at, st, kt);
#pragma unroll
          for (int g = 0; g < 2; ++g) s[g][kt] = mfma(a, q[st][g], s[g][kt]);
        }
      uint32_t p[2][4];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float top = m[g];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool on = bits >> (u * 32 + (e >> 2) * 16 + h4 * 4 + (e & 3)) & 1;
          s[g][e >> 2][e & 3] = on ? s[g][e >> 2][e & 3] * kLog2e : -INFINITY;
          top = fmaxf(top, s[g][e >> 2][e & 3]);
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float f = __builtin_amdgcn_exp2f(m[g] - top);
        m[g] = top;
        l[g] *= f;
        l_exact[g] *= f;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) acc[dt][g] *= f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x0 = __builtin_amdgcn_exp2f(s[g][e >> 1][(e & 1) * 2] - top);
          const float x1 = __builtin_amdgcn_exp2f(s[g][e >> 1][(e & 1) * 2 + 1] - top);
          l[g] += (float)(T)x0 + (float)(T)x1;
          l_exact[g] += x0 + x1;
          p[g][e] = pack<T>(x0, x1);
        }
      }
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        const vec8<T> a = col_operand<T>(smem + kTileBytes + u * kUnitBytes, at, dt);
#pragma unroll
        for (int g = 0; g < 2; ++g)
          acc[dt][g] = mfma(a, __builtin_bit_cast(vec8<T>, make_uint4(p[g][0], p[g][1], p[g][2], p[g][3])), acc[dt][g]);
      }
    }
  }
  float scale[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const float sum = across(l[g]), exact = across(l_exact[g]);
    scale[g] = sum > 0.0f ? 1.0f / sum : 0.0f;
    const int r = q0 + g * 16 + (lane & 15);
    if (A.lse && h4 == 0 && r < A.queries)
      A.lse[(int64_t)bh * A.queries + r] = sum > 0.0f ? (m[g] + __builtin_amdgcn_logf(exact)) * kLn2 : -INFINITY;
  }
  T* low = static_cast<T*>(A.low);
  if (low) low += ((int64_t)b * A.queries * A.heads + h) * kD;
  store_rows<T>(acc, scale, A.o.at<T>(b, h), A.o.row, q0, A.queries, low, (int64_t)A.heads * kD);
}

// dq, and the stats that attention_dkv_kernel reads.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_dq_kernel(const Args A) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * kTileBytes];
  const int lane = threadIdx.x & 63, h4 = lane >> 4;
  const int blocks = (A.queries + kBlock - 1) / kBlock;
  const int bh = blockIdx.x / blocks, b = bh / A.heads, h = bh - b * A.heads;
  const int q0 = (blockIdx.x - bh * blocks) * kBlock + (threadIdx.x >> 6) * 32;
  vec8<T> q[4][2], g0[4][2], o[4][2], low[4][2];
  load_rows<T>(q, A.q.at<T>(b, h), A.q.row, q0, A.queries);
  load_rows<T>(g0, A.dO.at<T>(b, h), A.dO.row, q0, A.queries);
  load_rows<T>(o, A.o.at<T>(b, h), A.o.row, q0, A.queries);
  load_rows<T>(low, static_cast<const T*>(A.low) + ((int64_t)b * A.queries * A.heads + h) * kD, (int64_t)A.heads * kD, q0,
               A.queries);
  float lse[2], delta[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int r = q0 + g * 16 + (lane & 15);
    const float x = r < A.queries ? A.lse[(int64_t)bh * A.queries + r] : -INFINITY;
    lse[g] = x == -INFINITY ? INFINITY : x * kLog2e;
    float sum = 0.0f;
#pragma unroll
    for (int st = 0; st < 4; ++st)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += (float)g0[st][g][e] * ((float)o[st][g][e] + (float)low[st][g][e]);
    delta[g] = x == -INFINITY ? 0.0f : across(sum);
    if (h4 == 0 && r < A.units * kUnit) {
      float* st = A.stats + ((int64_t)bh * A.units + r / kUnit) * 2 * kUnit + r % kUnit;
      st[0] = lse[g];
      st[kUnit] = -delta[g];
    }
  }
  const Places at = places();
  f32x4 acc[8][2] = {};
  const int n = live_tiles(A, b);
  for (int i = 0; i < n; ++i) {
    const int t = live_tile(A, b, i);
    const uint64_t bits = kept(A, b, t);
    __syncthreads();
    stage(smem, A.k.at<uint16_t>(b, h / A.group), A.k.row, t * kTile, bits);
    stage(smem + kTileBytes, A.v.at<uint16_t>(b, h / A.group), A.v.row, t * kTile, bits);
    __syncthreads();
    for (int u = 0; u < 2; ++u) {
      f32x4 s[2][2] = {}, dp[2][2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int g = 0; g < 2; ++g) dp[g][kt] = f32x4{-delta[g], -delta[g], -delta[g], -delta[g]};
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          const vec8<T> a = row_operand<T>(smem + u * kUnitBytes, at, st, kt);
          const vec8<T> c = row_operand<T>(smem + kTileBytes + u * kUnitBytes, at, st, kt);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            s[g][kt] = mfma(a, q[st][g], s[g][kt]);
            dp[g][kt] = mfma(c, g0[st][g], dp[g][kt]);
          }
        }
      }
      uint32_t ds[2][4];
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          float x[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const bool on = bits >> (u * 32 + (e >> 2) * 16 + h4 * 4 + (e & 3) + j) & 1;
            x[j] = on ? __builtin_amdgcn_exp2f(s[g][e >> 2][(e & 3) + j] * kLog2e - lse[g]) * dp[g][e >> 2][(e & 3) + j]
                      : 0.0f;
          }
          ds[g][e >> 1] = pack<T>(x[0], x[1]);
        }
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        const vec8<T> a = col_operand<T>(smem + u * kUnitBytes, at, dt);
#pragma unroll
        for (int g = 0; g < 2; ++g)
          acc[dt][g] = mfma(a, __builtin_bit_cast(vec8<T>, make_uint4(ds[g][0], ds[g][1], ds[g][2], ds[g][3])), acc[dt][g]);
      }
    }
  }
  const float one[2] = {1.0f, 1.0f};
  store_rows<T>(acc, one, A.dq.at<T>(b, h), A.dq.row, q0, A.queries);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void attention_dkv_kernel(const Args A) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * kTileBytes];
  const int lane = threadIdx.x & 63, h4 = lane >> 4;
  const int blocks = (A.keys + kBlock - 1) / kBlock;
  const int bh = blockIdx.x / blocks, b = bh / A.kv_heads, h = bh - b * A.kv_heads;
  const int first = (blockIdx.x - bh * blocks) * kBlock, k0 = first + (threadIdx.x >> 6) * 32;
  vec8<T> k[4][2], v[4][2];
  load_rows<T>(k, A.k.at<T>(b, h), A.k.row, k0, A.keys);
  load_rows<T>(v, A.v.at<T>(b, h), A.v.row, k0, A.keys);
  bool on[2];
  float one[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int r = k0 + g * 16 + (lane & 15);
    on[g] = r < A.keys && (kept(A, b, r / kTile) >> (r % kTile) & 1);
    one[g] = 1.0f;
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      k[st][g] = on[g] ? k[st][g] : vec8<T>{};
      v[st][g] = on[g] ? v[st][g] : vec8<T>{};
    }
  }
  const Places at = places();
  f32x4 dk[8][2] = {}, dv[8][2] = {};
  bool any = false;
  for (int t = first / kTile; t < min(A.tiles, (first + kBlock) / kTile); ++t) any |= kept(A, b, t) != 0;
  const int tiles = (A.queries + kTile - 1) / kTile, n = any ? tiles * A.group : 0;
  for (int i = 0; i < n; ++i) {
    const int hq = h * A.group + i / tiles, t = i % tiles;
    const int left = A.queries - t * kTile;
    const uint64_t bits = left >= 64 ? ~0ull : (1ull << left) - 1;
    __syncthreads();
    stage(smem, A.q.at<uint16_t>(b, hq), A.q.row, t * kTile, bits);
    stage(smem + kTileBytes, A.dO.at<uint16_t>(b, hq), A.dO.row, t * kTile, bits);
    __syncthreads();
    for (int u = 0; u < 2 && t * 2 + u < A.units; ++u) {
      const float* stats = A.stats + (((int64_t)b * A.heads + hq) * A.units + t * 2 + u) * 2 * kUnit;
      f32x4 s[2][2] = {}, dp[2][2], lse[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        lse[kt] = *reinterpret_cast<const f32x4*>(stats + kt * 16 + h4 * 4);
#pragma unroll
        for (int g = 0; g < 2; ++g) dp[g][kt] = *reinterpret_cast<const f32x4*>(stats + kUnit + kt * 16 + h4 * 4);
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          const vec8<T> a = row_operand<T>(smem + u * kUnitBytes, at, st, kt);
          const vec8<T> c = row_operand<T>(smem + kTileBytes + u * kUnitBytes, at, st, kt);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            s[g][kt] = mfma(a, k[st][g], s[g][kt]);
            dp[g][kt] = mfma(c, v[st][g], dp[g][kt]);
          }
        }
      }
      uint32_t p[2][4], ds[2][4];
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          float x[2], y[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            x[j] = __builtin_amdgcn_exp2f(s[g][e >> 2][(e & 3) + j] * kLog2e - lse[e >> 2][(e & 3) + j]);
            y[j] = x[j] * dp[g][e >> 2][(e & 3) + j];
          }
          p[g][e >> 1] = pack<T>(x[0], x[1]);
          ds[g][e >> 1] = pack<T>(y[0], y[1]);
        }
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        const vec8<T> a = col_operand<T>(smem + kTileBytes + u * kUnitBytes, at, dt);
        const vec8<T> c = col_operand<T>(smem + u * kUnitBytes, at, dt);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          dv[dt][g] = mfma(a, __builtin_bit_cast(vec8<T>, make_uint4(p[g][0], p[g][1], p[g][2], p[g][3])), dv[dt][g]);
          dk[dt][g] = mfma(c, __builtin_bit_cast(vec8<T>, make_uint4(ds[g][0], ds[g][1], ds[g][2], ds[g][3])), dk[dt][g]);
        }
      }
    }
  }
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      dk[dt][g] = on[g] ? dk[dt][g] : f32x4{};
      dv[dt][g] = on[g] ? dv[dt][g] : f32x4{};
    }
  store_rows<T>(dk, one, A.dk.at<T>(b, h), A.dk.row, k0, A.keys);
  store_rows<T>(dv, one, A.dv.at<T>(b, h), A.dv.row, k0, A.keys);
}

// The mask's words and live tiles of one batch entry a block; a thread a tile, 1024 tiles a turn.
constexpr int kPlanWaves = 16;
__global__ __launch_bounds__(64 * kPlanWaves) void attention_mask_kernel(const uint8_t* mask, int64_t batch_stride, int keys,
                                                                         int tiles, uint64_t* words, int* live, int* counts) {
  __shared__ int found[kPlanWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint8_t* row = mask + blockIdx.x * batch_stride;
  words += (int64_t)blockIdx.x * tiles;
  live += (int64_t)blockIdx.x * tiles;
  int count = 0;
  for (int t0 = 0; t0 < tiles; t0 += 64 * kPlanWaves) {
    uint64_t mine = 0;   // of tile t0 + threadIdx.x
#pragma unroll 8
    for (int i = 0; i < 64; ++i) {
      const int key = (t0 + wave * 64 + i) * kTile + lane;   // at most keys + 65535
      const uint64_t bits = __ballot(key < keys && row[key] != 0);
      mine = lane == i ? bits : mine;
    }
    const int t = t0 + threadIdx.x;
    const uint64_t any = __ballot(mine != 0);
    if (t < tiles) words[t] = mine;
    if (lane == 0) found[wave] = __popcll(any);
    __syncthreads();
    int at = count;
    for (int w = 0; w < kPlanWaves; ++w) {
      if (w < wave) at += found[w];
      count += found[w];
    }
    if (mine) live[at + __popcll(any & ((1ull << lane) - 1))] = t;
    __syncthreads();
  }
  if (threadIdx.x == 0) counts[blockIdx.x] = count;
}

int64_t mask_bytes(int batch, int keys) {
  const int64_t tiles = (keys + kTile - 1) / kTile;
  return (batch * (tiles * 12 + 4) + 255) / 256 * 256;
}
int64_t stats_bytes(int batch, int heads, int queries) {
  return (int64_t)batch * heads * ((queries + kUnit - 1) / kUnit) * 2 * kUnit * 4;
}

// Lays the mask's words and lists out in `workspace` and starts the kernel that fills them.
int plan_mask(const void* mask, int64_t batch_stride, Args& A, uint8_t* workspace, hipStream_t s) {
  if (!mask) return FLK_OK;
  uint64_t* words = reinterpret_cast<uint64_t*>(workspace);
  int* live = reinterpret_cast<int*>(words + (int64_t)A.batch * A.tiles);
  int* counts = live + (int64_t)A.batch * A.tiles;
  A.mask = Mask{words, live, counts};
  attention_mask_kernel<<<A.batch, 64 * kPlanWaves, 0, s>>>(static_cast<const uint8_t*>(mask), batch_stride, A.keys, A.tiles,
                                                            words, live, counts);
  return flk_launch_status();
}

bool sizes_ok(int batch, int heads, int kv_heads, int queries, int keys) {
  if (batch < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || queries < 0 || keys < 0) return false;
  if (queries > 1 << 28 || keys > 1 << 28 || batch > 1 << 20) return false;
  const int64_t rows = (int64_t)batch * heads, kv = (int64_t)batch * kv_heads;
  return rows * ((queries + 31) / 32) <= kMaxItems / 512 && kv * ((keys + 31) / 32) <= kMaxItems / 512;
}

int check_tensor(const void* p, const int64_t* strides) {
  if (!p || !strides) return FLK_E_INVALID;
  if (!flk_host_aligned(p, 16) || strides[0] % 8 || strides[1] % 8 || strides[2] % 8) return FLK_E_ALIGN;
  return FLK_OK;
}
Tensor tensor(const void* p, const int64_t* s) { return Tensor{const_cast<void*>(p), s[0], s[1], s[2]}; }

Args sizes(int batch, int heads, int kv_heads, int queries, int keys) {
  Args A{};
  A.batch = batch;
  A.heads = heads;
  A.kv_heads = kv_heads;
  A.group = heads / kv_heads;
  A.queries = queries;
  A.keys = keys;
  A.tiles = (keys + kTile - 1) / kTile;
  A.units = (queries + kUnit - 1) / kUnit;
  return A;
}

}  // namespace

extern "C" int flk_attention_plan(int batch, int heads, int kv_heads, int queries, int keys, int masked, int backward,
                                  int64_t* workspace_bytes) {
  if (!workspace_bytes || !sizes_ok(batch, heads, kv_heads, queries, keys)) return FLK_E_INVALID;
  *workspace_bytes = (masked ? mask_bytes(batch, keys) : 0) + (backward ? stats_bytes(batch, heads, queries) : 0);
  return FLK_OK;
}

extern "C" int flk_attention(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                             const void* v, const int64_t* v_strides, int dtype, const void* key_mask,
                             int64_t mask_batch_stride, int batch, int heads, int kv_heads, int queries, int keys,
                             int head_dim, void* o, const int64_t* o_strides, void* low, float* lse, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  if (dtype != FLK_BF16 && dtype != FLK_F16) return FLK_E_INVALID;
  if (head_dim != kD) return FLK_E_UNSUPPORTED;
  if (!sizes_ok(batch, heads, kv_heads, queries, keys)) return FLK_E_INVALID;
  if (batch == 0 || queries == 0) return FLK_OK;
  if (const int st = check_tensor(q, q_strides)) return st;
  if (const int st = check_tensor(o, o_strides)) return st;
  Args A = sizes(batch, heads, kv_heads, queries, keys);
  if (keys) {
    if (const int st = check_tensor(k, k_strides)) return st;
    if (const int st = check_tensor(v, v_strides)) return st;
    A.k = tensor(k, k_strides);
    A.v = tensor(v, v_strides);
  }
  if (!flk_host_aligned(low, 16) || !flk_host_aligned(lse, 4)) return FLK_E_ALIGN;
  const int64_t need = key_mask ? mask_bytes(batch, keys) : 0;
  if (need && (!workspace || workspace_bytes < need)) return FLK_E_SCRATCH;
  if (!flk_host_aligned(workspace, 256)) return FLK_E_ALIGN;
  A.q = tensor(q, q_strides);
  A.o = tensor(o, o_strides);
  A.low = low;
  A.lse = lse;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (const int st = plan_mask(key_mask, mask_batch_stride, A, static_cast<uint8_t*>(workspace), s)) return st;
  const dim3 grid((unsigned)((int64_t)batch * heads * ((queries + kBlock - 1) / kBlock)));
  if (dtype == FLK_BF16) attention_kernel<__bf16><<<grid, kThreads, 0, s>>>(A);
  else attention_kernel<_Float16><<<grid, kThreads, 0, s>>>(A);
  return flk_launch_status();
}

extern "C" int flk_attention_backward(const void* d_o, const int64_t* d_o_strides, const void* q, const int64_t* q_strides,
                                      const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                      const void* o, const int64_t* o_strides, const void* low, const float* lse, int dtype,
                                      const void* key_mask, int64_t mask_batch_stride, int batch, int heads, int kv_heads,
                                      int queries, int keys, int head_dim, void* dq, const int64_t* dq_strides, void* dk,
                                      const int64_t* dk_strides, void* dv, const int64_t* dv_strides, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  if (dtype != FLK_BF16 && dtype != FLK_F16) return FLK_E_INVALID;
  if (head_dim != kD) return FLK_E_UNSUPPORTED;
  if (!sizes_ok(batch, heads, kv_heads, queries, keys)) return FLK_E_INVALID;
  if (batch == 0 || queries == 0 || keys == 0) return FLK_OK;   // gradients over nothing are the caller's to clear
  const struct {
    const void* p;
    const int64_t* strides;
  } all[] = {{d_o, d_o_strides}, {q, q_strides}, {k, k_strides}, {v, v_strides},
             {o, o_strides},     {dq, dq_strides}, {dk, dk_strides}, {dv, dv_strides}};
  for (const auto& t : all)
    if (const int st = check_tensor(t.p, t.strides)) return st;
  if (!low || !lse) return FLK_E_INVALID;
  if (!flk_host_aligned(low, 16) || !flk_host_aligned(lse, 4)) return FLK_E_ALIGN;
  const int64_t of_mask = key_mask ? mask_bytes(batch, keys) : 0;
  if (!workspace || workspace_bytes < of_mask + stats_bytes(batch, heads, queries)) return FLK_E_SCRATCH;
  if (!flk_host_aligned(workspace, 256)) return FLK_E_ALIGN;
  Args A = sizes(batch, heads, kv_heads, queries, keys);
  A.dO = tensor(d_o, d_o_strides);
  A.q = tensor(q, q_strides);
  A.k = tensor(k, k_strides);
  A.v = tensor(v, v_strides);
  A.o = tensor(o, o_strides);
  A.dq = tensor(dq, dq_strides);
  A.dk = tensor(dk, dk_strides);
  A.dv = tensor(dv, dv_strides);
  A.low = const_cast<void*>(low);
  A.lse = const_cast<float*>(lse);
  A.stats = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + of_mask);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (const int st = plan_mask(key_mask, mask_batch_stride, A, static_cast<uint8_t*>(workspace), s)) return st;
  const dim3 of_q((unsigned)((int64_t)batch * heads * ((queries + kBlock - 1) / kBlock)));
  const dim3 of_k((unsigned)((int64_t)batch * kv_heads * ((keys + kBlock - 1) / kBlock)));
  if (dtype == FLK_BF16) {
    attention_dq_kernel<__bf16><<<of_q, kThreads, 0, s>>>(A);
    attention_dkv_kernel<__bf16><<<of_k, kThreads, 0, s>>>(A);
  } else {
    attention_dq_kernel<_Float16><<<of_q, kThreads, 0, s>>>(A);
    attention_dkv_kernel<_Float16><<<of_k, kThreads, 0, s>>>(A);
  }
  return flk_launch_status();
}

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
// The residual form (modules.py:157-167, between a block's two halves) takes x + gate * branch for x, with a gate row like
// the factor's; it stores that sum as r beside y.  Backward, with the gradient dr of r that comes in beside dy,
// everything of the sum's gradient d = dr + dx is known row by row: dx = d, dbranch = gate d, dgate = sum of d branch.  The sum
// is recomputed in float32 from x and branch, which have to be read anyway for dgate, rather than from the rounded r.
//
// All arithmetic is float32 and every output is rounded once.  Sums of squares of an uncentred residual
// stream, whose tokens sit off zero, would cancel, so each wave centres its part of the row on its own
// mean, and the waves' (mean, centred squares) are joined by the parallel form of the variance:
//   m = sum_w k_w m_w / K,   K v = sum_w s_w + k_w (m_w - m)^2
// and likewise sum t (x - m) = sum_w [sum t (x - m_w) + (m_w - m) sum t]: one exchange through LDS and
// one barrier a row, forwards and backwards.
//
// HBM bounds both directions: a row is read once and held in registers, one 8-element chunk a lane
// (two past 8192 columns, where the backward pass spills 14 registers, 28 with float32 rows), so a lane owns
// few columns and a CU has many rows in flight.  The backward pass recomputes m and q from the row it has to read anyway, so the forward pass
// keeps nothing.  Its column sums stay in the lanes that own the columns while a block walks its
// rows; blocks write them as partial rows, which a second kernel adds in a fixed order: the
// gradients do not depend on timing.
//
// 16-bit y and dx are stored past the caches: 4608 rows forward 13.3 -> 11.0 us, and no slower a product that reads y
// next (float32: see kStreamBytes).  Past 50 MB an elementwise reader finds less of it: 9216 rows 22.0 us alone (through
// the caches 25.0), 47.5 with such a reader (42.4); 4608 rows 22.1 (22.4).  The rows read are not (13.3 -> 16.7: the last
// cache often has them), nor the partial rows, read again at once.
//
// The residual form of 16-bit rows reads past the caches and stores through them: both outputs are read next, and they
// stay in the last cache where the operands would have pushed them out.  us alone, and with what adds the two outputs up
// behind it (as the norm alone does it; both past the caches): 4608 rows 25.0 and 37.7 (25.1, 42.0; 24.3, 41.5), their
// gradients 44.5 and 57.4 (45.7, 64.7; 45.3, 60.4), 4 x 4096 rows 83.5 and 126 (81.6, 137; 80.0, 133).  Rows off 16 bytes
// share words between lanes, which are then fetched twice: 3 x 1157 x 1111 float32 gradients 28.7 us, past the caches 34.
//
// Measured (bf16, width 3 * 1024, among other passes): forward 4 x 4096 rows in 41.7 us, 4.8 TB/s (a large copy's
// rate is 5.2), backward 4608 rows in 24.9 us (85 MB of operands, and 13 MB of partial rows written and read); 512
// rows in 4.1 and 11 us: a launch and three latencies one after the other, the factor's, the offset's and the first
// row's.  Widths past 8192, 1000 x 16384: 12.6 us forward, 39 backward (2.5 TB/s), float32 27 and 77.  What it took, at 4 x 4096 rows: a wave a
// row held 48 columns a lane and waited for its reductions with 2 waves a SIMD (65 us forward, 176
// backward); several waves a row that each add up the others' values from LDS, one after the other, spend 1800
// cycles a row on that (53, 94), where sixteen lanes take one wave's values each and add them by DPP (46, 69).
// Fetching more than two rows ahead gains nothing as the loop is: its fetches are conditional, and once a turn it waits
// for all that is outstanding, stores included.  A join of 16 columns a block gains nothing at this width (96 blocks
// of 64 columns; at 1000 columns they are 32 on 256 CUs, and the join takes 5 us all the same).
//
// A row's last chunk starts 8 columns before its end, so that every load is a whole one; the columns that
// it shares with the lane before are left out of its sums and stores.

#include <algorithm>

#include "elems.h"

namespace {

using flk::f32x4;

constexpr int kMaxWaves = 16;   // of a row: kV chunks of 8 x 64 columns each

struct Rows {            // row t of batch entry b at p + b * batch_stride + t * row_stride
  const void* p;
  int64_t batch_stride, row_stride;
};

struct NormArgs {
  Rows x, dy, y;         // y: the output (dx backwards)
  Rows branch, dr, r;    // the residual form's; r: the sum (dbranch backwards)
  const void* factor;    // NULL: 1
  const void* offset;    // NULL: 0
  const void* gate;      // the residual form's
  int64_t param_stride;  // elements from one batch entry's row to the next (0: one row for all)
  float add;             // a = factor + add
  float eps, inv_width;
  int length, width;
  // Blocks walk `per_block` rows of one group: of one batch entry's, or, where all share the parameters, of all.
  int64_t group_rows;
  int per_block, blocks_per_group;
  float* partial;        // backward: column sums (block, 2, width; the residual form 3), or NULL
};

// Sum over 64 lanes without leaving the registers; every lane ends with the same value.
__device__ __forceinline__ float wave_sum(float v) {
  v = flk::row16_sum(v);
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A lane's chunks of a row of `width` >= 8 columns (kNarrow: of fewer, one lane's), kV of them a block's lanes apart.
template <int kV, bool kNarrow>
struct Chunks {
  int at[kV];      // first column; past the end: the row's last 8 columns
  int skip[kV];    // leading columns that another lane has too (8: all)
  bool live[kV];
  __device__ __forceinline__ Chunks(int width, int lane, int lanes) {
#pragma unroll
    for (int c = 0; c < kV; ++c) {
      const int first = (lane + lanes * c) * 8;
      live[c] = first < width;
      at[c] = kNarrow ? first : min(first, width - 8);
      skip[c] = kNarrow ? 0 : min(first - at[c], 8);
    }
  }
  template <bool kStream = false, typename T>
  __device__ __forceinline__ flk::Raw8<T> load(const T* row, int c, int width) const {
    if constexpr (kNarrow) return flk::load8(row + at[c], width - at[c]);
    return flk::load8<kStream>(row + at[c], 8);
  }
  template <bool kStream, typename T>
  __device__ __forceinline__ void store(T* row, int c, int width, const float (&x)[8]) const {
    if (!live[c]) return;
    if constexpr (kNarrow) {
      flk::store8(row + at[c], width - at[c], x);
    } else if (skip[c] == 0) {
      flk::store8<kStream>(row + at[c], 8, x);
    } else {
#pragma unroll
      for (int i = 1; i < 8; ++i)
        if (i >= skip[c]) row[at[c] + i] = (T)x[i];
    }
  }
  // Whether element i of chunk c counts in the row's sums.
  __device__ __forceinline__ bool counts(int c, int i, int width) const {
    return kNarrow ? at[c] + i < width : i >= skip[c];
  }
};

// What a row's waves exchange, in turns of two: a wave's turn ends for all at the next row's barrier.
struct Exchange {
  f32x4 values[2][kMaxWaves];   // of the waves there are; zeros in the other places
};

// The row's mean and 1 / sqrt(v + eps), and with kGrads the sums of t and of t (x - mean).  own: this wave's
// mean, centred squares, sum of t, sum of t (x - own mean).
struct Stats {
  float mean, rstd, t, tx;
};

// columns: of wave lane % 16.
template <bool kOne, bool kGrads>
__device__ __forceinline__ Stats join(const f32x4& own, float columns, const NormArgs& A, Exchange& ex, int& turn) {
  float mean = own[0], square = own[1], t = own[2], tx = own[3];
  if constexpr (!kOne) {   // each 16 lanes take one wave's values a lane
    if ((threadIdx.x & 63) == 0) ex.values[turn][threadIdx.x >> 6] = own;
    __syncthreads();
    const f32x4 v = ex.values[turn][threadIdx.x & 15];
    mean = flk::row16_sum(v[0] * columns) * A.inv_width;
    const float d = v[0] - mean;
    square = flk::row16_sum(v[1] + columns * d * d);
    if constexpr (kGrads) {
      t = flk::row16_sum(v[2]);
      tx = flk::row16_sum(v[3] + d * v[2]);
    }
    turn ^= 1;
  }
  // rsqrtf, not the bare instruction, which takes the subnormal variances that eps = 0 lets through for zero
  return Stats{mean, rsqrtf(square * A.inv_width + A.eps), t, tx};
}

// A block's rows: slot's of every kSlots, first .. end - 1 of a group.
struct Walk {
  int64_t group, first, end;
  __device__ __forceinline__ Walk(const NormArgs& A, int slot) {
    group = blockIdx.x / A.blocks_per_group;
    const int64_t begin = (int64_t)(blockIdx.x - group * A.blocks_per_group) * A.per_block;
    first = begin + slot;
    end = min(begin + A.per_block, A.group_rows);
  }
  template <typename T>
  __device__ __forceinline__ T* row(const NormArgs& A, const Rows& r, int64_t at) const {
    int64_t b = group, t = at;
    if (A.group_rows != A.length) {   // one group of all entries' rows
      b = (uint32_t)at / (uint32_t)A.length;
      t = at - b * A.length;
    }
    return static_cast<T*>(const_cast<void*>(r.p)) + b * r.batch_stride + t * r.row_stride;
  }
};

// Which accesses leave the caches to others (nontemporal): none, the stores of y and dx, or the loads of all rows.
enum Access { kCached, kStorePast, kLoadPast };

// kOne: a wave takes a row alone, kSlots rows a block; otherwise all of the block's waves take one.
template <typename T, typename P, int kV, bool kOne, bool kNarrow, bool kBackward, Access kAccess, bool kResidual>
__global__ __launch_bounds__(kOne ? 256 : 64 * kMaxWaves) void norm_kernel(const NormArgs A) {
  constexpr int kSlots = kOne ? 4 : 1, kSums = kResidual ? 3 : 2;
  constexpr bool kStream = kAccess == kStorePast, kPast = kAccess == kLoadPast;
  __shared__ Exchange ex;
  __shared__ float sums[kOne && kBackward ? kSums * kV * 8 * 64 : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = kOne ? 1 : blockDim.x >> 6, slot = kOne ? wave : 0;
  const int lanes = 64 * waves, width = A.width;
  const Chunks<kV, kNarrow> chunks(width, kOne ? lane : (int)threadIdx.x, lanes);
  auto columns_of = [&](int w) {
    float n = 0.0f;
#pragma unroll
    for (int c = 0; c < kV; ++c) n += (float)max(0, min(width - (lanes * c + w * 64) * 8, 512));
    return n;
  };
  const float count = columns_of(kOne ? 0 : wave), inv_count = 1.0f / count;
  const float columns = (lane & 15) < waves ? columns_of(lane & 15) : 0.0f;
  if (!kOne && wave == 0 && lane >= 32 && (lane & 15) >= waves) ex.values[lane >> 4 & 1][lane & 15] = f32x4{};
  int turn = 0;
  const Walk walk(A, slot);

  const P* factor = static_cast<const P*>(A.factor);
  const P* offset = static_cast<const P*>(A.offset);
  const P* gate = static_cast<const P*>(A.gate);
  float a[kV][8], o[kBackward ? 1 : kV][8], gt[kResidual ? kV : 1][8];
#pragma unroll
  for (int c = 0; c < kV; ++c) {
    flk::Raw8<P> raw{};
    if (factor) raw = chunks.load(factor + walk.group * A.param_stride, c, width);
#pragma unroll
    for (int i = 0; i < 8; ++i) a[c][i] = factor ? (float)raw.v[i] + A.add : 1.0f;
    if constexpr (!kBackward) {
      if (offset) raw = chunks.load(offset + walk.group * A.param_stride, c, width);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[c][i] = offset ? (float)raw.v[i] : 0.0f;
    }
    if constexpr (kResidual) {
      raw = chunks.load(gate + walk.group * A.param_stride, c, width);
#pragma unroll
      for (int i = 0; i < 8; ++i) gt[c][i] = (float)raw.v[i];
    }
  }
  float da[kBackward ? kV : 1][8] = {}, dc[kBackward ? kV : 1][8] = {}, dg[kBackward && kResidual ? kV : 1][8] = {};
  // Whether all of this wave's columns count in the row's sums; where not, the others enter as zeros.
  const bool whole = count == (float)(kV * 512);

  // The next kDepth rows are asked for, one as each row is begun; those of the loop's next turn are waited for before it.
  constexpr int kDepth = sizeof(T) == 2 && kV == 1 ? 2 : 1;
  flk::Raw8<T> x[kDepth][kV], g[kBackward ? kDepth : 1][kV], br[kResidual ? kDepth : 1][kV];
  flk::Raw8<T> gr[kBackward && kResidual ? kDepth : 1][kV];
  auto fetch = [&](int d, int64_t r) {
    const T* px = walk.template row<T>(A, A.x, r);
    const T* pg = kBackward ? walk.template row<T>(A, A.dy, r) : nullptr;
    const T* pb = kResidual ? walk.template row<T>(A, A.branch, r) : nullptr;
    const T* pr = kResidual && kBackward ? walk.template row<T>(A, A.dr, r) : nullptr;
#pragma unroll
    for (int c = 0; c < kV; ++c) {
      x[d][c] = chunks.template load<kPast>(px, c, width);
      if constexpr (kResidual) br[d][c] = chunks.template load<kPast>(pb, c, width);
      if constexpr (kBackward) g[d][c] = chunks.template load<kPast>(pg, c, width);
      if constexpr (kBackward && kResidual) gr[d][c] = chunks.template load<kPast>(pr, c, width);
    }
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d)
    if (walk.first + d * kSlots < walk.end) fetch(d, walk.first + d * kSlots);
  auto work = [&](int d, int64_t r) {
    float xs[kV][8], gs[kBackward ? kV : 1][8];
    flk::Raw8<T> bs[kResidual ? kV : 1], rs[kBackward && kResidual ? kV : 1];
#pragma unroll
    for (int c = 0; c < kV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        xs[c][i] = (float)x[d][c].v[i];
        if constexpr (kResidual) xs[c][i] += gt[c][i] * (float)br[d][c].v[i];
        if constexpr (kBackward) gs[c][i] = (float)g[d][c].v[i];
      }
    if constexpr (kResidual) {
#pragma unroll
      for (int c = 0; c < kV; ++c) {
        bs[c] = br[d][c];
        if constexpr (kBackward) rs[c] = gr[d][c];
        else chunks.template store<kStream>(walk.template row<T>(A, A.r, r), c, width, xs[c]);
      }
    }
    if (r + kDepth * kSlots < walk.end) fetch(d, r + kDepth * kSlots);
    auto leave_out = [&](float (&v)[8], int c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = chunks.counts(c, i, width) ? v[i] : 0.0f;
    };
    f32x4 own{};
#pragma unroll
    for (int c = 0; c < kV; ++c) {
      if (!whole) {
        leave_out(xs[c], c);
        if constexpr (kBackward) leave_out(gs[c], c);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) own[0] += xs[c][i];
    }
    own[0] = wave_sum(own[0]) * inv_count;
#pragma unroll
    for (int c = 0; c < kV; ++c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) xs[c][i] -= own[0];
      if (!whole) leave_out(xs[c], c);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        own[1] += xs[c][i] * xs[c][i];
        if constexpr (kBackward) {
          dc[c][i] += gs[c][i];
          const float t = gs[c][i] * a[c][i];
          own[2] += t;
          own[3] += t * xs[c][i];
        }
      }
    }
    own[1] = wave_sum(own[1]);
    if constexpr (kBackward) {
      own[2] = wave_sum(own[2]);
      own[3] = wave_sum(own[3]);
    }
    const Stats st = join<kOne, kBackward>(own, columns, A, ex, turn);
    const float shift = (own[0] - st.mean) * st.rstd;
    const float mt = st.t * A.inv_width * st.rstd, mtn = st.rstd * st.tx * A.inv_width * st.rstd;
    T* y = walk.template row<T>(A, A.y, r);
#pragma unroll
    for (int c = 0; c < kV; ++c) {
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = xs[c][i] * st.rstd + shift;
        if constexpr (kBackward) {
          out[i] = gs[c][i] * a[c][i] * st.rstd - mt - n * mtn;
          da[c][i] += gs[c][i] * n;
          if constexpr (kResidual) {
            out[i] += (float)rs[c].v[i];
            dg[c][i] += out[i] * (float)bs[c].v[i];
          }
        } else {
          out[i] = n * a[c][i] + o[c][i];
        }
      }
      chunks.template store<kStream>(y, c, width, out);
      if constexpr (kBackward && kResidual) {
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] *= gt[c][i];
        chunks.template store<kStream>(walk.template row<T>(A, A.r, r), c, width, out);
      }
    }
  };
  for (int64_t r = walk.first; r < walk.end; r += kDepth * kSlots) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
      if (r + d * kSlots < walk.end) work(d, r + d * kSlots);
  }
  if constexpr (kBackward) {
    if (!A.partial) return;
    if constexpr (kOne) {   // slot 0 adds the other slots' sums, one slot at a time
      for (int s = 1; s < kSlots; ++s) {
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kV; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (slot == s) {
              sums[(c * 8 + i) * 64 + lane] = da[c][i];
              sums[(kV * 8 + c * 8 + i) * 64 + lane] = dc[c][i];
              if constexpr (kResidual) sums[(kV * 16 + c * 8 + i) * 64 + lane] = dg[c][i];
            }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kV; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (slot == 0) {
              da[c][i] += sums[(c * 8 + i) * 64 + lane];
              dc[c][i] += sums[(kV * 8 + c * 8 + i) * 64 + lane];
              if constexpr (kResidual) dg[c][i] += sums[(kV * 16 + c * 8 + i) * 64 + lane];
            }
      }
      if (slot) return;
    }
    float* out = A.partial + (int64_t)blockIdx.x * kSums * width;
#pragma unroll
    for (int c = 0; c < kV; ++c) {
      chunks.template store<false>(out, c, width, da[c]);
      chunks.template store<false>(out + width, c, width, dc[c]);
      if constexpr (kResidual) chunks.template store<false>(out + 2 * width, c, width, dg[c]);
    }
  }
}

// Adds a group's partial rows in a fixed order: 64 columns a block, its waves every kJoinWaves-th row each, then the
// waves' sums in order.
constexpr int kJoinWaves = 16;
template <typename P>
__global__ __launch_bounds__(64 * kJoinWaves) void norm_params_kernel(const float* __restrict__ partial, int blocks, int width,
                                                                      int cuts, P* dfactor, P* doffset, P* dgate) {
  __shared__ float part[kJoinWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t group = blockIdx.x / cuts;
  const int col = (int)(blockIdx.x - group * cuts) * 64 + lane;
  const int which = blockIdx.y, sums = gridDim.y;   // 0: factor, 1: offset, 2: gate
  P* out = which == 2 ? dgate : which ? doffset : dfactor;
  if (!out) return;
  const float* src = partial + group * blocks * sums * width + (int64_t)which * width + col;
  float sum = 0.0f;
  if (col < width) {
#pragma unroll 4
    for (int i = wave; i < blocks; i += kJoinWaves) sum += src[(int64_t)i * sums * width];
  }
  part[wave][lane] = sum;
  __syncthreads();
  if (wave || col >= width) return;
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w) sum += part[w][lane];
  out[group * width + col] = (P)sum;
}

constexpr int kMaxWidth = 2 * kMaxWaves * 512;
constexpr int kMaxRows = INT32_MAX;
constexpr int kMaxGroups = 1 << 22;       // batch entries with parameters of their own
// Float32 outputs up to this size pass the caches by, as 16-bit ones of any size do: 1200 x 24 * 128 forward 7.0 us
// (through the caches 8.2), backward 15.8 (16.4).  Larger ones do not: 2048 rows 10.5 and 21.4 us (past the caches
// 11.0 and 22.4), with what reads the output next 19.7 and 29.3 (21.0 and 32.3); 16384 x 1000 47 and 70 (56 and 78).
constexpr int64_t kStreamBytes = 18 << 20;
constexpr int64_t kMaxItems = 1LL << 31;  // of one launch, whose work-items are counted in 32 bits

// Rows a block walks.  Of the numbers of blocks a CU that keep up to `waves` waves on it, the one whose CUs
// all get nearly the same number of rows, and then the largest; `least` rows a block at any rate.
int rows_per_block(int64_t group_rows, int64_t groups, int width, int waves, int least) {
  const int slots = width <= 512 ? 4 : 1, of_block = width <= 512 ? 4 : std::min((width + 511) / 512, kMaxWaves);
  int64_t best = 0, load = INT64_MAX;
  for (int per_cu = std::max(1, waves / of_block); per_cu >= std::max(1, waves / 2 / of_block); --per_cu) {
    const int64_t blocks = std::max<int64_t>(1, 256 * per_cu / groups);
    const int64_t per = (std::max<int64_t>(least, (group_rows + blocks - 1) / blocks) + slots - 1) / slots * slots;
    const int64_t all = groups * ((group_rows + per - 1) / per), cu = (all + 255) / 256 * per;
    if (cu < load) {
      load = cu;
      best = per;
    }
  }
  return (int)best;
}
int forward_rows(int64_t group_rows, int64_t groups, int width) {
  return rows_per_block(group_rows, groups, width, 24, 1);
}
int backward_rows(int64_t group_rows, int64_t groups, int width) {
  return rows_per_block(group_rows, groups, width, 12, (int)std::min<int64_t>(4, 1 + group_rows * groups / 128));
}

// Threads of a block.
int threads_of(int width) { return width <= 512 ? 256 : std::min(((width + 7) / 8 + 63) / 64, kMaxWaves) * 64; }

int sums_of(const NormArgs& a) { return a.gate ? 3 : 2; }   // column sums of the backward pass

// Group g's rows and parameters.
template <typename T, typename P>
NormArgs from_group(NormArgs a, int64_t g) {
  if (g == 0) return a;   // the only one where the groups are not batch entries
  for (Rows* r : {&a.x, &a.dy, &a.y, &a.branch, &a.dr, &a.r})
    if (r->p) r->p = static_cast<const T*>(r->p) + g * r->batch_stride;
  for (const void** p : {&a.factor, &a.offset, &a.gate})
    if (*p) *p = static_cast<const P*>(*p) + g * a.param_stride;
  if (a.partial) a.partial += g * a.blocks_per_group * sums_of(a) * a.width;
  return a;
}

template <typename T, typename P, bool kBackward, Access kAccess, bool kResidual>
int launch(const NormArgs& all, int64_t groups, hipStream_t s) {
  const int threads = threads_of(all.width);
  const int64_t most = kMaxItems / threads / all.blocks_per_group;   // groups of one launch
  for (int64_t first = 0; first < groups; first += most) {
    const NormArgs a = from_group<T, P>(all, first);
    const dim3 grid((unsigned)(std::min(most, groups - first) * a.blocks_per_group));
    if (a.width < 8)
      norm_kernel<T, P, 1, true, true, kBackward, kAccess, kResidual><<<grid, threads, 0, s>>>(a);
    else if (a.width <= 512)
      norm_kernel<T, P, 1, true, false, kBackward, kAccess, kResidual><<<grid, threads, 0, s>>>(a);
    else if (a.width <= 512 * kMaxWaves)
      norm_kernel<T, P, 1, false, false, kBackward, kAccess, kResidual><<<grid, threads, 0, s>>>(a);
    else
      norm_kernel<T, P, 2, false, false, kBackward, kAccess, kResidual><<<grid, threads, 0, s>>>(a);
    if (const int st = flk_launch_status()) return st;
  }
  return FLK_OK;
}

// Whether every chunk of a row is a 16-byte word of its own.
template <typename T>
bool rows_aligned(const NormArgs& a) {
  for (const Rows* r : {&a.x, &a.branch, &a.dy, &a.dr}) {
    const int64_t bytes = (int64_t)(reinterpret_cast<uintptr_t>(r->p) | r->row_stride * sizeof(T) | r->batch_stride * sizeof(T));
    if (r->p && bytes % 16) return false;
  }
  return a.width % 8 == 0;
}

template <typename T, typename P, bool kBackward, bool kResidual>
int dispatch(const NormArgs& a, int64_t groups, hipStream_t s) {
  if constexpr (sizeof(T) == 4) {
    if (a.group_rows * groups * a.width * 4 > kStreamBytes) return launch<T, P, kBackward, kCached, kResidual>(a, groups, s);
  } else if constexpr (kResidual) {
    if (rows_aligned<T>(a)) return launch<T, P, kBackward, kLoadPast, true>(a, groups, s);
  }
  return launch<T, P, kBackward, kStorePast, kResidual>(a, groups, s);
}

template <typename P>
int join_params(const NormArgs& a, int64_t groups, void* dfactor, void* doffset, void* dgate, hipStream_t s) {
  const int cuts = (a.width + 63) / 64;
  const int64_t most = kMaxItems / (64 * kJoinWaves) / sums_of(a) / cuts;
  for (int64_t first = 0; first < groups; first += most) {
    const dim3 grid((unsigned)(std::min(most, groups - first) * cuts), sums_of(a));
    auto rows = [&](void* p) { return p ? static_cast<P*>(p) + first * a.width : nullptr; };
    norm_params_kernel<P><<<grid, 64 * kJoinWaves, 0, s>>>(a.partial + first * a.blocks_per_group * sums_of(a) * a.width,
                                                           a.blocks_per_group, a.width, cuts, rows(dfactor),
                                                           rows(doffset), rows(dgate));
    if (const int st = flk_launch_status()) return st;
  }
  return FLK_OK;
}

// Adds the column sums up, where there are any.
int join_types(int params, const NormArgs& a, int64_t groups, void* dfactor, void* doffset, void* dgate, hipStream_t s) {
  if (!a.partial) return FLK_OK;
  if (params == FLK_F32) return join_params<float>(a, groups, dfactor, doffset, dgate, s);
  if (params == FLK_BF16) return join_params<__bf16>(a, groups, dfactor, doffset, dgate, s);
  return join_params<_Float16>(a, groups, dfactor, doffset, dgate, s);
}

template <bool kBackward, bool kResidual>
int dispatch_types(int dtype, int params, const NormArgs& a, int64_t groups, hipStream_t s) {
  if (dtype == FLK_F32) return params == FLK_F32 ? dispatch<float, float, kBackward, kResidual>(a, groups, s) : FLK_E_UNSUPPORTED;
  if (dtype == FLK_BF16) {
    if (params == FLK_BF16) return dispatch<__bf16, __bf16, kBackward, kResidual>(a, groups, s);
    if (params == FLK_F32) return dispatch<__bf16, float, kBackward, kResidual>(a, groups, s);
  }
  if (dtype == FLK_F16) {
    if (params == FLK_F16) return dispatch<_Float16, _Float16, kBackward, kResidual>(a, groups, s);
    if (params == FLK_F32) return dispatch<_Float16, float, kBackward, kResidual>(a, groups, s);
  }
  return FLK_E_UNSUPPORTED;
}

unsigned elem_bytes(int dtype) { return dtype == FLK_F32 ? 4 : 2; }

int check(int dtype, int params, const void* x, const void* y, const void* factor, const void* offset,
          int64_t param_stride, float eps, int batch, int length, int width) {
  if (dtype < FLK_BF16 || dtype > FLK_F32 || params < FLK_BF16 || params > FLK_F32) return FLK_E_INVALID;
  if (batch < 0 || length < 0 || width <= 0 || !(eps >= 0.0f) || param_stride < 0) return FLK_E_INVALID;
  if (param_stride && param_stride < width) return FLK_E_INVALID;
  if ((int64_t)batch * length > kMaxRows || (param_stride && batch > kMaxGroups)) return FLK_E_INVALID;
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
  a.group_rows = param_stride ? length : (int64_t)batch * length;
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
  const int64_t groups = param_batch_stride ? batch : 1;
  a.per_block = forward_rows(a.group_rows, groups, width);
  a.blocks_per_group = (int)((a.group_rows + a.per_block - 1) / a.per_block);
  return dispatch_types<false, false>(dtype, params_dtype, a, groups, static_cast<hipStream_t>(stream));
}

extern "C" int flk_layer_norm_backward_plan(int batch, int length, int width, int shared_params,
                                            int64_t* workspace_bytes) {
  if (batch < 0 || length < 0 || width <= 0 || !workspace_bytes) return FLK_E_INVALID;
  if ((int64_t)batch * length > kMaxRows || (!shared_params && batch > kMaxGroups)) return FLK_E_INVALID;
  *workspace_bytes = 0;
  if (batch == 0 || length == 0) return FLK_OK;
  const int64_t groups = shared_params ? 1 : batch, group_rows = shared_params ? (int64_t)batch * length : length;
  const int per = backward_rows(group_rows, groups, width);
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
  const int64_t groups = param_batch_stride ? batch : 1;
  a.per_block = backward_rows(a.group_rows, groups, width);
  a.blocks_per_group = (int)((a.group_rows + a.per_block - 1) / a.per_block);
  if (dfactor || doffset) {
    const int64_t need = groups * a.blocks_per_group * 2 * width * 4;
    if (!workspace || workspace_bytes < need) return FLK_E_SCRATCH;
    if (!flk_host_aligned(workspace, 16)) return FLK_E_ALIGN;
    a.partial = static_cast<float*>(workspace);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (const int st = dispatch_types<true, false>(dtype, params_dtype, a, groups, s)) return st;
  return join_types(params_dtype, a, groups, dfactor, doffset, nullptr, s);
}

extern "C" int flk_residual_norm(const void* x, int64_t x_batch_stride, int64_t x_row_stride, const void* branch,
                                 int64_t branch_batch_stride, int64_t branch_row_stride, int dtype, const void* gate,
                                 const void* factor, const void* offset, int params_dtype, int64_t param_batch_stride,
                                 int add_one, float eps, int batch, int length, int width, void* r, int64_t r_batch_stride,
                                 int64_t r_row_stride, void* y, int64_t y_batch_stride, int64_t y_row_stride,
                                 void* stream) {
  if (const int st = check(dtype, params_dtype, x, y, factor, offset, param_batch_stride, eps, batch, length, width))
    return st;
  if (const int st = check(dtype, params_dtype, branch, r, gate, nullptr, param_batch_stride, eps, batch, length, width))
    return st;
  if (batch == 0 || length == 0) return FLK_OK;
  if (!gate) return FLK_E_INVALID;
  NormArgs a = common_args(x, x_batch_stride, x_row_stride, factor, offset, param_batch_stride, add_one, eps, batch,
                           length, width);
  a.y = Rows{y, y_batch_stride, y_row_stride};
  a.branch = Rows{branch, branch_batch_stride, branch_row_stride};
  a.r = Rows{r, r_batch_stride, r_row_stride};
  a.gate = gate;
  const int64_t groups = param_batch_stride ? batch : 1;
  a.per_block = forward_rows(a.group_rows, groups, width);
  a.blocks_per_group = (int)((a.group_rows + a.per_block - 1) / a.per_block);
  return dispatch_types<false, true>(dtype, params_dtype, a, groups, static_cast<hipStream_t>(stream));
}

extern "C" int flk_residual_norm_backward_plan(int batch, int length, int width, int shared_params,
                                               int64_t* workspace_bytes) {
  if (const int st = flk_layer_norm_backward_plan(batch, length, width, shared_params, workspace_bytes)) return st;
  *workspace_bytes = *workspace_bytes / 2 * 3;
  return FLK_OK;
}

extern "C" int flk_residual_norm_backward(const void* dr, int64_t dr_batch_stride, int64_t dr_row_stride, const void* dy,
                                          int64_t dy_batch_stride, int64_t dy_row_stride, const void* x,
                                          int64_t x_batch_stride, int64_t x_row_stride, const void* branch,
                                          int64_t branch_batch_stride, int64_t branch_row_stride, int dtype,
                                          const void* gate, const void* factor, int params_dtype,
                                          int64_t param_batch_stride, int add_one, float eps, int batch, int length,
                                          int width, void* dx, int64_t dx_batch_stride, int64_t dx_row_stride,
                                          void* dbranch, int64_t dbranch_batch_stride, int64_t dbranch_row_stride,
                                          void* dgate, void* dfactor, void* doffset, void* workspace,
                                          int64_t workspace_bytes, void* stream) {
  const struct {
    const void *in, *out, *row, *sum;
  } all[] = {{x, dx, factor, dfactor}, {branch, dbranch, gate, dgate}, {dy, dx, nullptr, doffset}, {dr, dx, nullptr, nullptr}};
  for (const auto& t : all)
    if (const int st = check(dtype, params_dtype, t.in, t.out, t.row, t.sum, param_batch_stride, eps, batch, length, width))
      return st;
  if (batch == 0 || length == 0) return FLK_OK;   // the sums over no rows are the caller's to clear
  if (!gate) return FLK_E_INVALID;
  NormArgs a = common_args(x, x_batch_stride, x_row_stride, factor, nullptr, param_batch_stride, add_one, eps, batch,
                           length, width);
  a.dy = Rows{dy, dy_batch_stride, dy_row_stride};
  a.dr = Rows{dr, dr_batch_stride, dr_row_stride};
  a.branch = Rows{branch, branch_batch_stride, branch_row_stride};
  a.y = Rows{dx, dx_batch_stride, dx_row_stride};
  a.r = Rows{dbranch, dbranch_batch_stride, dbranch_row_stride};
  a.gate = gate;
  const int64_t groups = param_batch_stride ? batch : 1;
  a.per_block = backward_rows(a.group_rows, groups, width);
  a.blocks_per_group = (int)((a.group_rows + a.per_block - 1) / a.per_block);
  if (dgate || dfactor || doffset) {
    const int64_t need = groups * a.blocks_per_group * 3 * width * 4;
    if (!workspace || workspace_bytes < need) return FLK_E_SCRATCH;
    if (!flk_host_aligned(workspace, 16)) return FLK_E_ALIGN;
    a.partial = static_cast<float*>(workspace);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (const int st = dispatch_types<true, true>(dtype, params_dtype, a, groups, s)) return st;
  return join_types(params_dtype, a, groups, dfactor, doffset, dgate, s);
}

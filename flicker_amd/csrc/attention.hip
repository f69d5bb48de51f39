// attention: softmax(q k^T) v of any lengths, over the keys that a mask keeps, and its gradients.
//
// Per (b, h) and query i, over the kept keys j of key head h / (heads / kv_heads); q comes scaled:
//   S_ij = q_i . k_j,  lse_i = log sum_j exp S_ij,  P_ij = exp(S_ij - lse_i),  o_i = sum_j P_ij v_j
// and backwards, for the gradient g_i of o_i,
//   delta_i = g_i . o_i,  dP_ij = g_i . v_j,  dS_ij = P_ij (dP_ij - delta_i)
//   dq_i = sum_j dS_ij k_j,  dk_j = sum_i dS_ij q_i,  dv_j = sum_i P_ij g_i
// (dk and dv also over the query heads that share the key head).  A query that keeps no key has o = 0, lse = -inf and
// no gradient.
//
// The products run on the 16x16x32 matrix instructions, whose accumulators hold a lane's four rows of one column.  Every
// product is laid out so that what one leaves is what the next takes: with keys as rows, S^T = K Q^T leaves a lane P of one
// query and 4 + 4 keys of a 32-key unit, packed the right operand of O^T += V^T P^T; with queries as rows, S = Q K^T leaves
// it P of one key and 4 + 4 queries, the right operand of dV^T += dO^T P.  So P and dS never pass through LDS to be
// turned, and a wave keeps its own 32 rows (Q and dO; or K, or V) as right operands in registers.  Left operands come from
// LDS: rows as they are (b128), columns through the transposing b64 read, both conflict-free by the swizzle below.
//
// LDS holds rings of 32-row units, filled by copies straight from memory that were started phases earlier.  A phase is 16
// or 24 slots of two matrix instructions on one left operand, read four slots before; between them, one element a slot,
// the vector units turn the last unit's S into P.  Loops are unrolled over the rings, which makes LDS addresses constants
// of a lane (4608 tokens: 249 -> 240 us forwards, 880 -> 790 backwards).
//
// The running maximum is one that lags: P are taken against the maximum of an earlier unit until one passes a limit, and
// only then is what has been summed scaled and the unit's P formed again, after the fact (a check before each unit's
// exponents sat ahead of its matrix work: 265 -> 249).  l, the sum that divides o, is of the rounded P (two more matrix
// instructions with a row of ones); lse is of the unrounded, added up in float32.
//
// Gradients take 7 products where 5 would do: dq has blocks of queries, dk and dv blocks of keys, and both form S and dP.
// Sharing them would mean 4 bytes of dq added to memory per key block and query and d, 2 GB at 4608 tokens and 24 heads,
// in an order that timing decides; the two products cost 0.2 ms there.  In a block of 128 keys pairs of waves share 32: one
// holds K and dV, forms S and P and leaves P (float32) in LDS for the other, which holds V and dK and forms dP and dS a unit
// later.  One wave with all four would need 320 registers at two waves a SIMD.  delta needs o closer
// than its type holds it where few keys carry a row (at two keys its rounding would cost dq, by estimate, twice all else),
// so the forward pass keeps what o's rounding left.
//
// Masks: bytes become one word of bits a unit and a list of the units that keep any, in a launch of their own past 64 units
// (attention_mask_kernel), and blocks walk that list.  In a unit that keeps part, the rows left out are cleared in LDS
// before anyone reads them (0 * inf), and their S set to -inf.
//
// Blocks that would leave CUs idle are cut along the units they walk, and a second kernel adds the float32 partial sums up in
// order; which and how many is estimated from a unit's time (plan_cut, search_gradients).  The gradients' two kinds of
// blocks share a launch, so that neither's last round leaves CUs idle (1536 tokens, forward and gradients: 172 -> 153 us).
//
// Bound: the matrix pipe, and over whole rounds of blocks the chip's power: random operands hold it there, where a large
// library product reaches 1.24 PFLOP/s.  Measured at 24 heads in bfloat16, PFLOP/s over all products that run: forward
// 4608 tokens 237 us (1.10), 16896 2.75 ms (1.28), with what the gradients need 261 us and 2.91 ms; gradients 741 us
// (1.23) and 9.6 ms (1.28), of which 15 and 66 us are the rows' stats.  1536 tokens are 192 blocks of queries for 256 CUs:
// 46 us and 113.  Few rows are bound by memory, and have a kernel of their own: one query on 4608 keys 17 us.

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace {

constexpr int kD = 128;
constexpr int kRowBytes = kD * 2;
constexpr int kUnit = 32;              // rows of a unit: the contraction length of one MFMA, keys of a mask word
constexpr int kUnitBytes = kUnit * kRowBytes;
constexpr int kWaves = 8;              // two a SIMD
constexpr int kThreads = 64 * kWaves;
constexpr int kQueries = 32 * kWaves;  // queries of a block, 32 a wave
constexpr int kKeys = 16 * kWaves;     // keys of a block, 32 a pair of waves
constexpr int kFewRows = 16;           // rows of a block of attention_few_kernel
constexpr int kLead = 4;               // slots between an operand's LDS read and its MFMAs
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;   // a running maximum of no keys
constexpr int64_t kMaxItems = 1LL << 31;
constexpr int64_t kMaxRow = 1LL << 25;   // elements between two rows: a unit's byte offsets stay below 2^31

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

// What the mask's bytes come to: of batch entry b the words bits[b * units + u], bit i of word u set where key 32 u + i is
// kept, and the units live[b * units + n].x, n < counts[b], whose words (.y) are not zero, in order.  Where `bytes` is set,
// each wave finds the list by itself, in rows of at most 64 units.  All NULL: all keys are kept.
struct Mask {
  const uint32_t* bits;
  const uint2* live;
  const int* counts;
  const uint8_t* bytes;
  int64_t batch_stride;
  __host__ __device__ bool none() const { return !bits && !bytes; }
};

// The blocks from `whole` on are cut into `splits` along the units they walk: partial sums of `pitch` rows, in order, which
// attention_join_kernel adds up.
struct Cuts {
  int whole, splits, tile;   // tile: rows of a block
  float* part;               // (cut, pitch, 128)
};
constexpr int pitch_of(int tile) { return tile == kFewRows ? kFewRows : kQueries; }

struct Args {
  Tensor q, k, v, o, dO, dq, dk, dv;
  void* low;        // (batch, queries, heads, 128): what o's rounding left, in the same type
  float* lse;       // (batch, heads, queries)
  float* stats;     // (batch * heads * q_units + 1, 2, 32): a unit's lse and -delta; inf and 0 in rows past the
                    // end and in the last unit
  float* norms;     // float16's gradients, of a quarter of a unit's rows each: the most |do|^2 and delta^2,
                    // (batch * heads * q_units, 4, 2), and |v|^2 of kept keys, (batch * kv_heads * k_units, 4)
  Mask mask;
  int batch, heads, kv_heads, group, queries, keys, q_units, k_units;
  Cuts of_q, of_k;  // of the blocks of queries, and of keys (backwards)
  float* part_top;  // (cut, pitch, 4): in the forward pass each row's (top, l, sum)
  int q_grid;       // backwards: hardware blocks that take queries, the first ones or, with k_first, the last
  bool k_first;
};

// Which keys of unit u are kept.
__device__ __forceinline__ uint32_t kept(const Args& A, int b, int u) {
  if (A.mask.bits) return A.mask.bits[(int64_t)b * A.k_units + u];
  const int left = A.keys - u * kUnit;
  return left >= kUnit ? ~0u : (1u << left) - 1;
}

// Hardware deals blocks round-robin over the 8 XCDs, each with an L2 of its own: this numbering gives each XCD
// neighbouring blocks, which read the same head's rows.
__device__ __forceinline__ int by_xcd(int p, int total) {
  const int xcd = p & 7, per = total >> 3, extra = total & 7;
  return xcd * per + min(xcd, extra) + (p >> 3);
}

// What a hardware block takes: a block, or one of its cuts.
struct Piece {
  int block, cut, split, splits;   // cut: its place among the partial sums, -1 for a whole block
  // p: which of `total` pieces.
  __device__ __forceinline__ Piece(const Cuts& c, int p, int total) {
    if (p < c.whole) {
      block = by_xcd(p, c.whole);
      cut = -1;
      split = 0;
      splits = 1;
    } else {
      const int i = by_xcd(p - c.whole, total - c.whole);
      splits = c.splits;
      block = c.whole + i / splits;
      split = i % splits;
      cut = splits > 1 ? i : -1;
    }
  }
  // Its part of n units.
  __device__ __forceinline__ int first(int n) const { return split * (n / splits) + min(split, n % splits); }
  __device__ __forceinline__ int count(int n) const { return n / splits + (split < n % splits); }
};

// A wave's queries in a block of of_q.tile: 256, 32 a wave, or 192, of which the waves 4-7 take 16 each, so that every
// SIMD holds 48.
struct Rows {
  int b, h, first, end, q0;
  bool wide;
  __device__ __forceinline__ Rows(const Args& A, const Piece& piece) {
    const int tile = A.of_q.tile, blocks = (A.queries + tile - 1) / tile, bh = piece.block / blocks;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    b = bh / A.heads;
    h = bh - b * A.heads;
    first = (piece.block - bh * blocks) * tile;
    end = min(A.queries, first + tile);
    wide = tile == kQueries || wave < 4;
    q0 = first + (wide ? wave * 32 : 64 + wave * 16);
  }
};

__device__ __forceinline__ int swz(int row) { return ((row & 7) << 1) | ((row >> 3) & 1); }

// LDS holds units of 32 rows of 256 bytes, whose 16-byte chunk c of row r sits in place c ^ swz(r).
struct Places {   // a lane's byte offsets of its operands within a unit
  int row[4];     // 16 rows x 32 d as they are: row lane % 16, d step st
  int col[8];     // 16 d x 32 rows transposed: d tile dt
};
__device__ __forceinline__ Places places() {
  Places at;
  const int lane = threadIdx.x & 63, h = lane >> 4, col = lane & 15;
  // k-slots 8h .. 8h + 7 of a row operand are d chunk 4 st + hperm, 0, 2, 1, 3 for h = 0 .. 3: lanes l and l + 32 then read
  // neighbouring chunks, on distinct banks however the read is split.
  const int hperm = ((h & 1) << 1) | (h >> 1);
#pragma unroll
  for (int st = 0; st < 4; ++st) {
    at.row[st] = col * kRowBytes + ((((st << 2) | hperm) ^ swz(col)) << 4);
    asm volatile("" : "+v"(at.row[st]));
  }
  // The transposing read hands lane 4a + b of a lane group element b of its source lanes a, a + 4, a + 8, a + 12: source lane
  // s of group h points at row 4h + s / 4, d 16 dt + 4 (s % 4), so the k-slots are rows 4h .. + 3 and those + 16.
  const int r = h * 4 + (col >> 2);
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) {
    at.col[dt] = r * kRowBytes + (((2 * dt + ((col & 3) >> 1)) ^ swz(r)) << 4) + (col & 1) * 8;
    asm volatile("" : "+v"(at.col[dt]));
  }
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
// P^T or dS^T of group g as the right operand of a product over a unit's rows: the packed words of its two accumulators.
template <typename T, int N>
__device__ __forceinline__ vec8<T> packed(const uint32_t (&p)[N], int g) {
  return __builtin_bit_cast(vec8<T>, make_uint4(p[4 * g], p[4 * g + 1], p[4 * g + 2], p[4 * g + 3]));
}

// Copies of a tensor's units into LDS: each wave 4 rows of 32, 16 bytes a lane, straight from memory.
struct Copies {
  const char* head;
  uint32_t step;          // bytes from one unit to the next
  uint32_t at, at_last;   // a lane's source offset in a unit, and in the last, whose rows past the end repeat the last row
  int last;               // that unit
  __device__ __forceinline__ Copies(const uint16_t* head, int64_t row, int rows)
      : head(reinterpret_cast<const char*>(head)), step((uint32_t)row * kUnit * 2) {
    const int lane = threadIdx.x & 63, r = (threadIdx.x >> 6) * 4 + (lane >> 4);
    const uint32_t chunk = ((lane & 15) ^ swz(r)) << 4;
    last = (rows - 1) / kUnit;
    at = (uint32_t)(r * row * 2) + chunk;
    at_last = (uint32_t)(min(r, rows - 1 - last * kUnit) * row * 2) + chunk;
  }
  // Unit `unit` of the head into the slot whose byte 0 of this wave's rows is `lds`.  kInside: it is not the last.
  template <bool kInside>
  __device__ __forceinline__ void start(unsigned lds, int unit) const {
    flk::dma16_lds(head + (uint64_t)(uint32_t)unit * step, kInside || unit != last ? at : at_last, lds);
  }
};

// Where this wave's 4 rows of the unit at the start of LDS go.
__device__ __forceinline__ unsigned wave_rows(const uint8_t* smem) {
  return __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)smem + (threadIdx.x >> 6) * 4 * kRowBytes);
}

// Clears this wave's rows of a unit that `bits` leaves out: 0 * what they hold would be NaN for infinities.  Their copy has
// landed; the others see zeros after the next barrier.
__device__ __forceinline__ void clear_rows(uint8_t* slot, uint32_t bits) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t mine = bits >> (4 * wave) & 15;
  if (mine == 15) return;
  if (!(mine >> (lane >> 4) & 1))
    *reinterpret_cast<uint4*>(slot + wave * 4 * kRowBytes + lane * 16) = make_uint4(0, 0, 0, 0);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// S of the keys that `bits` leaves out of a unit's accumulators (group, 16-key tile): -inf.
template <int N>
__device__ __forceinline__ void leave_out(f32x4 (&s)[N], uint32_t bits) {
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const uint32_t mine = bits >> (16 * kt + (threadIdx.x >> 4 & 3) * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int g = 0; g < N / 2; ++g) s[2 * g + kt][i] = mine >> i & 1 ? s[2 * g + kt][i] : -INFINITY;
  }
}

// The word of unit `lane` of a row's 64 from `first` on.  Bytes past the row's end are not read, and none is waited for before
// half of the others are asked for.
__device__ __forceinline__ uint32_t mask_word(const uint8_t* row, int first, int keys) {
  const int lane = threadIdx.x & 63;
  uint32_t mine = 0;
  for (int half = 0; half < 32; half += 16) {
    const int from = (first + 2 * half) * kUnit + lane;
    if (from - lane >= keys) break;
    uint8_t x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = row[min(from + 64 * i, keys - 1)];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint64_t both = __ballot(from + 64 * i < keys && x[i] != 0);
      if (lane >> 1 == half + i) mine = (uint32_t)(lane & 1 ? both >> 32 : both);
    }
  }
  return mine;
}
// A row's units that have kept keys, one a lane, and how many they are; the lanes behind them hold the others.
__device__ __forceinline__ uint2 find_live(const Args& A, int b, int& count) {
  const int lane = threadIdx.x & 63;
  const uint32_t mine = mask_word(A.mask.bytes + b * A.mask.batch_stride, 0, A.keys);
  const uint64_t any = __ballot(mine != 0);
  const int before = __popcll(any & ((1ull << lane) - 1));
  count = __popcll(any);
  const int to = 4 * (mine ? before : count + lane - before);
  return make_uint2(__builtin_amdgcn_ds_permute(to, lane), __builtin_amdgcn_ds_permute(to, (int)mine));
}

// The key units of a batch entry that have kept keys, asked for one after the other from 0; past the last: the last one with
// no key kept.  A masked entry's list is fetched 64 units at a time, one a lane.
template <bool kMasked>
struct Units {
  const uint2* live;
  int first, n;
  uint32_t tail;
  uint2 some;
  __device__ __forceinline__ Units(const Args& A, int b, const Piece& piece) {
    int all = A.k_units;
    if constexpr (kMasked) {
      if (A.mask.bytes) some = find_live(A, b, all);
      else all = A.mask.counts[b];
      all = __builtin_amdgcn_readfirstlane(all);
    }
    first = piece.first(all);
    n = piece.count(all);
    if constexpr (kMasked) {
      live = A.mask.bytes ? nullptr : A.mask.live + (int64_t)b * A.k_units + first;
      const int from = first + min((int)(threadIdx.x & 63), n - 1);
      if (!live) some = make_uint2(__shfl(some.x, from), __shfl(some.y, from));
    } else {
      tail = first + n == all ? kept(A, b, all - 1) : ~0u;
    }
  }
  __device__ __forceinline__ void get(int i, int& unit, uint32_t& bits) {
    if constexpr (kMasked) {
      if ((i & 63) == 0 && live) some = live[min(i + (int)(threadIdx.x & 63), n - 1)];
      unit = __builtin_amdgcn_readlane(some.x, i & 63);
      bits = i < n ? __builtin_amdgcn_readlane(some.y, i & 63) : 0u;
    } else {
      unit = first + min(i, n - 1);
      bits = i < n - 1 ? ~0u : i == n - 1 ? tail : 0u;
    }
  }
  // The units of u .. u + 4, of which a masked entry has fetched the first four.
  __device__ __forceinline__ void look(int u, int (&unit)[5], uint32_t (&bits)[5]) {
#pragma unroll
    for (int i = kMasked ? 4 : 0; i < 5; ++i) get(u + i, unit[i], bits[i]);
  }
  static __device__ __forceinline__ void shift(int (&unit)[5], uint32_t (&bits)[5]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unit[i] = unit[i + 1];
      bits[i] = bits[i + 1];
    }
  }
};

// The wave's G groups of 16 rows from row0 as the right operand: row lane % 16 of group g, d step st; zeros past `end`.
template <typename T, int G>
__device__ __forceinline__ void load_rows(vec8<T> (&x)[4][G], const T* src, int64_t stride, int row0, int end) {
  const int lane = threadIdx.x & 63, h = lane >> 4, hperm = ((h & 1) << 1) | (h >> 1);
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int r = row0 + g * 16 + (lane & 15);
#pragma unroll
    for (int st = 0; st < 4; ++st)
      x[st][g] = r < end ? *reinterpret_cast<const vec8<T>*>(src + (int64_t)r * stride + st * 32 + hperm * 8) : vec8<T>{};
  }
}

// acc (d tile, group) of the wave's rows, times scale[g], as rows of 128: 4 d values a store.
template <typename T, int G>
__device__ __forceinline__ void store_rows(const f32x4 (&acc)[8][G], const float (&scale)[G], T* dst, int64_t stride,
                                           int row0, int end, T* low = nullptr, int64_t low_stride = 0) {
  const int lane = threadIdx.x & 63, h = lane >> 4;
#pragma unroll
  for (int g = 0; g < G; ++g) {
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

// The same as float32 rows of a cut's partial sums, for rows below `end`.
template <int G>
__device__ __forceinline__ void store_part(const f32x4 (&acc)[8][G], const float (&scale)[G], float* dst, int row0, int end) {
  const int lane = threadIdx.x & 63, h = lane >> 4;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int r = row0 + g * 16 + (lane & 15);
    if (r >= end) continue;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(dst + r * kD + dt * 16 + h * 4) = acc[dt][g] * scale[g];
  }
}

__device__ __forceinline__ float across(float x) {   // the four lane groups' sum
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// The end of an iteration: the copies started one iteration ago have landed (`kCopies` of them a wave and iteration), and
// every wave's; no wait for LDS reads, which touch nothing that the next copies write.
template <int kCopies>
__device__ __forceinline__ void landed() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kCopies) : "memory");
}
__device__ __forceinline__ void barrier() { asm volatile("s_barrier" ::: "memory"); }

template <typename T, int G>   // of G groups of 16 queries
struct Forward {
  vec8<T> x[4][G];         // Q^T
  f32x4 acc[8][G];         // O^T
  vec8<T> ops[2 * kLead];  // operand of slot n in ops[n % (2 kLead)]
  f32x4 l[G];              // sums of the rounded P (register 0 of lanes 0-15)
  vec8<T> ones;            // row 0 ones, rows 1-15 zeros
  float sum[G];            // with kKeep: of the unrounded P, this lane's
  float top[G], base[G];   // the maximum that P is taken against, and -log2(e) times it less kShift
  bool far;                // whether base holds one of them too coarsely, or there is none yet
  Places at;
};

// P is held as exp2(log2(e) (S - top) - kShift<T>), where top is the maximum of an earlier unit's row, which has to rise where
// that passes a limit.  bfloat16 has float32's range: P 2^-20 and a limit of 2 leave 2^21 for S to rise by, and 2^-106 for P v, the sums'
// smallest terms (2^-60 takes the same time); past 2 is one bit of the packed form.  In float16 P 2^8 keeps all bits of P down to
// 2^-22 and some of them to 2^-33, and exponents are compared with kLimit, its range, which leaves 2^7 for S to rise by (as fast as P
// itself with 2^9, and zero below 2^-25; P 2^11 and 2^4: 4608 tokens 249 -> 258 us).
template <typename T>
constexpr float kShift = __is_same(T, __bf16) ? 20.0f : -8.0f;
constexpr float kLimit = 15.0f;
template <typename T>
__device__ __forceinline__ float shifted(float x, float y) {   // x y - kShift; in float16 by 4s that take no register from the loop
  return __is_same(T, __bf16) ? __builtin_fmaf(x, y, -kShift<T>) : __builtin_fmaf(x, y, -0.5f * kShift<T>) - 0.5f * kShift<T>;
}
// base is rounded, by up to 2^-12 at this size of top, which takes 2^-12 off the exponents of P, and past 2^28 their range.  Beyond it
// (and before the first maximum) each unit's P are formed again from the differences S - top, which are exact where it matters.
// From the differences at once: 4608 tokens 244 us rather than 237.
constexpr float kFar = 4096.0f;

// What divides a row's sums, and its lse.  l, the sum of the rounded P, is 0 where no key is kept; a NaN among them stays one.
__device__ __forceinline__ float inverse_of(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }
template <typename T>
__device__ __forceinline__ float lse_of(float top, float l, float sum) {
  return l == 0.0f ? -INFINITY : top + (__builtin_amdgcn_logf(sum) + kShift<T>) * kLn2;
}

// Slot n's share of the 8 G elements that a phase of 16 slots turns into P: one multiplied, the one before it
// exponentiated, and the two before that packed.
template <int G, typename Scaled, typename Exp, typename Put>
__device__ __forceinline__ void elements(int n, Scaled&& scaled, Exp&& exp, Put&& put) {
  if constexpr (G == 2) {
    if (n + 2 < 16) scaled(n + 2);
    if (n + 1 < 16) exp(n + 1);
    if (n < 16 && n & 1) put(n - 1);
  } else {
    const int m = n >> 1;
    if ((n & 1) == 0) {
      if (m + 2 < 8) scaled(m + 2);
      if (m + 1 < 8) exp(m + 1);
    } else if (m < 8 && m & 1) {
      put(m - 1);
    }
  }
}

// Phase u: S(u+1) = K(u+1) Q^T and O^T += V(u-1)^T P(u-1)^T on the matrix pipe while the vector units turn S(u) into P(u).
template <bool kPartial, bool kKeep, typename T, int G, typename Hook>
__device__ __forceinline__ void forward_phase(Forward<T, G>& w, const f32x4 (&s_cur)[2 * G], f32x4 (&s_next)[2 * G],
                                              const uint32_t (&p_prev)[4 * G], uint32_t (&p_cur)[4 * G], const uint8_t* k_unit,
                                              const uint8_t* v_unit, const uint8_t* k_after, uint32_t bits,
                                              Hook&& hook) {
  f32x4 sv[2 * G];
#pragma unroll
  for (int i = 0; i < 2 * G; ++i) {
    sv[i] = s_cur[i];
    asm volatile("" : "+v"(sv[i]));
  }
  if constexpr (kPartial)
    if (bits != ~0u) leave_out(sv, bits);
  constexpr int kElems = 8 * G;   // of a lane: one a slot, every other slot with one group
  constexpr bool kBits = __is_same(T, __bf16);
  float t[kElems], e[kElems], high = -INFINITY, sum[G] = {};
  uint32_t any = 0;
  auto scaled = [&](int n) { t[n] = __builtin_fmaf(sv[n >> 2][n & 3], kLog2e, w.base[n >> 3]); };
  auto exp = [&](int n) { e[n] = __builtin_amdgcn_exp2f(t[n]); };
  auto put = [&](int n) {
    p_cur[n >> 1] = pack<T>(e[n], e[n + 1]);
    asm volatile("" : "+v"(p_cur[n >> 1]));   // keeps the pack in its slot
    if constexpr (!kBits) high = fmaxf(fmaxf(high, t[n]), t[n + 1]);
    else if (n & 2) any |= p_cur[n >> 1] | p_cur[(n >> 1) - 1];
    if constexpr (kKeep) sum[n >> 3] += e[n] + e[n + 1];
  };
  vec8<T> pb[G];
#pragma unroll
  for (int g = 0; g < G; ++g) pb[g] = packed<T>(p_prev, g);
  scaled(0);
  scaled(1);
  exp(0);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int n = 0; n < 16; ++n) {
    const vec8<T>& a = w.ops[n % (2 * kLead)];
    if (n < 8) {
      const int st = n >> 1, kt = n & 1;
#pragma unroll
      for (int g = 0; g < G; ++g)
        s_next[2 * g + kt] = mfma(a, w.x[st][g], st ? s_next[2 * g + kt] : f32x4{});
    } else {
#pragma unroll
      for (int g = 0; g < G; ++g) w.acc[n - 8][g] = mfma(a, pb[g], w.acc[n - 8][g]);
      if (n == 15) {
#pragma unroll
        for (int g = 0; g < G; ++g) w.l[g] = mfma(w.ones, pb[g], w.l[g]);
      }
    }
    const int m = n + kLead;
    vec8<T>& to = w.ops[m % (2 * kLead)];
    if (m < 8) to = row_operand<T>(k_unit, w.at, m >> 1, m & 1);
    else if (m < 16) to = col_operand<T>(v_unit, w.at, m - 8);
    else to = row_operand<T>(k_after, w.at, (m - 16) >> 1, m & 1);
    elements<G>(n, scaled, exp, put);
    hook(n);
    __builtin_amdgcn_sched_barrier(0);
  }
  // top rises to the row's maximum, what has been summed is scaled, and this unit's P are formed again
  if (w.far || __any(kBits ? (any & 0x40004000u) != 0 : high > kLimit)) {
    bool far = false;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float x = sv[2 * g][0];
#pragma unroll
      for (int n = 1; n < 8; ++n) x = fmaxf(x, sv[2 * g + (n >> 2)][n & 3]);
      x = fmaxf(x, __shfl_xor(x, 16));
      x = fmaxf(fmaxf(x, __shfl_xor(x, 32)), w.top[g]);
      const float factor = __builtin_amdgcn_exp2f((w.top[g] - x) * kLog2e);
      w.top[g] = x;
      w.base[g] = shifted<T>(x, -kLog2e);
      far |= fabsf(x) > kFar;
      sum[g] = 0.0f;
      w.sum[g] *= factor;
      w.l[g] *= factor;   // row 0 of l sits in the lanes 0-15, whose columns are these queries
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) w.acc[dt][g] *= factor;
#pragma unroll
      for (int n = 8 * g; n < 8 * g + 8; ++n) {
        t[n] = shifted<T>(sv[n >> 2][n & 3] - x, kLog2e);
        exp(n);
        if (n & 1) put(n - 1);
      }
    }
    w.far = __any(far);
  }
  if constexpr (kKeep) {
#pragma unroll
    for (int g = 0; g < G; ++g) w.sum[g] += sum[g];
  }
}

constexpr int kKRing = 4, kVRing = 4;   // forward: units of K and of V in LDS

// One wave's 16 G queries from q0, of a block's `first` .. `end` - 1.
template <typename T, bool kMasked, bool kKeep, int G>
__device__ __forceinline__ void forward_wave(const Args& A, uint8_t* smem, const Piece& piece, int b, int h, int first,
                                             int end, int q0) {
  const int lane = threadIdx.x & 63, h4 = lane >> 4, bh = b * A.heads + h;
  Units<kMasked> units(A, b, piece);
  const int n = units.n;
  Forward<T, G> w;
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) w.acc[dt][g] = f32x4{};
    w.l[g] = f32x4{};
    w.sum[g] = 0.0f;
    w.top[g] = kLowest;
    w.base[g] = 0.0f;
  }
  w.far = true;
  if (n) {
    auto k_slot = [&](int i) { return smem + (i & (kKRing - 1)) * kUnitBytes; };
    auto v_slot = [&](int i) { return smem + (kKRing + (i & (kVRing - 1))) * kUnitBytes; };
    const unsigned lds = wave_rows(smem);
    auto k_lds = [&](int i) { return lds + (i & (kKRing - 1)) * kUnitBytes; };
    auto v_lds = [&](int i) { return lds + (kKRing + (i & (kVRing - 1))) * kUnitBytes; };
    const Copies kc(A.k.at<uint16_t>(b, h / A.group), A.k.row, A.keys), vc(A.v.at<uint16_t>(b, h / A.group), A.v.row, A.keys);
    int unit[5];          // of the iterations u .. u + 4
    uint32_t bits[5];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      units.get(i, unit[i], bits[i]);
      kc.start<false>(k_lds(i), unit[i]);
    }
    for (int i = 0; i < 2; ++i) vc.start<false>(v_lds(i), unit[i]);
    load_rows<T>(w.x, A.q.at<T>(b, h), A.q.row, q0, end);
    w.at = places();
    const T one = (T)((lane & 15) == 0 ? 1.0f : 0.0f);
    w.ones = vec8<T>{one, one, one, one, one, one, one, one};
    reinterpret_cast<uint4*>(v_slot(-1))[threadIdx.x] = make_uint4(0, 0, 0, 0);   // V(-1), times P(-1) = 0
    landed<0>();
    for (int i = 0; i < 4; ++i) clear_rows(k_slot(i), bits[i]);
    for (int i = 0; i < 2; ++i) clear_rows(v_slot(i), bits[i]);
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(q0) >= end) {   // no queries: this wave's share of the copies
      __syncthreads();
      const int turns = n > 8 ? (n - 5) / 4 * 4 : 0, all = turns + (n - turns + 2) / 2 * 2;   // as the loops below
      for (int u = 0; u < all; ++u) {
        units.look(u, unit, bits);
        kc.start<false>(k_lds(u), unit[4]);
        vc.start<false>(v_lds(u + 2), unit[2]);
        landed<2>();
        clear_rows(k_slot(u + 3), bits[3]);
        clear_rows(v_slot(u + 1), bits[1]);
        barrier();
        if constexpr (kMasked) units.shift(unit, bits);
      }
    } else {
      f32x4 s0[2 * G], s1[2 * G];
      uint32_t p0[4 * G], p1[4 * G] = {};
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          const vec8<T> a = row_operand<T>(k_slot(0), w.at, st, kt);
#pragma unroll
          for (int g = 0; g < G; ++g) s0[2 * g + kt] = mfma(a, w.x[st][g], st ? s0[2 * g + kt] : f32x4{});
        }
      }
#pragma unroll
      for (int m = 0; m < kLead; ++m) w.ops[m] = row_operand<T>(k_slot(1), w.at, m >> 1, m & 1);
      __syncthreads();   // K(0) has been read: iteration 0 copies K(4) over it
      // r: u's place in the rings; a literal in the unrolled loop, where LDS addresses are then a lane's constants
      auto iteration = [&](auto partial, int u, int r, const f32x4(&s_cur)[2 * G], f32x4(&s_next)[2 * G], const uint32_t(&p_prev)[4 * G],
                           uint32_t(&p_cur)[4 * G]) __attribute__((always_inline)) {
        constexpr bool kPartial = decltype(partial)::value, kAhead = !kMasked && !kPartial;
        if constexpr (!kAhead) units.look(u, unit, bits);
        forward_phase<kPartial, kKeep>(w, s_cur, s_next, p_prev, p_cur, k_slot(r + 1), v_slot(r - 1), k_slot(r + 2), bits[0],
                                    [&](int slot) {
                                      if (slot == 1) kc.start<kAhead>(k_lds(r), kAhead ? units.first + u + 4 : unit[4]);
                                      if (slot == 3) vc.start<kAhead>(v_lds(r + 2), kAhead ? units.first + u + 2 : unit[2]);
                                    });
        landed<2>();
        if constexpr (kPartial) {
          clear_rows(k_slot(r + 3), bits[3]);
          clear_rows(v_slot(r + 1), bits[1]);
        }
        barrier();
        if constexpr (kMasked) units.shift(unit, bits);
      };
      auto turn = [&](auto partial, int u) __attribute__((always_inline)) {
        iteration(partial, u, 0, s0, s1, p1, p0);
        iteration(partial, u + 1, 1, s1, s0, p0, p1);
        iteration(partial, u + 2, 2, s0, s1, p1, p0);
        iteration(partial, u + 3, 3, s1, s0, p0, p1);
      };
      int u = 0;
      // the last unit is out of reach of what a turn copies, clears and starts from
      for (; u + 8 < n; u += 4) turn(std::bool_constant<kMasked>{}, u);
      for (; u <= n; u += 2) {
        iteration(std::true_type{}, u, u, s0, s1, p1, p0);
        iteration(std::true_type{}, u + 1, u + 1, s1, s0, p0, p1);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no copy writes LDS that the block has left
  }
  if (piece.cut >= 0) {
    float one[G];
#pragma unroll
    for (int g = 0; g < G; ++g) one[g] = 1.0f;
    store_part(w.acc, one, A.of_q.part + (int64_t)piece.cut * kQueries * kD, q0 - first, end - first);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int r = q0 - first + g * 16 + (lane & 15);
      const f32x4 x = {w.top[g], __shfl(w.l[g][0], lane & 15), across(w.sum[g]), 0.0f};
      if (h4 == 0 && r < end - first) reinterpret_cast<f32x4*>(A.part_top)[(int64_t)piece.cut * kQueries + r] = x;
    }
    return;
  }
  float scale[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const float l = __shfl(w.l[g][0], lane & 15);
    scale[g] = inverse_of(l);
    if constexpr (kKeep) {
      const float sum = across(w.sum[g]);
      const int r = q0 + g * 16 + (lane & 15);
      if (h4 == 0 && r < end) A.lse[(int64_t)bh * A.queries + r] = lse_of<T>(w.top[g], l, sum);
    }
  }
  T* low = nullptr;
  if constexpr (kKeep) low = static_cast<T*>(A.low) + ((int64_t)b * A.queries * A.heads + h) * kD;
  store_rows<T>(w.acc, scale, A.o.at<T>(b, h), A.o.row, q0, end, low, (int64_t)A.heads * kD);
}

// o of 256 or 192 queries: 32 a wave rather than 64, which leaves a SIMD two waves, whose phases fill each other's gaps; all
// eight read the same K and V units, so LDS is read once per 256 queries x 32 keys.  What kKeep adds: 16 additions a lane and
// phase for lse, and o's second store (4608 tokens: 237 -> 261 us).
template <typename T, bool kMasked, bool kKeep>
__global__ __launch_bounds__(kThreads, 2) void attention_kernel(const Args A) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[(kKRing + kVRing) * kUnitBytes];
  const Piece piece(A.of_q, blockIdx.x, gridDim.x);
  const Rows rows(A, piece);
  if (rows.wide)
    forward_wave<T, kMasked, kKeep, 2>(A, smem, piece, rows.b, rows.h, rows.first, rows.end, rows.q0);
  else
    forward_wave<T, kMasked, kKeep, 1>(A, smem, piece, rows.b, rows.h, rows.first, rows.end, rows.q0);
}

// o of 16 rows, among the queries of all heads that share a key head, so that for a single query of each every key is read
// once.  For few rows: bound by memory, and where few blocks walk many units by its latency.  The four waves walk units of their
// own (every fourth of the block's), each copied into the wave's own LDS two ahead: no barrier, and 64 to 128 KB on their
// way to a CU.  The waves' sums are joined at the end.  One query of 24 heads: 4608 keys 17 us with the join (57 MB, 14 of
// them this kernel), 16896 keys 44 us (4.7 TB/s), 8 x 4608 81 us (5.6 TB/s).  Two blocks of two waves a CU take 5-17% more.
constexpr int kFewWaves = 4, kFewRing = 2;
constexpr int kFewBytes = (2 * kFewRing * kUnit + kFewRows) * kRowBytes;   // of a wave: K ring, V ring, Q

// Starts the copy of a unit's 32 rows by one wave; rows past the last of `rows` repeat it.
__device__ __forceinline__ void start_unit(const Tensor& t, const uint16_t* head, int rows, int unit, unsigned lds) {
  const int lane = threadIdx.x & 63, end = min(rows - 1 - unit * kUnit, kUnit - 1);
  const uint32_t row = (uint32_t)t.row * 2;
  const char* base = reinterpret_cast<const char*>(head) + (uint64_t)(uint32_t)unit * (row * kUnit);
#pragma unroll
  for (int i = 0; i < kUnit / 4; ++i) {
    const int r = 4 * i + (lane >> 4);
    flk::dma16_lds(base, min(r, end) * row + (((lane & 15) ^ swz(r)) << 4), lds + i * 4 * kRowBytes);
  }
}

template <typename T, bool kMasked>
__global__ __launch_bounds__(64 * kFewWaves) void attention_few_kernel(const Args A) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kFewWaves * kFewBytes];
  const int lane = threadIdx.x & 63, h4 = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int p = by_xcd(blockIdx.x, gridDim.x), splits = A.of_q.splits, split = p % splits, block = p / splits;
  const int rows = A.group * A.queries, tiles = (rows + kFewRows - 1) / kFewRows, bk = block / tiles;
  const int b = bk / A.kv_heads, hk = bk - b * A.kv_heads, row0 = (block - bk * tiles) * kFewRows;
  uint2 some;   // of a masked entry: 64 of the wave's units, one a lane
  int all = A.k_units;
  if constexpr (kMasked) {
    if (A.mask.bytes) some = find_live(A, b, all);
    else all = A.mask.counts[b];
    all = __builtin_amdgcn_readfirstlane(all);
  }
  const int first = split * (all / splits) + min(split, all % splits), count = all / splits + (split < all % splits);
  const int n = count > wave ? (count - wave + kFewWaves - 1) / kFewWaves : 0;
  uint8_t* mine = smem + wave * kFewBytes;
  const unsigned lds = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)mine);
  uint8_t* const q_rows = mine + 2 * kFewRing * kUnitBytes;

  f32x4 acc[8], l{};
  float sum = 0.0f, top = kLowest;
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) acc[dt] = f32x4{};
  if (n) {
    const uint16_t *k = A.k.at<uint16_t>(b, hk), *v = A.v.at<uint16_t>(b, hk);
    if (kMasked && A.mask.bytes) {
      const int from = first + min(wave + kFewWaves * lane, count - 1);
      some = make_uint2(__shfl(some.x, from), __shfl(some.y, from));
    }
    int unit[3];  // of the iterations i, i + 1 and i + 2
    uint32_t bits[3];
    auto get = [&](int i, int& unit, uint32_t& bits) {
      if constexpr (kMasked) {
        if ((i & 63) == 0 && !A.mask.bytes)
          some = A.mask.live[(int64_t)b * A.k_units + first + min(wave + kFewWaves * (i + lane), count - 1)];
        unit = __builtin_amdgcn_readlane(some.x, i & 63);
        bits = __builtin_amdgcn_readlane(some.y, i & 63);
      } else {
        unit = first + min(wave + kFewWaves * i, count - 1);
        bits = kept(A, b, unit);
      }
    };
    auto k_at = [&](int i) { return (i & (kFewRing - 1)) * kUnitBytes; };
    auto v_at = [&](int i) { return (kFewRing + (i & (kFewRing - 1))) * kUnitBytes; };
    get(0, unit[0], bits[0]);
    get(1, unit[1], bits[1]);
#pragma unroll
    for (int i = 0; i < kFewRows / 4; ++i) {   // row gi * queries + qi is query qi of the key head's query head gi
      const int r = 4 * i + h4, at = min(row0 + r, rows - 1), gi = at / A.queries;
      const uint16_t* src = A.q.at<uint16_t>(b, hk * A.group + gi) + (at - gi * A.queries) * A.q.row;
      flk::dma16(src + (((lane & 15) ^ swz(r)) << 3), q_rows + i * 4 * kRowBytes);
    }
    for (int i = 0; i < min(n, 2); ++i) {
      start_unit(A.k, k, A.keys, unit[i], lds + k_at(i));
      start_unit(A.v, v, A.keys, unit[i], lds + v_at(i));
    }
    const Places at = places();
    const T one = (T)((lane & 15) == 0 ? 1.0f : 0.0f);
    const vec8<T> ones = {one, one, one, one, one, one, one, one};
    vec8<T> x[4];
    for (int i = 0; i < n; ++i) {
      get(i + 2, unit[2], bits[2]);
      // a unit is 16 copies, K's before V's; those of later units may still be on their way
      if (i + 1 < n) landed<24>();
      else landed<8>();
      if (i == 0)
#pragma unroll
        for (int st = 0; st < 4; ++st) x[st] = row_operand<T>(q_rows, at, st, 0);
      f32x4 s[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int st = 0; st < 4; ++st)
          s[kt] = mfma(row_operand<T>(mine + k_at(i), at, st, kt), x[st], st ? s[kt] : f32x4{});
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // K(i) has been read
      if (i + 2 < n) start_unit(A.k, k, A.keys, unit[2], lds + k_at(i));
      if (bits[0] != ~0u) leave_out(s, bits[0]);
      float most = top;
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, s[e >> 2][e & 3]);
      most = fmaxf(most, __shfl_xor(most, 16));
      most = fmaxf(most, __shfl_xor(most, 32));
      if (__any(most > top)) {
        const float f = __builtin_amdgcn_exp2f((top - most) * kLog2e);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) acc[dt] *= f;
        l *= f;
        sum *= f;
        top = most;
      }
      float e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j >> 2][j & 3] - top, kLog2e, -kShift<T>));
        sum += e[j];
      }
      const uint32_t words[4] = {pack<T>(e[0], e[1]), pack<T>(e[2], e[3]), pack<T>(e[4], e[5]), pack<T>(e[6], e[7])};
      const vec8<T> w = packed<T>(words, 0);
      l = mfma(ones, w, l);
      if (i + 2 < n) landed<24>();
      else if (i + 1 < n) landed<16>();
      else landed<0>();
      if (bits[0] != ~0u) {   // 0 * what the rows left out hold would be NaN for infinities
#pragma unroll
        for (int j = 0; j < kUnit / 4; ++j)
          if (!(bits[0] >> (4 * j + h4) & 1))
            *reinterpret_cast<uint4*>(mine + v_at(i) + j * 4 * kRowBytes + lane * 16) = make_uint4(0, 0, 0, 0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) acc[dt] = mfma(col_operand<T>(mine + v_at(i), at, dt), w, acc[dt]);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // V(i) has been read
      if (i + 2 < n) start_unit(A.v, v, A.keys, unit[2], lds + v_at(i));
      unit[0] = unit[1];
      bits[0] = bits[1];
      unit[1] = unit[2];
      bits[1] = bits[2];
    }
  }

  // the waves' sums, through LDS that the wave itself has done with
  constexpr int kPitch = kD + 4;   // floats of a row
  float* sums = reinterpret_cast<float*>(mine);
  sum = across(sum);
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(sums + (lane & 15) * kPitch + dt * 16 + h4 * 4) = acc[dt];
  if (h4 == 0) *reinterpret_cast<f32x4*>(sums + kFewRows * kPitch + lane * 4) = f32x4{top, l[0], sum, 0.0f};
  __syncthreads();
  const int row = threadIdx.x >> 4, d = (threadIdx.x & 15) * 8;
  if (row0 + row >= rows) return;
  f32x4 t[kFewWaves], o[2] = {};
  top = kLowest;
#pragma unroll
  for (int i = 0; i < kFewWaves; ++i) {
    t[i] = *reinterpret_cast<const f32x4*>(smem + i * kFewBytes + (kFewRows * kPitch + row * 4) * 4);
    top = fmaxf(top, t[i][0]);
  }
  float total = 0.0f;
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kFewWaves; ++i) {
    const float f = __builtin_amdgcn_exp2f((t[i][0] - top) * kLog2e);
    const f32x4* from = reinterpret_cast<const f32x4*>(smem + i * kFewBytes + (row * kPitch + d) * 4);
    o[0] += from[0] * f;
    o[1] += from[1] * f;
    total += t[i][1] * f;
    sum += t[i][2] * f;
  }
  const int gi = (row0 + row) / A.queries, qi = row0 + row - gi * A.queries, h = hk * A.group + gi;
  if (splits > 1) {   // as if a head's queries had blocks of their own
    const int blocks = (A.queries + kFewRows - 1) / kFewRows;
    const int64_t of = (int64_t)(b * A.heads + h) * blocks + qi / kFewRows, at = (of * splits + split) * kFewRows + qi % kFewRows;
    f32x4* part = reinterpret_cast<f32x4*>(A.of_q.part + at * kD + d);
    part[0] = o[0];
    part[1] = o[1];
    if (d == 0) reinterpret_cast<f32x4*>(A.part_top)[at] = f32x4{top, total, sum, 0.0f};
    return;
  }
  const float scale = inverse_of(total);
  uint32_t high[4], low[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y0 = o[i >> 1][2 * (i & 1)] * scale, y1 = o[i >> 1][2 * (i & 1) + 1] * scale;
    high[i] = pack<T>(y0, y1);
    low[i] = pack<T>(y0 - (float)(T)y0, y1 - (float)(T)y1);
  }
  *reinterpret_cast<uint4*>(A.o.at<T>(b, h) + (int64_t)qi * A.o.row + d) = make_uint4(high[0], high[1], high[2], high[3]);
  if (!A.lse) return;
  *reinterpret_cast<uint4*>(static_cast<T*>(A.low) + (((int64_t)b * A.queries + qi) * A.heads + h) * kD + d) =
      make_uint4(low[0], low[1], low[2], low[3]);
  if (d == 0) A.lse[(int64_t)(b * A.heads + h) * A.queries + qi] = lse_of<T>(top, total, sum);
}

// float16 holds P and dS backwards times powers of two, undone at the end: P 2^kUp, and dS 2^e where
//   |dS_ij| <= |g_i| |v_j| + |delta_i| <= 2 max(|g_i| |v_j|, |delta_i|)
// shows that 2^e may take it to 2^15.  Unscaled, P and dS of 2^-14 and less lose bits and those below 2^-25 all, at 4608 tokens already for
// gradients of 2^-10.  e is a row's own for dq, by the v that its wave walks, and one for dk's wave of 32 keys, by the rows that
// it walks: a block reads as many norms as units.  They cost the stats' launch a pass over v, and the second wave of dk a
// multiplication an element, us of fp16 with gradients, 24 heads: 4608 tokens 1106 rather than 1073, 512 60 and 58, 40 queries of
// 16896 keys 302 and 271.
template <typename T>
constexpr bool kHalf = !__is_same(T, __bf16);
constexpr int kUp = 14;
__device__ __forceinline__ int up_of(float x) {   // x: that max, squared
  return kUp - ((__builtin_amdgcn_frexp_expf(x) + 1) >> 1);
}
__device__ __forceinline__ float power_of(int e) { return __builtin_ldexpf(1.0f, e); }
__device__ __forceinline__ float uniform(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}
template <typename T>
__device__ __forceinline__ float square_of(const vec8<T>& x) {
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum += (float)x[e] * (float)x[e];
  return sum;
}
__device__ __forceinline__ float most_lane(float x, int lanes) {   // of `lanes` neighbours
  for (int d = lanes >> 1; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}

// The most |v|^2 of the units that a wave walks.
template <bool kMasked>
__device__ __forceinline__ float most_v(const Args& A, int b, int h, const Units<kMasked>& units) {
  const f32x4* at = reinterpret_cast<const f32x4*>(A.norms) + (int64_t)A.batch * A.heads * A.q_units * 2 +
                    ((int64_t)b * A.kv_heads + h) * A.k_units;
  float x = 0.0f;
  for (int i = threadIdx.x & 63; i < units.n; i += 256) {
    f32x4 y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = min(i + 64 * j, units.n - 1);
      y[j] = at[kMasked ? units.live[n].x : units.first + n];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) x = fmaxf(fmaxf(fmaxf(x, y[j][0]), y[j][1]), fmaxf(y[j][2], y[j][3]));
  }
  return most_lane(x, 64);
}
// The most |do|^2 and delta^2 of n units.
__device__ __forceinline__ float2 most_do(const Args& A, int64_t first, int n) {
  const f32x4* at = reinterpret_cast<const f32x4*>(A.norms) + first * 2;
  float x = 0.0f, y = 0.0f;
  for (int i = threadIdx.x & 63; i < 2 * n; i += 256) {
    f32x4 z[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] = at[min(i + 64 * j, 2 * n - 1)];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x = fmaxf(fmaxf(x, z[j][0]), z[j][2]);
      y = fmaxf(fmaxf(y, z[j][1]), z[j][3]);
    }
  }
  return make_float2(most_lane(x, 64), most_lane(y, 64));
}

// kFrom: dP's sums start from -delta, which spares an addition an element and takes six registers that a masked pass's loop does
// not have (16896 tokens with gradients 12.40 ms rather than 12.53).
template <typename T, int G, bool kFrom>
struct Dq {
  vec8<T> x[4][G], g[4][G];   // Q^T, dO^T
  f32x4 acc[8][G];            // dQ^T
  vec8<T> ops[2 * kLead];
  float lse[G];               // in float16 less the logarithm of what dS is held times
  std::conditional_t<kFrom, f32x4, float> delta[G];   // -delta
  Places at;
};

template <typename T, int G, bool kFrom>
__device__ __forceinline__ f32x4 start_of(const Dq<T, G, kFrom>& w, int g) {
  if constexpr (kFrom) return w.delta[g];
  return f32x4{};
}

// Phase u: S(u+1) = K(u+1) Q^T, dP(u+1) = V(u+1) dO^T and dQ^T += K(u-1)^T dS(u-1)^T, while dS(u) is formed.
template <bool kPartial, typename T, int G, bool kFrom, typename Hook>
__device__ __forceinline__ void dq_phase(Dq<T, G, kFrom>& w, const f32x4 (&s_cur)[2 * G], const f32x4 (&d_cur)[2 * G],
                                         f32x4 (&s_next)[2 * G], f32x4 (&d_next)[2 * G], const uint32_t (&p_prev)[4 * G],
                                         uint32_t (&p_cur)[4 * G], const uint8_t* k_unit, const uint8_t* v_unit,
                                         const uint8_t* k_before, const uint8_t* k_after, uint32_t bits,
                                         Hook&& hook) {
  f32x4 sv[2 * G], dv[2 * G];
#pragma unroll
  for (int i = 0; i < 2 * G; ++i) {
    sv[i] = s_cur[i];
    dv[i] = d_cur[i];
    asm volatile("" : "+v"(sv[i]), "+v"(dv[i]));
  }
  if constexpr (kPartial)
    if (bits != ~0u) leave_out(sv, bits);
  float t[8 * G], e[8 * G];
  auto scaled = [&](int n) { t[n] = (sv[n >> 2][n & 3] - w.lse[n >> 3]) * kLog2e; };
  auto exp = [&](int n) { e[n] = __builtin_amdgcn_exp2f(t[n]); };
  auto put = [&](int n) {
    float x = dv[n >> 2][n & 3], y = dv[n >> 2][(n & 3) + 1];
    if constexpr (!kFrom) {
      x += w.delta[n >> 3];
      y += w.delta[n >> 3];
    }
    p_cur[n >> 1] = pack<T>(e[n] * x, e[n + 1] * y);
    asm volatile("" : "+v"(p_cur[n >> 1]));
  };
  vec8<T> pb[G];
#pragma unroll
  for (int g = 0; g < G; ++g) pb[g] = packed<T>(p_prev, g);
  scaled(0);
  scaled(1);
  exp(0);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int n = 0; n < 24; ++n) {
    const vec8<T>& a = w.ops[n % (2 * kLead)];
    const int st = (n & 7) >> 1, kt = n & 1;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (n < 8) s_next[2 * g + kt] = mfma(a, w.x[st][g], st ? s_next[2 * g + kt] : f32x4{});
      else if (n < 16) d_next[2 * g + kt] = mfma(a, w.g[st][g], st ? d_next[2 * g + kt] : start_of(w, g));
      else w.acc[n - 16][g] = mfma(a, pb[g], w.acc[n - 16][g]);
    }
    const int m = n + kLead;
    vec8<T>& to = w.ops[m % (2 * kLead)];
    if (m < 8) to = row_operand<T>(k_unit, w.at, m >> 1, m & 1);
    else if (m < 16) to = row_operand<T>(v_unit, w.at, (m - 8) >> 1, m & 1);
    else if (m < 24) to = col_operand<T>(k_before, w.at, m - 16);
    else to = row_operand<T>(k_after, w.at, (m - 24) >> 1, m & 1);
    elements<G>(n, scaled, exp, put);
    hook(n);
    __builtin_amdgcn_sched_barrier(0);
  }
}

constexpr int kDqKRing = 6, kDqVRing = 3;

template <typename T, bool kMasked, int G>
__device__ __forceinline__ void dq_wave(const Args& A, uint8_t* smem, const Piece& piece, int b, int h, int first, int end,
                                        int q0) {
  const int lane = threadIdx.x & 63, bh = b * A.heads + h;
  Units<kMasked> units(A, b, piece);
  const int n = units.n;
  Dq<T, G, !kMasked> w;
  load_rows<T>(w.g, A.dO.at<T>(b, h), A.dO.row, q0, end);
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int r = q0 + g * 16 + (lane & 15);
    const float* st = A.stats + ((int64_t)bh * A.q_units + r / kUnit) * 2 * kUnit + r % kUnit;
    w.lse[g] = r < end ? st[0] : INFINITY;
    const float delta = r < end ? st[kUnit] : 0.0f;
    if constexpr (kMasked) w.delta[g] = delta;
    else w.delta[g] = f32x4{delta, delta, delta, delta};
  }
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) w.acc[dt][g] = f32x4{};
  if (n) {
    // i: 0 .. 11, a place in K's ring plus up to 5; V's divides it
    auto k_slot = [&](int i) { return smem + (i >= kDqKRing ? i - kDqKRing : i) * kUnitBytes; };
    auto v_slot = [&](int i) { return smem + (kDqKRing + i % kDqVRing) * kUnitBytes; };
    const unsigned lds = wave_rows(smem);
    auto k_lds = [&](int i) { return lds + (i >= kDqKRing ? i - kDqKRing : i) * kUnitBytes; };
    auto v_lds = [&](int i) { return lds + (kDqKRing + i % kDqVRing) * kUnitBytes; };
    const Copies kc(A.k.at<uint16_t>(b, h / A.group), A.k.row, A.keys), vc(A.v.at<uint16_t>(b, h / A.group), A.v.row, A.keys);
    int unit[5];
    uint32_t bits[5];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      units.get(i, unit[i], bits[i]);
      kc.start<false>(k_lds(i), unit[i]);
      if (i < 3) vc.start<false>(v_lds(i), unit[i]);
    }
    load_rows<T>(w.x, A.q.at<T>(b, h), A.q.row, q0, end);
    w.at = places();
    reinterpret_cast<uint4*>(k_slot(kDqKRing - 1))[threadIdx.x] = make_uint4(0, 0, 0, 0);   // K(-1), times dS(-1) = 0
    if constexpr (kHalf<T>) {
      const float v2 = most_v(A, b, h / A.group, units);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float g2 = 0.0f, delta;
#pragma unroll
        for (int st = 0; st < 4; ++st) g2 += square_of<T>(w.g[st][g]);
        if constexpr (kMasked) delta = w.delta[g];
        else delta = w.delta[g][0];
        w.lse[g] -= (float)up_of(fmaxf(across(g2) * v2, delta * delta)) * kLn2;
      }
    }
    landed<0>();
    for (int i = 0; i < 4; ++i) {
      clear_rows(k_slot(i), bits[i]);
      if (i < 3) clear_rows(v_slot(i), bits[i]);
    }
    __syncthreads();
    f32x4 s0[2 * G], s1[2 * G], d0[2 * G], d1[2 * G];
    uint32_t p0[4 * G], p1[4 * G] = {};
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        const vec8<T> a = row_operand<T>(k_slot(0), w.at, st, kt), c = row_operand<T>(v_slot(0), w.at, st, kt);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          s0[2 * g + kt] = mfma(a, w.x[st][g], st ? s0[2 * g + kt] : f32x4{});
          d0[2 * g + kt] = mfma(c, w.g[st][g], st ? d0[2 * g + kt] : start_of(w, g));
        }
      }
    }
#pragma unroll
    for (int m = 0; m < kLead; ++m) w.ops[m] = row_operand<T>(k_slot(1), w.at, m >> 1, m & 1);
    __syncthreads();   // V(0) has been read: iteration 0 copies V(3) over it
    // r: u's place in K's ring
    auto iteration = [&](auto partial, int u, int r, const f32x4(&s_cur)[2 * G], const f32x4(&d_cur)[2 * G],
                         f32x4(&s_next)[2 * G],
                         f32x4(&d_next)[2 * G], const uint32_t(&p_prev)[4 * G], uint32_t(&p_cur)[4 * G]) __attribute__((always_inline)) {
      constexpr bool kPartial = decltype(partial)::value, kAhead = !kMasked && !kPartial;
      if constexpr (!kAhead) units.look(u, unit, bits);
      dq_phase<kPartial>(w, s_cur, d_cur, s_next, d_next, p_prev, p_cur, k_slot(r + 1), v_slot(r + 1), k_slot(r + 5),
                      k_slot(r + 2), bits[0], [&](int slot) {
                        if (slot == 1) kc.start<kAhead>(k_lds(r + 4), kAhead ? units.first + u + 4 : unit[4]);
                        if (slot == 3) vc.start<kAhead>(v_lds(r), kAhead ? units.first + u + 3 : unit[3]);
                      });
      landed<2>();
      if constexpr (kPartial) {
        clear_rows(k_slot(r + 3), bits[3]);
        clear_rows(v_slot(r + 2), bits[2]);
      }
      barrier();
      if constexpr (kMasked) units.shift(unit, bits);
    };
    auto turn = [&](auto partial, int u) __attribute__((always_inline)) {
#pragma unroll
      for (int r = 0; r < kDqKRing; r += 2) {
        iteration(partial, u + r, r, s0, d0, s1, d1, p1, p0);
        iteration(partial, u + r + 1, r + 1, s1, d1, s0, d0, p0, p1);
      }
    };
    int u = 0, r = 0;
    for (; u + 10 < n; u += kDqKRing) turn(std::bool_constant<kMasked>{}, u);
    for (; u <= n; u += 2) {
      iteration(std::true_type{}, u, r, s0, d0, s1, d1, p1, p0);
      iteration(std::true_type{}, u + 1, r + 1, s1, d1, s0, d0, p0, p1);
      r = r + 2 == kDqKRing ? 0 : r + 2;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  float down[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    down[g] = 1.0f;
    if constexpr (kHalf<T>) {   // what the difference came to: none of it where lse is far past it
      const int r = q0 + g * 16 + (lane & 15);
      const float lse = r < end ? A.stats[((int64_t)bh * A.q_units + r / kUnit) * 2 * kUnit + r % kUnit] : INFINITY;
      if (lse != INFINITY) down[g] = __builtin_amdgcn_exp2f((w.lse[g] - lse) * kLog2e);
    }
  }
  if (piece.cut >= 0) {
    store_part(w.acc, down, A.of_q.part + (int64_t)piece.cut * kQueries * kD, q0 - first, end - first);
    return;
  }
  store_rows<T>(w.acc, down, A.dq.at<T>(b, h), A.dq.row, q0, end);
}

// dk and dv of 128 keys, 32 a pair of waves: the first holds K^T and dV^T, forms S and P and hands P on through LDS, the
// second holds V^T and dK^T, forms dP and dS one unit later.
template <typename T>
struct Dkv {
  vec8<T> x[4][2];         // K^T (V^T)
  f32x4 acc[8][2];         // dV^T (dK^T)
  vec8<T> ops[2 * kLead];
  f32x4 stat[2];           // this phase's lse (-delta) of the rows of each accumulator
  float more;              // the second wave's: what float16's dS is held times beside P's 2^kUp
  Places at;
};

// The first wave's phase u: S(u+1) = Q(u+1) K^T, then dV^T += dO(u-1)^T P(u-1), while P(u) is formed.  The second's:
// dK^T += Q(u-2)^T dS(u-2), then dP(u) = dO(u) V^T, which starts from -delta, while dS(u-1) = P(u-1) (dP(u-1) - delta) is
// formed from what the first wave left in `hand`.  `after`: the next phase's first operands, `stats` its stats.
template <bool kSecond, typename T, typename Hook>
__device__ __forceinline__ void dkv_phase(Dkv<T>& w, const f32x4 (&s_cur)[4], f32x4 (&s_next)[4], const uint32_t (&p_prev)[8],
                                          uint32_t (&p_cur)[8], const uint8_t* rows, const uint8_t* cols, const uint8_t* after,
                                          const uint8_t* stats, uint8_t* hand, Hook&& hook) {
  const int lane = threadIdx.x & 63;
  f32x4* const mine = reinterpret_cast<f32x4*>(hand) + lane;   // accumulator i at mine[64 i]
  f32x4 sv[4], e4[4], stat_next[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sv[i] = s_cur[i];
    asm volatile("" : "+v"(sv[i]));
    if constexpr (kSecond) e4[i] = mine[64 * i];
  }
  float t[16];
  auto scaled = [&](int n) {
    const float x = sv[n >> 2][n & 3] - w.stat[n >> 2 & 1][n & 3];
    t[n] = kHalf<T> ? __builtin_fmaf(x, kLog2e, (float)kUp) : x * kLog2e;
  };
  auto exp = [&](int n) { e4[n >> 2][n & 3] = __builtin_amdgcn_exp2f(t[n]); };
  auto put = [&](int n) {
    float x = e4[n >> 2][n & 3], y = e4[n >> 2][(n & 3) + 1];
    if constexpr (kSecond) {
      if constexpr (kHalf<T>) {
        x *= w.more;
        y *= w.more;
      }
      x *= sv[n >> 2][n & 3];
      y *= sv[n >> 2][(n & 3) + 1];
    }
    p_cur[n >> 1] = pack<T>(x, y);
    asm volatile("" : "+v"(p_cur[n >> 1]));
  };
  const vec8<T> pb[2] = {packed<T>(p_prev, 0), packed<T>(p_prev, 1)};
  if constexpr (!kSecond) {
    scaled(0);
    scaled(1);
    exp(0);
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int n = 0; n < 16; ++n) {
    const vec8<T>& a = w.ops[n % (2 * kLead)];
    if ((n < 8) != kSecond) {
      const int st = (n & 7) >> 1, kt = n & 1;
#pragma unroll
      for (int g = 0; g < 2; ++g)
        s_next[2 * g + kt] = mfma(a, w.x[st][g], st ? s_next[2 * g + kt] : kSecond ? w.stat[kt] : f32x4{});
    } else {
#pragma unroll
      for (int g = 0; g < 2; ++g) w.acc[n & 7][g] = mfma(a, pb[g], w.acc[n & 7][g]);
    }
    const int m = n + kLead;
    vec8<T>& to = w.ops[m % (2 * kLead)];
    const bool of_rows = (m & 8) == (kSecond ? 8 : 0);
    if (of_rows) to = row_operand<T>(m < 16 ? rows : after, w.at, (m & 7) >> 1, m & 1);
    else to = col_operand<T>(m < 16 ? cols : after, w.at, m & 7);
    if (n >= 9 && n < 11) stat_next[n - 9] = *reinterpret_cast<const f32x4*>(
        stats + (kSecond ? kUnit * 4 : 0) + (n - 9) * 64 + (lane >> 4) * 16);
    if constexpr (kSecond) {
      if (n >= 8) put(2 * (n - 8));
    } else {
      if (n + 2 < 16) scaled(n + 2);
      if (n + 1 < 16) exp(n + 1);
      if (n & 1) put(n - 1);
      if ((n & 3) == 3) mine[64 * (n >> 2)] = e4[n >> 2];
    }
    hook(n);
    __builtin_amdgcn_sched_barrier(0);
  }
  w.stat[0] = stat_next[0];
  w.stat[1] = stat_next[1];
}

constexpr int kQRing = 8, kORing = 4, kStatRing = 8;   // units of Q, of dO and of their stats in LDS
constexpr int kStatBytes = 2 * kUnit * 4, kHandBytes = 4096;
constexpr int kDkvStats = (kQRing + kORing) * kUnitBytes, kDkvHands = kDkvStats + kStatRing * kStatBytes;
constexpr int kDkvBytes = kDkvHands + kWaves * kHandBytes;   // two hands a pair of waves

// The units of the query heads that share a key head, one after the other.
struct Queries {
  const char* at;        // the next unit
  int64_t step, wrap;    // bytes to the one after it, and from a head's last unit to the next head's first
  int units, unit, left; // its index in its head; heads from its on
  __device__ __forceinline__ Queries(const Tensor& t, int b, int h, int units, int heads, int first)
      : step(t.row * kUnit * 2), wrap((t.head - (units - 1) * (t.row * kUnit)) * 2), units(units) {
    const int skipped = first / units;
    unit = first - skipped * units;
    left = heads - skipped;
    at = reinterpret_cast<const char*>(t.at<uint16_t>(b, h + skipped)) + unit * step;
  }
  template <bool kInside>
  __device__ __forceinline__ void next() {   // past the last unit of all: the last; selects, not branches, inside a phase
    if constexpr (kInside) {
      at += step;
      ++unit;
    } else {
      const bool more = unit + 1 < units, wraps = !more && left > 1;
      at += more ? step : wraps ? wrap : 0;
      unit = more ? unit + 1 : wraps ? 0 : unit;
      left -= wraps;
    }
  }
};

template <bool kSecond, bool kGrouped, typename T>
__device__ __forceinline__ void dkv_wave(const Args& A, uint8_t* smem, const Piece& piece, int b, int h, int first, int k0,
                                         bool any) {
  const int lane = threadIdx.x & 63, pair = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
  Dkv<T> w;
  const Tensor& own = kSecond ? A.v : A.k;
  load_rows<T>(w.x, own.at<T>(b, h), own.row, k0, A.keys);
  bool on[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int r = k0 + g * 16 + (lane & 15);
    on[g] = r < A.keys && (kept(A, b, r / kUnit) >> (r % kUnit) & 1);
#pragma unroll
    for (int st = 0; st < 4; ++st) w.x[st][g] = on[g] ? w.x[st][g] : vec8<T>{};
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) w.acc[dt][g] = f32x4{};
  }
  float down[2] = {1.0f, 1.0f};
  if (any) {
    const int from = piece.first(A.q_units * A.group), n = piece.count(A.q_units * A.group);
    auto q_slot = [&](int i) { return smem + (i & (kQRing - 1)) * kUnitBytes; };
    auto o_slot = [&](int i) { return smem + (kQRing + (i & (kORing - 1))) * kUnitBytes; };
    auto stat_slot = [&](int i) { return smem + kDkvStats + (i & (kStatRing - 1)) * kStatBytes; };
    auto hand = [&](int i) { return smem + kDkvHands + (pair * 2 + (i & 1)) * kHandBytes; };
    const unsigned lds = wave_rows(smem);
    auto q_lds = [&](int i) { return lds + (i & (kQRing - 1)) * kUnitBytes; };
    auto o_lds = [&](int i) { return lds + (kQRing + (i & (kORing - 1))) * kUnitBytes; };
    const unsigned stat_lds = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)smem) + kDkvStats;
    const Copies qc(nullptr, A.q.row, A.queries), oc(nullptr, A.dO.row, A.queries);
    Queries qs(A.q, b, h * A.group, A.q_units, A.group, from), os(A.dO, b, h * A.group, A.q_units, A.group, from);
    const char* stats =
        reinterpret_cast<const char*>(A.stats + (((int64_t)b * A.heads + h * A.group) * A.q_units + from) * 2 * kUnit);
    const char* none = reinterpret_cast<const char*>(A.stats + (int64_t)A.batch * A.heads * A.q_units * 2 * kUnit);
    auto copy = [&](auto inside, const Copies& c, Queries& from, unsigned to) __attribute__((always_inline)) {
      constexpr bool kInside = decltype(inside)::value;
      flk::dma16_lds(from.at, kInside || from.unit != c.last ? c.at : c.at_last, to);
      from.template next<kInside>();
    };
    // every wave copies all of a unit's stats: as many copies a wave as the waits count
    auto copy_stats = [&](auto inside, int i, int r) __attribute__((always_inline)) {
      const char* from = stats + (int64_t)i * kStatBytes;
      if constexpr (!decltype(inside)::value) from = i < n ? from : none;
      flk::dma4_lds(from, lane * 4, stat_lds + (r & (kStatRing - 1)) * kStatBytes);
    };
    for (int i = 0; i < 4; ++i) copy(std::false_type{}, qc, qs, q_lds(i));
    for (int i = 0; i < 3; ++i) {
      if (i < 2) copy(std::false_type{}, oc, os, o_lds(i));
      copy_stats(std::false_type{}, i, i);
    }
    w.at = places();
    // Q(-1), Q(-2), dO(-1) and P(-1), which the first iterations read, times zeros
    reinterpret_cast<uint4*>(q_slot(-1))[threadIdx.x] = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4*>(q_slot(-2))[threadIdx.x] = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4*>(o_slot(-1))[threadIdx.x] = make_uint4(0, 0, 0, 0);
    if (!kSecond)
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<f32x4*>(hand(1))[64 * i + lane] = f32x4{};
    if constexpr (kHalf<T>) {
      int up = kUp;
      if constexpr (kSecond) {
        const float2 most = most_do(A, ((int64_t)b * A.heads + h * A.group) * A.q_units + from, n);
        float v2 = 0.0f;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          float sum = 0.0f;
#pragma unroll
          for (int st = 0; st < 4; ++st) sum += square_of<T>(w.x[st][g]);
          v2 = fmaxf(v2, across(sum));
        }
        up = up_of(fmaxf(most.x * most_lane(v2, 16), most.y));
        w.more = uniform(power_of(up - kUp));
      }
      down[0] = down[1] = uniform(power_of(-up));
    }
    landed<0>();
    __syncthreads();
    f32x4 s0[4] = {}, s1[4];
    uint32_t p0[8], p1[8] = {};
    if constexpr (!kSecond) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          const vec8<T> a = row_operand<T>(q_slot(0), w.at, st, kt);
#pragma unroll
          for (int g = 0; g < 2; ++g) s0[2 * g + kt] = mfma(a, w.x[st][g], s0[2 * g + kt]);
        }
    }
#pragma unroll
    for (int m = 0; m < kLead; ++m)
      w.ops[m] = kSecond ? col_operand<T>(q_slot(-2), w.at, m) : row_operand<T>(q_slot(1), w.at, m >> 1, m & 1);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
      w.stat[kt] = *reinterpret_cast<const f32x4*>(stat_slot(0) + (kSecond ? kUnit * 4 : 0) + kt * 64 + (lane >> 4) * 16);
    // r: u's place in the rings, 8 more or less; inside: no copy of it is of a head's last unit
    auto iteration = [&](auto inside, int u, int r, const f32x4(&s_cur)[4], f32x4(&s_next)[4], const uint32_t(&p_prev)[8],
                         uint32_t(&p_cur)[8]) __attribute__((always_inline)) {
      const uint8_t* rows = kSecond ? o_slot(r) : q_slot(r + 1);
      const uint8_t* cols = kSecond ? q_slot(r - 2) : o_slot(r - 1);
      const uint8_t* after = kSecond ? q_slot(r - 1) : q_slot(r + 2);
      dkv_phase<kSecond>(w, s_cur, s_next, p_prev, p_cur, rows, cols, after, stat_slot(r + 1), hand(kSecond ? r - 1 : r),
                         [&](int slot) {
                           if (slot == 1) copy(inside, qc, qs, q_lds(r + 4));
                           if (slot == 3) copy(inside, oc, os, o_lds(r + 2));
                           if (slot == 5) copy_stats(inside, u + 3, r + 3);
                         });
      if constexpr (!kSecond) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // P is in its hand
      landed<3>();
      barrier();
    };
    int u = 0;
    // A turn copies kQRing units from qs.unit and os.unit on, none a head's last, and the stats of up to u + kQRing + 2, all
    // below n (those of units from n on are `none`); where heads share the keys a turn may pass from one to the next.
    const int inside = kGrouped ? n + 3 - kQRing : min(A.q_units - max(qs.unit, os.unit), n - 2) - kQRing;
    const int end = inside > 0 ? inside : 0;
    for (; u < end; u += kQRing)
#pragma unroll
      for (int r = 0; r < kQRing; r += 2) {
        iteration(std::bool_constant<!kGrouped>{}, u + r, r, s0, s1, p1, p0);
        iteration(std::bool_constant<!kGrouped>{}, u + r + 1, r + 1, s1, s0, p0, p1);
      }
    for (; u < n + 2; u += 2) {   // the second wave's last unit goes into dK at u = n + 1
      iteration(std::false_type{}, u, u, s0, s1, p1, p0);
      iteration(std::false_type{}, u + 1, u + 1, s1, s0, p0, p1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) w.acc[dt][g] = on[g] ? w.acc[dt][g] : f32x4{};
  if (piece.cut >= 0) {   // dv's 128 rows, then dk's
    float* part = A.of_k.part + ((int64_t)piece.cut * 2 + kSecond) * kKeys * kD;
    store_part(w.acc, down, part, k0 - first, min(A.keys - first, kKeys));
    return;
  }
  const Tensor& out = kSecond ? A.dk : A.dv;
  store_rows<T>(w.acc, down, out.at<T>(b, h), out.row, k0, A.keys);
}

// All gradients: blocks of queries and blocks of keys in one launch, so that neither kind's last round leaves CUs idle (a
// launch each, with the stats in the first: 1536 tokens with their forward pass 172 us, now 153; 4608: 1026 and 997).
// 4608 tokens, 24 heads: 726 us without the stats, 1.26 PFLOP/s over the 7 products.
template <typename T, bool kMasked, bool kGrouped>   // kGrouped: query heads share key heads
__global__ __launch_bounds__(kThreads, 2) void attention_backward_kernel(const Args A) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kDkvBytes];
  static_assert(kDkvBytes >= (kDqKRing + kDqVRing) * kUnitBytes);
  const int k_grid = gridDim.x - A.q_grid, p = blockIdx.x;
  const int q_p = A.k_first ? p - k_grid : p, k_p = A.k_first ? p : p - A.q_grid;
  if (A.k_first ? q_p >= 0 : k_p < 0) {
    const Piece piece(A.of_q, q_p, A.q_grid);
    const Rows rows(A, piece);
    if (rows.wide) dq_wave<T, kMasked, 2>(A, smem, piece, rows.b, rows.h, rows.first, rows.end, rows.q0);
    else dq_wave<T, kMasked, 1>(A, smem, piece, rows.b, rows.h, rows.first, rows.end, rows.q0);
    return;
  }
  const int blocks = (A.keys + kKeys - 1) / kKeys;
  const Piece piece(A.of_k, k_p, k_grid);
  const int bh = piece.block / blocks, b = bh / A.kv_heads, h = bh - b * A.kv_heads;
  const int first = (piece.block - bh * blocks) * kKeys;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  bool any = false;
  for (int u = first / kUnit; u < min(A.k_units, (first + kKeys) / kUnit); ++u) any |= kept(A, b, u) != 0;
  const int k0 = first + (wave & 3) * 32;
  if (wave < 4) dkv_wave<false, kGrouped, T>(A, smem, piece, b, h, first, k0, any);
  else dkv_wave<true, kGrouped, T>(A, smem, piece, b, h, first, k0, any);
}

// Partial sums that are `step` floats apart, the first n of kJoined, all asked for at once: a load after the other is a way to
// memory each.
constexpr int kJoined = 8;
__device__ __forceinline__ void parts(const float* at, int step, int n, f32x4 (&y)[kJoined]) {
#pragma unroll
  for (int j = 0; j < kJoined; ++j) {
    const f32x4 t = *reinterpret_cast<const f32x4*>(at + min(j, n - 1) * step);
    y[j] = j < n ? t : f32x4{};
  }
}

// Adds the cuts' partial sums in order: 32 lanes a row, 8 rows of a cut block a block.  kForward: of o, or of the
// gradients, the queries' cut blocks first.  4 us, most of it the launch and the first loads' way to memory.
template <typename T, bool kForward, bool kKeep>
__global__ __launch_bounds__(256) void attention_join_kernel(const Args A, int q_blocks) {
  const int pitch = kForward ? pitch_of(A.of_q.tile) : kQueries;
  const int lane = threadIdx.x & 31, r = blockIdx.x % (pitch / 8) * 8 + (threadIdx.x >> 5);
  int cut_block = blockIdx.x / (pitch / 8);
  const bool of_keys = !kForward && cut_block >= q_blocks;
  if (of_keys) cut_block -= q_blocks;
  const Cuts& cuts = of_keys ? A.of_k : A.of_q;
  const int block = cuts.whole + cut_block, rows = of_keys ? A.keys : A.queries;
  const int per = cuts.tile, heads = of_keys ? A.kv_heads : A.heads;
  const int blocks = (rows + per - 1) / per, bh = block / blocks, b = bh / heads, h = bh - b * heads;
  const int row = (block - bh * blocks) * per + (of_keys ? r % kKeys : r);
  if (row >= rows || (!of_keys && r >= per)) return;
  const int64_t first = ((int64_t)cut_block * cuts.splits * pitch + r) * kD;
  f32x4 x{};
  if constexpr (kForward) {
    // lane i of the row's 32 holds the factors of the cuts i and i + 32
    const f32x4* tops = reinterpret_cast<const f32x4*>(A.part_top) + (int64_t)cut_block * cuts.splits * pitch + r;
    f32x4 t[2];
    float top = kLowest, l = 0.0f, sum = 0.0f, f[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = lane + 32 * i;
      t[i] = at < cuts.splits ? tops[(int64_t)at * pitch] : f32x4{kLowest, 0.0f, 0.0f, 0.0f};
      top = fmaxf(top, t[i][0]);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 32));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[i] = __builtin_amdgcn_exp2f((t[i][0] - top) * kLog2e);
      l += t[i][1] * f[i];
      sum += t[i][2] * f[i];
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      l += __shfl_xor(l, d, 32);
      sum += __shfl_xor(sum, d, 32);
    }
    const float* at = cuts.part + first + lane * 4;
    for (int i = 0; i < cuts.splits; i += kJoined) {
      f32x4 y[kJoined];
      parts(at + (int64_t)i * pitch * kD, pitch * kD, cuts.splits - i, y);
#pragma unroll
      for (int j = 0; j < kJoined; ++j) x += y[j] * __shfl(i + j < 32 ? f[0] : f[1], (i + j) & 31, 32);
    }
    x *= inverse_of(l);
    if constexpr (kKeep) {
      if (lane == 0) A.lse[(int64_t)bh * A.queries + row] = lse_of<T>(top, l, sum);
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = x[i] - (float)(T)x[i];
      T* low = static_cast<T*>(A.low) + (((int64_t)b * A.queries + row) * A.heads + h) * kD + lane * 4;
      *reinterpret_cast<uint2*>(low) = make_uint2(pack<T>(y[0], y[1]), pack<T>(y[2], y[3]));
    }
  } else {
    for (int i = 0; i < cuts.splits; i += kJoined) {
      f32x4 y[kJoined];
      parts(cuts.part + first + (int64_t)i * pitch * kD + lane * 4, pitch * kD, cuts.splits - i, y);
#pragma unroll
      for (int j = 0; j < kJoined; ++j) x += y[j];
    }
  }
  const Tensor& out = kForward ? A.o : !of_keys ? A.dq : r < kKeys ? A.dv : A.dk;
  *reinterpret_cast<uint2*>(out.at<T>(b, h) + (int64_t)row * out.row + lane * 4) =
      make_uint2(pack<T>(x[0], x[1]), pack<T>(x[2], x[3]));
}

// The mask's words and live units, one batch entry a block of 16 waves, a thread a unit, 1024 units a turn: one place
// knows the order of an entry's live units without a second launch.  5 us traced at 3473 keys, a launch and two ways
// to memory.
constexpr int kPlanWaves = 16;
struct MaskBytes {
  const uint8_t* mask;   // NULL: none
  int64_t batch_stride;
  uint32_t* bits;
  uint2* live;
  int* counts;
};
__device__ __forceinline__ void plan_entry(const MaskBytes& m, int entry, int keys, int units, int (&found)[kPlanWaves]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint8_t* row = m.mask + entry * m.batch_stride;
  uint32_t* bits = m.bits + (int64_t)entry * units;
  uint2* live = m.live + (int64_t)entry * units;
  int count = 0;
  for (int u0 = 0; u0 < units; u0 += 64 * kPlanWaves) {
    const uint32_t mine = mask_word(row, u0 + wave * 64, keys);   // keys up to keys + 32767
    const int u = u0 + threadIdx.x;
    const uint64_t any = __ballot(mine != 0);
    if (u < units) bits[u] = mine;
    if (lane == 0) found[wave] = __popcll(any);
    __syncthreads();
    int at = count;
    for (int w = 0; w < kPlanWaves; ++w) {
      if (w < wave) at += found[w];
      count += found[w];
    }
    if (mine) live[at + __popcll(any & ((1ull << lane) - 1))] = make_uint2(u, mine);
    __syncthreads();
  }
  if (threadIdx.x == 0) m.counts[entry] = count;
}

__global__ __launch_bounds__(64 * kPlanWaves) void attention_mask_kernel(const MaskBytes m, int keys, int units) {
  __shared__ int found[kPlanWaves];
  plan_entry(m, blockIdx.x, keys, units, found);
}

// What the gradients need first: the mask's words and lists, in the first A.batch blocks where there is a mask, and every
// row's stats, 16 lanes a row and 128 rows (four units) a block, which reads do, o and low once; in float16 the norms of do's
// rows beside them and, in the blocks behind those, of v's.  Bound by memory: 4608
// tokens of 24 heads 15 us for 85 MB, which the caches partly hold; 16896 66 us, 4.7 TB/s.
template <typename T>
__global__ __launch_bounds__(64 * kPlanWaves) void attention_prepare_kernel(const MaskBytes m, const Args A) {
  __shared__ int found[kPlanWaves];
  const int masks = m.mask ? A.batch : 0;
  if ((int)blockIdx.x < masks) {
    plan_entry(m, blockIdx.x, A.keys, A.k_units, found);
    return;
  }
  const int64_t all = (int64_t)A.batch * A.heads * A.q_units;
  const int64_t unit = (int64_t)(blockIdx.x - masks) * 4 + (threadIdx.x >> 8);   // `all` itself: the unit of no rows
  const int lane = threadIdx.x & 15;
  if constexpr (kHalf<T>) {
    const int64_t of_v = unit - (all + 4) / 4 * 4;
    if (of_v >= (int64_t)A.batch * A.kv_heads * A.k_units) return;
    if (of_v >= 0) {
      const int bh = (int)(of_v / A.k_units), b = bh / A.kv_heads, h = bh - b * A.kv_heads;
      const int first = (int)(of_v - (int64_t)bh * A.k_units) * kUnit + (threadIdx.x >> 4 & 15);
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = first + 16 * i;
        vec8<T> x{};
        if (r < A.keys && (!m.mask || m.mask[b * m.batch_stride + r]))
          x = *reinterpret_cast<const vec8<T>*>(A.v.at<T>(b, h) + (int64_t)r * A.v.row + lane * 8);
        most = fmaxf(most, flk::row16_sum(square_of<T>(x)));
      }
      most = fmaxf(most, __shfl_xor(most, 16));
      most = fmaxf(most, __shfl_xor(most, 32));
      if ((threadIdx.x & 63) == 0) A.norms[all * 8 + of_v * 4 + (threadIdx.x >> 6 & 3)] = most;
      return;
    }
  }
  if (unit > all) return;
  const int bh = (int)(unit / A.q_units), b = bh / A.heads, h = bh - b * A.heads;
  const int first = (int)(unit - (int64_t)bh * A.q_units) * kUnit + (threadIdx.x >> 4 & 15);
  float most_g = 0.0f, most_delta = 0.0f;
  float* st = A.stats + unit * 2 * kUnit + (threadIdx.x >> 4 & 15);
  vec8<T> x[2][3];
  float lse[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = first + 16 * i;
    const bool live = unit < all && r < A.queries;
    lse[i] = -INFINITY;
    if (live) {
      x[i][0] = *reinterpret_cast<const vec8<T>*>(A.dO.at<T>(b, h) + (int64_t)r * A.dO.row + lane * 8);
      x[i][1] = *reinterpret_cast<const vec8<T>*>(A.o.at<T>(b, h) + (int64_t)r * A.o.row + lane * 8);
      x[i][2] = *reinterpret_cast<const vec8<T>*>(static_cast<const T*>(A.low) +
                                                  (((int64_t)b * A.queries + r) * A.heads + h) * kD + lane * 8);
      lse[i] = A.lse[(int64_t)bh * A.queries + r];
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float sum = 0.0f;
    const bool live = lse[i] != -INFINITY;   // a row that keeps no key has no gradient, whatever do holds
#pragma unroll
    for (int e = 0; e < 8; ++e)
      sum += live ? (float)x[i][0][e] * ((float)x[i][1][e] + (float)x[i][2][e]) : 0.0f;
    sum = flk::row16_sum(sum);
    if constexpr (kHalf<T>) {
      most_g = fmaxf(most_g, flk::row16_sum(live ? square_of<T>(x[i][0]) : 0.0f));
      most_delta = fmaxf(most_delta, sum * sum);
    }
    if (lane == 0) {
      st[16 * i] = live ? lse[i] : INFINITY;
      st[16 * i + kUnit] = -sum;
    }
  }
  if constexpr (kHalf<T>) {
    for (int d = 16; d <= 32; d <<= 1) {
      most_g = fmaxf(most_g, __shfl_xor(most_g, d));
      most_delta = fmaxf(most_delta, __shfl_xor(most_delta, d));
    }
    if (unit < all && (threadIdx.x & 63) == 0)
      *reinterpret_cast<float2*>(A.norms + unit * 8 + (threadIdx.x >> 6 & 3) * 2) = make_float2(most_g, most_delta);
  }
}

int units_of(int rows) { return (rows + kUnit - 1) / kUnit; }
int64_t mask_bytes(int batch, int keys) { return ((int64_t)batch * (units_of(keys) * 12LL + 4) + 255) / 256 * 256; }
int64_t stats_bytes(int batch, int heads, int queries) {
  return ((int64_t)batch * heads * units_of(queries) + 1) * 2 * kUnit * 4;
}
int64_t norms_bytes(const Args& A) {
  return (int64_t)A.batch * (2LL * A.heads * A.q_units + (int64_t)A.kv_heads * A.k_units) * 16;
}

// Where the mask's words and lists lie in `workspace`.
MaskBytes mask_in(const void* mask, int64_t batch_stride, Args& A, uint8_t* workspace) {
  MaskBytes m{static_cast<const uint8_t*>(mask), batch_stride, nullptr, nullptr, nullptr};
  if (!mask) return m;
  m.live = reinterpret_cast<uint2*>(workspace);
  m.bits = reinterpret_cast<uint32_t*>(m.live + (int64_t)A.batch * A.k_units);
  m.counts = reinterpret_cast<int*>(m.bits + (int64_t)A.batch * A.k_units);
  A.mask = Mask{m.bits, m.live, m.counts, nullptr, 0};
  return m;
}

// How a launch of equal blocks of `tile` rows, each walking n units, is cut: whole rounds of the 256 CUs, and what is left
// in pieces, where that is estimated to be faster.  Forward and gradients of 1536 tokens: 166 us uncut, 163 cut; of 4608:
// 1071 and 1046.
struct Cut {
  int whole, splits, tile;
  int64_t blocks;
  double time;
  int64_t grid() const { return whole + (blocks - whole) * splits; }
  int64_t cuts() const { return splits > 1 ? (blocks - whole) * splits : 0; }
  int64_t part_rows() const { return cuts() * pitch_of(tile); }
  int64_t bytes() const { return part_rows() * (kD + 4) * 4; }
  Cuts in(uint8_t* workspace) const { return Cuts{whole, splits, tile, reinterpret_cast<float*>(workspace)}; }
};
constexpr int kCUs = 256, kMaxSplits = 64;
// us of a block's first loads and last stores, of the join's launch, and bytes of partial sums written and read a us
constexpr double kFixed = 6.0, kJoin = 5.0, kBytes = 4e6;
double join_time(int64_t cuts, int rows) { return cuts ? cuts * (double)rows * kD * 8 / kBytes : 0.0; }
// unit: us of one.
Cut plan_cut(int64_t blocks, int64_t n, double unit, int rows, int tile) {
  auto rounds = [&](int64_t grid) { return (double)((grid + kCUs - 1) / kCUs); };
  Cut best{(int)blocks, 1, tile, blocks, rounds(blocks) * (n * unit + kFixed)};
  const int64_t whole = blocks / kCUs * kCUs, rest = blocks - whole;
  if (rest == 0 || blocks > 16 * kCUs) return best;
  for (int s = 2; s <= kMaxSplits && 4 * s <= n; ++s) {
    const double time = rounds(whole) * (n * unit + kFixed) + rounds(rest * s) * ((n + s - 1) / s * unit + kFixed) + kJoin +
                        join_time(rest * s, rows);
    if (time < best.time) best = Cut{(int)whole, s, tile, blocks, time};
  }
  return best;
}
// Blocks of 192 queries are considered where they fit one round: there each takes less time than one of 256 (1536 tokens,
// forward and gradients: 163 us, with 256 alone 179; 987 of 36 heads: 147 and 158), while over more rounds the chip's power
// limit lets go of what they would save.
Cut plan_queries(const Args& A, double unit, double unit192) {
  auto plan = [&](int tile, double us) {
    const int64_t blocks = (int64_t)A.batch * A.heads * ((A.queries + tile - 1) / tile);
    return plan_cut(blocks, A.k_units, us, std::min(A.queries, tile), tile);
  };
  const Cut wide = plan(kQueries, unit), narrow = plan(192, unit192);
  return narrow.blocks <= kCUs && narrow.time < wide.time ? narrow : wide;
}
// us of a unit: of a block alone, more for every other that reads other keys, and at memory's rate of a block on each CU that
// does; of the first round of blocks, with its launch, and of each other; of the join's launch, and its for each cut.
constexpr double kFewUnit = 0.32, kFewMore = 0.0013, kFewFull = 0.72, kFewFixed = 4.0, kFewRound = 2.8, kFewJoin = 4.0,
                 kFewCut = 0.06;
int64_t few_blocks(const Args& A) {
  return (int64_t)A.batch * A.kv_heads * (((int64_t)A.group * A.queries + kFewRows - 1) / kFewRows);
}
Cut plan_few(const Args& A) {
  const int64_t blocks = few_blocks(A), joined = (int64_t)A.batch * A.heads * ((A.queries + kFewRows - 1) / kFewRows);
  Cut best{(int)joined, 1, kFewRows, joined, 1e300};
  for (int s = 1; s <= kMaxSplits && (s == 1 || (kFewWaves * s <= A.k_units && blocks * s <= 4 * kCUs)); ++s) {
    const int64_t grid = blocks * s, rounds = (grid + kCUs - 1) / kCUs;
    const int turns = ((A.k_units + s - 1) / s + kFewWaves - 1) / kFewWaves;
    const double others = (double)std::min<int64_t>(grid, kCUs) * A.batch * A.kv_heads / blocks;
    const double unit = std::max(kFewUnit + kFewMore * others, kFewFull * others / kCUs);
    const double time = rounds * (turns * kFewWaves * unit + kFewRound) + kFewFixed - kFewRound +
                        (s > 1 ? kFewJoin + kFewCut * s : 0.0);
    if (time < best.time) best = Cut{s > 1 ? 0 : (int)joined, s, kFewRows, joined, time};
  }
  return best;
}
// Blocks of 16 rows where they take less, by the estimates and kStart more for blocks of 256.  24 heads, us in blocks of 16
// and 256: one query of 512 keys 8.5 and 12.9, of 4608 17 and 20.5 (on 4 key heads 11.4 and 18.9, of 8 entries 85 and 101),
// 64 queries of 4608 33.5 and 23; 128 tokens 5.2 and 11.6, 256 11.1 and 16.6, 384 19.8 and 19.0, 512 24.4 and 21.0.
constexpr double kStart = 3.0;
Cut forward_cut(const Args& A) {
  const Cut few = plan_few(A), many = plan_queries(A, 0.82, 0.69);
  return few.time < many.time + kStart ? few : many;
}

// When the CUs, each taking the next block as it ends one, have done runs of equal blocks.
class Schedule {
  struct Some {
    double at;
    int64_t count;
  } some_[kCUs + 1];   // CUs that are free at the same time, soonest first
  int n_ = 1;

 public:
  Schedule() { some_[0] = Some{0.0, kCUs}; }
  void run(int64_t blocks, double time) {
    while (blocks > 0) {
      const int64_t take = std::min(some_[0].count, blocks);
      const double at = some_[0].at + time;
      blocks -= take;
      if ((some_[0].count -= take) == 0) {
        --n_;
        for (int i = 0; i < n_; ++i) some_[i] = some_[i + 1];
      }
      int i = 0;
      while (i < n_ && some_[i].at < at) ++i;
      if (i < n_ && some_[i].at == at) {
        some_[i].count += take;
      } else {
        for (int j = n_; j > i; --j) some_[j] = some_[j - 1];
        some_[i] = Some{at, take};
        ++n_;
      }
    }
  }
  double end() const { return some_[n_ - 1].at; }
};

// The gradients' launch: how its blocks of queries and of keys are cut, and which come first.
struct Gradients {
  Cut q, k;
  bool k_first;
  double time;
  int64_t bytes() const { return q.bytes() + k.bytes(); }
};
// us of a unit of 32 keys for 256 and for 192 queries, and of 32 queries for 128 keys
constexpr double kDqUnit = 1.1, kDqUnit192 = 0.9, kDkvUnit = 0.85;

Gradients search_gradients(const Args& A) {
  const int64_t k_n = (int64_t)A.q_units * A.group, q_n = A.k_units;
  const int64_t k_blocks = (int64_t)A.batch * A.kv_heads * ((A.keys + kKeys - 1) / kKeys);
  auto q_blocks = [&](int tile) { return (int64_t)A.batch * A.heads * ((A.queries + tile - 1) / tile); };
  const double k_time = k_n * kDkvUnit + kFixed;
  Gradients best{Cut{(int)q_blocks(kQueries), 1, kQueries, q_blocks(kQueries), 0.0},
                 Cut{(int)k_blocks, 1, kKeys, k_blocks, 0.0}, k_time > q_n * kDqUnit + kFixed, 1e300};
  if (best.q.blocks + k_blocks > 32 * kCUs) return best;   // the last round is little of it
  auto consider = [&](const Cut& q, const Cut& k) {
    const double unit = q.tile == kQueries ? kDqUnit : kDqUnit192;
    const double join = q.cuts() + k.cuts() == 0 ? 0.0
                                                 : kJoin + join_time(q.cuts(), std::min(A.queries, q.tile)) +
                                                       join_time(k.cuts(), 2 * std::min(A.keys, kKeys));
    const double q_time = (q_n + q.splits - 1) / q.splits * unit + kFixed;
    const double cut_time = (k_n + k.splits - 1) / k.splits * kDkvUnit + kFixed;
    const double work = q.grid() * q_time + k.whole * k_time + k.cuts() * cut_time;
    if (std::max(work / kCUs, std::max(q_time, k.whole ? k_time : cut_time)) + join >= best.time) return;
    for (const bool k_first : {false, true}) {
      Schedule s;
      if (!k_first) s.run(q.grid(), q_time);
      s.run(k.whole, k_time);
      s.run(k.cuts(), cut_time);
      if (k_first) s.run(q.grid(), q_time);
      if (s.end() + join < best.time) best = Gradients{q, k, k_first, s.end() + join};
    }
  };
  for (const int tile : {kQueries, 192})
    for (const int sq : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
      const int64_t blocks = q_blocks(tile);
      if (sq > 1 && (4 * sq > q_n || blocks * sq > 2 * kCUs)) break;
      const Cut q{sq == 1 ? (int)blocks : 0, sq, tile, blocks, 0.0};
      consider(q, Cut{(int)k_blocks, 1, kKeys, k_blocks, 0.0});
      for (const int sk : {2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
        if (4 * sk > k_n) break;
        if (k_blocks * sk <= 4 * kCUs) consider(q, Cut{0, sk, kKeys, k_blocks, 0.0});
        for (const int rest : {16, 32, 64, 96, 128, 192, 256})
          if (rest < k_blocks) consider(q, Cut{(int)k_blocks - rest, sk, kKeys, k_blocks, 0.0});
      }
    }
  return best;
}

// The search takes up to 25 us, and a call plans twice; a thread keeps what it found for the last shapes.
Gradients plan_gradients(const Args& A) {
  struct Found {
    int sizes[5];
    Gradients plan;
  };
  constexpr int kFound = 32;
  static thread_local Found found[kFound];   // batch 0: none
  const int sizes[5] = {A.batch, A.heads, A.kv_heads, A.queries, A.keys};
  uint32_t hash = 0;
  for (const int x : sizes) hash = hash * 2654435761u + (uint32_t)x;
  Found& f = found[(hash >> 16) % kFound];
  if (!std::equal(sizes, sizes + 5, f.sizes)) {
    f.plan = search_gradients(A);
    std::copy(sizes, sizes + 5, f.sizes);
  }
  return f.plan;
}

bool sizes_ok(int batch, int heads, int kv_heads, int queries, int keys) {
  if (batch < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || queries < 0 || keys < 0) return false;
  if (queries > 1 << 28 || keys > 1 << 28 || batch > 1 << 20) return false;
  auto fits = [&](int heads, int length) {   // batch * heads stays below 2^51
    const int64_t units = (length + 31) / 32, most = kMaxItems / 512;
    return units == 0 || (int64_t)batch * heads <= most / units;
  };
  return fits(heads, queries) && fits(kv_heads, keys);
}

int check_tensor(const void* p, const int64_t* strides) {
  if (!p || !strides) return FLK_E_INVALID;
  if (!flk_host_aligned(p, 16) || strides[0] % 8 || strides[1] % 8 || strides[2] % 8) return FLK_E_ALIGN;
  if (strides[2] < 0 || strides[2] > kMaxRow) return FLK_E_INVALID;
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
  A.q_units = units_of(queries);
  A.k_units = units_of(keys);
  return A;
}

int64_t join_blocks(const Cut& cut) { return cut.splits > 1 ? cut.blocks - cut.whole : 0; }

template <typename T>
void forward(const Args& A, const Cut& cut, hipStream_t s) {
  const bool few = cut.tile == kFewRows;
  const dim3 grid((unsigned)(few ? few_blocks(A) * cut.splits : cut.grid()));
  if (few) {
    if (!A.mask.none()) attention_few_kernel<T, true><<<grid, 64 * kFewWaves, 0, s>>>(A);
    else attention_few_kernel<T, false><<<grid, 64 * kFewWaves, 0, s>>>(A);
  } else if (!A.mask.none()) {
    if (A.lse) attention_kernel<T, true, true><<<grid, kThreads, 0, s>>>(A);
    else attention_kernel<T, true, false><<<grid, kThreads, 0, s>>>(A);
  } else {
    if (A.lse) attention_kernel<T, false, true><<<grid, kThreads, 0, s>>>(A);
    else attention_kernel<T, false, false><<<grid, kThreads, 0, s>>>(A);
  }
  const int joined = (int)join_blocks(cut);
  if (!joined) return;
  const dim3 join((unsigned)(joined * (pitch_of(cut.tile) / 8)));
  if (A.lse) attention_join_kernel<T, true, true><<<join, 256, 0, s>>>(A, joined);
  else attention_join_kernel<T, true, false><<<join, 256, 0, s>>>(A, joined);
}

template <typename T>
void backward(const MaskBytes& mask, const Args& A, const Gradients& plan, hipStream_t s) {
  const int64_t units = (int64_t)A.batch * A.heads * A.q_units + 1;
  const int64_t of_v = kHalf<T> ? (int64_t)A.batch * A.kv_heads * A.k_units : 0;
  const dim3 prepare((unsigned)((mask.mask ? A.batch : 0) + (units + 3) / 4 + (of_v + 3) / 4));
  attention_prepare_kernel<T><<<prepare, 64 * kPlanWaves, 0, s>>>(mask, A);
  auto launch = [&](const Args& of, int64_t blocks) {
    const dim3 grid((unsigned)blocks);
    if (of.mask.bits) {
      if (of.group > 1) attention_backward_kernel<T, true, true><<<grid, kThreads, 0, s>>>(of);
      else attention_backward_kernel<T, true, false><<<grid, kThreads, 0, s>>>(of);
    } else {
      if (of.group > 1) attention_backward_kernel<T, false, true><<<grid, kThreads, 0, s>>>(of);
      else attention_backward_kernel<T, false, false><<<grid, kThreads, 0, s>>>(of);
    }
  };
  const int64_t q_grid = plan.q.grid(), k_grid = plan.k.grid();
  if ((q_grid + k_grid) * kThreads <= kMaxItems) {
    launch(A, q_grid + k_grid);
  } else {   // more work-items than a launch counts: each kind fits one, by sizes_ok
    Args one = A;
    one.k_first = false;
    launch(one, q_grid);
    one.q_grid = 0;
    launch(one, k_grid);
  }
  const int q = (int)join_blocks(plan.q), k = (int)join_blocks(plan.k);
  if (q + k) attention_join_kernel<T, false, false><<<(unsigned)((q + k) * (kQueries / 8)), 256, 0, s>>>(A, q);
}

// Whether the forward pass's waves find the live units themselves, one a lane, which spares a launch (3 x 12 heads of 77
// tokens 9.8 us, with the launch 11.9; 2 x 24 of 512 23.3 and 25.7, 8 x 24 of 2048 406 and 405).
bool waves_find(const Args& A) { return A.k_units <= 64; }

int64_t workspace_of(const Args& A, bool masked, bool backward) {
  if (A.batch == 0 || A.queries == 0 || (A.keys == 0 && backward)) return 0;
  const int64_t mask = masked ? mask_bytes(A.batch, A.keys) : 0;
  if (!backward) return (waves_find(A) ? 0 : mask) + forward_cut(A).bytes();
  return mask + stats_bytes(A.batch, A.heads, A.queries) + norms_bytes(A) + plan_gradients(A).bytes();
}

}  // namespace

extern "C" int flk_attention_plan(int batch, int heads, int kv_heads, int queries, int keys, int masked, int backward,
                                  int64_t* workspace_bytes) {
  if (!workspace_bytes || !sizes_ok(batch, heads, kv_heads, queries, keys)) return FLK_E_INVALID;
  const Args A = sizes(batch, heads, kv_heads, queries, keys);
  *workspace_bytes = workspace_of(A, masked, backward);
  return FLK_OK;
}

extern "C" int flk_attention_blocks(int batch, int heads, int kv_heads, int queries, int keys, int backward, int* blocks) {
  if (!blocks || !sizes_ok(batch, heads, kv_heads, queries, keys)) return FLK_E_INVALID;
  std::fill(blocks, blocks + 8, 0);
  if (batch == 0 || queries == 0 || (keys == 0 && backward)) return FLK_OK;
  const Args A = sizes(batch, heads, kv_heads, queries, keys);
  auto report = [](const Cut& cut, int64_t all, int* to) {
    to[0] = cut.tile;
    to[1] = (int)(all - join_blocks(cut));
    to[2] = (int)join_blocks(cut);
    to[3] = cut.splits;
  };
  if (backward) {
    const Gradients plan = plan_gradients(A);
    report(plan.q, plan.q.blocks, blocks);
    report(plan.k, plan.k.blocks, blocks + 4);
    return FLK_OK;
  }
  const Cut cut = forward_cut(A);
  report(cut, cut.blocks, blocks);
  if (cut.tile == kFewRows) blocks[cut.splits > 1 ? 2 : 1] = (int)few_blocks(A);   // all of them are cut or none
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
  if (!low != !lse) return FLK_E_INVALID;
  if (!flk_host_aligned(low, 16) || !flk_host_aligned(lse, 4)) return FLK_E_ALIGN;
  const int64_t need = workspace_of(A, key_mask, false);
  if (need && (!workspace || workspace_bytes < need)) return FLK_E_SCRATCH;
  if (!flk_host_aligned(workspace, 256)) return FLK_E_ALIGN;
  A.q = tensor(q, q_strides);
  A.o = tensor(o, o_strides);
  A.low = low;
  A.lse = lse;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Cut cut = forward_cut(A);
  uint8_t* parts = static_cast<uint8_t*>(workspace);
  if (key_mask && waves_find(A)) {
    A.mask = Mask{nullptr, nullptr, nullptr, static_cast<const uint8_t*>(key_mask), mask_batch_stride};
  } else if (key_mask) {
    const MaskBytes mask = mask_in(key_mask, mask_batch_stride, A, parts);
    attention_mask_kernel<<<batch, 64 * kPlanWaves, 0, s>>>(mask, keys, A.k_units);
    parts += mask_bytes(batch, keys);
  }
  A.of_q = cut.in(parts);
  A.part_top = A.of_q.part + cut.part_rows() * kD;
  if (dtype == FLK_BF16) forward<__bf16>(A, cut, s);
  else forward<_Float16>(A, cut, s);
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
  Args A = sizes(batch, heads, kv_heads, queries, keys);
  if (!workspace || workspace_bytes < workspace_of(A, key_mask, true)) return FLK_E_SCRATCH;
  if (!flk_host_aligned(workspace, 256)) return FLK_E_ALIGN;
  const int64_t of_mask = key_mask ? mask_bytes(batch, keys) : 0;
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
  const MaskBytes mask = mask_in(key_mask, mask_batch_stride, A, static_cast<uint8_t*>(workspace));
  const Gradients plan = plan_gradients(A);
  A.norms = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(A.stats) + stats_bytes(batch, heads, queries));
  uint8_t* parts = reinterpret_cast<uint8_t*>(A.norms) + norms_bytes(A);
  A.of_q = plan.q.in(parts);
  A.of_k = plan.k.in(parts + plan.q.bytes());
  A.q_grid = (int)plan.q.grid();
  A.k_first = plan.k_first;
  if (dtype == FLK_BF16) backward<__bf16>(mask, A, plan, s);
  else backward<_Float16>(mask, A, plan, s);
  return flk_launch_status();
}

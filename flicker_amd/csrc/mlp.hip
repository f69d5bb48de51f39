// The matrix products of the gated MLP and of its gradients, on bf16 / fp16 MFMA.
//
//   forward   [g | u] = x Win,  h = silu(g) u,  y = h Wout
//   backward  dh = dy Wout^T,  [dg | du] from dh, g, u (swiglu.hip's formulas),
//             dWout = h^T dy,  dWin = x^T [dg | du],  dx = [dg | du] Win^T
//
// Each is D (rows, cols) = A B with float32 sums, computed transposed (D^T = B^T A^T: the MFMA's A
// operand holds 16 columns of D, its B operand 16 rows), so that a lane ends with four neighbouring
// columns of one row.  The gate's product takes g's and u's columns into one tile: a lane that holds
// g of a column holds u of the same column, and h leaves the registers as the only output.  h, y, dgu
// and the gradients are rounded once, to the operands' type, which the matrix cores take; g and u are kept in
// float32 for the backward pass: rounded to 16 bits they would add 1.5 roundings to dg and du.
//
// What bounds them (4096 tokens, width 3 * 1024, hidden 9 * 1024, random bf16; times of one box):
//   * Large products, the MFMA under the chip's power limit: gate 354 us (1.31 PFLOP/s), y 167 us
//     (1.39), dWin 366 us (1.27); the same launches on constant operands take 20% less, at higher
//     clocks.  A library product of 8192^3 reaches 1.37 on the same box.  Whole rounds of tiles count
//     as much: 18 * 16 tiles of 256 x 256 on 256 CUs take two rounds for one and an eighth.
//   * The gate's backward pass (294 us) and the forward pass that keeps g and u (404 us): also the
//     float32 g and u, 302 MB each way, in the epilogue, which no MFMA of the same block covers.
//   * 512 tokens: the weights' latency, one stage ahead (95 us with the weights in the caches, 134 without).
//   * One token: HBM, the weights read once (42 us for 170 MB, two split products and two joins).
// Timed and left: 192 x 192 tiles (no faster a column than 192 x 256), stages of 32 terms in three buffers
// with two 256 x 128 blocks a CU (20% slower), fragment rings of 4 to 8 read 3 to 6 groups ahead
// (all within 3%), barriers 2 to 4 groups before a stage's end (within 2%).

#include <algorithm>
#include <type_traits>

#include "elems.h"

namespace {

using flk::f32x4;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// A block's tile: WN x WM waves across the columns and rows of D, each NF x MF fragments of 16 x 16.
template <int WN, int WM, int NF, int MF, int BUFFERS, int PER_CU, int RING, int LEAD, int BAR, int AHEAD>
struct Geometry {
  static constexpr int kWN = WN, kWM = WM, kNF = NF, kMF = MF;
  static constexpr int kBuffers = BUFFERS;   // stages in LDS
  static constexpr int kPerCU = PER_CU;      // blocks a CU holds
  static constexpr int kRing = RING, kLead = LEAD, kBar = BAR;   // column fragments in flight, see mlp_kernel
  static constexpr int kAhead = AHEAD;       // stages that a touch is ahead of the stage worked on (0: none)
  static constexpr int kWaves = WN * WM, kThreads = 64 * kWaves;
  static constexpr int kTB = 16 * NF * WN, kTA = 16 * MF * WM;
};
typedef Geometry<2, 4, 8, 4, 2, 1, 4, 3, 3, 2> Large;    // 256 columns x 256 rows
typedef Geometry<2, 4, 6, 4, 2, 1, 3, 2, 2, 2> Medium;   // 192 x 256
typedef Geometry<2, 2, 4, 4, 2, 2, 4, 3, 3, 0> Small;    // 128 x 128, two blocks a CU
typedef Geometry<2, 2, 4, 4, 4, 1, 4, 3, 3, 0> Deep;     // 128 x 128, one block a CU with more stages in flight
typedef Geometry<4, 1, 2, 2, 4, 2, 4, 2, 1, 0> Few;      // 128 x 32: few rows, the columns' operand streams through

constexpr int kK = 64;                // inner terms a stage
constexpr int kKBytes = kK * 2;       // of one operand row: a 128-byte line
constexpr int kXcds = 8;
constexpr int kGroup = 4;             // row tiles that sweep the column tiles together

enum Epilogue { kPlain, kGate, kGateBackward, kPartial };

struct Operand {      // rows x inner: element (r, k) at r * stride + k, or, across its memory, k * stride + r
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
  bool stream;        // whether what the launch writes (kGateBackward: gu, which it reads) passes the caches by
  float* partial;     // kPartial: (splits, rows, cols) sums over `stages` stages each
  int splits, stages;
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

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  typedef T pair __attribute__((ext_vector_type(2)));
  const pair p = {(T)lo, (T)hi};
  return __builtin_bit_cast(uint32_t, p);
}

// The 8-term chunk of an inner step's 32 that lane group h4 holds.  The LDS serves a b128 read's lanes l
// and l + 32 together: groups 0 and 2 take neighbouring chunks.
__device__ __forceinline__ int slot_chunk(int h4) { return ((h4 & 1) << 1) | (h4 >> 1); }

// One operand's half of a stage: kT rows x 64 inner terms of 16 bits, in 16-byte chunks.
//
// Along its memory (a row's inner terms are contiguous) the half holds kT lines of 128 bytes, whose 8
// chunks are XOR-swizzled by the row: an operand read takes one chunk each of 16 rows
// (ds_read_b128) and lanes l, l + 32 take neighbouring chunks of the same 8 rows.
//
// Across its memory (neighbouring rows are contiguous) it holds 64 lines of kT elements, one per
// inner term, and an operand read is two ds_read_b64_tr_b16: in each 16 lanes, source lane s points at
// term s / 4 and columns 4 (s % 4) .. +3, and lane i receives column i of the four terms.  32 lanes
// read 8 lines (four terms and the same + 16) x 2 chunks, which the swizzle puts on the 16
// chunk positions of the 256-byte bank line: lines of whole 256 bytes need three bits of the
// term, lines of odd multiples of 128 alternate between the halves and need two.
//
// Copies go from global memory straight into LDS (dma16_at), a wave instruction filling 64 chunks in
// order, so the swizzle chooses what a lane fetches.  Both forms give the same k slots: lane groups
// 0, 1, 2, 3 of an MFMA operand hold terms 0-7, 16-23, 8-15, 24-31 (slot_chunk).
template <typename T, bool kAcross, int kT, int kWaves>
struct Half {
  typedef typename Mfma<T>::vec vec;
  static constexpr int kRows = kT;
  static constexpr int kBytes = kT * kKBytes;
  static constexpr int kCopies = kBytes / 1024 / kWaves;   // copy instructions per wave
  static constexpr int kLine = kAcross ? kT * 2 : kKBytes;
  static constexpr int kLineChunks = kLine / 16;
  static_assert(kBytes % (1024 * kWaves) == 0, "whole copies per wave");

  static __device__ __forceinline__ int swizzle(int line) {
    if constexpr (!kAcross) return (line & 7) ^ ((line >> 3) & 1);
    if constexpr (kLine % 256 == 0) return 2 * ((line & 3) | ((line >> 2) & 4));
    return 2 * (((line >> 1) & 1) | ((line >> 3) & 2));
  }

  const uint8_t* base;          // the tile's first row / column
  int64_t step;                 // bytes from one stage to the next
  uint32_t from[kCopies];       // what this lane fetches, from base
  uint32_t touched;

  // rows / terms beyond the operand repeat its last one; results of repeated rows are never stored, and
  // repeated terms are never fetched (tail).
  template <typename Column>
  __device__ __forceinline__ void init(const Operand& o, int64_t first, int wave, int lane, Column column) {
    const int64_t pitch = o.stride * 2;
    base = static_cast<const uint8_t*>(o.p) + (kAcross ? 0 : first * pitch);
    step = kAcross ? kK * pitch : kKBytes;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int at = (wave * kCopies + i) * 64 + lane, line = at / kLineChunks, chunk = (at % kLineChunks) ^ swizzle(line);
      if constexpr (kAcross)
        from[i] = (uint32_t)(line * (uint32_t)pitch) + 2u * (uint32_t)column(chunk * 8);
      else
        from[i] = (uint32_t)column(line) * (uint32_t)pitch + chunk * 16;
    }
  }
  // Touches one 128-byte line a lane of a stage far ahead, so that the L2 has it when the copies come: line i of
  // the half.  What it brings lands in LDS that nothing reads.  Across, where a half's columns are 48 of g and 48 of
  // u in turn (the gate on Medium), columns 64 i are not where its lines begin: some of them are left out.
  template <typename Column>
  __device__ __forceinline__ void init_touch(const Operand& o, int i, Column column) {
    if constexpr (kAcross)
      touched = (uint32_t)(i / (kT / 64)) * (uint32_t)(o.stride * 2) + 2u * (uint32_t)column(i % (kT / 64) * 64);
    else
      touched = (uint32_t)column(i) * (uint32_t)(o.stride * 2);
  }
  __device__ __forceinline__ void touch(int stage, uint8_t* lds) const { flk::dma4_at(base + stage * step, touched, lds); }
  __device__ __forceinline__ void copy(int i, int stage, uint8_t* lds, int wave) const {
    flk::dma16_at(base + stage * step, from[i], lds + (wave * kCopies + i) * 1024);
  }
  // The last stage where `left` < 64 terms are left: zeros in place of the terms that are not there.
  __device__ __forceinline__ void tail(int stage, int left, uint8_t* lds, int wave, int lane) const {
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int at = (wave * kCopies + i) * 64 + lane, line = at / kLineChunks;
      const int term = kAcross ? line : ((at % kLineChunks) ^ swizzle(line)) * 8;
      uint4 v = {0, 0, 0, 0};
      if (term < left) v = *reinterpret_cast<const uint4*>(base + stage * step + from[i]);
      *reinterpret_cast<uint4*>(lds + at * 16) = v;
    }
  }
};

// A wave's fragments of 16 rows x 32 terms of a half: fragment f, inner step ks.
template <typename T, typename H, bool kAcross, int kFrags>
struct Frags {
  typedef typename Mfma<T>::vec vec;
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  int off[kAcross ? kFrags : 2];   // along: of inner steps 0, 1; across: of fragment f
  __device__ __forceinline__ void init(int first, int lane) {   // first: the wave's first row in the tile
    const int l16 = lane & 15, c4 = slot_chunk(lane >> 4);
    if constexpr (!kAcross) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) off[ks] = (first + l16) * kKBytes + (((4 * ks + c4) ^ H::swizzle(l16)) * 16);
    } else {
      const int line = 8 * c4 + (l16 >> 2);
#pragma unroll
      for (int f = 0; f < kFrags; ++f) {
        const int chunk = (first + f * 16) / 8 + ((l16 >> 1) & 1);
        off[f] = line * H::kLine + ((chunk ^ H::swizzle(line)) * 16) + (l16 & 1) * 8;
      }
    }
  }
  __device__ __forceinline__ vec read(const uint8_t* half, int f, int ks) const {
    if constexpr (!kAcross) {
      return *reinterpret_cast<const vec*>(half + off[ks] + f * 16 * kKBytes);
    } else {
      const uint8_t* p = half + off[f] + ks * 32 * H::kLine;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * H::kLine));
      const s16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(vec, both);
    }
  }
};

// Column tiles of the gate's product: a wave's kCols columns are kCols / 2 of g, then the same of u.
template <int kCols, int kWN>
__device__ __forceinline__ int pair_column(int tile, int c, int hidden) {
  const int wave = c / kCols, i = c % kCols, half = kCols / 2;
  const int col = min(tile * (kWN * half) + wave * half + i % half, hidden - 8 + i % 8);
  return i < half ? col : hidden + col;
}

// Finished values leave through the wave's part of the LDS as rows of kChunks 16-byte chunks, written
// four columns a lane and read back a chunk a lane, so that every store is 16 bytes of a
// contiguous row.
template <int kChunks>
__device__ __forceinline__ int out_swizzle(int row) {
  constexpr int mask = kChunks % 16 == 0 ? 15 : kChunks % 8 == 0 ? 7 : kChunks % 4 == 0 ? 3 : 1;
  return row & mask;
}

// Accesses that leave the caches to others where kStream is set.
template <bool kStream, typename V>
__device__ __forceinline__ void store(V* p, const V& v) {
  if constexpr (kStream)
    __builtin_nontemporal_store(v, p);
  else
    *p = v;
}
template <bool kStream, typename V>
__device__ __forceinline__ V load(const V* p) {
  if constexpr (kStream) return __builtin_nontemporal_load(p);
  return *p;
}

template <bool kStream, typename T, int kChunks, int kRows>
__device__ __forceinline__ void store_rows(const uint8_t* lds, T* d, int64_t stride, int64_t row0, int64_t rows,
                                           int col0, int cols, int lane) {
#pragma unroll
  for (int it = 0; it < (kRows * kChunks + 63) / 64; ++it) {
    const int at = it * 64 + lane, r = at / kChunks, c = at % kChunks;
    if (kRows * kChunks % 64 && r >= kRows) break;
    const u32x4 v = *reinterpret_cast<const u32x4*>(lds + (r * kChunks + (c ^ out_swizzle<kChunks>(r))) * 16);
    if (row0 + r < rows && col0 + c * 8 < cols)
      store<kStream>(reinterpret_cast<u32x4*>(d + (row0 + r) * stride + col0 + c * 8), v);
  }
}

template <typename T, int kChunks>
__device__ __forceinline__ void put4(uint8_t* lds, int row, int col, const float (&x)[4]) {
  *reinterpret_cast<uint2*>(lds + (row * kChunks + ((col >> 3) ^ out_swizzle<kChunks>(row))) * 16 + (col & 4) * 2) =
      uint2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
}

// Logical tile u -> its row and column tiles: kGroup row tiles sweep the column tiles together.
__device__ __forceinline__ void tile_of(int u, int tiles_a, int tiles_b, int& ta, int& tb) {
  const int group_tiles = kGroup * tiles_b, group = u / group_tiles, first = group * kGroup;
  const int rows = min(kGroup, tiles_a - first), in_group = u - group * group_tiles;
  ta = first + in_group % rows;
  tb = in_group / rows;
}

// One tile of D; kPartial: its sum over one range of the inner axis.
template <typename T, bool kAAcross, bool kBAcross, Epilogue kE, typename G>
__global__ __launch_bounds__(G::kThreads, G::kThreads * G::kPerCU / 256) void mlp_kernel(const Product P) {
  constexpr int kNF = G::kNF, kMF = G::kMF, kWM = G::kWM, kTB = G::kTB, kTA = G::kTA, kBuffers = G::kBuffers;
  typedef Half<T, kBAcross, kTB, G::kWaves> HB;
  typedef Half<T, kAAcross, kTA, G::kWaves> HA;
  constexpr int kStage = HB::kBytes + HA::kBytes, kCopies = HB::kCopies + HA::kCopies;
  // A stage is kGroups groups of kMF MFMAs, inner step by inner step, each on one column fragment.  Fragments
  // are read kLead groups ahead into a ring; kBar groups of a stage follow its barrier.
  constexpr int kGroups = 2 * kNF, kRing = G::kRing, kLead = G::kLead, kBar = G::kBar;
  static_assert(kGroups % kRing == 0 && kLead < kRing && kBar <= kLead && kMF <= kNF, "the fragment ring divides a stage");
  constexpr int kAhead = G::kAhead;
  static_assert(kAhead == 0 || (kBuffers == 2 && G::kWaves == 8), "two waits: with a touch in flight, or without");
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kBuffers * kStage + (kAhead ? 2048 : 0)];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wb = wave / kWM, wa = wave % kWM, l16 = lane & 15, h4 = lane >> 4;

  // Blocks are dealt round-robin over the XCDs; each XCD runs a contiguous range of logical tiles, the
  // ranges of a split tile's inner axis one after the other.
  const int xcd = blockIdx.x % kXcds, per = gridDim.x / kXcds, extra = gridDim.x % kXcds;
  int unit = xcd * per + min(xcd, extra) + blockIdx.x / kXcds, ta, tb, range = 0;
  if constexpr (kE == kPartial) {
    range = unit / (P.tiles_a * P.tiles_b);
    unit -= range * (P.tiles_a * P.tiles_b);
  }
  tile_of(unit, P.tiles_a, P.tiles_b, ta, tb);

  HB hb;
  HA ha;
  const int64_t row0 = (int64_t)ta * kTA, col0 = (int64_t)tb * kTB;
  // Blocks of a sweep share their row and column operands.  Each touches its share of both a little before
  // all of them copy the lines, so that one miss serves all (forward and backward 2-4% faster at 4096
  // and 16384 tokens; further ahead, or every block all of its lines, slower).  Sweeps of fewer rows gain nothing.
  const int share_b = min(kGroup, P.tiles_a), share_a = min(8, P.tiles_b);
  const int part_b = (kTB + share_b - 1) / share_b, part_a = (kTA + share_a - 1) / share_a;
  const int turn = (wave & 3) * 64, part = wave < 4 ? part_b : part_a;
  const bool touches = kAhead > 0 && turn < part && P.tiles_a >= kGroup;
  const int line = min((wave < 4 ? ta % share_b : tb % share_a) * part + min(turn + lane, part - 1), (wave < 4 ? kTB : kTA) - 1);
  auto init = [&](auto& half, const Operand& o, int64_t first, auto column) __attribute__((always_inline)) {
    half.init(o, first, wave, lane, column);
    if constexpr (kAhead > 0) half.init_touch(o, min(line, half.kRows - 1), column);
  };
  if constexpr (kE == kGate)
    init(hb, P.b, 0, [&](int c) { return pair_column<16 * kNF, G::kWN>(tb, c, P.hidden); });
  else if constexpr (kBAcross)
    init(hb, P.b, 0, [&](int c) { return min((int)col0 + c, P.b.rows - 8); });
  else
    init(hb, P.b, col0, [&](int r) { return min(r, P.b.rows - 1 - (int)col0); });
  if constexpr (kAAcross)
    init(ha, P.a, 0, [&](int c) { return min((int)row0 + c, P.a.rows - 8); });
  else
    init(ha, P.a, row0, [&](int r) { return min(r, P.a.rows - 1 - (int)row0); });

  // Stages first .. first + stages - 1 of the inner axis; the axis' last may have fewer terms (left).
  const int all = (P.inner + kK - 1) / kK, left = P.inner - (all - 1) * kK;
  const int first = kE == kPartial ? range * P.stages : 0;
  const int stages = kE == kPartial ? min(P.stages, all - first) : all;
  const int whole = first + stages == all && left < kK ? stages - 1 : stages;   // stages that are copied by DMA
  auto copy_some = [&](int s, int from, int to) {   // copy instructions [from, to) of a whole stage
    uint8_t* lds = smem + s % kBuffers * kStage;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      if (i < from || i >= to) continue;
      constexpr int kBoth = 2 * (HB::kCopies < HA::kCopies ? HB::kCopies : HA::kCopies);   // alternating, then the rest
      const bool b = i < kBoth ? i % 2 == 0 : HB::kCopies > HA::kCopies;
      const int k = i < kBoth ? i / 2 : i - kBoth / 2;
      if (b)
        hb.copy(k, first + s, lds, wave);
      else
        ha.copy(k, first + s, lds + HB::kBytes, wave);
    }
  };
  auto tail_stage = [&](int s) {
    uint8_t* lds = smem + s % kBuffers * kStage;
    hb.tail(first + s, left, lds, wave, lane);
    ha.tail(first + s, left, lds + HB::kBytes, wave, lane);
  };
  Frags<T, HB, kBAcross, kNF> fb;
  Frags<T, HA, kAAcross, kMF> fa;
  fb.init(wb * 16 * kNF, lane);
  fa.init(wa * 16 * kMF, lane);

  f32x4 acc[kNF][kMF];
#pragma unroll
  for (int n = 0; n < kNF; ++n)
#pragma unroll
    for (int m = 0; m < kMF; ++m) acc[n][m] = f32x4{};

  // kBuffers stages of two inner steps each.  Fragments are read from the stage as the groups before go; kBar
  // groups before its end -- every wave done reading the stage, the next one landed everywhere (the
  // barrier) -- the stage's buffer begins to take the stage kBuffers on, a copy instruction or two a
  // group (all at once they fill the address units and stall the MFMAs: 4%), and the next stage's
  // first fragments are read.  After the last stage those reads take what is there; nothing uses it.
  // Copies return in order: while kLater whole stages follow the awaited one, theirs may be in flight.
  constexpr int kLater = kBuffers - 2;
  constexpr int kTouch = kGroups - kBar - 4;   // the touch follows the stage's copies
  constexpr int kSpread = (kCopies + kBar + kNF - 1) / (kBar + kNF);   // copy instructions a group
  static_assert(kAhead == 0 || (kBar + kTouch) * kSpread >= kCopies, "the touch comes after the last copy");
#pragma unroll
  for (int s = 0; s < kBuffers; ++s) {
    if (s < whole)
      copy_some(s, 0, kCopies);
    else if (s < stages)
      tail_stage(s);
  }
  if (kLater > 0 && kBuffers <= whole)
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"((kLater + 1) * kCopies) : "memory");
  else
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
  typedef typename Mfma<T>::vec vec;
  vec ring[kRing], a[2][kMF];
  auto read_b = [&](const uint8_t* stage, int g) { return fb.read(stage, g % kNF, g / kNF); };
#pragma unroll
  for (int m = 0; m < kMF; ++m) a[0][m] = fa.read(smem + HB::kBytes, m, 0);
#pragma unroll
  for (int g = 0; g < kLead; ++g) ring[g] = read_b(smem, g);
  for (int s = 0; s < stages; ++s) {
    const uint8_t* cs = smem + s % kBuffers * kStage;
    const uint8_t* ns = smem + (s + 1) % kBuffers * kStage;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int after = g - (kGroups - kBar);   // groups since the barrier
      if (after == 0) {
        if (kLater > 0 && s + kBuffers <= whole)
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(kLater * kCopies) : "memory");
        else if (touches && s + kAhead < whole)
          asm volatile("s_waitcnt vmcnt(1) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (s + kBuffers >= whole && s + kBuffers < stages) tail_stage(s + kBuffers);
      }
      if (after >= 0) {
        if (s + kBuffers < whole) copy_some(s + kBuffers, after * kSpread, (after + 1) * kSpread);
      } else if (kAhead > 0 && g == kTouch) {
        if (touches && s + kAhead < whole) {
          if (wave < 4)
            hb.touch(first + s + kAhead, smem + kBuffers * kStage + wave * 256);
          else
            ha.touch(first + s + kAhead, smem + kBuffers * kStage + wave * 256);
        }
      } else if ((kBar + g) * kSpread < kCopies) {
        if (s > 0 && s + kBuffers - 1 < whole) copy_some(s + kBuffers - 1, (kBar + g) * kSpread, (kBar + g + 1) * kSpread);
      }
#pragma unroll
      for (int m = 0; m < kMF; ++m) acc[g % kNF][m] = Mfma<T>::run(ring[g % kRing], a[g / kNF][m], acc[g % kNF][m]);
      if (after < 0) {
        if (g + kLead < kGroups) ring[(g + kLead) % kRing] = read_b(cs, g + kLead);
        if (g < kMF) a[1][g] = fa.read(cs + HB::kBytes, g, 1);
      } else {
#pragma unroll
        for (int i = 0; i < kLead; ++i)
          if (i * kBar / kLead == after) ring[i % kRing] = read_b(ns, i);
#pragma unroll
        for (int m = 0; m < kMF; ++m)
          if (m * kBar / kMF == after) a[0][m] = fa.read(ns + HB::kBytes, m, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();   // every wave is done reading the stages

  // The lane owns row l16 and columns 4 h4 .. +3 of each 16 x 16 fragment.
  constexpr int kRows = 16 * kMF;
  T* d = static_cast<T*>(P.d);
  const int64_t wrow = row0 + wa * kRows;
  auto finish = [&](auto stream) __attribute__((always_inline)) {
    constexpr bool kStream = decltype(stream)::value;
    (void)kStream;
    if constexpr (kE == kPartial) {
      float* out = P.partial + (int64_t)range * P.a.rows * P.b.rows;
  #pragma unroll
      for (int m = 0; m < kMF; ++m) {
        const int64_t row = wrow + m * 16 + l16;
        if (row >= P.a.rows) continue;
  #pragma unroll
        for (int n = 0; n < kNF; ++n) {
          const int col = (int)col0 + wb * 16 * kNF + n * 16 + h4 * 4;
          if (col < P.b.rows) *reinterpret_cast<f32x4*>(out + row * P.b.rows + col) = acc[n][m];
        }
      }
    } else if constexpr (kE == kPlain) {
      constexpr int kChunks = 2 * kNF;
      uint8_t* out = smem + wave * (kRows * kChunks * 16);
  #pragma unroll
      for (int n = 0; n < kNF; ++n)
  #pragma unroll
        for (int m = 0; m < kMF; ++m) {
          const float x[4] = {acc[n][m][0], acc[n][m][1], acc[n][m][2], acc[n][m][3]};
          put4<T, kChunks>(out, m * 16 + l16, n * 16 + h4 * 4, x);
        }
      store_rows<kStream, T, kChunks, kRows>(out, d, P.d_stride, wrow, P.a.rows, (int)col0 + wb * 16 * kNF, P.b.rows, lane);
    } else if constexpr (kE == kGateBackward) {
      // dh leaves as float32 rows of half the wave's columns at a time; a lane takes 8 columns of a row
      // back, so that g and u are read, and dg and du written, in whole lines.
      constexpr int kPass = kNF / 2, kChunks = kPass * 4, kParts = kPass * 2;   // chunks of 4, parts of 8 columns
      constexpr int kTurns = (kRows * kParts + 63) / 64, kBatch = kTurns % 4 == 0 ? 4 : 3;
      uint8_t* out = smem + wave * (kRows * kChunks * 16);
  #pragma unroll
      for (int pass = 0; pass < 2; ++pass) {
  #pragma unroll
        for (int n = 0; n < kPass; ++n)
  #pragma unroll
          for (int m = 0; m < kMF; ++m) {
            const int r = m * 16 + l16;
            *reinterpret_cast<f32x4*>(out + (r * kChunks + ((n * 4 + h4) ^ out_swizzle<kChunks>(r))) * 16) =
                acc[pass * kPass + n][m];
          }
        const int wcol = (int)col0 + wb * 16 * kNF + pass * kPass * 16;
  #pragma unroll
        for (int first = 0; first < kTurns; first += kBatch) {
          f32x4 g[kBatch][2], u[kBatch][2];
  #pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const int at = (first + i) * 64 + lane, r = at / kParts, col = wcol + at % kParts * 8;
            if (r >= kRows || wrow + r >= P.a.rows || col >= P.hidden) continue;
            const f32x4* src = reinterpret_cast<const f32x4*>(P.gu + (wrow + r) * 2 * P.hidden + col);
            const f32x4* usrc = reinterpret_cast<const f32x4*>(P.gu + (wrow + r) * 2 * P.hidden + P.hidden + col);
            g[i][0] = load<kStream>(src);
            g[i][1] = load<kStream>(src + 1);
            u[i][0] = load<kStream>(usrc);
            u[i][1] = load<kStream>(usrc + 1);
          }
  #pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const int at = (first + i) * 64 + lane, r = at / kParts, part = at % kParts, col = wcol + part * 8;
            if (r >= kRows || wrow + r >= P.a.rows || col >= P.hidden) continue;
            float dg[8], du[8];
  #pragma unroll
            for (int c = 0; c < 2; ++c) {
              const f32x4 dh = *reinterpret_cast<const f32x4*>(
                  out + (r * kChunks + ((part * 2 + c) ^ out_swizzle<kChunks>(r))) * 16);
  #pragma unroll
              for (int j = 0; j < 4; ++j) flk::gate_backward(dh[j], g[i][c][j], u[i][c][j], dg[c * 4 + j], du[c * 4 + j]);
            }
            T* dst = d + (wrow + r) * P.d_stride + col;
            *reinterpret_cast<uint4*>(dst) = uint4{pack2<T>(dg[0], dg[1]), pack2<T>(dg[2], dg[3]), pack2<T>(dg[4], dg[5]),
                                                   pack2<T>(dg[6], dg[7])};
            *reinterpret_cast<uint4*>(dst + P.hidden) = uint4{pack2<T>(du[0], du[1]), pack2<T>(du[2], du[3]),
                                                              pack2<T>(du[4], du[5]), pack2<T>(du[6], du[7])};
          }
        }
      }
    } else {
      constexpr int kHalf = kNF / 2, kChunks = kNF;
      uint8_t* out = smem + wave * (kRows * kChunks * 16);
      const int wcol = tb * (kTB / 2) + wb * 16 * kHalf;
  #pragma unroll
      for (int n = 0; n < kHalf; ++n)
  #pragma unroll
        for (int m = 0; m < kMF; ++m) {
          const f32x4 g = acc[n][m], u = acc[n + kHalf][m];
          const int64_t row = wrow + m * 16 + l16;
          const int col = wcol + n * 16 + h4 * 4;
          if (P.gu && row < P.a.rows && col < P.hidden) {
            float* dst = P.gu + row * 2 * P.hidden + col;
            store<kStream>(reinterpret_cast<f32x4*>(dst), g);
            store<kStream>(reinterpret_cast<f32x4*>(dst + P.hidden), u);
          }
          float x[4];
  #pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = flk::gate(g[i], u[i]);
          put4<T, kChunks>(out, m * 16 + l16, n * 16 + h4 * 4, x);
        }
      store_rows<kStream, T, kChunks, kRows>(out, d, P.d_stride, wrow, P.a.rows, wcol, P.hidden, lane);
    }
  };
  if (P.stream)
    finish(std::true_type{});
  else
    finish(std::false_type{});
}

// Adds the ranges' partial sums in order and finishes as kE says, four columns a lane: of one row of D,
// or for the gate's product four of g and the same four of u.
template <typename T, Epilogue kE>
__global__ __launch_bounds__(256) void mlp_join_kernel(const Product P) {
  const int cols = kE == kGate ? P.hidden : P.b.rows, quads = cols / 4;
  const int64_t range = (int64_t)P.a.rows * P.b.rows, total = (int64_t)P.a.rows * quads;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (int64_t)gridDim.x * 256) {
    const int64_t row = at / quads;
    const int col = (int)(at - row * quads) * 4;
    const float* src = P.partial + row * P.b.rows + col;
    f32x4 x{}, y{};
#pragma unroll 4
    for (int r = 0; r < P.splits; ++r) {
      x += *reinterpret_cast<const f32x4*>(src + r * range);
      if constexpr (kE == kGate) y += *reinterpret_cast<const f32x4*>(src + r * range + P.hidden);
    }
    T* d = static_cast<T*>(P.d) + row * P.d_stride + col;
    float a[4], b[4];
    if constexpr (kE == kGate) {
      if (P.gu) {
        float* gu = P.gu + row * 2 * P.hidden + col;
        *reinterpret_cast<f32x4*>(gu) = x;
        *reinterpret_cast<f32x4*>(gu + P.hidden) = y;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = flk::gate(x[i], y[i]);
    } else if constexpr (kE == kGateBackward) {
      const float* gu = P.gu + row * 2 * P.hidden + col;
      const f32x4 g = *reinterpret_cast<const f32x4*>(gu), u = *reinterpret_cast<const f32x4*>(gu + P.hidden);
#pragma unroll
      for (int i = 0; i < 4; ++i) flk::gate_backward(x[i], g[i], u[i], a[i], b[i]);
      *reinterpret_cast<uint2*>(d + P.hidden) = uint2{pack2<T>(b[0], b[1]), pack2<T>(b[2], b[3])};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = x[i];
    }
    *reinterpret_cast<uint2*>(d) = uint2{pack2<T>(a[0], a[1]), pack2<T>(a[2], a[3])};
  }
}

constexpr int kMaxDim = INT32_MAX - 256;
constexpr int64_t kMaxStride = 1 << 22;   // 256 rows of one operand are addressed in 32 bits
constexpr int64_t kMaxBlocks = 1 << 22;   // work-items of a launch are counted in 32 bits
constexpr int kCUs = 256;
// Outputs larger than this leave the caches alone (nontemporal): what follows reads them from HBM anyway, and
// the operands stay.  4096 tokens, float32 g and u: 464 -> 404 us; at 65 MB the same costs 13%.
constexpr int64_t kStreamBytes = 80 << 20;

enum Tile { kLarge, kMedium, kSmall, kDeep, kFew, kTiles };

struct Choice {
  Tile tile;
  int splits;       // ranges of the inner axis; 1: no partial sums
  int stages;       // of each range
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The tile and the split of a product of `rows` x `cols` (all columns, both of the gate's halves): the least
// estimated time over tiles and numbers of ranges.  A tile's blocks run in rounds of what the GPU
// holds; a stage takes the measured time below with one or two blocks on a CU, a round some more to
// fill its first stages and to write its tiles, and split products pay a second launch and write
// and read their partial sums (6 TB/s, mostly from the caches).  What an epilogue reads and writes is not counted: of
// 2961 tokens, 1000 wide, the gate that keeps g and u over 2728 columns takes 72 us where this says 47, its
// backward pass 52 for 24; the tiles compared pay about the same for it.  splits 0: no tile's launch holds the product.
Choice choose(int64_t rows, int64_t cols, int64_t inner, bool a_across) {
  struct Cost {
    int rows, cols, per_cu;
    double stage[2], round;   // microseconds: a stage with one / two blocks on the CU, a round
    bool whole, split;
  };
  static constexpr Cost kCost[kTiles] = {
      {Large::kTA, Large::kTB, Large::kPerCU, {1.42, 0}, 4.0, true, false},
      {Medium::kTA, Medium::kTB, Medium::kPerCU, {1.26, 0}, 3.5, true, false},
      {Small::kTA, Small::kTB, Small::kPerCU, {0.66, 0.92}, 3.0, true, true},
      {Deep::kTA, Deep::kTB, Deep::kPerCU, {0.56, 0}, 3.0, true, true},
      {Few::kTA, Few::kTB, Few::kPerCU, {0.55, 0.95}, 2.0, false, true},
  };
  static constexpr int kSplits[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48};
  const int64_t all = ceil_div(inner, kK);
  Choice best{kLarge, 0, (int)all};
  double least = 1e300;
  for (int tile = 0; tile < kTiles; ++tile) {
    const Cost& c = kCost[tile];
    if (tile == kFew && a_across) continue;
    const int64_t tiles = ceil_div(rows, c.rows) * ceil_div(cols, c.cols), slots = (int64_t)kCUs * c.per_cu;
    for (const int want : kSplits) {
      if (want == 1 ? !c.whole : !c.split || want > all) continue;
      const int64_t stages = ceil_div(all, want), splits = ceil_div(all, stages);
      const int64_t blocks = tiles * splits, rounds = blocks / slots, rest = blocks - rounds * slots;
      if (blocks > kMaxBlocks) continue;
      double us = rounds * (c.stage[c.per_cu - 1] * stages + c.round);
      if (rest) us += c.stage[rest > kCUs] * stages + c.round;
      if (splits > 1) us += 3.0 + 8.0 * splits * rows * cols / 6e6;
      if (us < least) {
        least = us;
        best = Choice{(Tile)tile, (int)splits, (int)stages};
      }
    }
  }
  return best;
}

int64_t partial_bytes(const Choice& c, int64_t rows, int64_t cols) { return c.splits > 1 ? 4 * c.splits * rows * cols : 0; }

template <typename T, bool kAAcross, bool kBAcross, Epilogue kE, typename G>
int launch_tiles(Product& p, hipStream_t s) {
  p.tiles_a = (int)ceil_div(p.a.rows, G::kTA);
  p.tiles_b = (int)(kE == kGate ? ceil_div(p.hidden, G::kTB / 2) : ceil_div(p.b.rows, G::kTB));
  const int64_t blocks = (int64_t)p.tiles_a * p.tiles_b * p.splits;
  mlp_kernel<T, kAAcross, kBAcross, kE, G><<<dim3((unsigned)blocks), G::kThreads, 0, s>>>(p);
  return flk_launch_status();
}

template <typename T, bool kAAcross, bool kBAcross, Epilogue kE>
int launch_typed(Product& p, const Choice& c, hipStream_t s) {
  p.splits = c.splits;
  p.stages = c.stages;
  if (c.splits == 1) {
    switch (c.tile) {
      case kLarge: return launch_tiles<T, kAAcross, kBAcross, kE, Large>(p, s);
      case kMedium: return launch_tiles<T, kAAcross, kBAcross, kE, Medium>(p, s);
      case kSmall: return launch_tiles<T, kAAcross, kBAcross, kE, Small>(p, s);
      default: return launch_tiles<T, kAAcross, kBAcross, kE, Deep>(p, s);
    }
  }
  int st = FLK_OK;
  if (c.tile == kSmall) {
    st = launch_tiles<T, kAAcross, kBAcross, kPartial, Small>(p, s);
  } else if (c.tile == kDeep) {
    st = launch_tiles<T, kAAcross, kBAcross, kPartial, Deep>(p, s);
  } else if constexpr (!kAAcross) {
    st = launch_tiles<T, kAAcross, kBAcross, kPartial, Few>(p, s);
  }
  if (st) return st;
  const int64_t quads = (int64_t)p.a.rows * ((kE == kGate ? p.hidden : p.b.rows) / 4);
  mlp_join_kernel<T, kE><<<dim3((unsigned)std::min(ceil_div(quads, 256), kMaxBlocks)), 256, 0, s>>>(p);
  return flk_launch_status();
}

template <bool kAAcross, bool kBAcross, Epilogue kE>
int launch(Product& p, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  if (p.a.stride > kMaxStride || p.b.stride > kMaxStride) return FLK_E_INVALID;
  const Choice c = choose(p.a.rows, p.b.rows, p.inner, kAAcross);
  if (!c.splits) return FLK_E_INVALID;
  p.stream = (kE == kPlain || !p.gu ? 2LL * p.a.rows * (kE == kGate ? p.hidden : p.b.rows) : 8LL * p.a.rows * p.hidden) > kStreamBytes;
  const int64_t need = partial_bytes(c, p.a.rows, p.b.rows);
  if (need) {
    if (!workspace || workspace_bytes < need) return FLK_E_SCRATCH;
    if (!flk_host_aligned(workspace, 16)) return FLK_E_ALIGN;
    p.partial = static_cast<float*>(workspace);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == FLK_BF16) return launch_typed<__bf16, kAAcross, kBAcross, kE>(p, c, s);
  return launch_typed<_Float16, kAAcross, kBAcross, kE>(p, c, s);
}

bool odd8(int64_t v) { return v % 8 != 0; }

}  // namespace

extern "C" int flk_mlp_plan(int product, int rows, int cols, int inner, int64_t* workspace_bytes) {
  if (product < FLK_MLP_GATE || product > FLK_MLP_MATMUL_AT || rows < 0 || cols < 0 || inner < 0 || !workspace_bytes)
    return FLK_E_INVALID;
  const int64_t columns = product == FLK_MLP_GATE ? 2LL * cols : cols;
  if (rows > kMaxDim || columns > kMaxDim || inner > kMaxDim) return FLK_E_INVALID;
  *workspace_bytes = 0;
  if (!rows || !cols || !inner) return FLK_OK;
  const Choice c = choose(rows, columns, inner, product == FLK_MLP_MATMUL_AT);
  *workspace_bytes = partial_bytes(c, rows, columns);
  return c.splits ? FLK_OK : FLK_E_INVALID;
}

extern "C" const char* flk_mlp_kernel(int product, int rows, int cols, int inner) {
  static constexpr const char* kNames[kTiles][2] = {{"256x256", ""}, {"192x256", ""}, {"128x128 x2", "128x128 x2 split"},
                                                    {"128x128 deep", "128x128 deep split"}, {"", "128x32 split"}};
  int64_t bytes = 0;
  if (flk_mlp_plan(product, rows, cols, inner, &bytes) != FLK_OK || !rows || !cols || !inner) return "";
  const Choice c = choose(rows, product == FLK_MLP_GATE ? 2LL * cols : cols, inner, product == FLK_MLP_MATMUL_AT);
  return kNames[c.tile][c.splits > 1];
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
  return launch<false, true, kGate>(p, dtype, workspace, workspace_bytes, stream);
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
  return launch<false, false, kGateBackward>(p, dtype, workspace, workspace_bytes, stream);
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
  if (a_transposed) return launch<true, true, kPlain>(p, dtype, workspace, workspace_bytes, stream);
  if (b_transposed) return launch<false, false, kPlain>(p, dtype, workspace, workspace_bytes, stream);
  return launch<false, true, kPlain>(p, dtype, workspace, workspace_bytes, stream);
}

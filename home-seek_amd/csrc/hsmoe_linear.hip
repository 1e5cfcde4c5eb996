// Matrix products with bias, activation and residual in their epilogue, dense
// or with one matrix per expert over rows sorted by expert, and their
// gradients.  All three products are one tile kernel: with "rows" the index of
// the output's rows and "cols" that of its contiguous dimension,
//   forward   out[m, n] = sum_k x[m, k] w[n, k]      reduction contiguous in both
//   input     dx[m, k]  = sum_n dz[m, n] w[n, k]     cols operand transposed
//   weights   dw[n, k]  = sum_m dz[m, n] x[m, k]     both transposed
// A transposed operand lies in LDS as it lies in memory and is read through
// ds_read_b64_tr_b16, which hands a lane four values down a column.
#include "hsmoe_common.h"
#include "hsmoe_internal.h"
#include "hsmoe_stage.h"

namespace hsmoe {
namespace {

constexpr int kBK = 64;                     // reduction steps per stage
constexpr int64_t kMaxRange = 0x7fffffe0;   // bytes that one resource covers at most
constexpr int kMaxGroups = 1024;

typedef short s16x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- tiles
// One stage of one operand: kBK reduction steps of kRows rows, bf16.
//   contiguous  [kRows][kBK]: a row's 16-byte chunk c at place c ^ turn(row)
//   transposed  [kBK][kRows]: chunk c of step r at place c ^ turn(r)
// so that the lanes which read together touch different banks.  The loads write
// LDS in lane order, so the lane that fills a place loads that place's chunk.
//
// The matrix instruction hands a lane four results: rows 4 (lane / 16) ..+3 of
// its first operand, the tile's columns.  kCols: block j of that operand takes
// its 16 columns such that the lane's four of blocks 2 P and 2 P + 1 are eight
// in a row (column 32 P + 8 (i / 4) + 4 (j & 1) + i % 4 is row i of block j), so
// that results leave in 16-byte stores of 64 bytes per output row.
template <int kRows, int kWaves, bool kTrans, bool kCols, bool kGated>
struct Operand {
  static constexpr int kBytes = kRows * kBK * 2;
  static constexpr int kLoads = kBytes / 1024 / kWaves;  // 1 KiB instructions per wave and stage
  static_assert(kBytes % (1024 * kWaves) == 0, "every wave loads whole instructions");
  static_assert(!kTrans || kRows >= 128, "a transposed step has the 16 chunks that turn() permutes");

  static constexpr bool kTransposed = kTrans;

  // Contiguous: lanes read 16 rows 0-15, or with kCols 0-3, 8-11, 16-19, 24-27
  // (+ 4).  Transposed: 4 steps r .. r + 3 of one 32-byte piece, or with kCols of
  // four pieces of 8 bytes 16 apart, in four groups 8 steps apart.
  static __device__ __forceinline__ int turn(int row) {
    if (kTrans) return kCols ? (row & 3) << 2 : (row & 3) << 1 | (row & 8);
    return kCols ? (row & 3) | (row >> 1 & 4) : row & 7;
  }

  // Load i of a wave fills 1 KiB of LDS: the lane's row (step, if transposed) and
  // chunk of it there, and the row that it comes from.
  static __device__ __forceinline__ int place(int i, int wave, int lane) {
    const int q = wave * kLoads + i;
    return kTrans ? q * (512 / kRows) + lane / (kRows / 8) : 8 * q + (lane >> 3);
  }
  static __device__ __forceinline__ int chunk(int i, int wave, int lane) {
    return (kTrans ? lane % (kRows / 8) : lane & 7) ^ turn(place(i, wave, lane));
  }
  // kGated: LDS rows are blocks of 16 rows of two matrices in turn.
  static __device__ __forceinline__ int line(int i, int wave, int lane) {
    const int r = place(i, wave, lane);
    return kGated ? (r >> 5) * 16 + (r & 15) : r;
  }
  // Two loads per wave: a wave loads one matrix, which Source::open makes its
  // first (a choice at each load: 49 instead of 36 us, 500 rows, 2 x 4096 x 4096).
  static constexpr bool kOneMatrix = kGated && kLoads == 2;
  static __device__ __forceinline__ bool second(int i) { return kGated && !kOneMatrix && (i >> 1 & 1); }

  // The MFMA operand of block j of a wave whose rows begin at row0 (a multiple
  // of 32): reduction steps 32 kk + 8 (lane / 16) ..+7 of 16 rows.  kGated:
  // blocks j and j + 1 are the same columns of both matrices.
  static __device__ __forceinline__ bf16x8 frag(const char* stage, int row0, int j, int kk, int lane) {
    const int i = lane & 15;
    if (!kTrans) {
      int row = row0 + 16 * j + i;
      if (kCols && kGated)
        row = row0 + 64 * (j >> 2) + 16 * (j & 1) + 4 * (j >> 1 & 1) + 32 * (i >> 3) + 8 * (i >> 2 & 1) + (i & 3);
      else if (kCols)
        row = row0 + 32 * (j >> 1) + 4 * (j & 1) + 8 * (i >> 2) + (i & 3);
      const int place = (4 * kk + (lane >> 4)) ^ (kCols ? (i & 7) : turn(i));
      return *reinterpret_cast<const bf16x8*>(stage + row * (kBK * 2) + place * 16);
    }
    // the 16 lanes of a group address four values each of steps r .. r + 3 and
    // get four values down one column each
    const int r = 32 * kk + 8 * (lane >> 4) + (i >> 2);
    int at;
    if (kCols)
      at = (((row0 >> 3) + 4 * (j >> 1) + (i & 3)) ^ turn(r)) * 16 + 8 * (j & 1);
    else
      at = ((((row0 >> 3) + 2 * j + (i >> 1 & 1)) ^ turn(r)) * 16) + 8 * (i & 1);
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const char* p = stage + r * (kRows * 2) + at;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * kRows * 2));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, v);
  }
};

// What a tile reads of one operand, stage by stage: kRows rows of `count`
// reduction steps, `ld` bytes apart (rows, or steps if transposed).  Reads
// beyond the rows or the steps that there are give zeros: past the resource's
// end, or (steps of contiguous rows) by an offset beyond kFar, ORed in since the
// compiler makes divergent branches around the load of a select.  Stages beyond
// the last read nothing.
template <typename Op>
struct Source {
  static_assert(Op::kLoads % 2 == 0, "two loads of a wave in turn have the lane's chunk at its two places");
  const char* base[2];  // the second matrix: kGated
  uint32_t ld, width;   // width: bytes of a step (transposed), of the whole operand (contiguous)
  uint32_t at[Op::kLoads];
  int edge[2];  // contiguous: the first step of the lane's chunk, in even and odd loads

  // contiguous: `rows` rows of `bytes` each; transposed: steps of `bytes` each
  __device__ __forceinline__ void open(const char* p, const char* second, int64_t ld_, int rows, int64_t bytes, int wave,
                                       int lane) {
    const bool odd = Op::kOneMatrix && (wave & 1);
    base[0] = odd ? second : p;
    base[1] = odd ? p : second;
    ld = (uint32_t)ld_;
    width = Op::kTransposed ? (uint32_t)bytes : (uint32_t)(rows - 1) * ld + (uint32_t)bytes;
#pragma unroll
    for (int i = 0; i < Op::kLoads; ++i)
      at[i] = (uint32_t)Op::line(i, wave, lane) * ld + (uint32_t)Op::chunk(i, wave, lane) * 16;
    edge[0] = Op::chunk(0, wave, lane) * 8;
    edge[1] = Op::chunk(1, wave, lane) * 8;
  }
  // Loads kFrom .. kTo - 1 of the stage of steps first ..+63, `left` of them there
  // (first: times 2 bytes, or ld if transposed, from base).
  template <int kFrom, int kTo>
  __device__ __forceinline__ void load(int64_t first, int left, char* stage, int wave) const {
    if (Op::kTransposed) {
      const int n = left < kBK ? left : kBK;
      const i32x4 r = lds_buf(base[0] + first * ld, n > 0 ? (uint32_t)(n - 1) * ld + width : 0u);
#pragma unroll
      for (int i = kFrom; i < kTo; ++i) lds_load16(r, at[i], stage + (wave * Op::kLoads + i) * 1024);
    } else {
      const uint32_t k = (uint32_t)first * 2, far[2] = {past(edge[0], left), past(edge[1], left)};
#pragma unroll
      for (int i = kFrom; i < kTo; ++i) {
        const i32x4 r = lds_buf(Op::second(i) ? base[1] : base[0], width);
        lds_load16(r, (at[i] + k) | far[i & 1], stage + (wave * Op::kLoads + i) * 1024);
      }
    }
  }
};

// Which of a stage's loads: all, the first or second half of either operand's,
// one operand's.
enum { kPartAll, kPartFirst, kPartSecond, kPartRows, kPartCols };
template <int kValue>
struct Part {
  static constexpr int value = kValue;
};
constexpr Part<kPartAll> kAll;
constexpr Part<kPartFirst> kFirst;
constexpr Part<kPartSecond> kSecond;
constexpr Part<kPartRows> kRowsOnly;
constexpr Part<kPartCols> kColsOnly;

// kStages_: the stages, or one of these (reduce_turns with two or three stages
// of the columns' operand).
constexpr int kTurnsNear = 0, kTurnsFar = -1;

template <int kBR, int kBC, int kWR, int kWC, int kStages_, bool kTR, bool kTC, bool kGated = false>
struct Tile {
  static constexpr int kStages = kStages_ <= 0 ? 2 : kStages_;
  static constexpr bool kTurns = kStages_ <= 0;
  static constexpr int kColStages = kStages_ == kTurnsFar ? 3 : kStages;
  static constexpr int kWaves = kWR * kWC;
  static constexpr int kThreads = kWaves * 64;
  static constexpr int kFR = kBR / kWR / 16, kFC = kBC / kWC / 16;  // 16 x 16 blocks per wave
  static_assert(kFC % (kGated ? 4 : 2) == 0, "eight columns in a row per lane");
  static constexpr bool kRowsTrans = kTR, kColsTrans = kTC;
  using R = Operand<kBR, kWaves, kTR, false, false>;
  using C = Operand<kBC, kWaves, kTC, true, kGated>;
  static constexpr int kStage = R::kBytes + C::kBytes;
  static constexpr int kLds = kStages * R::kBytes + kColStages * C::kBytes;
  static constexpr int kLoads = R::kLoads + C::kLoads;  // per wave and stage

  // Loads of a stage into r_stage and c_stage.
  template <int kPart>
  static __device__ __forceinline__ void load(const Source<R>& rs, int64_t r_first, const Source<C>& cs, int64_t c_first,
                                              int left, char* r_stage, char* c_stage, int wave) {
    constexpr bool kHalf0 = kPart == kPartFirst, kHalf1 = kPart == kPartSecond;
    if constexpr (kPart != kPartCols)
      rs.template load<kHalf1 ? R::kLoads / 2 : 0, kHalf0 ? R::kLoads / 2 : R::kLoads>(r_first, left, r_stage, wave);
    if constexpr (kPart != kPartRows)
      cs.template load<kHalf1 ? C::kLoads / 2 : 0, kHalf0 ? C::kLoads / 2 : C::kLoads>(c_first, left, c_stage, wave);
  }

  static __device__ __forceinline__ void read(const char* r_stage, const char* c_stage, int wr, int wc, int kk, int lane,
                                              bf16x8 (&c)[kFC], bf16x8 (&r)[kFR]) {
#pragma unroll
    for (int j = 0; j < kFC; ++j) c[j] = C::frag(c_stage, wc * kFC * 16, j, kk, lane);
#pragma unroll
    for (int i = 0; i < kFR; ++i) r[i] = R::frag(r_stage, wr * kFR * 16, i, kk, lane);
  }
  static __device__ __forceinline__ void product(const bf16x8 (&c)[kFC], const bf16x8 (&r)[kFR],
                                                 f32x4 (&acc)[kFR][kFC]) {
#pragma unroll
    for (int i = 0; i < kFR; ++i)
#pragma unroll
      for (int j = 0; j < kFC; ++j) acc[i][j] = mfma16x16x32(c[j], r[i], acc[i][j]);
  }
  // One stage's products.
  static __device__ __forceinline__ void multiply(const char* stage, int wr, int wc, int lane, f32x4 (&acc)[kFR][kFC]) {
#pragma unroll
    for (int kk = 0; kk < kBK / 32; ++kk) {
      bf16x8 c[kFC], r[kFR];
      read(stage, stage + R::kBytes, wr, wc, kk, lane, c, r);
      product(c, r, acc);
    }
  }
};

// The reduction with two stages: one is on its way while the other is
// multiplied, and the second workgroup of the CU fills what that leaves idle.
// Every wave waits for its own loads of a stage (and for its LDS reads, whose
// products may come later), then all meet: the stage is whole, and nobody reads
// the one that is loaded next.
template <typename T, typename Load>
__device__ __forceinline__ void reduce_stages(char* lds, int steps, int wr, int wc, int lane, const Load& load,
                                              f32x4 (&acc)[T::kFR][T::kFC]) {
  static_assert(T::kStages == 2, "a stage in use, a stage on its way");
  auto fill = [&](int s, int slot, auto part) {
    load(s, lds + slot * T::kStage, lds + slot * T::kStage + T::R::kBytes, part);
  };
  if (steps > 0) fill(0, 0, kAll);
  for (int s = 0; s < steps; ++s) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (s + 1 < steps) fill(s + 1, (s + 1) & 1, kAll);
    T::multiply(lds + (s & 1) * T::kStage, wr, wc, lane, acc);
  }
}

// The reduction with three stages or more: operands of the next 32 reduction
// steps are read, and half a stage's loads are issued, between the products of
// the current ones.  A stage's first half is read before the stage before it is
// done, so the wait and the barrier for it come in mid-stage; the place of the
// stage that is loaded was read to its end before the last barrier.
template <typename T, typename Load>
__device__ __forceinline__ void reduce_ahead(char* lds, int steps, int wr, int wc, int lane, const Load& load,
                                             f32x4 (&acc)[T::kFR][T::kFC]) {
  constexpr int S = T::kStages, kHalf = T::kLoads / 2;
  static_assert(S >= 3 && T::kLoads % 2 == 0, "a stage is waited for while two others are in use");
  constexpr int kReads = T::kFC * (T::kColsTrans ? 2 : 1) + T::kFR * (T::kRowsTrans ? 2 : 1);
  constexpr int kGroups = kHalf, kMfma = T::kFR * T::kFC / kGroups;
  bf16x8 c[2][T::kFC], r[2][T::kFR];
  auto wait = [&](bool all) {
    __builtin_amdgcn_sched_barrier(0);
    if (all)
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    else
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S - 3) * T::kLoads + kHalf) : "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
  };
  auto fill = [&](int s, int slot, auto part) {
    load(s, lds + slot * T::kStage, lds + slot * T::kStage + T::R::kBytes, part);
  };
  auto mix = [&]() {  // the order of what stands between two barriers
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);                                   // a load
      __builtin_amdgcn_sched_group_barrier(0x100, (kReads + kGroups - 1) / kGroups, 0);  // LDS reads
      __builtin_amdgcn_sched_group_barrier(0x008, kMfma, 0);                               // products
    }
  };
  if (steps == 0) return;
  for (int s = 0; s < S - 1; ++s) fill(s, s, kAll);
  wait(true);
  auto read = [&](int slot, int kk) {
    const char* stage = lds + slot * T::kStage;
    T::read(stage, stage + T::R::kBytes, wr, wc, kk, lane, c[kk], r[kk]);
  };
  read(0, 0);
  int at = 0, next = S - 1;
  for (int s = 0; s < steps; ++s) {
    const int after = at + 1 == S ? 0 : at + 1;
    fill(s + S - 1, next, kFirst);
    read(at, 1);
    T::product(c[0], r[0], acc);
    mix();
    wait(false);
    fill(s + S - 1, next, kSecond);
    read(after, 0);
    T::product(c[1], r[1], acc);
    mix();
    at = after;
    next = next + 1 == S ? 0 : next + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may reach LDS after the workgroup's end
}

// The reduction by eight waves of which two share a SIMD (w and w + 4), in turns:
// one half's waves read a stage's operands and issue the next stage's loads
// while the other half's multiply, with a barrier between the turns.  The second
// half is one turn behind.  Turns of one stage, first half / second half:
//   read 0, load / multiply 1 of the stage before;  multiply 0 / read 0, load;
//   read 1 / multiply 0;  multiply 1 / read 1
// so both have read a stage when the first half starts on the next but one,
// which goes into its place: a stage's loads have two turns at least between
// their issue and the wait for them at the end of the last turn.
// Three stages of the columns' operand (kTurnsFar, for matrices that are read
// once): its loads are issued a stage earlier, behind the rows' of the stage
// before, and the wait leaves them in flight (loads return in order); stages
// beyond the last are loaded too, from nowhere, to keep the count.  Experts of
// 192 rows: 273 -> 258 us (w), 289 -> 272 (dx); a dense product of 4096^3, which
// finds w in the caches, 110 -> 118.
template <typename T, typename Load>
__device__ __forceinline__ void reduce_turns(char* lds, int steps, int rows, int wave, int wr, int wc, int lane,
                                             const Load& load, f32x4 (&acc)[T::kFR][T::kFC]) {
  static_assert(T::kWaves == 8, "two waves per SIMD");
  const bool second = wave >= 4;
  bf16x8 c[T::kFC], r[T::kFR];
  char* const c_lds = lds + 2 * T::R::kBytes;
  auto load_rows = [&](int s) { load(s, lds + (s & 1) * T::R::kBytes, c_lds, kRowsOnly); };
  auto load_cols = [&](int s, int slot) { load(s, lds, c_lds + slot * T::C::kBytes, kColsOnly); };
  constexpr bool kAhead = T::kColStages == 3;
  // (a wave without rows in the tile only keeps the turns; skipping half of its
  // blocks too costs the registers of a second copy of the products)
  const bool live = rows > wr * T::kFR * 16;
  auto multiply = [&]() {
    __builtin_amdgcn_s_setprio(1);
    if (live) T::product(c, r, acc);
    __builtin_amdgcn_s_setprio(0);
  };
  auto turn = [&](bool loads) {  // ends a turn; loads: the next stage, as far as the wave loads it, is in LDS
    if (loads) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kAhead ? T::C::kLoads : 0) : "memory");
    else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
  };
  if (steps == 0) return;
  load_cols(0, 0);
  load_rows(0);
  if (kAhead) load_cols(1, 1);
  turn(true);
  if (second) turn(false);
  int at = 0;  // s modulo the columns' stages
  for (int s = 0; s < steps; ++s) {
    const char* rs = lds + (s & 1) * T::R::kBytes;
    const char* cs = c_lds + at * T::C::kBytes;
    const int before = at == 0 ? T::kColStages - 1 : at - 1;  // the stage that was read to its end
    T::read(rs, cs, wr, wc, 0, lane, c, r);
    if (kAhead || s + 1 < steps) {
      load_rows(s + 1);
      load_cols(s + T::kColStages - 1, before);
    }
    turn(false);
    multiply();
    turn(false);
    T::read(rs, cs, wr, wc, 1, lane, c, r);
    turn(second);
    multiply();
    turn(!second);
    at = at == T::kColStages - 1 ? 0 : at + 1;
  }
  if (!second) turn(false);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may reach LDS after the workgroup's end
}

// ---------------------------------------------------------------- groups
// Rows [0, n_rows) in groups: offsets[g] .. offsets[g + 1] belong to group g
// (offsets NULL: all to group 0), what lies behind offsets[n_groups] to none.
// Bounds out of [0, n_rows] or out of order are cut, so no offsets lead outside.
struct Span {
  int group;       // n_groups: rows of no group
  int64_t row, end;  // first row of the tile, end of its group
};

__device__ __forceinline__ int64_t cut(int64_t v, int64_t n) { return v < 0 ? 0 : v > n ? n : v; }

// Tiles of kBR rows: group by group, then the rows of no group.  Every wave
// works it out for itself: lane l sums the tiles of its share of the groups.
struct TileScan {
  int total;      // tiles in all
  int incl;       // tiles up to this lane's share, inclusive
  int own;        // of this lane's share
};
template <int kBR>
__device__ __forceinline__ TileScan scan_tiles(const int* offsets, int n_groups, int64_t n_rows, int lane) {
  TileScan s;
  if (!offsets) {
    s.total = (int)((n_rows + kBR - 1) / kBR);
    s.incl = s.own = s.total;
    return s;
  }
  const int per = (n_groups + 64) / 64;  // n_groups + 1 groups, the last one the rows of none
  int tiles = 0;
  for (int i = 0; i < per; ++i) {
    const int g = lane * per + i;
    if (g <= n_groups) {
      const int64_t a = cut(offsets[g], n_rows), b = g < n_groups ? cut(offsets[g + 1], n_rows) : n_rows;
      tiles += b > a ? (int)((b - a + kBR - 1) / kBR) : 0;
    }
  }
  // (a launch has 2^22 at most; groups that overlap could name more than an int counts)
  tiles = tiles < 1 << 24 ? tiles : 1 << 24;
  int v = tiles;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(v, off, 64);
    if (lane >= off) v += o;
  }
  s.incl = v;
  s.own = tiles;
  s.total = __builtin_amdgcn_readlane(v, 63);
  return s;
}
template <int kBR>
__device__ __forceinline__ Span find_tile(const TileScan& s, int tile, const int* offsets, int n_groups, int64_t n_rows) {
  if (!offsets) return {0, (int64_t)tile * kBR, n_rows};
  const uint64_t reach = __ballot(s.incl > tile);  // not empty: tile < total
  const int l = __builtin_ctzll(reach);
  int t = tile - (__builtin_amdgcn_readlane(s.incl, l) - __builtin_amdgcn_readlane(s.own, l));
  const int per = (n_groups + 64) / 64;
  for (int i = 0; i < per; ++i) {
    const int g = l * per + i;
    if (g > n_groups) break;
    const int64_t a = cut(offsets[g], n_rows), b = g < n_groups ? cut(offsets[g + 1], n_rows) : n_rows;
    const int tiles = b > a ? (int)((b - a + kBR - 1) / kBR) : 0;
    if (t < tiles)
      return {__builtin_amdgcn_readfirstlane(g), uniform64(a + (int64_t)t * kBR), uniform64(b)};
    t -= tiles;
  }
  return {n_groups, n_rows, n_rows};
}

template <typename T, typename Load>
__device__ __forceinline__ void reduce(char* lds, int steps, int rows, int wave, int wr, int wc, int lane,
                                       const Load& load, f32x4 (&acc)[T::kFR][T::kFC]) {
  if constexpr (T::kTurns)
    reduce_turns<T>(lds, steps, rows, wave, wr, wc, lane, load, acc);
  else if constexpr (T::kStages == 2)
    reduce_stages<T>(lds, steps, wr, wc, lane, load, acc);
  else
    reduce_ahead<T>(lds, steps, wr, wc, lane, load, acc);
}

// The reduction in `splits` parts: where few tiles would leave CUs idle, that
// many workgroups share a tile and a join adds their fp32 sums in order.
struct Steps {
  int first, count;
};
__device__ __forceinline__ Steps part_of(int steps, int splits, int part) {
  const int per = (steps + splits - 1) / splits, first = part * per;
  return {first, steps - first < per ? (steps > first ? steps - first : 0) : per};
}

// ---------------------------------------------------------------- forward
struct LinearParams {
  const char* x;         // [n_rows] rows of k, ldx bytes apart
  const char* w[2];      // weight, and the up weight of swiglu; [n_groups][n][k]
  const char* bias[2];   // bf16 [n_groups][n] or NULL
  const char* residual;  // bf16 [n_rows][n] or NULL
  char* out;             // [n_rows][n]
  uint16_t* pre;         // bf16 [n_rows][n * mats] or NULL
  const int* offsets;
  int64_t n_rows, n, k, ldx, ldw, w_group, ld_res;
  int n_groups, act, out_f32;
  float limit;
  float* part;  // fp32 [splits][n_rows][n * mats]: the reduction in parts, or NULL
  int splits;
};

// A gate as sigmoid() and the products with it take it: finite values below -86 as
// -86.  Their sigmoid is a number that fp32 does not hold, 2^-124 there: with the
// gate at -86 too, z sigmoid(z) stays below 2^-117 however far the gate is (with
// z itself: -7 at -3e38), and not 0 (0 times an infinite up value would be NaN).
// -inf and NaN stay.
__device__ __forceinline__ float near_gate(float z) { return z > -__builtin_inff() ? __builtin_fmaxf(z, -86.0f) : z; }

// Of a near_gate, from t = exp(-z) by the hardware's exp2 and reciprocal (1 ulp
// each).  kFine: the product with log2(e) as a head and what its rounding left,
// which keeps t good to 3 ulp; without it the error of t is |z| 2^-24, nothing
// beside the half step of a bf16 result.
template <bool kFine>
__device__ __forceinline__ float sigmoid(float z) {
  const float kLog2e = 1.4426950408889634f, kLog2eLow = 1.9259629911e-8f;
  const float h = -z * kLog2e;
  float t = __builtin_amdgcn_exp2f(h);
  if (kFine) {
    const float rest = __builtin_fmaf(-z, kLog2eLow, __builtin_fmaf(-z, kLog2e, -h));  // NaN for infinities: 0.5 then
    t = __builtin_fmaf(t, __builtin_fminf(rest, 0.5f) * 0.6931471805599453f, t);
  }
  return __builtin_amdgcn_rcpf(1.0f + t);
}

// min / max that hand a NaN on, as torch's clamp does
__device__ __forceinline__ float clamp_top(float v, float l) { return v > l ? l : v; }
__device__ __forceinline__ float clamp_both(float v, float l) { return v > l ? l : v < -l ? -l : v; }

// Eight values of a row: sums, or what eight bf16 stand for.
struct Row8 {
  float v[8];
};
__device__ __forceinline__ Row8 row8(f32x4 a, f32x4 b) { return {{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}}; }
__device__ __forceinline__ Row8 unpack8(uint4 u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  Row8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = i & 1 ? __uint_as_float(w[i >> 1] & 0xffff0000u) : bf16_bits_to_f32(w[i >> 1] & 0xffffu);
  return r;
}
__device__ __forceinline__ uint4 pack8(const Row8& r) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = f32_to_bf16_bits(r.v[2 * i]) | f32_to_bf16_bits(r.v[2 * i + 1]) << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 load16(const void* p) { return ldg<uint4>(p); }
__device__ __forceinline__ void store8(char* base, int64_t at, const Row8& r, bool f32) {
  if (f32) {
    float4* o = reinterpret_cast<float4*>(base + at * 4);
    o[0] = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
    o[1] = make_float4(r.v[4], r.v[5], r.v[6], r.v[7]);
  } else {
    *reinterpret_cast<uint4*>(base + at * 2) = pack8(r);
  }
}

template <bool kFine>
__device__ __forceinline__ Row8 activate(const LinearParams& p, const Row8& z, const Row8& zu) {
  Row8 y;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (p.act == HSMOE_ACT_SILU) {
      const float g = near_gate(z.v[i]);
      y.v[i] = g * sigmoid<kFine>(g);
    } else {
      const float g = near_gate(clamp_top(z.v[i], p.limit));
      y.v[i] = g * sigmoid<kFine>(g) * clamp_both(zu.v[i], p.limit);
    }
  }
  return y;
}

// Eight outputs of a row: z (and zu) are the sums with bias.
__device__ __forceinline__ Row8 outputs8(const LinearParams& p, const Row8& z, const Row8& zu, uint4 residual) {
  Row8 y = z;
  if (p.act != HSMOE_ACT_NONE) y = p.out_f32 ? activate<true>(p, z, zu) : activate<false>(p, z, zu);
  if (p.residual) {
    const Row8 r = unpack8(residual);
#pragma unroll
    for (int i = 0; i < 8; ++i) y.v[i] += r.v[i];
  }
  return y;
}

// Row m's from column n on.
__device__ __forceinline__ void finish8(const LinearParams& p, int64_t m, int64_t n, const Row8& z, const Row8& zu,
                                        uint4 residual) {
  if (p.pre) {
    const int64_t ldp = p.act == HSMOE_ACT_SWIGLU ? 2 * p.n : p.n;
    *reinterpret_cast<uint4*>(p.pre + m * ldp + n) = pack8(z);
    if (p.act == HSMOE_ACT_SWIGLU) *reinterpret_cast<uint4*>(p.pre + m * ldp + p.n + n) = pack8(zu);
  }
  store8(p.out, m * p.n + n, outputs8(p, z, zu, residual), p.out_f32);
}

// Two rows of eight bf16 per lane, columns 8 g ..+7 and 32 + 8 g ..+7 of row r of
// a block of 16 x 64 (r = lane % 16, g = lane / 16), to memory in whole 128-byte
// lines: lanes r and r ^ 8 exchange one of theirs, and each store takes eight
// rows.  `out` is the block's first value; rows and cols are what there is of it.
template <bool kStream>
__device__ __forceinline__ void store_lines(char* out, int64_t width, int rows, int cols, uint4 a, uint4 b, int lane) {
  const int r = lane & 15, g = lane >> 4;
  const bool low = r < 8;
  const uint32_t va[4] = {a.x, a.y, a.z, a.w}, vb[4] = {b.x, b.y, b.z, b.w};
  u32x4 first, second;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // row_ror:8, lane ^ 8
    const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)(low ? vb[i] : va[i]), 0x128, 0xf, 0xf, true);
    first[i] = low ? va[i] : got;
    second[i] = low ? got : vb[i];
  }
  const int col = 8 * g + (low ? 0 : 32), row = r & 7;
  if (col >= cols) return;
  u32x4* o = reinterpret_cast<u32x4*>(out + (row * width + col) * 2);
  u32x4* o8 = reinterpret_cast<u32x4*>(out + ((row + 8) * width + col) * 2);
  if (kStream) {
    if (row < rows) __builtin_nontemporal_store(first, o);
    if (row + 8 < rows) __builtin_nontemporal_store(second, o8);
  } else {
    if (row < rows) *o = first;
    if (row + 8 < rows) *o8 = second;
  }
}

// One output; a row of no group gets zeros.
__device__ __forceinline__ void finish1(const LinearParams& p, int group, int64_t m, int64_t n, float z, float zu) {
  const bool none = group >= p.n_groups;
  auto bf = [](const void* q, int64_t at) { return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(q)[at]); };
  if (!none && p.bias[0]) z += bf(p.bias[0], group * p.n + n);
  if (!none && p.bias[1]) zu += bf(p.bias[1], group * p.n + n);
  if (p.pre) {
    const int64_t at = m * (p.act == HSMOE_ACT_SWIGLU ? 2 * p.n : p.n) + n;
    p.pre[at] = (uint16_t)f32_to_bf16_bits(z);
    if (p.act == HSMOE_ACT_SWIGLU) p.pre[at + p.n] = (uint16_t)f32_to_bf16_bits(zu);
  }
  float y = z;
  if (p.act == HSMOE_ACT_SILU) {
    const float g = near_gate(z);
    y = g * sigmoid<true>(g);
  } else if (p.act == HSMOE_ACT_SWIGLU) {
    const float g = near_gate(clamp_top(z, p.limit));
    y = g * sigmoid<true>(g) * clamp_both(zu, p.limit);
  }
  if (!none && p.residual) y += bf(p.residual + m * p.ld_res, n);
  if (p.out_f32)
    reinterpret_cast<float*>(p.out)[m * p.n + n] = y;
  else
    reinterpret_cast<uint16_t*>(p.out)[m * p.n + n] = (uint16_t)f32_to_bf16_bits(y);
}

// Rows of no group: zeros.
__device__ __forceinline__ void clear8(const LinearParams& p, int64_t m, int64_t n) {
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  store8(p.out, m * p.n + n, Row8{}, p.out_f32);
  if (p.pre) {
    const int64_t ldp = p.act == HSMOE_ACT_SWIGLU ? 2 * p.n : p.n;
    *reinterpret_cast<uint4*>(p.pre + m * ldp + n) = zero;
    if (p.act == HSMOE_ACT_SWIGLU) *reinterpret_cast<uint4*>(p.pre + m * ldp + p.n + n) = zero;
  }
}

// kGated: the column tile is made of blocks of 16 gate columns and the same 16
// up columns in turn, so that a lane holds a gate sum and its up sum.
template <int kBR, int kBC, int kWR, int kWC, int kStages, bool kGated>
__global__ void __launch_bounds__(kWR* kWC * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) linear_kernel(LinearParams p) {
  using T = Tile<kBR, kBC, kWR, kWC, kStages, false, false, kGated>;
  __shared__ __align__(1024) char lds[T::kLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int kCols = kGated ? kBC / 2 : kBC;  // output columns per tile
  const TileScan scan = scan_tiles<kBR>(p.offsets, p.n_groups, p.n_rows, lane);
  int rt, ct;
  const int col_tiles = (int)((p.n + kCols - 1) / kCols);
  if (!place_tile(blockIdx.x, scan.total, col_tiles * p.splits, rt, ct)) return;
  const Span sp = find_tile<kBR>(scan, rt, p.offsets, p.n_groups, p.n_rows);
  const int split = ct / col_tiles;
  const int64_t n0 = (int64_t)(ct % col_tiles) * kCols;
  const int rows = (int)imin64(kBR, sp.end - sp.row);
  const int cols = (int)imin64(kCols, p.n - n0);
  if (sp.group >= p.n_groups) {  // (the join clears them)
    for (int i = p.part ? rows * cols : threadIdx.x; i < rows * (cols / 8); i += T::kThreads)
      clear8(p, sp.row + i / (cols / 8), n0 + i % (cols / 8) * 8);
    return;
  }
  const Steps steps = part_of((int)((p.k + kBK - 1) / kBK), p.splits, split);
  // Rows are often a power of two apart, and workgroups in step then read the
  // same few memory channels.  With experts, each XCD begins at an eighth of the
  // reduction of its own (64 matrices of 2048 x 4096 for 32 rows each: 262 -> 224
  // us); the XCDs of a dense product read the same w, once in step (500 rows, two
  // such matrices: 24 against 27 us turned), and the kernels with more stages, for
  // few tiles, do without.
  const int turned = T::kStages == 2 && p.offsets ? (blockIdx.x & 7) * steps.count >> 3 : 0;
  const int64_t wo = sp.group * p.w_group + n0 * p.ldw;
  Source<typename T::R> xs;
  xs.open(p.x + sp.row * p.ldx, nullptr, p.ldx, rows, p.k * 2, wave, lane);
  Source<typename T::C> ws;
  ws.open(p.w[0] + wo, p.w[1] + wo, p.ldw, cols, p.k * 2, wave, lane);
  auto load = [&](int s, char* r_stage, char* c_stage, auto part) {
    const int at = s + turned < steps.count ? s + turned : s + turned - steps.count;
    const int first = (steps.first + at) * kBK;
    T::template load<decltype(part)::value>(xs, first, ws, first, s < steps.count ? (int)p.k - first : 0,
                                            r_stage, c_stage,
                                            wave);
  };
  const int wr = wave / kWC, wc = wave % kWC;
  f32x4 acc[T::kFR][T::kFC] = {};
  reduce<T>(lds, steps.count, rows, wave, wr, wc, lane, load, acc);
  if (p.part) {
    const int64_t width = kGated ? 2 * p.n : p.n;
    char* base = (char*)(p.part + split * p.n_rows * width);
#pragma unroll
    for (int i = 0; i < T::kFR; ++i) {
      const int r = (wr * T::kFR + i) * 16 + (lane & 15);
      if (r >= rows) continue;
#pragma unroll
      for (int j = 0; j < T::kFC; j += kGated ? 4 : 2) {
        const int c = (wc * T::kFC + j) * (kGated ? 8 : 16) + 8 * (lane >> 4);
        if (c >= cols) continue;
        const int64_t at = (sp.row + r) * width + n0 + c;
        store8(base, at, kGated ? row8(acc[i][j], acc[i][j + 2]) : row8(acc[i][j], acc[i][j + 1]), true);
        if (kGated) store8(base, at + p.n, row8(acc[i][j + 1], acc[i][j + 3]), true);
      }
    }
    return;
  }
  // a lane has kE times eight columns of kFR rows; the next row's residual is on
  // its way while a row is finished
  constexpr int kStep = kGated ? 4 : 2, kE = T::kFC / kStep;
  const int r0 = wr * T::kFR * 16 + (lane & 15), cw = wc * kE * 32 + 8 * (lane >> 4);
  Row8 bias[2][kE];
#pragma unroll
  for (int e = 0; e < kE; ++e)
#pragma unroll
    for (int s = 0; s < (kGated ? 2 : 1); ++s) {
      const int64_t at = sp.group * p.n + n0 + cw + 32 * e;
      bias[s][e] = p.bias[s] && cw + 32 * e < cols ? unpack8(load16(p.bias[s] + at * 2)) : Row8{};
    }
  uint4 res[2][kE] = {};
  auto load_res = [&](int i) {
    if (p.residual && r0 + 16 * i < rows) {
#pragma unroll
      for (int e = 0; e < kE; ++e)
        if (cw + 32 * e < cols)
          res[i & 1][e] = load16(p.residual + (sp.row + r0 + 16 * i) * p.ld_res + (n0 + cw + 32 * e) * 2);
    }
  };
  load_res(0);
#pragma unroll
  for (int i = 0; i < T::kFR; ++i) {
    if (i + 1 < T::kFR) load_res(i + 1);
    Row8 z[kE], zu[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      z[e] = kGated ? row8(acc[i][4 * e], acc[i][4 * e + 2]) : row8(acc[i][2 * e], acc[i][2 * e + 1]);
      zu[e] = kGated ? row8(acc[i][4 * e + 1], acc[i][4 * e + 3]) : Row8{};
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        z[e].v[v] += bias[0][e].v[v];
        if (kGated) zu[e].v[v] += bias[1][e].v[v];
      }
    }
    if constexpr (!kGated) {
      static_assert(kE == 2, "a wave has 64 columns");
      const int64_t at = (sp.row + wr * T::kFR * 16 + 16 * i) * p.n + n0 + wc * 64;
      const int left = rows - (wr * T::kFR + i) * 16, width = cols - wc * 64;
      if (p.pre) store_lines<false>((char*)(p.pre + at), p.n, left, width, pack8(z[0]), pack8(z[1]), lane);
      if (!p.out_f32) {
        const uint4 a = pack8(outputs8(p, z[0], z[0], res[i & 1][0])), b = pack8(outputs8(p, z[1], z[1], res[i & 1][1]));
        store_lines<false>(p.out + at * 2, p.n, left, width, a, b, lane);
        continue;
      }
    }
    if (r0 + 16 * i >= rows) continue;
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      if (cw + 32 * e >= cols) continue;
      const int64_t m = sp.row + r0 + 16 * i, n = n0 + cw + 32 * e;
      if (kGated) finish8(p, m, n, z[e], zu[e], res[i & 1][e]);
      else store8(p.out, m * p.n + n, outputs8(p, z[e], z[e], res[i & 1][e]), true);
    }
  }
}

__device__ __forceinline__ Row8 load8(const float* p) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
// The sum of `splits` values of eight, `stride` apart, in order.
__device__ __forceinline__ Row8 sum_parts(const float* p, int64_t stride, int splits) {
  Row8 z = load8(p);
  for (int s = 1; s < splits; ++s) {
    const Row8 q = load8(p + s * stride);
#pragma unroll
    for (int v = 0; v < 8; ++v) z.v[v] += q.v[v];
  }
  return z;
}
__device__ __forceinline__ int64_t end_of_groups(const int* offsets, int n_groups, int64_t n_rows) {
  return offsets ? cut(offsets[n_groups], n_rows) : n_rows;
}

// The parts of a split reduction added, and the epilogue: eight columns per thread.
__global__ void __launch_bounds__(256) linear_join_kernel(LinearParams p) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, per = p.n / 8, m = at / per, n = at % per * 8;
  if (m >= p.n_rows) return;
  if (m >= end_of_groups(p.offsets, p.n_groups, p.n_rows)) return clear8(p, m, n);
  const bool gated = p.act == HSMOE_ACT_SWIGLU;
  const int64_t width = gated ? 2 * p.n : p.n;
  const float* part = p.part + m * width + n;
  Row8 z = sum_parts(part, p.n_rows * width, p.splits), zu{};
  if (gated) zu = sum_parts(part + p.n, p.n_rows * width, p.splits);
  if (p.bias[0] || p.bias[1]) {
    int lo = 0;  // the row's group: the last one that begins at or before it
    for (int hi = p.n_groups; p.offsets && hi - lo > 1;) {
      const int mid = (lo + hi) >> 1;
      if (p.offsets[mid] <= m) lo = mid;
      else hi = mid;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (!p.bias[s]) continue;
      const Row8 b = unpack8(load16(p.bias[s] + (lo * p.n + n) * 2));
#pragma unroll
      for (int v = 0; v < 8; ++v) (s ? zu : z).v[v] += b.v[v];
    }
  }
  finish8(p, m, n, z, zu, p.residual ? load16(p.residual + m * p.ld_res + n * 2) : make_uint4(0u, 0u, 0u, 0u));
}

// ---------------------------------------------------------------- few rows
// Up to 16 rows (of a group) against all of w: what counts is w's stream.  A
// tile is 16 rows of w (kGated: 8 of each matrix), and a workgroup's eight waves
// share its reduction, a wave's part in batches of kBatch units of 128 steps, 16
// bytes per lane and load, a batch's loads in flight before its first product.
// w goes to the matrix cores straight from registers as their first operand; its
// lanes read 64 bytes of 16 rows per load, a unit's four loads 256 in a row.
// Two workgroups per CU go through the tiles in turn (one launch of a workgroup
// per tile costs a quarter more where experts bring thousands of them).
constexpr int kNarrowRows = 16, kNarrowWaves = 8, kUnit = 128, kBatch = 2;

// bf16 x 8 from p, zeros where !there
__device__ __forceinline__ bf16x8 load_frag(const char* p, bool there) {
  const uint4 u = there ? load16(p) : make_uint4(0u, 0u, 0u, 0u);
  return __builtin_bit_cast(bf16x8, u);
}

template <bool kGated>
__global__ void __launch_bounds__(kNarrowWaves * 64) __attribute__((amdgpu_waves_per_eu(4)))
linear_narrow_kernel(LinearParams p) {
  constexpr int kCols = kGated ? 8 : 16;
  __shared__ float s_part[2][kNarrowWaves][kNarrowRows][17];  // [tile's parity][wave][row][row of w], padded
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TileScan scan = scan_tiles<kNarrowRows>(p.offsets, p.n_groups, p.n_rows, lane);
  const int col_tiles = (int)((p.n + kCols - 1) / kCols);
  const int64_t total = (int64_t)scan.total * col_tiles;
  int turn = 0;
  for (int64_t tile = blockIdx.x; tile < total; tile += gridDim.x, turn ^= 1) {
    const int rt = (int)(tile / col_tiles), ct = (int)(tile % col_tiles);
    const Span sp = find_tile<kNarrowRows>(scan, rt, p.offsets, p.n_groups, p.n_rows);
    const int rows = (int)imin64(kNarrowRows, sp.end - sp.row);
    const int64_t n0 = (int64_t)ct * kCols;
    const int cols = (int)imin64(kCols, p.n - n0);
    if (sp.group < p.n_groups) {
      const int i = lane & 15, g = lane >> 4, mat = kGated && i >= 8 ? 1 : 0;
      const int wrow = kGated ? i & 7 : i;
      // rows of w beyond the last one read the last one again; their sums go nowhere
      const char* wp = p.w[mat] + sp.group * p.w_group + (n0 + (wrow < cols ? wrow : cols - 1)) * p.ldw + 16 * g;
      const char* xp = p.x + (sp.row + i) * p.ldx + 16 * g;
      const int units = (int)((p.k + kUnit - 1) / kUnit), per = (units + kNarrowWaves - 1) / kNarrowWaves;
      const int u1 = units < (wave + 1) * per ? units : (wave + 1) * per;
      f32x4 acc = {};
      for (int u = wave * per; u < u1; u += kBatch) {
        bf16x8 w[kBatch][4], x[kBatch][4];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const int first = (u + b) * kUnit + 8 * g, left = u + b < u1 ? (int)p.k : 0;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const bool there = first + 32 * t < left;
            const int64_t at = (int64_t)(u + b) * (kUnit * 2) + 64 * t;
            w[b][t] = load_frag(wp + at, there);
            x[b][t] = load_frag(xp + at, there && i < rows);
          }
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
#pragma unroll
          for (int t = 0; t < 4; ++t) acc = mfma16x16x32(w[b][t], x[b][t], acc);
      }
#pragma unroll
      for (int v = 0; v < 4; ++v) s_part[turn][wave][i][4 * g + v] = acc[v];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * kCols; e += kNarrowWaves * 64) {
      const int r = e / kCols, c = e % kCols;
      if (c >= cols) continue;
      float z = 0.0f, zu = 0.0f;
      if (sp.group < p.n_groups) {
#pragma unroll
        for (int w = 0; w < kNarrowWaves; ++w) {
          z += s_part[turn][w][r][c];
          if (kGated) zu += s_part[turn][w][r][c + 8];
        }
      }
      finish1(p, sp.group, sp.row + r, n0 + c, z, zu);
    }
  }
}

// ---------------------------------------------------------------- gradients
struct LinearGradParams {
  const char* dz;       // bf16 [n_rows][n * mats], ldz bytes apart
  const char* x;        // bf16 [n_rows][k]
  const char* w[2];     // [n_groups][n][k]
  char* dx;             // bf16 [n_rows][k]
  char* dw[2];          // [n_groups][n][k], bf16 or fp32
  const int* offsets;
  int64_t n_rows, n, k, ldz, ldx, ldw, w_group;
  int n_groups, mats, dw_f32;
  float* part;  // fp32 [splits][n_rows][k], or [splits][n_groups][mats][n][k]: the reduction in parts, or NULL
  int splits;
};

// The sums of a tile to rows row0 .. and columns col0 .. of a matrix of `width`.
// kStream: past the caches (weights' gradients: far more than they hold, and
// what the tiles read would be driven out of them).
template <typename T, bool kStream>
__device__ __forceinline__ void store_tile(char* out, int64_t width, int64_t row0, int64_t col0, int rows, int cols,
                                           bool f32, int wr, int wc, int lane, const f32x4 (&acc)[T::kFR][T::kFC]) {
  static_assert(T::kFC == 4, "a wave has 64 columns");
  const int rb = wr * T::kFR * 16, cb = wc * 64;
#pragma unroll
  for (int i = 0; i < T::kFR; ++i) {
    const Row8 a = row8(acc[i][0], acc[i][1]), b = row8(acc[i][2], acc[i][3]);
    if (f32) {
      const int r = rb + 16 * i + (lane & 15), c = cb + 8 * (lane >> 4);
      const int64_t at = (row0 + r) * width + col0 + c;
      if (r < rows && c < cols) store8(out, at, a, true);
      if (r < rows && c + 32 < cols) store8(out, at + 32, b, true);
    } else {
      store_lines<kStream>(out + ((row0 + rb + 16 * i) * width + col0 + cb) * 2, width, rows - rb - 16 * i, cols - cb,
                           pack8(a), pack8(b), lane);
    }
  }
}

// dx = dz w (+ dz_up w_up): the reduction runs over the n columns of dz and the
// rows of w, then over those of up.
template <int kBR, int kBC, int kWR, int kWC, int kStages>
__global__ void __launch_bounds__(kWR* kWC * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) linear_grad_input_kernel(LinearGradParams p) {
  using T = Tile<kBR, kBC, kWR, kWC, kStages, false, true>;
  __shared__ __align__(1024) char lds[T::kLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TileScan scan = scan_tiles<kBR>(p.offsets, p.n_groups, p.n_rows, lane);
  int rt, ct;
  const int col_tiles = (int)((p.k + kBC - 1) / kBC);
  if (!place_tile(blockIdx.x, scan.total, col_tiles * p.splits, rt, ct)) return;
  const Span sp = find_tile<kBR>(scan, rt, p.offsets, p.n_groups, p.n_rows);
  const int split = ct / col_tiles;
  const int64_t c0 = (int64_t)(ct % col_tiles) * kBC;
  const int rows = (int)imin64(kBR, sp.end - sp.row), cols = (int)imin64(kBC, p.k - c0);
  if (sp.group >= p.n_groups) {  // (the join clears them)
    for (int i = p.part ? rows * cols : threadIdx.x; i < rows * (cols / 8); i += T::kThreads)
      store8(p.dx, (sp.row + i / (cols / 8)) * p.k + c0 + i % (cols / 8) * 8, Row8{}, false);
    return;
  }
  const int per = (int)((p.n + kBK - 1) / kBK);
  const Steps steps = part_of(per * p.mats, p.splits, split);
  Source<typename T::R> zs;
  zs.open(p.dz + sp.row * p.ldz, nullptr, p.ldz, rows, p.n * p.mats * 2, wave, lane);
  Source<typename T::C> ws;
  const int64_t wo = sp.group * p.w_group + c0 * 2;
  ws.open(p.w[0] + wo, nullptr, p.ldw, 0, cols * 2, wave, lane);
  auto load = [&](int s, char* r_stage, char* c_stage, auto part) {
    const int step = steps.first + s, mat = step >= per ? 1 : 0, first = (step - mat * per) * kBK;
    ws.base[0] = (mat ? p.w[1] : p.w[0]) + wo;
    T::template load<decltype(part)::value>(zs, mat * p.n + first, ws, first, s < steps.count ? (int)p.n - first : 0,
                                            r_stage, c_stage,
                                            wave);
  };
  const int wr = wave / kWC, wc = wave % kWC;
  f32x4 acc[T::kFR][T::kFC] = {};
  reduce<T>(lds, steps.count, rows, wave, wr, wc, lane, load, acc);
  char* out = p.part ? (char*)(p.part + split * p.n_rows * p.k) : p.dx;
  store_tile<T, false>(out, p.k, sp.row, c0, rows, cols, p.part != nullptr, wr, wc, lane, acc);
}

// dw[g] = dz^T x over the rows of group g: a tile of n x k per workgroup, all
// groups and both matrices in one launch; a group without rows gets zeros.
template <int kBR, int kBC, int kWR, int kWC, int kStages>
__global__ void __launch_bounds__(kWR* kWC * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) linear_grad_weight_kernel(LinearGradParams p) {
  using T = Tile<kBR, kBC, kWR, kWC, kStages, true, true>;
  __shared__ __align__(1024) char lds[T::kLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row_tiles = (int)((p.n + kBR - 1) / kBR), col_tiles = (int)((p.k + kBC - 1) / kBC);
  int rt, ct;
  if (!place_tile(blockIdx.x, p.n_groups * p.mats * row_tiles, col_tiles * p.splits, rt, ct)) return;
  const int gm = rt / row_tiles, group = gm / p.mats, mat = gm % p.mats, split = ct / col_tiles;
  const int64_t n0 = (int64_t)(rt % row_tiles) * kBR, c0 = (int64_t)(ct % col_tiles) * kBC;
  const int64_t first = p.offsets ? cut(p.offsets[group], p.n_rows) : 0;
  const int64_t end = p.offsets ? cut(p.offsets[group + 1], p.n_rows) : p.n_rows;
  const int64_t count = end > first ? end - first : 0;
  const int nrow = (int)imin64(kBR, p.n - n0), ncol = (int)imin64(kBC, p.k - c0);
  const Steps steps = part_of((int)((count + kBK - 1) / kBK), p.splits, split);
  Source<typename T::R> zs;
  zs.open(p.dz + first * p.ldz + (mat * p.n + n0) * 2, nullptr, p.ldz, 0, nrow * 2, wave, lane);
  Source<typename T::C> xs;
  xs.open(p.x + first * p.ldx + c0 * 2, nullptr, p.ldx, 0, ncol * 2, wave, lane);
  auto load = [&](int s, char* r_stage, char* c_stage, auto part) {
    const int first_step = (steps.first + s) * kBK;
    T::template load<decltype(part)::value>(zs, first_step, xs, first_step, s < steps.count ? (int)count - first_step : 0,
                                            r_stage, c_stage,
                                            wave);
  };
  const int wr = wave / kWC, wc = wave % kWC;
  f32x4 acc[T::kFR][T::kFC] = {};
  reduce<T>(lds, steps.count, nrow, wave, wr, wc, lane, load, acc);
  const bool f32 = p.part || p.dw_f32;
  char* out = p.part ? (char*)(p.part + ((int64_t)split * p.n_groups * p.mats + gm) * p.n * p.k)
                     : p.dw[mat] + (int64_t)group * p.n * p.k * (f32 ? 4 : 2);
  store_tile<T, true>(out, p.k, n0, c0, nrow, ncol, f32, wr, wc, lane, acc);
}

// The parts of a split reduction added: kWeight: dw (and dw_up), else dx.
template <bool kWeight>
__global__ void __launch_bounds__(256) linear_grad_join_kernel(LinearGradParams p) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  const int64_t total = (kWeight ? (int64_t)p.n_groups * p.mats * p.n : p.n_rows) * p.k;
  if (at >= total) return;
  if (kWeight) {
    const int64_t size = p.n * p.k, gm = at / size;
    store8(p.dw[gm % p.mats], gm / p.mats * size + at % size, sum_parts(p.part + at, total, p.splits), p.dw_f32);
  } else {
    const bool none = at / p.k >= end_of_groups(p.offsets, p.n_groups, p.n_rows);
    store8(p.dx, at, none ? Row8{} : sum_parts(p.part + at, total, p.splits), false);
  }
}

// dz = d_out act'(pre) and the column sums of dz over the rows of a group (the
// bias's gradient), from the unrounded values.  dz itself is rounded to bf16, as
// pre is: the matrix cores, to which it goes twice, take bf16, and its error of
// half a step is that of every other factor of those sums.  What the limit cuts
// off goes by pre as it is kept, rounded (hsmoe.h says what that means at the
// limit).  A workgroup has 256 columns and a share of a group's rows: 32 threads
// of 8 columns, 8 rows at a time; the shares' sums go to `part`
// [shares][n_groups][n * mats] and are added in order by a second launch (one
// share: straight to the result).
struct ActGradParams {
  const uint16_t* d_out;  // [n_rows][n]
  const uint16_t* pre;    // [n_rows][n * mats], NULL without an activation
  uint16_t* dz;           // [n_rows][n * mats] or NULL
  float* part;            // or NULL
  float* d_bias[2];
  const int* offsets;
  int64_t n_rows, n, ld_out;
  int n_groups, act, mats, shares;
  float limit;
};

constexpr int kActThreads = 256;

// kSums: the column sums are wanted (and with them dz before its rounding).
template <int kMats, bool kSums>
__global__ void __launch_bounds__(kActThreads) act_grad_kernel(ActGradParams p) {
  __shared__ float s_sum[kMats][8][256];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, group = blockIdx.y, share = blockIdx.z;
  const int64_t col = (int64_t)blockIdx.x * 256 + tx * 8;
  const int64_t first = p.offsets ? cut(p.offsets[group], p.n_rows) : 0;
  const int64_t end = p.offsets ? cut(p.offsets[group + 1], p.n_rows) : p.n_rows;
  const int64_t count = end > first ? end - first : 0;
  const int64_t a = first + count * share / p.shares, b = first + count * (share + 1) / p.shares;
  float sum[kMats][8] = {};
  // two rows' loads on their way before the first is used
  constexpr int kAhead = 2;
  for (int64_t r0 = a + ty; r0 < b && col < p.n; r0 += 8 * kAhead) {
    uint4 d_out[kAhead], pre[kAhead][kMats] = {};
#pragma unroll
    for (int h = 0; h < kAhead; ++h) {
      const int64_t r = r0 + 8 * h;
      if (r >= b) continue;
      d_out[h] = load16(p.d_out + r * p.ld_out + col);
      if (p.pre) {
#pragma unroll
        for (int t = 0; t < kMats; ++t) pre[h][t] = load16(p.pre + r * p.n * kMats + t * p.n + col);
      }
    }
#pragma unroll
    for (int h = 0; h < kAhead; ++h) {
      const int64_t r = r0 + 8 * h;
      if (r >= b) continue;
      const Row8 d = unpack8(d_out[h]), z = unpack8(pre[h][0]), zu = unpack8(pre[h][kMats - 1]);
      Row8 o[kMats];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (kMats == 2) {
          const float g = near_gate(clamp_top(z.v[i], p.limit)), s = sigmoid<kSums>(g), gs = g * s;
          o[0].v[i] = z.v[i] > p.limit ? 0.0f : d.v[i] * clamp_both(zu.v[i], p.limit) * (s + gs * (1.0f - s));
          o[kMats - 1].v[i] = zu.v[i] > p.limit || zu.v[i] < -p.limit ? 0.0f : d.v[i] * gs;
        } else if (p.act == HSMOE_ACT_SILU) {
          const float g = near_gate(z.v[i]), s = sigmoid<kSums>(g);
          o[0].v[i] = d.v[i] * (s + g * s * (1.0f - s));
        } else {
          o[0].v[i] = d.v[i];
        }
      }
#pragma unroll
      for (int t = 0; t < kMats; ++t) {
        if (kSums) {
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[t][i] += o[t].v[i];
        }
        if (p.dz) *reinterpret_cast<uint4*>(p.dz + r * p.n * kMats + t * p.n + col) = pack8(o[t]);
      }
    }
  }
  if (!kSums) return;
#pragma unroll
  for (int t = 0; t < kMats; ++t)
#pragma unroll
    for (int i = 0; i < 8; ++i) s_sum[t][ty][tx * 8 + i] = sum[t][i];
  __syncthreads();
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= p.n) return;
#pragma unroll
  for (int t = 0; t < kMats; ++t) {
    float v = 0.0f;
#pragma unroll
    for (int y = 0; y < 8; ++y) v += s_sum[t][y][threadIdx.x];
    if (p.part)
      p.part[(((int64_t)share * p.n_groups + group) * kMats + t) * p.n + c] = v;
    else if (p.d_bias[t])
      p.d_bias[t][group * p.n + c] = v;
  }
}

__global__ void __launch_bounds__(256) bias_sum_kernel(ActGradParams p) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x, width = p.n * p.mats;
  const int64_t total = width * p.n_groups;
  if (c >= total) return;
  float v = 0.0f;
#pragma unroll 8
  for (int s = 0; s < p.shares; ++s) v += p.part[s * total + c];
  const int64_t group = c / width, in = c % width;
  float* o = p.d_bias[in >= p.n ? 1 : 0];
  if (o) o[group * p.n + in % p.n] = v;
}

// ---------------------------------------------------------------- host
// Row tiles of `rows` rows at most: dense exactly, in groups one more for each
// group that has rows (their last tiles are not full) and one for the rest.
int64_t max_row_tiles(int64_t n_rows, int64_t rows, const void* offsets, int n_groups) {
  if (!offsets) return (n_rows + rows - 1) / rows;
  return n_rows / rows + (n_groups + 1 < n_rows ? n_groups + 1 : n_rows);
}

int check_counts(const char* what, int64_t m, int64_t n, int64_t k, int64_t n_groups, const void* offsets) {
  if (m < 0 || n < 1 || k < 1 || n_groups < 1) return fail(HSMOE_ERR_ARG, "%s: bad counts", what);
  if (n_groups > kMaxGroups) return fail(HSMOE_ERR_SHAPE, "%s: at most %d groups", what, kMaxGroups);
  if (!offsets && n_groups != 1) return fail(HSMOE_ERR_ARG, "%s: groups need their offsets", what);
  if (n % 8 != 0 || k % 8 != 0) return fail(HSMOE_ERR_SHAPE, "%s: n and k must be multiples of 8", what);
  // (steps are counted in 32 bits, up to four stages beyond the last one)
  if (m > INT32_MAX - 1024) return fail(HSMOE_ERR_SHAPE, "%s: m must be below 2^31 - 1024", what);
  if (offsets && !aligned(offsets, 4)) return fail(HSMOE_ERR_SHAPE, "%s: misaligned offsets", what);
  return HSMOE_OK;
}

// A matrix of rows of `cols` bf16, `stride` elements apart: whole 16-byte
// vectors, and a tile's rows within one resource.
int check_matrix(const char* what, const char* name, const void* p, int64_t cols, int64_t stride) {
  if (!p) return fail(HSMOE_ERR_ARG, "%s: null pointer (%s)", what, name);
  if (!aligned(p, 16) || stride % 8 != 0)
    return fail(HSMOE_ERR_SHAPE, "%s: rows of %s must be 16-byte aligned", what, name);
  if (stride < cols) return fail(HSMOE_ERR_ARG, "%s: row stride of %s is below its row", what, name);
  if (stride > kMaxRange / 2 / 256 || cols > kMaxRange / 2 / 256)
    return fail(HSMOE_ERR_SHAPE, "%s: rows of %s are too far apart", what, name);
  return HSMOE_OK;
}

// Workgroups for row_tiles x tiles of bc columns, as place_tile deals them out; 0
// if that is more than a launch can hold.
unsigned tile_grid(int64_t row_tiles, int64_t cols, int bc) {
  const int64_t total = row_tiles * ((cols + bc - 1) / bc), unit = total > 8 * (kChunk - 1) ? 8 * kChunk : 8;
  return total > (1 << 22) - unit ? 0 : (unsigned)((total + unit - 1) / unit * unit);
}

// How a product is done: the tile, and the parts of its reduction.
struct Plan {
  int tile;  // kNarrow or an index into kTiles
  int splits;
  size_t bytes;  // of the parts
};
constexpr int kNarrow = -1;

// The tiles, with what a round of workgroups (one or two per CU) takes for 64
// reduction steps and for the rest (first loads, epilogue), in us with every CU
// at work, the part of a step's time that is left with few at work, and the rate
// at which they stream matrices that are read once (swiglu's two):
//   256 x 256, turns of eight waves        1.45 + 16,  0.8, 5.0 (5.1) TB/s
//   128 x 128, 4 stages, eight waves       0.52 + 6.5, 0.6, 4.4 (4.6) TB/s (four waves: 0.56 + 7)
//   64 x 128, 4 stages, four waves         0.35 + 6,   0.8, 4.3 (4.5) TB/s
//   128 x 128, 2 stages, two per CU        1.02 + 8,   0.4, 5.7 (4.8) TB/s
//   256 x 128, 3 stages, eight waves       0.79 + 9,   0.6, 3.9 TB/s
// The kernel for few rows streams w at 5.3 TB/s less 3% per row, and takes 2.2 us
// for a tile of 16 of w's rows however short they are.  What takes the least time
// by these figures is taken; a split reduction costs the fp32 sums' way to memory
// and back and a launch.
struct TileCost {
  int rows, cols, per_cu;
  double step, rest, few, rate, rate_two;  // us, us, 1, bytes per us
};
constexpr TileCost kTiles[] = {{256, 256, 1, 1.45, 16.0, 0.8, 5.0e6, 5.1e6},
                               {128, 128, 1, 0.52, 6.5, 0.6, 4.4e6, 4.6e6},
                               {64, 128, 1, 0.35, 6.0, 0.8, 4.3e6, 4.5e6},
                               {128, 128, 2, 1.02, 8.0, 0.4, 5.7e6, 4.8e6},
                               {256, 128, 1, 0.79, 9.0, 0.6, 3.9e6, 3.9e6}};
constexpr int kAllTiles = 5, kGatedTiles = 4;  // (the last one does not hold swiglu's two sums in its registers)
// The same for the weights' gradients, whose experts often have one or two steps
// and whose tiles often end at the matrix's edge: what a round takes beside its
// steps is less there, and the results go out at 3 TB/s.  Over 800 shapes (1 to
// 16384 rows, up to 256 experts, 32 to 4400 columns either way) the choice by
// these takes 0.6% more than the best tile in the mean and 1.35 times at most;
// the 256 x 256 one alone takes 60% more in the mean, the 128 x 128 one 20%.
constexpr TileCost kWeightTiles[] = {{256, 256, 1, 1.9, 4.0, 0.65, 3.0e6, 3.0e6},
                                     {128, 128, 1, 0.61, 3.0, 0.72, 3.0e6, 3.0e6}};

// rows: of the output, in groups of which at most `active` have any (one: dense);
// cols: tiles' columns (twice the output's for swiglu: two); outputs: as many of
// them, each tiled for itself; bytes: of the groups' matrices; sums: fp32 values
// of one part; table: the tiles to choose from.
Plan plan_tiles(double rows, double active, int64_t cols, int64_t outputs, int64_t steps, double bytes, bool two,
                double sums, const TileCost* table, int n_tiles, double& least) {
  const double cus = device_cus();
  Plan best{0, 1, 0};
  least = 1e30;
  for (int t = 0; t < n_tiles; ++t) {
    const TileCost& c = table[t];
    // groups end inside a tile: half a tile more for each on average
    double row_tiles = active <= 1 ? __builtin_ceil(rows / c.rows) : rows / c.rows + 0.5 * active;
    if (row_tiles < active) row_tiles = active;
    const double tiles = row_tiles * (double)((cols + c.cols - 1) / c.cols * outputs);
    for (int s = 1; s <= 16; s *= 2) {
      const int64_t per = (steps + s - 1) / s;
      if (s > 1 && (per < 4 || (steps + per - 1) / per != s)) continue;
      const double fill = tiles * s / (cus * c.per_cu), rounds = __builtin_ceil(fill);
      double us = rounds * (per * c.step * (c.few + (1.0 - c.few) * fill / rounds) + c.rest);
      const double stream = bytes / (two ? c.rate_two : c.rate);
      if (us < stream) us = stream;
      if (s > 1) us += 2.5 + s * sums * 8.0 / 5e6;
      if (us < least) {
        least = us;
        best = {t, s, s > 1 ? (size_t)(s * sums * 4.0) : 0};
      }
    }
  }
  return best;
}

Plan plan_linear(int64_t m, int64_t n, int64_t k, int64_t n_groups, int act) {
  const int64_t active = n_groups < m ? n_groups : m, mats = act == HSMOE_ACT_SWIGLU ? 2 : 1;
  const double rows = (double)m / (double)active, bytes = 2.0 * active * n * mats * k;
  double tiled;
  const Plan plan = plan_tiles((double)m, (double)active, n * mats, 1, (k + kBK - 1) / kBK, bytes, mats == 2,
                               (double)m * n * mats, kTiles, mats == 2 ? kGatedTiles : kAllTiles, tiled);
  const double passes = (double)active * ((n * mats + 15) / 16) / (2.0 * device_cus()), stream = bytes / 5.3e6 * (1.0 + 0.03 * rows);
  const double narrow = 2.0 + (stream > 2.2 * passes ? stream : 2.2 * passes);
  return rows <= kNarrowRows && narrow < tiled ? Plan{kNarrow, 1, 0} : plan;
}
Plan plan_grad_input(int64_t m, int64_t n, int64_t k, int64_t n_groups, int mats) {
  const int64_t active = n_groups < m ? n_groups : m;
  double us;
  return plan_tiles((double)m, (double)active, k, 1, (n + kBK - 1) / kBK * mats, 2.0 * active * n * mats * k, false,
                    (double)m * k, kTiles, kAllTiles, us);
}
// (both operands transposed: no tile of 64 rows)
Plan plan_grad_weight(int64_t m, int64_t n, int64_t k, int64_t n_groups, int mats) {
  const int64_t rows = (m + n_groups - 1) / n_groups;
  const double values = (double)n_groups * mats * n * k;
  double us;
  return plan_tiles((double)n, 1, k, n_groups * mats, (rows + kBK - 1) / kBK, 2.0 * values, false, values, kWeightTiles, 2,
                    us);
}

int check_workspace(const char* what, const Plan& plan, const void* ws, size_t bytes) {
  if (!plan.bytes) return HSMOE_OK;
  if (!ws || bytes < plan.bytes) return fail(HSMOE_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", what, plan.bytes);
  if (!aligned(ws, 16)) return fail(HSMOE_ERR_SHAPE, "%s: the workspace must be 16-byte aligned", what);
  return HSMOE_OK;
}

unsigned join_grid(int64_t values) { return (unsigned)((values / 8 + 255) / 256); }

template <int kBR, int kBC, int kWR, int kWC, int kStages, bool kGated>
int launch_linear_as(const LinearParams& p, hipStream_t st) {
  const int64_t row_tiles = max_row_tiles(p.n_rows, kBR, p.offsets, p.n_groups) * p.splits;
  const unsigned grid = tile_grid(row_tiles, p.n, kGated ? kBC / 2 : kBC);
  if (!grid) return fail(HSMOE_ERR_SHAPE, "hsmoe_linear: too many tiles");
  hipLaunchKernelGGL((linear_kernel<kBR, kBC, kWR, kWC, kStages, kGated>), dim3(grid), dim3(kWR * kWC * 64), 0, st, p);
  if (p.part) hipLaunchKernelGGL(linear_join_kernel, dim3(join_grid(p.n_rows * p.n)), dim3(256), 0, st, p);
  return check_launch("hsmoe_linear");
}
template <int kBR, int kBC, int kWR, int kWC, int kStages>
int launch_linear(const LinearParams& p, hipStream_t st) {
  if (p.act == HSMOE_ACT_SWIGLU) return launch_linear_as<kBR, kBC, kWR, kWC, kStages, true>(p, st);
  return launch_linear_as<kBR, kBC, kWR, kWC, kStages, false>(p, st);
}

int launch_narrow(const LinearParams& p, hipStream_t st) {
  const bool gated = p.act == HSMOE_ACT_SWIGLU;
  const int64_t tiles = max_row_tiles(p.n_rows, kNarrowRows, p.offsets, p.n_groups), cols = gated ? 8 : 16;
  int64_t grid = tiles * ((p.n + cols - 1) / cols), most = 2 * device_cus();  // what the chip holds at once
  if (grid > most) grid = most;
  const dim3 block(kNarrowWaves * 64);
  if (gated)
    hipLaunchKernelGGL(linear_narrow_kernel<true>, dim3((unsigned)grid), block, 0, st, p);
  else
    hipLaunchKernelGGL(linear_narrow_kernel<false>, dim3((unsigned)grid), block, 0, st, p);
  return check_launch("hsmoe_linear");
}

template <int kBR, int kBC, int kWR, int kWC, int kStages>
int launch_grad_input(const LinearGradParams& p, hipStream_t st) {
  const unsigned grid = tile_grid(max_row_tiles(p.n_rows, kBR, p.offsets, p.n_groups) * p.splits, p.k, kBC);
  if (!grid) return fail(HSMOE_ERR_SHAPE, "hsmoe_linear_grad_input: too many tiles");
  hipLaunchKernelGGL((linear_grad_input_kernel<kBR, kBC, kWR, kWC, kStages>), dim3(grid), dim3(kWR * kWC * 64), 0, st, p);
  if (p.part)
    hipLaunchKernelGGL(linear_grad_join_kernel<false>, dim3(join_grid(p.n_rows * p.k)), dim3(256), 0, st, p);
  return check_launch("hsmoe_linear_grad_input");
}

template <int kBR, int kBC, int kWR, int kWC, int kStages>
int launch_grad_weight(const LinearGradParams& p, hipStream_t st) {
  const int64_t groups = (int64_t)p.n_groups * p.mats;
  const unsigned grid = tile_grid((p.n + kBR - 1) / kBR * groups * p.splits, p.k, kBC);
  if (!grid) return fail(HSMOE_ERR_SHAPE, "hsmoe_linear_grad_weight: too many tiles");
  hipLaunchKernelGGL((linear_grad_weight_kernel<kBR, kBC, kWR, kWC, kStages>), dim3(grid), dim3(kWR * kWC * 64), 0, st, p);
  if (p.part)
    hipLaunchKernelGGL(linear_grad_join_kernel<true>, dim3(join_grid(groups * p.n * p.k)), dim3(256), 0, st, p);
  return check_launch("hsmoe_linear_grad_weight");
}

// Shares of a group's rows in act_grad_kernel: enough workgroups for the chip,
// at least 64 rows each.
int act_shares(int64_t m, int64_t n, int64_t n_groups) {
  const int64_t blocks = (n + 255) / 256 * n_groups, rows = (m + n_groups - 1) / n_groups;
  int64_t shares = (4 * 256 + blocks - 1) / blocks;
  if (shares > (rows + 63) / 64) shares = (rows + 63) / 64;
  return (int)(shares < 1 ? 1 : shares > 256 ? 256 : shares);
}

}  // namespace
}  // namespace hsmoe

using namespace hsmoe;

// The rule's answer for a product, as the entry points ask for it below.
extern "C" int hsmoe_linear_plan(int product, int64_t m, int64_t n, int64_t k, int64_t n_groups, int act, int32_t plan[4]) {
  if (!plan) return fail(HSMOE_ERR_ARG, "hsmoe_linear_plan: null pointer");
  if (m < 1 || n < 1 || k < 1 || n_groups < 1) return fail(HSMOE_ERR_ARG, "hsmoe_linear_plan: bad counts");
  if (act != HSMOE_ACT_NONE && act != HSMOE_ACT_SILU && act != HSMOE_ACT_SWIGLU)
    return fail(HSMOE_ERR_ARG, "hsmoe_linear_plan: bad activation %d", act);
  const int mats = act == HSMOE_ACT_SWIGLU ? 2 : 1;
  Plan p{};
  if (product == HSMOE_LINEAR_OUT) p = plan_linear(m, n, k, n_groups, act);
  else if (product == HSMOE_LINEAR_DX) p = plan_grad_input(m, n, k, n_groups, mats);
  else if (product == HSMOE_LINEAR_DW) p = plan_grad_weight(m, n, k, n_groups, mats);
  else return fail(HSMOE_ERR_ARG, "hsmoe_linear_plan: bad product %d", product);
  if (p.tile == kNarrow) {
    plan[0] = plan[1] = kNarrowRows, plan[2] = 2, plan[3] = 1;
  } else {
    const TileCost& c = kTiles[p.tile];
    plan[0] = c.rows, plan[1] = c.cols, plan[2] = c.per_cu, plan[3] = p.splits;
  }
  return HSMOE_OK;
}

extern "C" size_t hsmoe_linear_workspace_size(int64_t m, int64_t n, int64_t k, int64_t n_groups, int act) {
  return m < 1 || n < 1 || k < 1 || n_groups < 1 ? 0 : plan_linear(m, n, k, n_groups, act).bytes;
}

extern "C" int hsmoe_linear(const void* x, int64_t x_row_stride, int64_t m, int64_t k, const void* w, const void* w_up,
                            int64_t w_row_stride, int64_t w_group_stride, int64_t n, const int32_t* offsets,
                            int64_t n_groups, const void* bias, const void* bias_up, const void* residual,
                            int64_t res_row_stride, int act, float limit, int out_kind, void* out, void* pre,
                            void* workspace, size_t workspace_bytes, hsmoe_stream_t stream) {
  if (int rc = check_counts("hsmoe_linear", m, n, k, n_groups, offsets)) return rc;
  if (act != HSMOE_ACT_NONE && act != HSMOE_ACT_SILU && act != HSMOE_ACT_SWIGLU)
    return fail(HSMOE_ERR_ARG, "hsmoe_linear: bad activation %d", act);
  if (out_kind != HSMOE_OUT_F32 && out_kind != HSMOE_OUT_BF16)
    return fail(HSMOE_ERR_ARG, "hsmoe_linear: bad output kind %d", out_kind);
  const bool gated = act == HSMOE_ACT_SWIGLU;
  if (gated != (w_up != nullptr) || (bias_up && !gated))
    return fail(HSMOE_ERR_ARG, "hsmoe_linear: an up weight goes with swiglu, and only with it");
  if (gated && !(limit > 0.0f)) return fail(HSMOE_ERR_ARG, "hsmoe_linear: the limit of swiglu must be positive");
  if (m == 0) return HSMOE_OK;
  if (int rc = check_matrix("hsmoe_linear", "x", x, k, x_row_stride)) return rc;
  if (int rc = check_matrix("hsmoe_linear", "w", w, k, w_row_stride)) return rc;
  if (gated)
    if (int rc = check_matrix("hsmoe_linear", "w_up", w_up, k, w_row_stride)) return rc;
  if (n_groups > 1 && w_group_stride % 8 != 0)
    return fail(HSMOE_ERR_SHAPE, "hsmoe_linear: the groups' matrices must be 16-byte aligned");
  if (residual)
    if (int rc = check_matrix("hsmoe_linear", "the residual", residual, n, res_row_stride)) return rc;
  if (int rc = check_matrix("hsmoe_linear", "out", out, n, n)) return rc;
  if ((bias && !aligned(bias, 16)) || (bias_up && !aligned(bias_up, 16)) || (pre && !aligned(pre, 16)))
    return fail(HSMOE_ERR_SHAPE, "hsmoe_linear: bias and pre must be 16-byte aligned");
  LinearParams p{};
  p.x = (const char*)x;
  p.w[0] = (const char*)w;
  p.w[1] = (const char*)w_up;
  p.bias[0] = (const char*)bias;
  p.bias[1] = (const char*)bias_up;
  p.residual = (const char*)residual;
  p.out = (char*)out;
  p.pre = (uint16_t*)pre;
  p.offsets = offsets;
  p.n_rows = m, p.n = n, p.k = k;
  p.ldx = x_row_stride * 2, p.ldw = w_row_stride * 2, p.w_group = w_group_stride * 2, p.ld_res = res_row_stride * 2;
  p.n_groups = (int)n_groups, p.act = act, p.out_f32 = out_kind == HSMOE_OUT_F32, p.limit = limit;
  const Plan plan = plan_linear(m, n, k, n_groups, act);
  if (int rc = check_workspace("hsmoe_linear", plan, workspace, workspace_bytes)) return rc;
  p.splits = plan.splits, p.part = plan.bytes ? (float*)workspace : nullptr;
  hipStream_t st = (hipStream_t)stream;
  if (plan.tile == kNarrow) return launch_narrow(p, st);
  if (plan.tile == 0 && offsets) return launch_linear<256, 256, 2, 4, kTurnsFar>(p, st);
  if (plan.tile == 0) return launch_linear<256, 256, 2, 4, kTurnsNear>(p, st);
  if (plan.tile == 1) return launch_linear<128, 128, 4, 2, 4>(p, st);
  if (plan.tile == 2) return launch_linear<64, 128, 2, 2, 4>(p, st);
  if (plan.tile == 3) return launch_linear<128, 128, 2, 2, 2>(p, st);
  return launch_linear_as<256, 128, 4, 2, 3, false>(p, st);
}

extern "C" size_t hsmoe_linear_act_grad_workspace_size(int64_t m, int64_t n, int64_t n_groups, int act) {
  if (m < 1 || n < 1 || n_groups < 1) return 0;
  const int shares = act_shares(m, n, n_groups);
  return shares == 1 ? 0 : (size_t)shares * n_groups * n * (act == HSMOE_ACT_SWIGLU ? 2 : 1) * 4;
}

extern "C" int hsmoe_linear_act_grad(const void* d_out, int64_t d_row_stride, const void* pre, int64_t m, int64_t n,
                                     int act, float limit, const int32_t* offsets, int64_t n_groups, void* dz,
                                     float* d_bias, float* d_bias_up, void* workspace, size_t workspace_bytes,
                                     hsmoe_stream_t stream) {
  if (int rc = check_counts("hsmoe_linear_act_grad", m, n, 8, n_groups, offsets)) return rc;
  if (act != HSMOE_ACT_NONE && act != HSMOE_ACT_SILU && act != HSMOE_ACT_SWIGLU)
    return fail(HSMOE_ERR_ARG, "hsmoe_linear_act_grad: bad activation %d", act);
  const bool gated = act == HSMOE_ACT_SWIGLU;
  if (d_bias_up && !gated) return fail(HSMOE_ERR_ARG, "hsmoe_linear_act_grad: an up bias goes with swiglu");
  if (gated && !(limit > 0.0f))
    return fail(HSMOE_ERR_ARG, "hsmoe_linear_act_grad: the limit of swiglu must be positive");
  if (!dz && !d_bias && !d_bias_up) return HSMOE_OK;
  if (m > 0) {
    if (int rc = check_matrix("hsmoe_linear_act_grad", "d_out", d_out, n, d_row_stride)) return rc;
    if (act != HSMOE_ACT_NONE)
      if (int rc = check_matrix("hsmoe_linear_act_grad", "pre", pre, n, n)) return rc;
    if (dz && !aligned(dz, 16)) return fail(HSMOE_ERR_SHAPE, "hsmoe_linear_act_grad: dz must be 16-byte aligned");
  }
  const bool sums = d_bias || d_bias_up;
  if (m == 0 && !sums) return HSMOE_OK;
  const int shares = m > 0 ? act_shares(m, n, n_groups) : 1;
  const size_t need = sums ? hsmoe_linear_act_grad_workspace_size(m, n, n_groups, act) : 0;
  if (need && (!workspace || workspace_bytes < need))
    return fail(HSMOE_ERR_WORKSPACE, "hsmoe_linear_act_grad: workspace of %zu bytes needed", need);
  if (need && !aligned(workspace, 4)) return fail(HSMOE_ERR_SHAPE, "hsmoe_linear_act_grad: misaligned workspace");
  ActGradParams p{};
  p.d_out = (const uint16_t*)d_out;
  p.pre = act == HSMOE_ACT_NONE ? nullptr : (const uint16_t*)pre;
  p.dz = (uint16_t*)dz;
  p.part = need ? (float*)workspace : nullptr;
  p.d_bias[0] = d_bias, p.d_bias[1] = d_bias_up;
  p.offsets = offsets;
  p.n_rows = m, p.n = n, p.ld_out = d_row_stride;
  p.n_groups = (int)n_groups, p.act = act, p.mats = gated ? 2 : 1, p.shares = shares, p.limit = limit;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)((n + 255) / 256), (unsigned)n_groups, (unsigned)shares);
  const dim3 block(kActThreads);
  if (gated && sums)
    hipLaunchKernelGGL((act_grad_kernel<2, true>), grid, block, 0, st, p);
  else if (gated)
    hipLaunchKernelGGL((act_grad_kernel<2, false>), grid, block, 0, st, p);
  else if (sums)
    hipLaunchKernelGGL((act_grad_kernel<1, true>), grid, block, 0, st, p);
  else
    hipLaunchKernelGGL((act_grad_kernel<1, false>), grid, block, 0, st, p);
  if (need)
    hipLaunchKernelGGL(bias_sum_kernel, dim3((unsigned)((n * p.mats * n_groups + 255) / 256)), dim3(256), 0, st, p);
  return check_launch("hsmoe_linear_act_grad");
}

extern "C" size_t hsmoe_linear_grad_workspace_size(int64_t m, int64_t n, int64_t k, int64_t n_groups, int act) {
  if (m < 1 || n < 1 || k < 1 || n_groups < 1) return 0;
  const int mats = act == HSMOE_ACT_SWIGLU ? 2 : 1;
  const size_t a = plan_grad_input(m, n, k, n_groups, mats).bytes, b = plan_grad_weight(m, n, k, n_groups, mats).bytes;
  return a > b ? a : b;
}

extern "C" int hsmoe_linear_grad_input(const void* dz, int64_t dz_row_stride, int64_t m, int64_t n, const void* w,
                                       const void* w_up, int64_t w_row_stride, int64_t w_group_stride, int64_t k,
                                       const int32_t* offsets, int64_t n_groups, void* dx, void* workspace,
                                       size_t workspace_bytes, hsmoe_stream_t stream) {
  if (int rc = check_counts("hsmoe_linear_grad_input", m, n, k, n_groups, offsets)) return rc;
  if (m == 0) return HSMOE_OK;
  const int mats = w_up ? 2 : 1;
  if (int rc = check_matrix("hsmoe_linear_grad_input", "dz", dz, n * mats, dz_row_stride)) return rc;
  if (int rc = check_matrix("hsmoe_linear_grad_input", "w", w, k, w_row_stride)) return rc;
  if (w_up)
    if (int rc = check_matrix("hsmoe_linear_grad_input", "w_up", w_up, k, w_row_stride)) return rc;
  if (n_groups > 1 && w_group_stride % 8 != 0)
    return fail(HSMOE_ERR_SHAPE, "hsmoe_linear_grad_input: the groups' matrices must be 16-byte aligned");
  if (int rc = check_matrix("hsmoe_linear_grad_input", "dx", dx, k, k)) return rc;
  LinearGradParams p{};
  p.dz = (const char*)dz;
  p.w[0] = (const char*)w, p.w[1] = (const char*)w_up;
  p.dx = (char*)dx;
  p.offsets = offsets;
  p.n_rows = m, p.n = n, p.k = k;
  p.ldz = dz_row_stride * 2, p.ldw = w_row_stride * 2, p.w_group = w_group_stride * 2;
  p.n_groups = (int)n_groups, p.mats = mats;
  const Plan plan = plan_grad_input(m, n, k, n_groups, mats);
  if (int rc = check_workspace("hsmoe_linear_grad_input", plan, workspace, workspace_bytes)) return rc;
  p.splits = plan.splits, p.part = plan.bytes ? (float*)workspace : nullptr;
  hipStream_t st = (hipStream_t)stream;
  if (plan.tile == 0 && offsets) return launch_grad_input<256, 256, 2, 4, kTurnsFar>(p, st);
  if (plan.tile == 0) return launch_grad_input<256, 256, 2, 4, kTurnsNear>(p, st);
  if (plan.tile == 1) return launch_grad_input<128, 128, 4, 2, 4>(p, st);
  if (plan.tile == 2) return launch_grad_input<64, 128, 2, 2, 4>(p, st);
  if (plan.tile == 3) return launch_grad_input<128, 128, 2, 2, 2>(p, st);
  return launch_grad_input<256, 128, 4, 2, 3>(p, st);
}

extern "C" int hsmoe_linear_grad_weight(const void* dz, int64_t dz_row_stride, const void* x, int64_t x_row_stride,
                                        int64_t m, int64_t n, int64_t k, const int32_t* offsets, int64_t n_groups,
                                        int out_kind, void* dw, void* dw_up, void* workspace, size_t workspace_bytes,
                                        hsmoe_stream_t stream) {
  if (int rc = check_counts("hsmoe_linear_grad_weight", m, n, k, n_groups, offsets)) return rc;
  if (out_kind != HSMOE_OUT_F32 && out_kind != HSMOE_OUT_BF16)
    return fail(HSMOE_ERR_ARG, "hsmoe_linear_grad_weight: bad output kind %d", out_kind);
  const int mats = dw_up ? 2 : 1;
  if (m > 0) {
    if (int rc = check_matrix("hsmoe_linear_grad_weight", "dz", dz, n * mats, dz_row_stride)) return rc;
    if (int rc = check_matrix("hsmoe_linear_grad_weight", "x", x, k, x_row_stride)) return rc;
  }
  if (int rc = check_matrix("hsmoe_linear_grad_weight", "dw", dw, k, k)) return rc;
  if (dw_up)
    if (int rc = check_matrix("hsmoe_linear_grad_weight", "dw_up", dw_up, k, k)) return rc;
  LinearGradParams p{};
  p.dz = (const char*)dz, p.x = (const char*)x;
  p.dw[0] = (char*)dw, p.dw[1] = (char*)dw_up;
  p.offsets = offsets;
  p.n_rows = m, p.n = n, p.k = k;
  p.ldz = dz_row_stride * 2, p.ldx = x_row_stride * 2;
  p.n_groups = (int)n_groups, p.mats = mats, p.dw_f32 = out_kind == HSMOE_OUT_F32;
  const Plan plan = plan_grad_weight(m > 0 ? m : 1, n, k, n_groups, mats);
  if (int rc = check_workspace("hsmoe_linear_grad_weight", plan, workspace, workspace_bytes)) return rc;
  p.splits = plan.splits, p.part = plan.bytes ? (float*)workspace : nullptr;
  hipStream_t st = (hipStream_t)stream;
  if (plan.tile == 0) return launch_grad_weight<256, 256, 2, 4, kTurnsNear>(p, st);
  return launch_grad_weight<128, 128, 4, 2, 4>(p, st);
}

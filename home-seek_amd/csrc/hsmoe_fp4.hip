// Microscaled 4-bit floating point: quantisation to the experts' format (e2m1
// codes, low nibble first, and one power of two (E8M0) per 32 values of a row)
// and the product of two such operands,
//   out[m, n] = sum_b 2^(ex[m, b] + ew[n, b] - 254) sum_j cx[m, b, j] cw[n, b, j]
// on the scaled matrix instructions, which take codes and exponents as they are.
// Their sums of e2m1 products are exact while the exponents of one instruction
// (two or four blocks of 32) lie within 2^10 of each other; beyond, what is lost is
// below 2^-20 of the largest product, whatever the distance (against 64 bits, k = 1024,
// both operands' exponents spread over +-4, +-10 .. +-60: results off by 2^-21.7 of the
// sum of their products' magnitudes at most, with the additions in fp32).
#include <algorithm>
#include <type_traits>

#include "hsmoe_common.h"
#include "hsmoe_internal.h"
#include "hsmoe_stage.h"

namespace hsmoe {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kStep = 256;   // values of the reduction per stage: 128 bytes of codes, 8 scales
constexpr int kUnit = 512;   // values that a wave quantises at a time, and few_kernel's stage

// ---------------------------------------------------------------- quantisation
// Scales where the tiles want them, "dealt": a lane (r, h) of a matrix
// instruction over 64 values takes 32 of row r; with the values of a stage dealt
// so that half h takes blocks 4 h .. 4 h + 3 in its four instructions, its four
// scales are one word.  Word (stage, row / 32, h, row % 32); zeros beyond the
// rows and beyond k.
__host__ __device__ __forceinline__ int64_t dealt_word(int64_t stage, int64_t row, int h, int64_t row_blocks) {
  return (stage * row_blocks + (row >> 5)) * 64 + h * 32 + (row & 31);
}

enum { kRowsF32 = HSMOE_OUT_F32, kRowsBf16 = HSMOE_OUT_BF16 };

struct Eight {
  uint32_t v[8];  // fp32 bits
};
template <int kKind>
__device__ __forceinline__ Eight load_eight(const char* p) {
  Eight e;
  if (kKind == kRowsBf16) {
    const uint4 u = ldg<uint4>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) e.v[2 * i] = w[i] << 16, e.v[2 * i + 1] = w[i] & 0xffff0000u;
  } else {
    const uint4 a = ldg<uint4>(p), b = ldg<uint4>(p + 16);
    e = {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
  }
  return e;
}

// Eight values per lane, a block per four lanes: the lane's codes, and the block's
// scale.  The exponent is the smallest with which the largest magnitude
// 1.f 2^(E - 127) is at most 6 = 1.5 * 2^2, so nothing saturates; rounding is the
// hardware's, to nearest with ties to the even code.  A block with an infinity or
// NaN has exponent 255, which is NaN whatever the codes.
__device__ __forceinline__ uint32_t quantise8(const Eight& x, uint32_t& exponent) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = x.v[i] & 0x7fffffffu;  // magnitudes in the order of their bits, NaN above all
    top = a > top ? a : top;
  }
  uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xf, 0xf, true);  // lane ^ 1
  top = o > top ? o : top;
  o = (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xf, 0xf, true);  // lane ^ 2
  top = o > top ? o : top;
  const int biased = (int)(top >> 23) - ((top & 0x7fffffu) > 0x400000u ? 1 : 2);
  const uint32_t e = top >= 0x7f800000u ? 255u : biased > 0 ? (uint32_t)biased : 0u;
  exponent = e;
  const float s = __uint_as_float(e << 23);  // (the conversion reads the exponent's bits: 0 is 2^-127)
  auto f = [&](int i) { return __uint_as_float(x.v[i]); };
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(0), f(1), s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(2), f(3), s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(4), f(5), s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(6), f(7), s, 3);
  return w;
}
// The exponents of 16 lanes' four blocks as one word, in every lane.
__device__ __forceinline__ uint32_t gather_exponents(uint32_t e, int lane) {
  uint32_t v = e << (8 * (lane >> 2 & 3));
  v |= (uint32_t)__shfl_xor((int)v, 4, 64);
  v |= (uint32_t)__shfl_xor((int)v, 8, 64);
  return v;
}

struct QuantParams {
  const char* x;      // [m] rows of k values, ldx bytes apart
  char* codes;        // [m][k / 2]
  uint8_t* scale;     // [m][ld_scale], or dealt words
  int64_t m, k, ldx, ld_scale;
  int64_t units;      // waves' units per row
  int across;         // of a workgroup's waves, so many side by side in a row, the others in further rows
  int64_t row_blocks; // dealt words: blocks of 32 rows (0: rows of scales)
};

// A wave takes 512 values of kRows rows: eight values per lane, 16 bytes in (bf16), 4
// out, whole lines both ways.  HBM-bound (8190 x 4096 bf16 with the weights' scales
// 19 us, 4.6 TB/s; the copy's rate would be 17); one row per wave where few rows would
// leave the chip idle (33 rows 2.9 us, 5.4 with four).
template <int kKind, int kRows>
__device__ __forceinline__ void quant_rows(const QuantParams& p, int64_t row0, int seg, int lane) {
  if (row0 >= p.m) return;
  const int64_t at = (int64_t)seg * kUnit + lane * 8;
  const int rows = p.m - row0 < kRows ? (int)(p.m - row0) : kRows;
  Eight x[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    x[i] = Eight{};
    if (i < rows && at < p.k) x[i] = load_eight<kKind>(p.x + (row0 + i) * p.ldx + at * (kKind == kRowsBf16 ? 2 : 4));
  }
  uint32_t words[kRows];
  const int64_t group = (int64_t)seg * 4 + (lane >> 4);  // of four blocks
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    uint32_t e;
    const uint32_t w = quantise8(x[i], e);
    if (i < rows && at < p.k) *reinterpret_cast<uint32_t*>(p.codes + (row0 + i) * (p.k / 2) + at / 2) = w;
    if (at >= p.k) e = 0;  // padding of the words
    words[i] = gather_exponents(e, lane);
    if (p.row_blocks || i >= rows) continue;
    uint8_t* to = p.scale + (row0 + i) * p.ld_scale;
    if (p.ld_scale % 4 == 0) {
      if ((lane & 15) == 0 && group * 4 < p.ld_scale) *reinterpret_cast<uint32_t*>(to + group * 4) = words[i];
    } else if ((lane & 3) == 0 && at < p.k) {
      to[at / 32] = (uint8_t)e;
    }
  }
  if (p.row_blocks && (lane & 15) == 0) {  // (rows beyond the last have words too)
    uint32_t* to = reinterpret_cast<uint32_t*>(p.scale) + dealt_word(group >> 1, row0, (int)(group & 1), p.row_blocks);
    if constexpr (kRows == 4)
      *reinterpret_cast<uint4*>(to) = make_uint4(words[0], words[1], words[2], words[3]);
    else
      to[0] = words[0];
  }
}

// Rows of scales [rows][blocks] dealt to words: a thread takes 16 blocks of a row.
struct DealParams {
  const uint8_t* scale;
  uint32_t* words;
  int64_t rows, blocks, row_blocks, groups;  // groups of 16 blocks
};
__device__ __forceinline__ void deal_scales(const DealParams& p, int64_t t) {
  const int64_t row = (t >> 5) / p.groups * 32 + (t & 31), g = (t >> 5) % p.groups;
  if (row >= p.row_blocks * 32) return;
  uint32_t w[4] = {0, 0, 0, 0};
  if (row < p.rows) {
    const uint8_t* s = p.scale + row * p.blocks + g * 16;
    if (p.blocks % 16 == 0) {
      const uint4 u = ldg<uint4>(s);
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (g * 16 + i < p.blocks) w[i >> 2] |= (uint32_t)s[i] << (8 * (i & 3));
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) p.words[dealt_word(2 * g + (i >> 1), row, i & 1, p.row_blocks)] = w[i];
}

constexpr int kQuantThreads = 256;
constexpr int kQuantWaves = kQuantThreads / 64;

// Workgroup b's part: four waves side by side read 4 KB of a row in one piece, and the
// workgroups go through the rows in the order of memory (65536 x 4096 bf16 149 us with
// the waves in further rows, 130 so; fp32 8190 x 4096 36 and 29).
template <int kKind, int kRows>
__device__ __forceinline__ void quant_group(const QuantParams& p, uint32_t b) {
  const uint32_t parts = (uint32_t)p.units / p.across, r = b / parts, wave = threadIdx.x >> 6, down = wave / p.across;
  const int seg = (int)((b - r * parts) * p.across + (wave - down * p.across));
  quant_rows<kKind, kRows>(p, ((int64_t)r * (kQuantWaves / p.across) + down) * kRows, seg, threadIdx.x & 63);
}
template <int kKind, int kRows>
__global__ void __launch_bounds__(kQuantThreads) fp4_quant_kernel(QuantParams p) {
  quant_group<kKind, kRows>(p, blockIdx.x);
}

// What a product wants before it: x quantised (kKind < 0: its scales dealt) by the
// first `first_blocks` workgroups, the weights' scales dealt by the others.
template <int kKind, int kRows>
__global__ void __launch_bounds__(kQuantThreads) fp4_ready_kernel(QuantParams q, DealParams x, DealParams w, uint32_t first_blocks) {
  if (blockIdx.x >= first_blocks) {
    deal_scales(w, (int64_t)(blockIdx.x - first_blocks) * kQuantThreads + threadIdx.x);
  } else if constexpr (kKind < 0) {
    deal_scales(x, (int64_t)blockIdx.x * kQuantThreads + threadIdx.x);
  } else {
    quant_group<kKind, kRows>(q, blockIdx.x);
  }
}

// ---------------------------------------------------------------- tiles
struct Fp4Params {
  const char* x;        // [m][k / 2]
  const char* w;        // [n][k / 2]
  const uint8_t* xs;    // few rows: [m][ld_xs]; tiles: dealt words from `words` on
  const uint8_t* ws;    // few rows: [n][k / 32]
  const char* words;    // both operands' dealt words
  uint32_t x_words, w_words, words_bytes;  // offsets of the operands' and size of it all
  char* out;            // [m][n]
  int64_t m, n, k, ld_xs;
  int out_f32;
};

__device__ __forceinline__ i32x8 widen(i32x4 v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }
template <int kByte>
__device__ __forceinline__ f32x16 mfma32(i32x4 a, i32x4 b, f32x16 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widen(a), widen(b), c, 4, 4, kByte, sa, kByte, sb);
}
template <int kByte>
__device__ __forceinline__ f32x4 mfma16(i32x4 a, i32x4 b, f32x4 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(a), widen(b), c, 4, 4, kByte, sa, kByte, sb);
}

// A tile of kBR rows of x by kBC rows of w, kWR x kWC waves, each 32 x 32 blocks of
// v_mfma_scale_f32_32x32x64.  A stage is 256 values of both operands: [row][128 bytes] with a row's 16-byte chunk
// c at place c ^ (row / 2 % 8), loaded straight to LDS, then the scales' words.
// Instruction s takes chunk 4 h + s of a row in lanes of half h.  Measured, 256 x 256
// tiles by eight waves: 8190 x 4096 x 4096 72 us, 3.8 PFLOP/s.  A loop of these
// instructions alone makes 6.2 PFLOP/s of random codes and 8.9 of zeros, and this
// kernel 3.9 and 5.0 at 8192^3, 63% and 56% of it: zeros save 22% there and 8% at the
// size above, so power is the smaller part of what is left; 8 us of a tile's 36 are
// its start and end, when nothing multiplies.  Two stages without
// turns, and four waves of 128 x 128 with the next operands read ahead, take as long.
// kStages_ 0: two stages, eight waves in turns.
template <int kBR, int kBC, int kWR, int kWC, int kStages_>
struct Fp4Tile {
  static constexpr bool kTurns = kStages_ == 0;
  static constexpr int kStages = kTurns ? 2 : kStages_;
  static constexpr int kWaves = kWR * kWC, kThreads = kWaves * 64;
  static_assert(!kTurns || kWaves == 8, "two waves per SIMD");
  static constexpr int kFR = kBR / kWR / 32, kFC = kBC / kWC / 32;
  static constexpr int kRowsBytes = kBR * 128, kColsBytes = kBC * 128, kScaleBytes = (kBR + kBC) * 8;
  static constexpr int kStage = kRowsBytes + kColsBytes + kScaleBytes;
  static constexpr int kLds = kStages * kStage;
  static constexpr int kRowLoads = kRowsBytes / 1024 / kWaves, kColLoads = kColsBytes / 1024 / kWaves;
  static constexpr int kScaleLanes = kScaleBytes / 16 / kWaves;  // of each wave, one load
  static constexpr int kLoads = kRowLoads + kColLoads + 1;
  static constexpr int kOutPitch = kFC * 32 + 4;  // fp32 words of a row on its way out
  static_assert(kScaleLanes <= 64 && kRowsBytes % (1024 * kWaves) == 0 && kColsBytes % (1024 * kWaves) == 0, "whole loads");
  static_assert(kWaves * 32 * kOutPitch * 4 <= kLds, "a wave's 32 rows on their way out");

  static __device__ __forceinline__ int turn(int row) { return row >> 1 & 7; }
  static __device__ __forceinline__ i32x4 frag(const char* part, int row0, int s, int lane) {
    const int row = row0 + (lane & 31), c = 4 * (lane >> 5) + s;
    return *reinterpret_cast<const i32x4*>(part + row * 128 + (c ^ turn(row)) * 16);
  }
};

// One operand's loads: `rows` rows of `bytes` bytes, zeros beyond both.
template <int kLoads>
struct Fp4Source {
  const char* base;
  uint32_t width, at[kLoads];
  int chunk[kLoads];
  __device__ __forceinline__ void open(const char* p, int rows, int64_t bytes, int wave, int lane) {
    base = p;
    width = (uint32_t)((rows - 1) * bytes + bytes);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = (wave * kLoads + i) * 8 + (lane >> 3);
      chunk[i] = (lane & 7) ^ (row >> 1 & 7);
      at[i] = (uint32_t)(row * bytes) + chunk[i] * 16;
    }
  }
  // stage s of which `left` blocks of 32 are there
  __device__ __forceinline__ void load(int s, int left, char* part, int wave) const {
    const i32x4 r = lds_buf(base, width);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      lds_load16(r, (at[i] + (uint32_t)s * 128) | past(chunk[i], left), part + (wave * kLoads + i) * 1024);
  }
};

// kSplit 2: twice the waves, of which the second half takes every other stage into
// memory of its own; the sums are joined at the end.
template <int kBR, int kBC, int kWR, int kWC, int kStages_, int kSplit>
__global__ void __launch_bounds__(kWR* kWC * 64 * kSplit) __attribute__((amdgpu_waves_per_eu(2, 2))) fp4_tile_kernel(Fp4Params p) {
  using T = Fp4Tile<kBR, kBC, kWR, kWC, kStages_>;
  constexpr int kStages = T::kStages;
  static_assert(kSplit == 1 || (kSplit == 2 && !T::kTurns && T::kWaves * T::kFR * T::kFC * 4096 <= T::kLds), "two halves, whose sums fit");
  __shared__ __align__(1024) char memory[kSplit * T::kLds];
  const int lane = threadIdx.x & 63, any = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = kSplit == 1 ? 0 : any / T::kWaves, wave = any - part * T::kWaves;
  char* lds = memory + part * T::kLds;
  int rt, ct;
  if (!place_tile(blockIdx.x, (int)((p.m + kBR - 1) / kBR), (int)((p.n + kBC - 1) / kBC), rt, ct)) return;
  const int64_t m0 = (int64_t)rt * kBR, n0 = (int64_t)ct * kBC, row_bytes = p.k / 2;
  const int rows = (int)imin64(kBR, p.m - m0), cols = (int)imin64(kBC, p.n - n0);
  const int blocks = (int)(p.k / 32), steps = (int)((p.k + kStep - 1) / kStep);
  Fp4Source<T::kRowLoads> xs;
  xs.open(p.x + m0 * row_bytes, rows, row_bytes, wave, lane);
  Fp4Source<T::kColLoads> ws;
  ws.open(p.w + n0 * row_bytes, cols, row_bytes, wave, lane);
  // the wave's share of a stage's words: the lane's 16 bytes of [rows | cols]
  const uint32_t mine = (uint32_t)(wave * T::kScaleLanes + lane) * 16;
  const bool of_rows = mine < kBR * 8;
  const uint32_t scale_step = (uint32_t)((of_rows ? p.m : p.n) + 31) / 32 * 256;
  const uint32_t scale_at = of_rows ? p.x_words + (uint32_t)(m0 / 32) * 256 + mine
                                    : p.w_words + (uint32_t)(n0 / 32) * 256 + mine - kBR * 8;
  auto load = [&](int s, int slot) {
    char* stage = lds + slot * T::kStage;
    const int left = blocks - 8 * s;
    xs.load(s, left, stage, wave);
    ws.load(s, left, stage + T::kRowsBytes, wave);
    const i32x4 r = lds_buf(p.words, p.words_bytes);
    if (lane < T::kScaleLanes)
      lds_load16(r, (scale_at + (uint32_t)s * scale_step) | past(s, steps),
                 stage + T::kRowsBytes + T::kColsBytes + wave * T::kScaleLanes * 16);
  };
  const int wr = wave / kWC, wc = wave % kWC;
  f32x16 acc[T::kFR][T::kFC] = {};
  int sr[T::kFR], sc[T::kFC];
  auto read_scales = [&](const char* stage) {
    const char* scales = stage + T::kRowsBytes + T::kColsBytes;
#pragma unroll
    for (int i = 0; i < T::kFR; ++i) sr[i] = *reinterpret_cast<const int*>(scales + (wr * T::kFR + i) * 256 + lane * 4);
#pragma unroll
    for (int j = 0; j < T::kFC; ++j)
      sc[j] = *reinterpret_cast<const int*>(scales + kBR * 8 + (wc * T::kFC + j) * 256 + lane * 4);
  };
  auto read = [&](const char* stage, int step, i32x4 (&r)[T::kFR], i32x4 (&c)[T::kFC]) {
#pragma unroll
    for (int j = 0; j < T::kFC; ++j) c[j] = T::frag(stage + T::kRowsBytes, (wc * T::kFC + j) * 32, step, lane);
#pragma unroll
    for (int i = 0; i < T::kFR; ++i) r[i] = T::frag(stage, (wr * T::kFR + i) * 32, step, lane);
  };
  auto multiply = [&](auto step, const i32x4 (&r)[T::kFR], const i32x4 (&c)[T::kFC]) {
    constexpr int kByte = decltype(step)::value;
#pragma unroll
    for (int i = 0; i < T::kFR; ++i)
#pragma unroll
      for (int j = 0; j < T::kFC; ++j) acc[i][j] = mfma32<kByte>(c[j], r[i], acc[i][j], sc[j], sr[i]);
  };
  constexpr std::integral_constant<int, 0> k0;
  constexpr std::integral_constant<int, 1> k1;
  constexpr std::integral_constant<int, 2> k2;
  constexpr std::integral_constant<int, 3> k3;
  if constexpr (T::kTurns) {
    // Two waves share a SIMD (w and w + 4): one half's waves read a stage's operands
    // while the other half's multiply, with a barrier between the turns; the second
    // half is one turn behind.  The first half reads stage i in turn 2 i and multiplies in
    // turn 2 i + 1, the second reads in 2 i + 1 and multiplies in 2 i + 2.  So stage i's
    // place is free from turn 2 i + 2 on: each half issues its part of stage i + 2 in that
    // turn and waits for it at the end of turn 2 i + 3, before anybody reads it.
    // (Half a stage in a turn: 291 us for 282 at 8192^3.  Workgroups that go on to another
    // tile, its first stage loaded during the last products: 281 to 285.)
    const bool second = wave >= 4;
    // (a wave without rows in the tile only keeps the turns; the branch also keeps the
    // products between the barriers, where the compiler would move them behind the last)
    const bool live = rows > wr * T::kFR * 32;
    i32x4 r[4][T::kFR], c[4][T::kFC];
    auto turn = [&](bool loads) {  // ends a turn; loads: what the wave loads of the next stage is in LDS
      if (loads) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("" ::: "memory");
    };
    load(0, 0);
    turn(true);
    if (second) {
      if (steps > 1) load(1, 1);
      turn(false);
    }
    for (int s = 0; s < steps; ++s) {
      const char* stage = lds + (s & 1) * T::kStage;
      read_scales(stage);
      read(stage, 0, r[0], c[0]);
      read(stage, 1, r[1], c[1]);
      read(stage, 2, r[2], c[2]);
      read(stage, 3, r[3], c[3]);
      if (!second && s + 1 < steps) load(s + 1, (s + 1) & 1);
      turn(second);
      if (second && s + 2 < steps) load(s + 2, s & 1);
      __builtin_amdgcn_s_setprio(1);
      if (live) multiply(k0, r[0], c[0]), multiply(k1, r[1], c[1]), multiply(k2, r[2], c[2]), multiply(k3, r[3], c[3]);
      __builtin_amdgcn_s_setprio(0);
      turn(!second);
    }
    if (!second) turn(false);
  } else {
    const int own = (steps + kSplit - 1) / kSplit;
    for (int s = 0; s < kStages - 1; ++s) load(s * kSplit + part, s);
    int at = 0, next = kStages - 1;
    for (int s = 0; s < own; ++s) {
      // stage s is whole when every wave's loads of it are, and nobody reads the one
      // before any more; stages beyond the last are loaded from nowhere, for the count
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kStages - 2) * T::kLoads) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      load((s + kStages - 1) * kSplit + part, next);
      const char* stage = lds + at * T::kStage;
      i32x4 r[T::kFR], c[T::kFC];
      read_scales(stage);
      read(stage, 0, r, c), multiply(k0, r, c);
      read(stage, 1, r, c), multiply(k1, r, c);
      read(stage, 2, r, c), multiply(k2, r, c);
      read(stage, 3, r, c), multiply(k3, r, c);
      at = at + 1 == kStages ? 0 : at + 1;
      next = next + 1 == kStages ? 0 : next + 1;
    }
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // no load may reach LDS once it is used for the results
  __syncthreads();
  if constexpr (kSplit == 2) {
    f32x4* sums = reinterpret_cast<f32x4*>(memory + T::kLds) + wave * T::kFR * T::kFC * 256 + lane;
#pragma unroll
    for (int i = 0; i < T::kFR; ++i)
#pragma unroll
      for (int j = 0; j < T::kFC; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (part) sums[((i * T::kFC + j) * 4 + q) * 64] = f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int i = 0; i < T::kFR; ++i)
#pragma unroll
      for (int j = 0; j < T::kFC; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 v = sums[((i * T::kFC + j) * 4 + q) * 64];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] += v[e];
        }
  }
  // A lane has row lane % 32 and columns 8 q + 4 h ..+3 of a block: 32 rows at a
  // time go through the wave's own part of LDS, to leave in whole lines.
  float* mem = reinterpret_cast<float*>(lds) + wave * 32 * T::kOutPitch;
  const int h = lane >> 5;
#pragma unroll
  for (int i = 0; i < T::kFR; ++i) {
    const int r0 = (wr * T::kFR + i) * 32;
#pragma unroll
    for (int j = 0; j < T::kFC; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(mem + (lane & 31) * T::kOutPitch + j * 32 + 8 * q + 4 * h) =
            f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    constexpr int kPer = T::kFC * 4;  // lanes of a row, eight columns each
    const int col = wc * T::kFC * 32 + lane % kPer * 8;
#pragma unroll
    for (int r = lane / kPer; r < 32; r += 64 / kPer) {
      const float* v = mem + r * T::kOutPitch + lane % kPer * 8;
      const f32x4 a = *reinterpret_cast<const f32x4*>(v), b = *reinterpret_cast<const f32x4*>(v + 4);
      if (r0 + r >= rows || col >= cols) continue;
      const int64_t o = (m0 + r0 + r) * p.n + n0 + col;
      if (p.out_f32) {
        f32x4* d = reinterpret_cast<f32x4*>(p.out + o * 4);
        d[0] = a, d[1] = b;
      } else {
        const uint32_t w[4] = {f32_to_bf16_bits(a[0]) | f32_to_bf16_bits(a[1]) << 16, f32_to_bf16_bits(a[2]) | f32_to_bf16_bits(a[3]) << 16,
                               f32_to_bf16_bits(b[0]) | f32_to_bf16_bits(b[1]) << 16, f32_to_bf16_bits(b[2]) | f32_to_bf16_bits(b[3]) << 16};
        *reinterpret_cast<uint4*>(p.out + o * 2) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

// ---------------------------------------------------------------- few rows
// Up to 16 kRB rows: a workgroup takes 16 columns, its four waves every fourth
// 512 values each, straight from memory to registers: a lane (row r, quarter g)
// has 64 bytes of its row, its four instructions' 32 values each, and one word of
// scales.  kFused: every workgroup quantises x for itself, into LDS, while its first
// weights are on their way: one launch.  What bounds it is the weights' stream, or for
// one small matrix the latency of one load of everything: 4096 x 4096 by one row 4.8 us,
// by 33 6.8 (of which the launch is 1.6).
constexpr int kFewLds = 8192;  // bytes of codes that a workgroup keeps of a quantised x
template <int kRB, int kKind, bool kAligned>
__global__ void __launch_bounds__(256) fp4_few_kernel(Fp4Params p, const char* x_raw, int64_t ldx) {
  constexpr bool kFused = kKind >= 0;
  __shared__ __align__(16) char codes[kFused ? kFewLds : 16];
  __shared__ __align__(16) uint32_t exps[kFused ? kFewLds / 64 + 64 : 4];
  __shared__ float sums[3][16][16 * kRB + 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16, blocks = p.k / 32, row_bytes = p.k / 2;
  const int units = (int)((p.k + kUnit - 1) / kUnit);
  const bool col_ok = n0 + r < p.n;
  const char* w_row = p.w + (n0 + (col_ok ? r : 0)) * row_bytes;
  const uint8_t* w_scale = p.ws + (n0 + (col_ok ? r : 0)) * blocks;
  struct Part {
    uint4 v[4];
    uint32_t scale;
  };
  auto load_w = [&](int u) {
    Part w{};
    const int64_t b0 = (int64_t)u * 16 + 4 * g;  // the lane's first block
    if (u < units && col_ok) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (b0 + i < blocks) w.v[i] = ldg<uint4>(w_row + (b0 + i) * 16);
      if (kAligned) {
        if (b0 < blocks) w.scale = ldg<uint32_t>(w_scale + b0);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (b0 + i < blocks) w.scale |= (uint32_t)w_scale[b0 + i] << (8 * i);
      }
    }
    return w;
  };
  Part w0 = load_w(wave), w1 = load_w(wave + 4);
  if constexpr (kFused) {
    for (int u = wave; u < p.m * units; u += 4) {
      const int row = u / units, seg = u % units, at = seg * kUnit + lane * 8;
      Eight x{};
      if (at < p.k) x = load_eight<kKind>(x_raw + row * ldx + (int64_t)at * (kKind == kRowsBf16 ? 2 : 4));
      uint32_t e;
      const uint32_t c = quantise8(x, e);
      if (at >= p.k) e = 0;
      const uint32_t word = gather_exponents(e, lane);
      *reinterpret_cast<uint32_t*>(codes + (row * units + seg) * 256 + lane * 4) = c;
      if ((lane & 15) == 0) exps[(row * units + seg) * 4 + g] = word;
    }
    __syncthreads();
  }
  f32x4 acc[kRB] = {};
  for (int u = wave; u < units; u += 8) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int v = u + 4 * half;
      if (v >= units) break;
      Part& w = half ? w1 : w0;
      i32x4 wv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) wv[i] = i32x4{(int)w.v[i].x, (int)w.v[i].y, (int)w.v[i].z, (int)w.v[i].w};
      const int w_scales = (int)w.scale;
#pragma unroll
      for (int b = 0; b < kRB; ++b) {
        const int row = 16 * b + r;
        i32x4 xv[4] = {};
        int x_scales = 0;
        if (row < p.m) {
          if constexpr (kFused) {
            const int unit = row * units + v;
#pragma unroll
            for (int i = 0; i < 4; ++i) xv[i] = *reinterpret_cast<const i32x4*>(codes + unit * 256 + g * 64 + i * 16);
            x_scales = (int)exps[unit * 4 + g];
          } else {
            const int64_t b0 = (int64_t)v * 16 + 4 * g;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (b0 + i < blocks) {
                const uint4 t = ldg<uint4>(p.x + row * row_bytes + (b0 + i) * 16);
                xv[i] = i32x4{(int)t.x, (int)t.y, (int)t.z, (int)t.w};
              }
            if (kAligned) {
              if (b0 < blocks) x_scales = (int)ldg<uint32_t>(p.xs + row * p.ld_xs + b0);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (b0 + i < blocks) x_scales |= (int)p.xs[row * p.ld_xs + b0 + i] << (8 * i);
            }
          }
        }
        acc[b] = mfma16<0>(wv[0], xv[0], acc[b], w_scales, x_scales);
        acc[b] = mfma16<1>(wv[1], xv[1], acc[b], w_scales, x_scales);
        acc[b] = mfma16<2>(wv[2], xv[2], acc[b], w_scales, x_scales);
        acc[b] = mfma16<3>(wv[3], xv[3], acc[b], w_scales, x_scales);
      }
      if (half) w1 = load_w(v + 8); else w0 = load_w(v + 8);
    }
  }
  // columns 4 g ..+3 of rows 16 b + r; the waves' sums in wave order
  if (wave > 0) {
#pragma unroll
    for (int b = 0; b < kRB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) sums[wave - 1][4 * g + i][16 * b + r] = acc[b][i];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int b = 0; b < kRB; ++b) {
    const int row = 16 * b + r;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = 4 * g + i;
      v[i] = acc[b][i] + sums[0][c][row] + sums[1][c][row] + sums[2][c][row];
    }
    const int64_t col = n0 + 4 * g;
    if (row >= p.m || col >= p.n) continue;
    const int64_t o = row * p.n + col;
    if (p.out_f32)
      *reinterpret_cast<f32x4*>(p.out + o * 4) = f32x4{v[0], v[1], v[2], v[3]};
    else
      *reinterpret_cast<uint2*>(p.out + o * 2) = make_uint2(f32_to_bf16_bits(v[0]) | f32_to_bf16_bits(v[1]) << 16,
                                                            f32_to_bf16_bits(v[2]) | f32_to_bf16_bits(v[3]) << 16);
  }
}

// ---------------------------------------------------------------- host
int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// Reductions that 64 x 64 tiles of which a CU has one at most share out to two halves of
// a workgroup: 128 rows by 4096 columns, k = 2048 8.3 us for 8.3, 4096 10.5 for 11.6, 16384
// 24.7 for 31.
bool halves(int64_t k) { return k > 8 * kStep; }

// Rows that fp4_few_kernel can take, and those that it does: its workgroups read x again
// for each 16 columns, so that many columns are for the tiles.  By estimated time: us
// from what a workgroup per CU takes (256 CUs), c of them one after the other (measured
// with k = 4096, kernel and tiles; 1, 16 and 64 rows by 4096 columns 4.3 and 9.6, 6.7
// and 9.7, 10.8 and 10.1; by 16384 8.7 and 11.3, 14.1 and 11.8, 29 and 12.5; by 129280 57 and
// 63, 93 and 61, 206 and 68; k = 1024, 4096 columns 3.0 and 6.3, 5.7 and 6.5, 7.2 and 6.7,
// 16384 columns 3.9 and 6.6, 7.9 and 6.7, 11.2 and 7.2; codes that are there 2 less with few).
constexpr int64_t kFewRows = 64;
bool takes_few(int64_t m, int64_t n, int64_t k, bool packed) {
  if (m > kFewRows) return false;
  if (up(n, 32) * up(k, kUnit) / 32 >= (1ll << 30)) return true;  // (more scales than the tiles' 32-bit offsets reach)
  const double c = (double)n / 4096, kk = (double)k / 4096, rows = 1.45 + 0.07 * m;
  const double few = packed ? 3.0 + c * kk * rows : 4.0 + c * kk * (m == 1 ? 1.5 : std::max(2.15, rows));
  return few <= std::max(5.1 + (halves(k) ? 4.8 : 5.9) * kk, 4.0 + 1.85 * c * kk);
}

// Rows per wave, waves side by side in a row and workgroups of a quantisation.
bool four_rows(int64_t m, int64_t units) { return m * units >= 8192; }
// Dealt words of sixteen rows are whole lines, so waves that write them take further rows.
int waves_across(int64_t units, bool dealt) { return dealt ? 1 : units % 4 == 0 ? 4 : units % 2 == 0 ? 2 : 1; }
int64_t quant_groups(int64_t m, int64_t units, bool dealt) {
  const int across = waves_across(units, dealt);
  const int64_t rows = kQuantWaves / across * (four_rows(m, units) ? 4 : 1);
  return (m + rows - 1) / rows * (units / across);
}
void launch_quant(const QuantParams& q, bool bf16, hipStream_t st) {
  const dim3 grid((unsigned)quant_groups(q.m, q.units, q.row_blocks)), block(kQuantThreads);
  if (bf16 && four_rows(q.m, q.units))
    hipLaunchKernelGGL((fp4_quant_kernel<kRowsBf16, 4>), grid, block, 0, st, q);
  else if (bf16)
    hipLaunchKernelGGL((fp4_quant_kernel<kRowsBf16, 1>), grid, block, 0, st, q);
  else if (four_rows(q.m, q.units))
    hipLaunchKernelGGL((fp4_quant_kernel<kRowsF32, 4>), grid, block, 0, st, q);
  else
    hipLaunchKernelGGL((fp4_quant_kernel<kRowsF32, 1>), grid, block, 0, st, q);
}

// What a product does and where its workspace keeps what.
struct Fp4Plan {
  bool few, fused, split;
  int tile;                    // 0: 256 x 256, 1: 128 x 128, 2: 64 x 64
  int64_t codes, xs, ws, bytes;  // offsets: x's codes, its scales, the weights' dealt words; size
};
Fp4Plan plan_fp4(int64_t m, int64_t n, int64_t k, bool packed) {
  Fp4Plan p{};
  p.few = takes_few(m, n, k, packed);
  p.fused = p.few && m <= 16 && !packed && m * up(k, kUnit) / 2 <= kFewLds;
  if (p.fused) return p;
  const int64_t stages = up(k, kUnit) / kStep;
  p.codes = 0;
  p.xs = packed ? 0 : up(m * (k / 2), 256);
  if (p.few) {
    p.ws = p.bytes = packed ? 0 : p.xs + up(m * up(k / 32, 16), 256);
    return p;
  }
  p.ws = p.xs + stages * ((m + 31) / 32) * 256;
  p.bytes = p.ws + stages * ((n + 31) / 32) * 256;
  // The tile by estimated time: us for k = 4096 on 256 CUs, from the rounds of tiles
  // that a CU takes (measured, with 4096 columns: 64 x 64 tiles 9 us for a round, 12 for
  // two at once, then 5 more each; 128 x 128 18, then 10 more each; 256 x 256 36 each.  700
  // rows: 19, 16 and 30 us; 4096 rows: 76, 46 and 40; 6000 rows: 113, 66 and 72).  Short
  // reductions keep the order (k = 512, 4096 rows: 31, 19 and 17 us with the quantisation).
  const int64_t cus = device_cus();
  auto rounds = [&](int64_t s) {
    return (((m + s - 1) / s) * ((n + s - 1) / s) + cus - 1) / cus;
  };
  const int64_t r64 = rounds(64), r128 = rounds(128), r256 = rounds(256);
  const double t64 = r64 <= 2 ? 6.5 + 2.6 * r64 : 3.0 + 5.0 * r64, t128 = 7.0 + 9.8 * r128, t256 = 3.0 + 36.0 * r256;
  p.tile = t256 <= t128 && t256 <= t64 ? 0 : t128 <= t64 ? 1 : 2;
  p.split = p.tile == 2 && r64 == 1 && halves(k);
  return p;
}

int check_quant(const char* who, int64_t m, int64_t k, const void* x, int64_t stride, int kind) {
  if (m < 0 || k < 1) return fail(HSMOE_ERR_ARG, "%s: bad arguments", who);
  if (k % 32 != 0 || k >= (1 << 22)) return fail(HSMOE_ERR_SHAPE, "%s: k must be a multiple of 32 below 2^22", who);
  if (m >= (1ll << 31)) return fail(HSMOE_ERR_SHAPE, "%s: m must be below 2^31", who);
  if (m == 0) return HSMOE_OK;
  if (!x) return fail(HSMOE_ERR_ARG, "%s: null pointer", who);
  const int64_t size = kind == HSMOE_OUT_BF16 ? 2 : 4;
  if (!aligned(x, 16) || stride < k || stride * size % 16 != 0)
    return fail(HSMOE_ERR_SHAPE, "%s: rows must be 16-byte aligned", who);
  return HSMOE_OK;
}

// Workgroups for rows by columns of tiles of kBR x kBC: place_tile's chunks, all eight XCDs'.
int64_t tile_groups(int64_t m, int64_t n, int64_t rows, int64_t cols) {
  const int64_t tiles = ((m + rows - 1) / rows) * ((n + cols - 1) / cols);
  const int64_t size = tiles >= 8 * kChunk ? kChunk : (tiles + 7) / 8;
  return (tiles + 8 * size - 1) / (8 * size) * 8 * size;
}
// .. and whether a launch holds those of a plan.
bool tiles_fit(const Fp4Plan& p, int64_t m, int64_t n) {
  const int64_t side = p.tile == 0 ? 256 : p.tile == 1 ? 128 : 64;
  return grid_fits(tile_groups(m, n, side, side), p.tile == 0 || p.split ? 512 : 256);
}
template <int kBR, int kBC, int kWR, int kWC, int kStages, int kSplit = 1>
void launch_tile(const Fp4Params& p, hipStream_t st) {
  const int64_t grid = tile_groups(p.m, p.n, kBR, kBC);
  hipLaunchKernelGGL((fp4_tile_kernel<kBR, kBC, kWR, kWC, kStages, kSplit>), dim3((unsigned)grid), dim3(kWR * kWC * 64 * kSplit), 0, st, p);
}

template <int kRB, int kKind>
void launch_few(const Fp4Params& p, const void* x, int64_t ldx, hipStream_t st) {
  const dim3 grid((unsigned)((p.n + 15) / 16)), block(256);
  if (p.k % 128 == 0 && aligned(p.ws, 4) && aligned(p.xs, 4))
    hipLaunchKernelGGL((fp4_few_kernel<kRB, kKind, true>), grid, block, 0, st, p, (const char*)x, ldx);
  else
    hipLaunchKernelGGL((fp4_few_kernel<kRB, kKind, false>), grid, block, 0, st, p, (const char*)x, ldx);
}

}  // namespace
}  // namespace hsmoe

using namespace hsmoe;

extern "C" int hsmoe_fp4_quant(const void* x, int64_t x_row_stride, int row_kind, int64_t m, int64_t k, void* codes,
                               void* scale, hsmoe_stream_t stream) {
  if (row_kind != HSMOE_OUT_F32 && row_kind != HSMOE_OUT_BF16)
    return fail(HSMOE_ERR_ARG, "hsmoe_fp4_quant: bad row kind %d", row_kind);
  if (int rc = check_quant("hsmoe_fp4_quant", m, k, x, x_row_stride, row_kind)) return rc;
  if (m == 0) return HSMOE_OK;
  if (!codes || !scale) return fail(HSMOE_ERR_ARG, "hsmoe_fp4_quant: null pointer");
  if (!aligned(codes, 4) || (k % 128 == 0 && !aligned(scale, 4)))
    return fail(HSMOE_ERR_SHAPE, "hsmoe_fp4_quant: codes and scales must be 4-byte aligned");
  if (!grid_fits(quant_groups(m, (k + kUnit - 1) / kUnit, false), kQuantThreads))
    return fail(HSMOE_ERR_SHAPE, "hsmoe_fp4_quant: too many rows for one launch");
  QuantParams q{};
  q.x = (const char*)x, q.codes = (char*)codes, q.scale = (uint8_t*)scale;
  q.m = m, q.k = k, q.ldx = x_row_stride * (row_kind == HSMOE_OUT_BF16 ? 2 : 4), q.ld_scale = k / 32;
  q.units = (k + kUnit - 1) / kUnit, q.across = waves_across(q.units, false);
  launch_quant(q, row_kind == HSMOE_OUT_BF16, (hipStream_t)stream);
  return check_launch("hsmoe_fp4_quant");
}

extern "C" size_t hsmoe_fp4_linear_workspace_size(int64_t m, int64_t n, int64_t k, int x_kind) {
  if (m < 1 || n < 1 || k < 1) return 0;
  return (size_t)plan_fp4(m, n, k, x_kind == HSMOE_ROWS_FP4).bytes;
}

extern "C" int hsmoe_fp4_linear(const void* x, int x_kind, int64_t x_row_stride, const void* x_scale, int64_t m,
                                int64_t k, const void* w, const void* w_scale, int64_t n, int out_kind, void* out,
                                void* workspace, size_t workspace_bytes, hsmoe_stream_t stream) {
  const char* who = "hsmoe_fp4_linear";
  const bool packed = x_kind == HSMOE_ROWS_FP4;
  if (!packed && x_kind != HSMOE_OUT_F32 && x_kind != HSMOE_OUT_BF16) return fail(HSMOE_ERR_ARG, "%s: bad kind of rows %d", who, x_kind);
  if (out_kind != HSMOE_OUT_F32 && out_kind != HSMOE_OUT_BF16) return fail(HSMOE_ERR_ARG, "%s: bad output kind %d", who, out_kind);
  if (int rc = check_quant(who, m, k, x, packed ? k : x_row_stride, packed ? HSMOE_OUT_F32 : x_kind)) return rc;
  if (n < 1) return fail(HSMOE_ERR_ARG, "%s: bad arguments", who);
  if (n % 8 != 0 || n >= (1ll << 31)) return fail(HSMOE_ERR_SHAPE, "%s: n must be a multiple of 8 below 2^31", who);
  if (m == 0) return HSMOE_OK;
  if (!w || !w_scale || !out || (packed && !x_scale)) return fail(HSMOE_ERR_ARG, "%s: null pointer", who);
  if (!aligned(w, 16) || !aligned(out, 16) || (k % 512 == 0 && (!aligned(w_scale, 16) || (packed && !aligned(x_scale, 16)))))
    return fail(HSMOE_ERR_SHAPE, "%s: operands must be 16-byte aligned", who);
  const Fp4Plan plan = plan_fp4(m, n, k, packed);
  if (plan.few && !grid_fits((n + 15) / 16, 256)) return fail(HSMOE_ERR_SHAPE, "%s: operands too large", who);
  if (!plan.few && (plan.bytes - plan.xs >= (1ll << 31) - 1024 || !tiles_fit(plan, m, n)))
    return fail(HSMOE_ERR_SHAPE, "%s: operands too large", who);
  if (plan.bytes && (!workspace || workspace_bytes < (size_t)plan.bytes))
    return fail(HSMOE_ERR_WORKSPACE, "%s: workspace of %lld bytes needed", who, (long long)plan.bytes);
  if (plan.bytes && !aligned(workspace, 16)) return fail(HSMOE_ERR_SHAPE, "%s: misaligned workspace", who);
  hipStream_t st = (hipStream_t)stream;
  char* mem = (char*)workspace;
  Fp4Params p{};
  p.x = packed ? (const char*)x : mem + plan.codes;
  p.w = (const char*)w, p.ws = (const uint8_t*)w_scale;
  p.out = (char*)out, p.m = m, p.n = n, p.k = k, p.out_f32 = out_kind == HSMOE_OUT_F32;
  const int64_t ldx = packed ? 0 : x_row_stride * (x_kind == HSMOE_OUT_BF16 ? 2 : 4);
  if (plan.fused) {
    if (x_kind == HSMOE_OUT_BF16)
      launch_few<1, kRowsBf16>(p, x, ldx, st);
    else
      launch_few<1, kRowsF32>(p, x, ldx, st);
    return check_launch(who);
  }
  QuantParams q{};
  q.x = (const char*)x, q.codes = mem + plan.codes, q.scale = (uint8_t*)mem + plan.xs;
  q.m = m, q.k = k, q.ldx = ldx, q.units = (k + kUnit - 1) / kUnit;
  q.ld_scale = up(k / 32, 16), q.row_blocks = plan.few ? 0 : (m + 31) / 32;
  q.across = waves_across(q.units, !plan.few);
  DealParams dx{}, dw{};
  dw.scale = (const uint8_t*)w_scale, dw.words = (uint32_t*)(mem + plan.ws);
  dw.rows = n, dw.blocks = k / 32, dw.row_blocks = (n + 31) / 32, dw.groups = q.units;
  dx = dw;
  dx.scale = (const uint8_t*)x_scale, dx.words = (uint32_t*)(mem + plan.xs), dx.rows = m, dx.row_blocks = (m + 31) / 32;
  auto deal_blocks = [&](const DealParams& d) { return (d.row_blocks * 32 * d.groups + kQuantThreads - 1) / kQuantThreads; };
  if (plan.few) {
    p.xs = (const uint8_t*)q.scale, p.ld_xs = q.ld_scale;
    if (packed)
      p.xs = (const uint8_t*)x_scale, p.ld_xs = k / 32;
    else
      launch_quant(q, x_kind == HSMOE_OUT_BF16, st);
    if (m <= 16)
      launch_few<1, -1>(p, nullptr, 0, st);
    else if (m <= 32)
      launch_few<2, -1>(p, nullptr, 0, st);
    else if (m <= 48)
      launch_few<3, -1>(p, nullptr, 0, st);
    else
      launch_few<4, -1>(p, nullptr, 0, st);
    return check_launch(who);
  }
  p.words = mem + plan.xs, p.x_words = 0, p.w_words = (uint32_t)(plan.ws - plan.xs);
  p.words_bytes = (uint32_t)(plan.bytes - plan.xs);
  const int64_t first = packed ? deal_blocks(dx) : quant_groups(m, q.units, true);
  const int64_t all = first + deal_blocks(dw);
  if (!grid_fits(all, kQuantThreads)) return fail(HSMOE_ERR_SHAPE, "%s: operands too large", who);
  auto ready = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)all), dim3(kQuantThreads), 0, st, q, dx, dw, (uint32_t)first); };
  const bool bf16 = x_kind == HSMOE_OUT_BF16, four = four_rows(m, q.units);
  if (packed) ready(fp4_ready_kernel<-1, 1>);
  else if (bf16) four ? ready(fp4_ready_kernel<kRowsBf16, 4>) : ready(fp4_ready_kernel<kRowsBf16, 1>);
  else four ? ready(fp4_ready_kernel<kRowsF32, 4>) : ready(fp4_ready_kernel<kRowsF32, 1>);
  if (plan.tile == 0)
    launch_tile<256, 256, 2, 4, 0>(p, st);
  else if (plan.tile == 1)
    launch_tile<128, 128, 2, 2, 2>(p, st);
  else if (plan.split)
    launch_tile<64, 64, 2, 2, 4, 2>(p, st);
  else
    launch_tile<64, 64, 2, 2, 4>(p, st);
  return check_launch(who);
}

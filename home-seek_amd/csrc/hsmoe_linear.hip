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

namespace hsmoe {
namespace {

constexpr int kBK = 64;                     // reduction steps per stage
constexpr uint32_t kFar = 0x7ffffff0u;      // an offset that no resource reaches: reads as zero
constexpr int64_t kMaxRange = 0x7fffffe0;   // bytes that one resource covers at most
constexpr int kMaxGroups = 1024;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

__device__ __forceinline__ int64_t imin64(int64_t a, int64_t b) { return a < b ? a : b; }

// kFar where step i is not below `left`, else 0.
__device__ __forceinline__ uint32_t past(int i, int left) { return (uint32_t)((left - 1 - i) >> 31) & kFar; }

// Values that are the same in every lane, in scalar registers.
__device__ __forceinline__ int64_t uniform64(int64_t v) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// ---------------------------------------------------------------- tiles
// One stage of one operand: kBK reduction steps of kRows rows, bf16.
//   contiguous  [kRows][64]: 128 bytes per row, its 16-byte chunk c at place c ^ (row & 7)
//   transposed  [64][kRows]: chunk c of step r at place c ^ 2 f(r), f = (r & 3) + 4 * (r >> 3 & 1)
// so that the lanes which read together (8 rows of a chunk, or 4 + 4 steps of a
// 32-byte piece) touch different banks.  The loads write LDS in lane order, so
// the lane that fills a place loads that place's chunk.
template <int kRows, int kWaves, bool kTrans>
struct Operand {
  static constexpr int kBytes = kRows * kBK * 2;
  static constexpr int kLoads = kBytes / 1024 / kWaves;  // 1 KiB instructions per wave and stage
  static_assert(kBytes % (1024 * kWaves) == 0, "every wave loads whole instructions");

  // Byte offset of the lane's chunk in load i (wave's), relative to the stage's
  // first row and step; beyond kFar past `left` reduction steps (an OR, since
  // the compiler makes divergent branches around the load of a select).
  static __device__ __forceinline__ uint32_t offset(int i, int wave, int lane, uint32_t ld, int left) {
    const int q = wave * kLoads + i;
    if (!kTrans) {
      const int chunk = (lane & 7) ^ (lane >> 3);
      return ((uint32_t)(8 * q + (lane >> 3)) * ld + chunk * 16) | past(chunk * 8, left);
    }
    constexpr int kPer = kRows / 8;  // chunks per step
    const int r = q * (64 / kPer) + lane / kPer;
    const int chunk = (lane % kPer) ^ (2 * ((r & 3) | ((r >> 1) & 4)));
    return ((uint32_t)r * ld + chunk * 16) | past(r, left);
  }

  // The MFMA operand of 16 rows from row0 on (a multiple of 16), reduction
  // steps 32 kk + 8 (lane / 16) ..+7.
  static __device__ __forceinline__ bf16x8 frag(const char* stage, int row0, int kk, int lane) {
    if (!kTrans) {
      const int place = (4 * kk + (lane >> 4)) ^ (lane & 7);
      return *reinterpret_cast<const bf16x8*>(stage + (row0 + (lane & 15)) * 128 + place * 16);
    }
    const int i = lane & 15, f = (i >> 2) | ((lane >> 2) & 4);
    const char* p = stage + (32 * kk + 8 * (lane >> 4) + (i >> 2)) * (kRows * 2) + (((row0 >> 4) ^ f) << 5) +
                    (i & 3) * 8;
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * kRows * 2));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, v);
  }
};

__device__ __forceinline__ void lds_load16(BufRsrc r, uint32_t off, char* dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16, (int)off, 0, 0, 0);
}

// A resource over what an operand has from `base` on, `bytes` of it.
__device__ __forceinline__ BufRsrc range(const char* base, int64_t bytes) {
  return make_buf((uint64_t)base, (uint32_t)imin64(bytes < 0 ? 0 : bytes, kMaxRange));
}

template <int kBR, int kBC, int kWR, int kWC, bool kTR, bool kTC>
struct Tile {
  static constexpr int kWaves = kWR * kWC;
  static constexpr int kThreads = kWaves * 64;
  static constexpr int kFR = kBR / kWR / 16, kFC = kBC / kWC / 16;  // 16 x 16 blocks per wave
  using R = Operand<kBR, kWaves, kTR>;
  using C = Operand<kBC, kWaves, kTC>;
  static constexpr int kStage = R::kBytes + C::kBytes;

  // One stage's products.
  static __device__ __forceinline__ void multiply(const char* stage, int wr, int wc, int lane, f32x4 (&acc)[kFR][kFC]) {
    const char* cs = stage + R::kBytes;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      bf16x8 c[kFC], r[kFR];
#pragma unroll
      for (int j = 0; j < kFC; ++j) c[j] = C::frag(cs, wc * kFC * 16 + 16 * j, kk, lane);
#pragma unroll
      for (int i = 0; i < kFR; ++i) r[i] = R::frag(stage, wr * kFR * 16 + 16 * i, kk, lane);
#pragma unroll
      for (int i = 0; i < kFR; ++i)
#pragma unroll
        for (int j = 0; j < kFC; ++j) acc[i][j] = mfma16x16x32(c[j], r[i], acc[i][j]);
    }
  }
};

// Every wave waits for its own loads (and its LDS reads, whose products may come
// later), then all meet: the stage that was loaded is whole, and nobody reads
// the other one any more.
__device__ __forceinline__ void stage_ready() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
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

// The workgroup's place among total tiles.  Workgroup b runs on XCD b % 8: each
// XCD takes a contiguous eighth, in which four row tiles go through the column
// tiles together, so that its L2 serves a row tile to several column tiles and
// a column tile to four row tiles.  False: nothing left for it.
__device__ __forceinline__ bool place_tile(int b, int row_tiles, int col_tiles, int& rt, int& ct) {
  const int total = row_tiles * col_tiles;
  const int q = total >> 3, rem = total & 7, x = b & 7, at = b >> 3;
  if (at >= q + (x < rem ? 1 : 0)) return false;
  const int t = x * q + (x < rem ? x : rem) + at;
  const int band = 4 * col_tiles, b0 = t / band, in = t % band;
  const int height = row_tiles - 4 * b0 < 4 ? row_tiles - 4 * b0 : 4;
  rt = 4 * b0 + in % height;
  ct = in / height;
  return true;
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
};

// From exp(-|z|), which does not overflow: below -88 the result is small, not 0
// (0 times an infinite up value would be NaN).
__device__ __forceinline__ float sigmoid(float z) {
  const float t = expf(-__builtin_fabsf(z));
  return (z < 0.0f ? t : 1.0f) / (1.0f + t);
}

// min / max that hand a NaN on, as torch's clamp does
__device__ __forceinline__ float clamp_top(float v, float l) { return v > l ? l : v; }
__device__ __forceinline__ float clamp_both(float v, float l) { return v > l ? l : v < -l ? -l : v; }

__device__ __forceinline__ f32x4 unpack4(uint2 u) {
  return f32x4{bf16_bits_to_f32(u.x & 0xffffu), __uint_as_float(u.x & 0xffff0000u), bf16_bits_to_f32(u.y & 0xffffu),
               __uint_as_float(u.y & 0xffff0000u)};
}
__device__ __forceinline__ uint2 pack4(f32x4 v) {
  return make_uint2(f32_to_bf16_bits(v[0]) | f32_to_bf16_bits(v[1]) << 16,
                    f32_to_bf16_bits(v[2]) | f32_to_bf16_bits(v[3]) << 16);
}

// Four outputs of row m from column n on: z (and z_up) are the sums.
__device__ __forceinline__ void finish4(const LinearParams& p, int group, int64_t m, int64_t n, f32x4 z, f32x4 zu) {
  if (p.bias[0]) z += unpack4(*reinterpret_cast<const uint2*>(p.bias[0] + (group * p.n + n) * 2));
  if (p.act == HSMOE_ACT_SWIGLU && p.bias[1])
    zu += unpack4(*reinterpret_cast<const uint2*>(p.bias[1] + (group * p.n + n) * 2));
  if (p.pre) {
    const int64_t ldp = p.act == HSMOE_ACT_SWIGLU ? 2 * p.n : p.n;
    *reinterpret_cast<uint2*>(p.pre + m * ldp + n) = pack4(z);
    if (p.act == HSMOE_ACT_SWIGLU) *reinterpret_cast<uint2*>(p.pre + m * ldp + p.n + n) = pack4(zu);
  }
  f32x4 y = z;
  if (p.act == HSMOE_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = z[i] * sigmoid(z[i]);
  } else if (p.act == HSMOE_ACT_SWIGLU) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float g = clamp_top(z[i], p.limit);
      y[i] = g * sigmoid(g) * clamp_both(zu[i], p.limit);
    }
  }
  if (p.residual) y += unpack4(*reinterpret_cast<const uint2*>(p.residual + m * p.ld_res + n * 2));
  if (p.out_f32)
    *reinterpret_cast<f32x4*>(p.out + (m * p.n + n) * 4) = y;
  else
    *reinterpret_cast<uint2*>(p.out + (m * p.n + n) * 2) = pack4(y);
}

// Rows of no group: zeros.
__device__ __forceinline__ void clear4(const LinearParams& p, int64_t m, int64_t n) {
  if (p.out_f32)
    *reinterpret_cast<f32x4*>(p.out + (m * p.n + n) * 4) = f32x4{};
  else
    *reinterpret_cast<uint2*>(p.out + (m * p.n + n) * 2) = make_uint2(0u, 0u);
  if (p.pre) {
    const int64_t ldp = p.act == HSMOE_ACT_SWIGLU ? 2 * p.n : p.n;
    *reinterpret_cast<uint2*>(p.pre + m * ldp + n) = make_uint2(0u, 0u);
    if (p.act == HSMOE_ACT_SWIGLU) *reinterpret_cast<uint2*>(p.pre + m * ldp + p.n + n) = make_uint2(0u, 0u);
  }
}

// kGated: the column tile is made of blocks of 16 gate columns and the same 16
// up columns in turn, so that a lane holds a gate sum and its up sum.
template <int kBR, int kBC, int kWR, int kWC, bool kGated>
__global__ void __launch_bounds__(kWR* kWC * 64) linear_kernel(LinearParams p) {
  using T = Tile<kBR, kBC, kWR, kWC, false, false>;
  __shared__ __align__(1024) char lds[2][T::kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int kCols = kGated ? kBC / 2 : kBC;  // output columns per tile
  const TileScan scan = scan_tiles<kBR>(p.offsets, p.n_groups, p.n_rows, lane);
  int rt, ct;
  if (!place_tile(blockIdx.x, scan.total, (int)((p.n + kCols - 1) / kCols), rt, ct)) return;
  const Span sp = find_tile<kBR>(scan, rt, p.offsets, p.n_groups, p.n_rows);
  const int64_t n0 = (int64_t)ct * kCols;
  const int rows = (int)imin64(kBR, sp.end - sp.row);
  const int cols = (int)imin64(kCols, p.n - n0);
  if (sp.group >= p.n_groups) {
    for (int i = threadIdx.x; i < rows * (cols / 4); i += T::kThreads)
      clear4(p, sp.row + i / (cols / 4), n0 + i % (cols / 4) * 4);
    return;
  }
  const char* xb = p.x + sp.row * p.ldx;
  const char* wb[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) wb[s] = p.w[kGated ? s : 0] + sp.group * p.w_group + n0 * p.ldw;
  const int64_t x_bytes = (rows - 1) * p.ldx + p.k * 2, w_bytes = (cols - 1) * p.ldw + p.k * 2;
  const int steps = (int)((p.k + kBK - 1) / kBK);

  auto load = [&](int s) {
    char* stage = lds[s & 1];
    const int64_t at = (int64_t)s * kBK * 2;
    const int left = (int)imin64(kBK, p.k - (int64_t)s * kBK);
    const BufRsrc xr = range(xb + at, x_bytes - at);
#pragma unroll
    for (int i = 0; i < T::R::kLoads; ++i)
      lds_load16(xr, T::R::offset(i, wave, lane, (uint32_t)p.ldx, left), stage + (wave * T::R::kLoads + i) * 1024);
    if (!kGated) {
      const BufRsrc wr = range(wb[0] + at, w_bytes - at);
#pragma unroll
      for (int i = 0; i < T::C::kLoads; ++i)
        lds_load16(wr, T::C::offset(i, wave, lane, (uint32_t)p.ldw, left),
                   stage + T::R::kBytes + (wave * T::C::kLoads + i) * 1024);
    } else {
      // load q fills LDS rows 8 q ..+7: rows 16 (q / 4) + 8 (q & 1) ..+7 of matrix (q >> 1) & 1
      const BufRsrc wr[2] = {range(wb[0] + at, w_bytes - at), range(wb[1] + at, w_bytes - at)};
      const int chunk = (lane & 7) ^ (lane >> 3);
#pragma unroll
      for (int i = 0; i < T::C::kLoads; ++i) {
        const int q = wave * T::C::kLoads + i;
        const uint32_t row = 16 * (q >> 2) + 8 * (q & 1) + (lane >> 3);
        const uint32_t off = (row * (uint32_t)p.ldw + chunk * 16) | past(chunk * 8, left);
        char* dst = stage + T::R::kBytes + q * 1024;
        if ((q >> 1) & 1) lds_load16(wr[1], off, dst);
        else lds_load16(wr[0], off, dst);
      }
    }
  };

  const int wr = wave / kWC, wc = wave % kWC;
  f32x4 acc[T::kFR][T::kFC] = {};
  load(0);
  for (int s = 0; s < steps; ++s) {
    stage_ready();
    if (s + 1 < steps) load(s + 1);
    T::multiply(lds[s & 1], wr, wc, lane, acc);
  }
#pragma unroll
  for (int i = 0; i < T::kFR; ++i) {
    const int r = (wr * T::kFR + i) * 16 + (lane & 15);
    if (r >= rows) continue;
    const int64_t m = sp.row + r;
    if (kGated) {
#pragma unroll
      for (int j = 0; j < T::kFC; j += 2) {
        const int c = (wc * T::kFC + j) * 8 + 4 * (lane >> 4);
        if (c < cols) finish4(p, sp.group, m, n0 + c, acc[i][j], acc[i][j + 1]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < T::kFC; ++j) {
        const int c = (wc * T::kFC + j) * 16 + 4 * (lane >> 4);
        if (c < cols) finish4(p, sp.group, m, n0 + c, acc[i][j], f32x4{});
      }
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
};

// dx = dz w (+ dz_up w_up): the reduction runs over the n columns of dz and the
// rows of w, then over those of up.
template <int kBR, int kBC, int kWR, int kWC>
__global__ void __launch_bounds__(kWR* kWC * 64) linear_grad_input_kernel(LinearGradParams p) {
  using T = Tile<kBR, kBC, kWR, kWC, false, true>;
  __shared__ __align__(1024) char lds[2][T::kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TileScan scan = scan_tiles<kBR>(p.offsets, p.n_groups, p.n_rows, lane);
  int rt, ct;
  if (!place_tile(blockIdx.x, scan.total, (int)((p.k + kBC - 1) / kBC), rt, ct)) return;
  const Span sp = find_tile<kBR>(scan, rt, p.offsets, p.n_groups, p.n_rows);
  const int64_t c0 = (int64_t)ct * kBC;
  const int rows = (int)imin64(kBR, sp.end - sp.row), cols = (int)imin64(kBC, p.k - c0);
  if (sp.group >= p.n_groups) {
    for (int i = threadIdx.x; i < rows * (cols / 4); i += T::kThreads)
      *reinterpret_cast<uint2*>(p.dx + ((sp.row + i / (cols / 4)) * p.k + c0 + i % (cols / 4) * 4) * 2) =
          make_uint2(0u, 0u);
    return;
  }
  const int per = (int)((p.n + kBK - 1) / kBK), steps = per * p.mats;
  auto load = [&](int s) {
    char* stage = lds[s & 1];
    const int mat = s >= per ? 1 : 0;
    const int64_t r0 = (int64_t)(s - mat * per) * kBK;
    const int left = (int)imin64(kBK, p.n - r0);
    const int64_t at = (mat * p.n + r0) * 2;
    const BufRsrc zr = range(p.dz + sp.row * p.ldz + at, (rows - 1) * p.ldz + left * 2);
#pragma unroll
    for (int i = 0; i < T::R::kLoads; ++i)
      lds_load16(zr, T::R::offset(i, wave, lane, (uint32_t)p.ldz, left), stage + (wave * T::R::kLoads + i) * 1024);
    const BufRsrc wr = range(p.w[mat] + sp.group * p.w_group + r0 * p.ldw + c0 * 2, (left - 1) * p.ldw + cols * 2);
#pragma unroll
    for (int i = 0; i < T::C::kLoads; ++i)
      lds_load16(wr, T::C::offset(i, wave, lane, (uint32_t)p.ldw, left),
                 stage + T::R::kBytes + (wave * T::C::kLoads + i) * 1024);
  };
  const int wr = wave / kWC, wc = wave % kWC;
  f32x4 acc[T::kFR][T::kFC] = {};
  load(0);
  for (int s = 0; s < steps; ++s) {
    stage_ready();
    if (s + 1 < steps) load(s + 1);
    T::multiply(lds[s & 1], wr, wc, lane, acc);
  }
#pragma unroll
  for (int i = 0; i < T::kFR; ++i) {
    const int r = (wr * T::kFR + i) * 16 + (lane & 15);
    if (r >= rows) continue;
#pragma unroll
    for (int j = 0; j < T::kFC; ++j) {
      const int c = (wc * T::kFC + j) * 16 + 4 * (lane >> 4);
      if (c < cols) *reinterpret_cast<uint2*>(p.dx + ((sp.row + r) * p.k + c0 + c) * 2) = pack4(acc[i][j]);
    }
  }
}

// dw[g] = dz^T x over the rows of group g: a tile of n x k per workgroup, all
// groups and both matrices in one launch; a group without rows gets zeros.
template <int kBR, int kBC, int kWR, int kWC>
__global__ void __launch_bounds__(kWR* kWC * 64) linear_grad_weight_kernel(LinearGradParams p) {
  using T = Tile<kBR, kBC, kWR, kWC, true, true>;
  __shared__ __align__(1024) char lds[2][T::kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row_tiles = (int)((p.n + kBR - 1) / kBR), col_tiles = (int)((p.k + kBC - 1) / kBC);
  int rt, ct;
  if (!place_tile(blockIdx.x, p.n_groups * p.mats * row_tiles, col_tiles, rt, ct)) return;
  const int gm = rt / row_tiles, group = gm / p.mats, mat = gm % p.mats;
  const int64_t n0 = (int64_t)(rt % row_tiles) * kBR, c0 = (int64_t)ct * kBC;
  const int64_t first = p.offsets ? cut(p.offsets[group], p.n_rows) : 0;
  const int64_t end = p.offsets ? cut(p.offsets[group + 1], p.n_rows) : p.n_rows;
  const int64_t count = end > first ? end - first : 0;
  const int nrow = (int)imin64(kBR, p.n - n0), ncol = (int)imin64(kBC, p.k - c0);
  const char* zb = p.dz + first * p.ldz + (mat * p.n + n0) * 2;
  const char* xb = p.x + first * p.ldx + c0 * 2;
  const int steps = (int)((count + kBK - 1) / kBK);
  auto load = [&](int s) {
    char* stage = lds[s & 1];
    const int64_t r0 = (int64_t)s * kBK;
    const int left = (int)imin64(kBK, count - r0);
    const BufRsrc zr = range(zb + r0 * p.ldz, (left - 1) * p.ldz + nrow * 2);
#pragma unroll
    for (int i = 0; i < T::R::kLoads; ++i)
      lds_load16(zr, T::R::offset(i, wave, lane, (uint32_t)p.ldz, left), stage + (wave * T::R::kLoads + i) * 1024);
    const BufRsrc xr = range(xb + r0 * p.ldx, (left - 1) * p.ldx + ncol * 2);
#pragma unroll
    for (int i = 0; i < T::C::kLoads; ++i)
      lds_load16(xr, T::C::offset(i, wave, lane, (uint32_t)p.ldx, left),
                 stage + T::R::kBytes + (wave * T::C::kLoads + i) * 1024);
  };
  const int wr = wave / kWC, wc = wave % kWC;
  f32x4 acc[T::kFR][T::kFC] = {};
  if (steps > 0) load(0);
  for (int s = 0; s < steps; ++s) {
    stage_ready();
    if (s + 1 < steps) load(s + 1);
    T::multiply(lds[s & 1], wr, wc, lane, acc);
  }
  const int es = p.dw_f32 ? 4 : 2;
  char* ob = p.dw[mat] + (int64_t)group * p.n * p.k * es;
#pragma unroll
  for (int i = 0; i < T::kFR; ++i) {
    const int r = (wr * T::kFR + i) * 16 + (lane & 15);
    if (r >= nrow) continue;
#pragma unroll
    for (int j = 0; j < T::kFC; ++j) {
      const int c = (wc * T::kFC + j) * 16 + 4 * (lane >> 4);
      if (c >= ncol) continue;
      char* o = ob + ((n0 + r) * p.k + c0 + c) * es;
      if (p.dw_f32)
        *reinterpret_cast<f32x4*>(o) = acc[i][j];
      else
        *reinterpret_cast<uint2*>(o) = pack4(acc[i][j]);
    }
  }
}

// dz = d_out act'(pre) and the column sums of dz over the rows of a group (the
// bias's gradient), from the unrounded values.  A workgroup has 256 columns and
// a share of a group's rows: 32 threads of 8 columns, 8 rows at a time; the
// shares' sums go to `part` [shares][n_groups][n * mats] and are added in order
// by a second launch (one share: straight to the result).
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

template <int kMats>
__global__ void __launch_bounds__(kActThreads) act_grad_kernel(ActGradParams p) {
  __shared__ float s_sum[kMats][8][256];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, group = blockIdx.y, share = blockIdx.z;
  const int64_t col = (int64_t)blockIdx.x * 256 + tx * 8;
  const int64_t first = p.offsets ? cut(p.offsets[group], p.n_rows) : 0;
  const int64_t end = p.offsets ? cut(p.offsets[group + 1], p.n_rows) : p.n_rows;
  const int64_t count = end > first ? end - first : 0;
  const int64_t a = first + count * share / p.shares, b = first + count * (share + 1) / p.shares;
  float sum[kMats][8] = {};
  if (col < p.n) {
    for (int64_t r = a + ty; r < b; r += 8) {
      const uint4 du = *reinterpret_cast<const uint4*>(p.d_out + r * p.ld_out + col);
      const uint32_t dw[4] = {du.x, du.y, du.z, du.w};
      uint32_t pw[kMats][4], ow[kMats][4];
      if (p.pre) {
#pragma unroll
        for (int t = 0; t < kMats; ++t) {
          const uint4 u = *reinterpret_cast<const uint4*>(p.pre + r * p.n * kMats + t * p.n + col);
          pw[t][0] = u.x, pw[t][1] = u.y, pw[t][2] = u.z, pw[t][3] = u.w;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        auto half = [&](uint32_t w) { return i & 1 ? __uint_as_float(w & 0xffff0000u) : bf16_bits_to_f32(w & 0xffffu); };
        const float d = half(dw[i >> 1]);
        float o[kMats];
        o[0] = d;
        if (kMats == 2) {
          const float z = half(pw[0][i >> 1]), zu = half(pw[kMats - 1][i >> 1]);
          const float g = clamp_top(z, p.limit), s = sigmoid(g);
          o[0] = z > p.limit ? 0.0f : d * clamp_both(zu, p.limit) * (s + g * s * (1.0f - s));
          o[kMats - 1] = zu > p.limit || zu < -p.limit ? 0.0f : d * (g * s);
        } else if (p.act == HSMOE_ACT_SILU) {
          const float z = half(pw[0][i >> 1]), s = sigmoid(z);
          o[0] = d * (s + z * s * (1.0f - s));
        }
#pragma unroll
        for (int t = 0; t < kMats; ++t) {
          sum[t][i] += o[t];
          const uint32_t h = f32_to_bf16_bits(o[t]);
          ow[t][i >> 1] = i & 1 ? ow[t][i >> 1] | h << 16 : h;
        }
      }
      if (p.dz) {
#pragma unroll
        for (int t = 0; t < kMats; ++t)
          *reinterpret_cast<uint4*>(p.dz + r * p.n * kMats + t * p.n + col) =
              make_uint4(ow[t][0], ow[t][1], ow[t][2], ow[t][3]);
      }
    }
  }
  if (!p.part && !p.d_bias[0] && !p.d_bias[1]) return;
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
  if (m > INT32_MAX) return fail(HSMOE_ERR_SHAPE, "%s: m must be below 2^31", what);
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

// Workgroups for tiles of bc columns, in whole rounds over the eight XCDs; 0 if
// that is more than a launch can hold.
unsigned tile_grid(int64_t row_tiles, int64_t cols, int bc) {
  const int64_t total = row_tiles * ((cols + bc - 1) / bc);
  return total > (1 << 22) - 8 ? 0 : (unsigned)((total + 7) / 8 * 8);
}

// Whether tiles of 256 x 256 still give every CU one (rows and cols of the
// output, in `groups` of equal size).
bool big_tiles(int64_t rows, int64_t cols, int64_t groups) {
  const int64_t per = (rows + groups - 1) / groups;
  return per > 128 && groups * ((per + 255) / 256) * ((cols + 255) / 256) >= device_cus();
}

template <int kBR, int kBC, int kWR, int kWC>
int launch_linear(const LinearParams& p, hipStream_t st) {
  const bool gated = p.act == HSMOE_ACT_SWIGLU;
  const unsigned grid = tile_grid(max_row_tiles(p.n_rows, kBR, p.offsets, p.n_groups), p.n, gated ? kBC / 2 : kBC);
  if (!grid) return fail(HSMOE_ERR_SHAPE, "hsmoe_linear: too many tiles");
  const dim3 block(kWR * kWC * 64);
  if (gated)
    hipLaunchKernelGGL((linear_kernel<kBR, kBC, kWR, kWC, true>), dim3(grid), block, 0, st, p);
  else
    hipLaunchKernelGGL((linear_kernel<kBR, kBC, kWR, kWC, false>), dim3(grid), block, 0, st, p);
  return check_launch("hsmoe_linear");
}

template <int kBR, int kBC, int kWR, int kWC>
int launch_grad_input(const LinearGradParams& p, hipStream_t st) {
  const unsigned grid = tile_grid(max_row_tiles(p.n_rows, kBR, p.offsets, p.n_groups), p.k, kBC);
  if (!grid) return fail(HSMOE_ERR_SHAPE, "hsmoe_linear_grad_input: too many tiles");
  hipLaunchKernelGGL((linear_grad_input_kernel<kBR, kBC, kWR, kWC>), dim3(grid), dim3(kWR * kWC * 64), 0, st, p);
  return check_launch("hsmoe_linear_grad_input");
}

template <int kBR, int kBC, int kWR, int kWC>
int launch_grad_weight(const LinearGradParams& p, hipStream_t st) {
  const unsigned grid = tile_grid((p.n + kBR - 1) / kBR * p.n_groups * p.mats, p.k, kBC);
  if (!grid) return fail(HSMOE_ERR_SHAPE, "hsmoe_linear_grad_weight: too many tiles");
  hipLaunchKernelGGL((linear_grad_weight_kernel<kBR, kBC, kWR, kWC>), dim3(grid), dim3(kWR * kWC * 64), 0, st, p);
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

extern "C" int hsmoe_linear(const void* x, int64_t x_row_stride, int64_t m, int64_t k, const void* w, const void* w_up,
                            int64_t w_row_stride, int64_t w_group_stride, int64_t n, const int32_t* offsets,
                            int64_t n_groups, const void* bias, const void* bias_up, const void* residual,
                            int64_t res_row_stride, int act, float limit, int out_kind, void* out, void* pre,
                            hsmoe_stream_t stream) {
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
  if (big_tiles(m, gated ? 2 * n : n, n_groups)) return launch_linear<256, 256, 2, 4>(p, (hipStream_t)stream);
  return launch_linear<128, 128, 2, 2>(p, (hipStream_t)stream);
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
  if (gated)
    hipLaunchKernelGGL(act_grad_kernel<2>, grid, dim3(kActThreads), 0, st, p);
  else
    hipLaunchKernelGGL(act_grad_kernel<1>, grid, dim3(kActThreads), 0, st, p);
  if (need)
    hipLaunchKernelGGL(bias_sum_kernel, dim3((unsigned)((n * p.mats * n_groups + 255) / 256)), dim3(256), 0, st, p);
  return check_launch("hsmoe_linear_act_grad");
}

extern "C" int hsmoe_linear_grad_input(const void* dz, int64_t dz_row_stride, int64_t m, int64_t n, const void* w,
                                       const void* w_up, int64_t w_row_stride, int64_t w_group_stride, int64_t k,
                                       const int32_t* offsets, int64_t n_groups, void* dx, hsmoe_stream_t stream) {
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
  if (big_tiles(m, k, n_groups)) return launch_grad_input<256, 256, 2, 4>(p, (hipStream_t)stream);
  return launch_grad_input<128, 128, 2, 2>(p, (hipStream_t)stream);
}

extern "C" int hsmoe_linear_grad_weight(const void* dz, int64_t dz_row_stride, const void* x, int64_t x_row_stride,
                                        int64_t m, int64_t n, int64_t k, const int32_t* offsets, int64_t n_groups,
                                        int out_kind, void* dw, void* dw_up, hsmoe_stream_t stream) {
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
  if (big_tiles(n * n_groups * mats, k, n_groups * mats)) return launch_grad_weight<256, 256, 2, 4>(p, (hipStream_t)stream);
  return launch_grad_weight<128, 128, 2, 2>(p, (hipStream_t)stream);
}

// What stands between two blocks of a residual network: the norm after the block,
// its gate and residual scale, the add to the stream, and the norm before the next
// block, in one pass, and the gradient of it all.
//   u  = post_w * f r1,  r1 = 1 / sqrt(mean(f^2) + eps)     (without post_w: u = f)
//   h' = h + scale * gate * u                                rounded to the stream's type
//   n  = pre_w * h' r2,  r2 = 1 / sqrt(mean(h'^2) + eps)    (without pre_w: none)
// The norm before the next block is that of the stream as it is held (rounded), so
// that the gradient, which has h' only, is that of the same function.  Gradient:
//   g   = pre_w dn;  dH = dh' + r2 (g - h' r2^2 mean(g h'));  d_pre = sum_rows dn h' r2
//   dt  = scale dH;  d_gate = dt u (summed over what the gate is broadcast to)
//   du  = dt gate;   d_post = sum_rows du f r1
//   df  = r1 (post_w du - f r1^2 mean(post_w du f))         (without post_w: du)
// Sums in fp32.  All of it is bound by HBM; few rows by the latency of two sums
// over a row, one after the other.  Measured: 8191 x 4096, rows and stream bf16, a gate
// per channel 47 us (5.7 TB/s), fp32 stream and a full gate 90 us (5.2 TB/s; a copy by
// workgroups of 4 KB runs at 6.2, torch's at 5.1); the gradient 84 us and 5 for the join
// (4.5 TB/s), with an fp32 stream 4.8 TB/s; three rows 3.2 us.
#include <algorithm>

#include "hsmoe_common.h"
#include "hsmoe_internal.h"

namespace hsmoe {
namespace {

constexpr int kMaxD = 16384;
enum { kGateNone = 0, kGateChannel = 1, kGateToken = 2, kGateFull = 3 };

struct BlockNormParams {
  const void *f, *h;             // [m][d]; h: the stream before (forward), after the block (gradient)
  const void *post_w, *pre_w;    // [d] or NULL
  const void* gate;              // [d], [m], [m][d] or NULL
  void *h_out, *n_out;           // forward
  const void *d_h, *d_n;         // gradient: [m][d] each, NULL for zeros
  void *d_f, *d_x;               // [m][d] of f and of the stream; NULL where not wanted
  void* d_gate;                  // kGateFull: [m][d]; kGateToken: fp32 [m]
  float* part;                   // fp32 [workgroups][3][d]: sums of d_pre, d_post, d_gate (kGateChannel)
  int64_t m;
  int d, gate_kind;
  bool w_f32, gate_f32;          // weights and gate of fp32 (else bf16)
  bool sum_pre, sum_post, sum_gate;
  float scale, eps, per;         // per: 1 / d
};

// Eight values of a row at a time.
struct V8 {
  float v[8];
};
// Eight values as they lie in memory.
template <bool kF32>
struct Raw8 {
  uint32_t w[kF32 ? 8 : 4];
  __device__ __forceinline__ float at(int i) const {
    if (kF32) return __uint_as_float(w[i]);
    return i & 1 ? __uint_as_float(w[i >> 1] & 0xffff0000u) : __uint_as_float(w[i >> 1] << 16);
  }
};

// Rows through a buffer resource over those that a workgroup takes at a time, a
// thread's place in them a 32-bit offset in values: one register instead of an
// address per tensor, and beyond the rows and columns reads give zeros and writes
// go nowhere.
constexpr uint32_t kNowhere = 0x0ffffff0u;
template <bool kF32>
__device__ __forceinline__ BufRsrc rows_buf(const void* base, int64_t first, int64_t left, int64_t d) {
  constexpr int64_t kSize = kF32 ? 4 : 2;
  return make_buf((uint64_t)base + (uint64_t)(first * d * kSize), left > 0 && base ? (uint32_t)(left * d * kSize) : 0u);
}
template <bool kF32>
__device__ __forceinline__ Raw8<kF32> raw8(BufRsrc buf, uint32_t at) {
  Raw8<kF32> r;
#pragma unroll
  for (int i = 0; i < (kF32 ? 2 : 1); ++i) {
    const uint4 a = bload128(buf, at * (kF32 ? 4 : 2) + 16 * i);
    r.w[4 * i] = a.x, r.w[4 * i + 1] = a.y, r.w[4 * i + 2] = a.z, r.w[4 * i + 3] = a.w;
  }
  return r;
}
template <bool kF32>
__device__ __forceinline__ V8 read8(BufRsrc buf, uint32_t at) {
  const Raw8<kF32> r = raw8<kF32>(buf, at);
  V8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v.v[i] = r.at(i);
  return v;
}
// Rows of either kind, decided at run time.
__device__ __forceinline__ V8 read8(const void* base, int64_t first, int64_t left, int64_t d, uint32_t at, bool f32) {
  return f32 ? read8<true>(rows_buf<true>(base, first, left, d), at) : read8<false>(rows_buf<false>(base, first, left, d), at);
}
__device__ __forceinline__ void store16(BufRsrc buf, uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
  __builtin_amdgcn_raw_buffer_store_b128(u32x4{a, b, c, d}, buf, (int)at, 0, 0);
}
template <bool kF32>
__device__ __forceinline__ void write8(BufRsrc buf, uint32_t at, const V8& r) {
  if (kF32) {
#pragma unroll
    for (int i = 0; i < 8; i += 4)
      store16(buf, at * 4 + i * 4, __float_as_uint(r.v[i]), __float_as_uint(r.v[i + 1]), __float_as_uint(r.v[i + 2]), __float_as_uint(r.v[i + 3]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = f32_to_bf16_bits(r.v[2 * i]) | f32_to_bf16_bits(r.v[2 * i + 1]) << 16;
    store16(buf, at * 2, w[0], w[1], w[2], w[3]);
  }
}
template <bool kF32>
__device__ __forceinline__ V8 rounded8(const V8& r) {
  if (kF32) return r;
  V8 o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o.v[i] = bf16_bits_to_f32(f32_to_bf16_bits(r.v[i]));
  return o;
}
__device__ __forceinline__ V8 ones8() { return V8{{1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f}}; }

__device__ __forceinline__ float inv_rms(float sum, float per, float eps) {
  return __fdiv_rn(1.0f, __fsqrt_rn(__fmaf_rn(sum, per, eps)));
}

// Sums over 8, 16, 32 or 64 lanes, in every one of them, in a fixed order: within
// sixteen by DPP, beyond by reading a lane of each.
template <int kCtrl>
__device__ __forceinline__ float moved(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), kCtrl, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_of(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }
template <int kLanes>
__device__ __forceinline__ float lanes_sum(float v) {
  v += moved<0xB1>(v);                       // lane ^ 1
  v += moved<0x4E>(v);                       // lane ^ 2
  v += moved<0x141>(v);                      // the other four of eight
  if (kLanes >= 16) v += moved<0x140>(v);    // the other eight of sixteen
  if (kLanes == 32) v += __shfl_xor(v, 16, 64);
  if (kLanes == 64) v = (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
  return v;
}

// kLanes threads share a row: 8 .. 64 of a wave (a workgroup of 256 then takes
// several rows at a time), or all of a workgroup (0), up to 1024 threads.  kC: a
// thread's chunks of eight columns, kLanes (the workgroup) apart.
// Sums over the row's threads; every thread gets them.
template <int kLanes, int kN>
__device__ __forceinline__ void row_sum(float (&s)[kN], float (*mem)[16], int threads) {
#pragma unroll
  for (int i = 0; i < kN; ++i) s[i] = lanes_sum<kLanes ? kLanes : 64>(s[i]);
  if (kLanes == 0) {
    const int waves = threads >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < kN; ++i) mem[i][wave] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kN; ++i) s[i] = lanes_sum<16>(lane % 16 < waves ? mem[i][lane % 16] : 0.0f);
  }
}

template <int kLanes, int kC, bool kF32, bool kS32>
__global__ void __launch_bounds__(kLanes ? 256 : 1024) block_norm_kernel(BlockNormParams p) {
  __shared__ float mem[2][1][16];
  constexpr int kRows = kLanes ? 256 / (kLanes ? kLanes : 1) : 1;
  const int threads = kLanes ? kLanes : (int)blockDim.x;
  const int t = kLanes ? threadIdx.x % kLanes : threadIdx.x;
  const int mine = kLanes ? threadIdx.x / (kLanes ? kLanes : 1) : 0;
  const int64_t first = (int64_t)blockIdx.x * kRows, left = p.m - first < kRows ? p.m - first : kRows;
  const bool live = mine < left;
  V8 f[kC], h[kC], gate[kC], wa[kC], wb[kC];
  uint32_t at[kC];
  float token = 1.0f;
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    const uint32_t col = (uint32_t)(t + c * threads) * 8;
    const bool in = col < (uint32_t)p.d;
    at[c] = live && in ? (uint32_t)(mine * p.d) + col : kNowhere;
    gate[c] = wa[c] = wb[c] = ones8();
    f[c] = read8<kF32>(rows_buf<kF32>(p.f, first, left, p.d), at[c]);
    h[c] = read8<kS32>(rows_buf<kS32>(p.h, first, left, p.d), at[c]);
    const uint32_t wcol = in ? col : kNowhere;
    if (p.gate_kind == kGateFull) gate[c] = read8(p.gate, first, left, p.d, at[c], p.gate_f32);
    if (p.gate_kind == kGateChannel) gate[c] = read8(p.gate, 0, 1, p.d, wcol, p.gate_f32);
    if (p.post_w) wa[c] = read8(p.post_w, 0, 1, p.d, wcol, p.w_f32);
    if (p.pre_w) wb[c] = read8(p.pre_w, 0, 1, p.d, wcol, p.w_f32);
  }
  if (p.gate_kind == kGateToken && live)
    token = p.gate_f32 ? ((const float*)p.gate)[first + mine] : bf16_bits_to_f32(((const uint16_t*)p.gate)[first + mine]);
  float r1 = 1.0f;
  if (p.post_w) {
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < kC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[0] = __fmaf_rn(f[c].v[i], f[c].v[i], s[0]);
    row_sum<kLanes, 1>(s, mem[0], threads);
    r1 = inv_rms(s[0], p.per, p.eps);
  }
  float s[1] = {0.0f};
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    const bool in = at[c] != kNowhere;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = f[c].v[i] * r1 * wa[c].v[i];
      h[c].v[i] = __fmaf_rn(p.scale, token * gate[c].v[i] * u, h[c].v[i]);
    }
    h[c] = rounded8<kS32>(h[c]);
    write8<kS32>(rows_buf<kS32>(p.h_out, first, left, p.d), at[c], h[c]);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[0] = __fmaf_rn(in ? h[c].v[i] : 0.0f, h[c].v[i], s[0]);
  }
  if (!p.pre_w) return;
  row_sum<kLanes, 1>(s, mem[1], threads);
  const float r2 = inv_rms(s[0], p.per, p.eps);
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    V8 n;
#pragma unroll
    for (int i = 0; i < 8; ++i) n.v[i] = h[c].v[i] * r2 * wb[c].v[i];
    write8<kF32>(rows_buf<kF32>(p.n_out, first, left, p.d), at[c], n);
  }
}

// Ones, and weights of either kind (bf16 ones as fp32 where kW32).
template <bool kW32>
__device__ __forceinline__ Raw8<kW32> ones() {
  Raw8<kW32> r;
#pragma unroll
  for (int i = 0; i < (kW32 ? 8 : 4); ++i) r.w[i] = kW32 ? 0x3f800000u : 0x3f803f80u;
  return r;
}
template <bool kW32>
__device__ __forceinline__ Raw8<kW32> weights8(const void* base, int64_t first, int64_t left, int64_t d, uint32_t at, bool f32) {
  if constexpr (kW32) {
    if (f32) return raw8<true>(rows_buf<true>(base, first, left, d), at);
    const Raw8<false> b = raw8<false>(rows_buf<false>(base, first, left, d), at);
    Raw8<true> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = __float_as_uint(b.at(i));
    return r;
  } else {
    return raw8<false>(rows_buf<false>(base, first, left, d), at);
  }
}

// The compiler unpacks it again behind this, instead of keeping eight floats over a sum.
template <bool kF32>
__device__ __forceinline__ void unpack_later(Raw8<kF32>& r) {
#pragma unroll
  for (int i = 0; i < (kF32 ? 8 : 4); ++i) asm volatile("" : "+v"(r.w[i]));
}

// No load moves over this.
__device__ __forceinline__ void apart() { asm volatile("" ::: "memory"); }

// The gradient.  A workgroup goes through every gridDim-th row (group of rows) and
// keeps its columns' part of the weights' gradients in registers; they leave once at
// its end, as one row of `part`, and a second kernel adds the workgroups' rows in
// their order.
template <int kLanes, int kC, int kMax, bool kF32, bool kS32, bool kW32>
__global__ void __launch_bounds__(kMax, kMax >= 512 ? 4 : 2) block_norm_grad_kernel(BlockNormParams p) {
  __shared__ float mem[2][3][16];
  __shared__ float sums[kLanes ? 256 * 8 * kC : 1];
  constexpr int kRows = kLanes ? 256 / (kLanes ? kLanes : 1) : 1;  // at a time
  const int threads = kLanes ? kLanes : (int)blockDim.x;
  const int t = kLanes ? threadIdx.x % kLanes : threadIdx.x;
  const int mine = kLanes ? threadIdx.x / (kLanes ? kLanes : 1) : 0;
  uint32_t at[kC], wcol[kC];  // the thread's places in the rows, and in the weights
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    const uint32_t col = (uint32_t)(t + c * threads) * 8;
    wcol[c] = col < (uint32_t)p.d ? col : kNowhere;
    at[c] = col < (uint32_t)p.d ? (uint32_t)(mine * p.d) + col : kNowhere;
  }
  auto left_at = [&](int64_t first) { return p.m - first < kRows ? p.m - first : (int64_t)kRows; };
  struct Row {
    Raw8<kF32> f[kC], dn[kC];
    Raw8<kS32> h[kC], dh[kC];
  };
  auto load_at = [&](Row& r, int c, int64_t first) {  // (zeros of what is not there)
    const int64_t left = left_at(first);
    r.f[c] = raw8<kF32>(rows_buf<kF32>(p.f, first, left, p.d), at[c]);
    r.dh[c] = raw8<kS32>(rows_buf<kS32>(p.d_h, first, left, p.d), at[c]);
    r.h[c] = raw8<kS32>(rows_buf<kS32>(p.d_n ? p.h : nullptr, first, left, p.d), at[c]);
    r.dn[c] = raw8<kF32>(rows_buf<kF32>(p.d_n, first, left, p.d), at[c]);
  };
  auto load = [&](int64_t first) {
    Row r;
#pragma unroll
    for (int c = 0; c < kC; ++c) load_at(r, c, first);
    return r;
  };
  const int64_t stride = (int64_t)gridDim.x * kRows;
  int64_t first = (int64_t)blockIdx.x * kRows;
  // Rows of more than 8192 (kLean): what is not summed is read again where it is needed,
  // the row a second and third time, from the caches: kept, it spills (2048 x 16384 bf16
  // 125 us, 3.2 TB/s, 283 with all of it kept; fp32 with a full gate 267, 4.0 TB/s, and
  // 441).  The next row is loaded ahead where several share a workgroup only: otherwise
  // it costs the registers with which two workgroups share a CU, which hides more (fp32
  // rows of 4096: 129 us with, 85 without).
  constexpr bool kLean = kC > 1 && kLanes == 0, kAhead = kLanes != 0 && kC == 1;
  Row next;
  if (kAhead) next = load(first);
  // (a_y: the rows' sums of dt y times what of the gate is a row's own; the norm's weight
  // and a channel's gate are factors of the whole sum)
  V8 a_pre[kC] = {}, a_y[kC] = {};
  Raw8<kW32> gate[kC], wa[kC], wb[kC];
  auto read_post = [&](int c) {
    gate[c] = p.gate_kind == kGateChannel ? weights8<kW32>(p.gate, 0, 1, p.d, wcol[c], p.gate_f32) : ones<kW32>();
    wa[c] = p.post_w ? weights8<kW32>(p.post_w, 0, 1, p.d, wcol[c], p.w_f32) : ones<kW32>();
  };
  auto read_pre = [&](int c) { wb[c] = p.d_n ? weights8<kW32>(p.pre_w, 0, 1, p.d, wcol[c], p.w_f32) : ones<kW32>(); };
  if (!kLean)
#pragma unroll
    for (int c = 0; c < kC; ++c) read_post(c), read_pre(c);
  for (; first < p.m; first += stride) {
    const int64_t left = left_at(first);
    const bool live = mine < left;
    Row r;
    if (kAhead) r = next, next = load(first + stride);
    else if (!kLean) r = load(first);
    float token = 1.0f;
    if (p.gate_kind == kGateToken && live)
      token = p.gate_f32 ? ((const float*)p.gate)[first + mine] : bf16_bits_to_f32(((const uint16_t*)p.gate)[first + mine]);
    if (!kLean && p.gate_kind == kGateFull)
#pragma unroll
      for (int c = 0; c < kC; ++c) gate[c] = weights8<kW32>(p.gate, first, left, p.d, at[c], p.gate_f32);
    if (!kLean)
#pragma unroll
      for (int c = 0; c < kC; ++c) unpack_later(wa[c]), unpack_later(wb[c]), unpack_later(gate[c]);
    float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      if (kLean) apart(), load_at(r, c, first), read_pre(c);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = r.f[c].at(i), h = r.h[c].at(i);
        s[0] = __fmaf_rn(f, f, s[0]);
        s[1] = __fmaf_rn(h, h, s[1]);
        s[2] = __fmaf_rn(r.dn[c].at(i) * wb[c].at(i), h, s[2]);
      }
    }
    row_sum<kLanes, 3>(s, mem[0], threads);
#pragma unroll
    for (int c = 0; c < kC; ++c)
      if (!kLean) unpack_later(r.f[c]), unpack_later(r.h[c]), unpack_later(r.dn[c]), unpack_later(wb[c]);
    // (a row that is not there adds nothing to the sums, without eps either)
    const float r1 = !live ? 0.0f : p.post_w ? inv_rms(s[0], p.per, p.eps) : 1.0f;
    const float r2 = live && p.d_n ? inv_rms(s[1], p.per, p.eps) : 0.0f;
    const float m2 = s[2] * p.per * r2 * r2;  // r2^2 mean(g h')
    float q[2] = {0.0f, 0.0f};                // sum of post_w du f, and of dt u
    V8 df[kC];
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      V8 dx, dg;
      if (kLean) {
        apart(), load_at(r, c, first), read_pre(c), read_post(c);
        if (p.gate_kind == kGateFull) gate[c] = weights8<kW32>(p.gate, first, left, p.d, at[c], p.gate_f32);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = r.h[c].at(i), g = r.dn[c].at(i), f = r.f[c].at(i);
        a_pre[c].v[i] = __fmaf_rn(g, x * r2, a_pre[c].v[i]);
        dx.v[i] = __fmaf_rn(r2, __fmaf_rn(-x, m2, g * wb[c].at(i)), r.dh[c].at(i));
        const float dt = p.scale * dx.v[i];
        const float y = f * r1;
        dg.v[i] = dt * (y * wa[c].at(i));
        const float du = dt * (token * gate[c].at(i));
        a_y[c].v[i] = __fmaf_rn(p.gate_kind == kGateFull ? du : dt * token, y, a_y[c].v[i]);
        df[c].v[i] = du * wa[c].at(i);
        q[0] = __fmaf_rn(df[c].v[i], f, q[0]);
        q[1] += dg.v[i];
      }
      if (kLean) {  // (the sums are made here, not kept as their terms until the end of the row)
#pragma unroll
        for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(a_pre[c].v[i]), "+v"(a_y[c].v[i]), "+v"(df[c].v[i]));
        asm volatile("" : "+v"(q[0]), "+v"(q[1]));
      }
      if (p.d_x) write8<kS32>(rows_buf<kS32>(p.d_x, first, left, p.d), at[c], dx);
      if (p.gate_kind == kGateFull && p.d_gate) {
        if (p.gate_f32) write8<true>(rows_buf<true>(p.d_gate, first, left, p.d), at[c], dg);
        else write8<false>(rows_buf<false>(p.d_gate, first, left, p.d), at[c], dg);
      }
    }
    row_sum<kLanes, 2>(q, mem[1], threads);
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      if (kLean) r.f[c] = raw8<kF32>(rows_buf<kF32>(p.f, first, left, p.d), at[c]);
      unpack_later(r.f[c]);
    }
    if (p.gate_kind == kGateToken && p.d_gate && live && t == 0) ((float*)p.d_gate)[first + mine] = q[1];
    if (p.d_f) {
      const float m1 = q[0] * p.per * r1 * r1;  // r1^2 mean(post_w du f)
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        if (p.post_w)  // (without it f is no factor: an infinity or NaN there may not reach d_f as a product with 0)
#pragma unroll
          for (int i = 0; i < 8; ++i) df[c].v[i] = r1 * __fmaf_rn(-r.f[c].at(i), m1, df[c].v[i]);
        write8<kF32>(rows_buf<kF32>(p.d_f, first, left, p.d), at[c], df[c]);
      }
    }
  }
  if (!p.part) return;
  float* out = p.part + (int64_t)blockIdx.x * 3 * p.d;
  auto leave = [&](const V8 (&a)[kC], float* to) {
    if (kLanes == 0) {
#pragma unroll
      for (int c = 0; c < kC; ++c) write8<true>(rows_buf<true>(to, 0, 1, p.d), wcol[c], a[c]);
    } else {  // the rows' groups in their order
      __syncthreads();
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[(mine * kC + c) * 8 * threads + i * threads + t] = a[c].v[i];
      __syncthreads();
      if (mine == 0)
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          V8 v = {};
          for (int g = 0; g < kRows; ++g)
#pragma unroll
            for (int i = 0; i < 8; ++i) v.v[i] += sums[(g * kC + c) * 8 * threads + i * threads + t];
          write8<true>(rows_buf<true>(to, 0, 1, p.d), wcol[c], v);
        }
    }
  };
  if (p.sum_pre) leave(a_pre, out);
  if (!p.sum_post && !p.sum_gate) return;
  V8 v[kC];
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    if (kLean) read_post(c);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[c].v[i] = a_y[c].v[i] * wa[c].at(i);
  }
  if (p.sum_gate) leave(v, out + 2 * p.d);
  if (!p.sum_post) return;
#pragma unroll
  for (int c = 0; c < kC; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[c].v[i] = p.gate_kind == kGateChannel ? a_y[c].v[i] * gate[c].at(i) : a_y[c].v[i];
  leave(v, out + p.d);
}

// Column sums of the workgroups' rows: 64 columns per workgroup, its 16 waves a
// sixteenth of the rows each, joined in wave order.
constexpr int kJoinWaves = 16;
struct JoinParams {
  const float* part;
  float* out[3];
  int rows[3];  // 0: a gradient of zeros
  int d;
};
__global__ void __launch_bounds__(kJoinWaves * 64) block_norm_join_kernel(JoinParams p) {
  __shared__ float mem[kJoinWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t col = blockIdx.x * 64 + lane, which = blockIdx.y;
  if (!p.out[which]) return;
  const int rows = p.rows[which], per = (rows + kJoinWaves - 1) / kJoinWaves;
  const int r0 = wave * per, r1 = r0 + per < rows ? r0 + per : rows;
  float s = 0.0f;
  if (col < (uint32_t)p.d)
#pragma unroll 8
    for (int r = r0; r < r1; ++r) s += p.part[((int64_t)r * 3 + which) * p.d + col];
  mem[wave][lane] = s;
  __syncthreads();
  if (wave || col >= (uint32_t)p.d) return;
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w) s += mem[w][lane];
  p.out[which][col] = s;
}

// How rows are shared out: threads per row (8 .. 64 of a wave, 0: the workgroup's),
// threads of a workgroup, its rows at a time, a thread's chunks of eight columns.
struct Shape {
  int lanes, threads, rows, chunks;
};
Shape shape_of(int64_t d, bool grad) {
  const int chunks = (int)(d / 8);
  if (chunks <= 8) return {8, 256, 32, 1};
  if (chunks <= 16) return {16, 256, 16, 1};
  if (chunks <= 32) return {32, 256, 8, 1};
  if (chunks <= 64) return {64, 256, 4, 1};
  // (a row of 512 to 1024 by a wave, which waits for no other: 32768 x 768 bf16 67 us, by two waves 158)
  if (grad && chunks <= 128) return {64, 256, 4, 2};
  // (half the threads with two chunks each take longer: forward 8191 x 4096 51.5 us for 47,
  // 8191 x 6144 89 for 72)
  const int per = chunks > 1024 ? 2 : 1;
  return {0, ((chunks + per - 1) / per + 63) / 64 * 64, 1, per};
}
// Workgroups of the gradient: with weights' gradients to sum, what the CUs hold (each
// leaves a row of sums); else one per row group.  Short rows of a workgroup each want
// more of them to wait with (bf16 21000 x 1536 90 us with four per CU, 111 with two), if
// they are not of fp32 (136 with two, 149 with four).  Few rows: four for a workgroup,
// since each of them leaves a row of sums to be joined (512 x 4096 captured 22 us by 512, 18 by 128).
int64_t grad_groups(int64_t m, const Shape& s, bool sums, bool f32) {
  const int per_cu = s.threads > 512 ? 1 : s.lanes || f32 ? 2 : std::max(2, 768 / s.threads);
  const int64_t all = (m + s.rows - 1) / s.rows, some = std::min(per_cu * (int64_t)device_cus(), std::max<int64_t>(128, all / 4));
  // (by 1024 threads 2^22 would be one thread more than a launch counts; workgroups go on to further rows)
  return sums && all > some ? some : std::min<int64_t>(all, (1 << 22) - 1);
}

template <bool kGrad, bool kF32, bool kS32, bool kW32>
void launch(const Shape& s, int64_t grid, const BlockNormParams& p, hipStream_t st) {
  const dim3 g((unsigned)grid), b(s.threads);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, b, 0, st, p); };
  if constexpr (kGrad) {
    if (s.lanes == 8) return go(block_norm_grad_kernel<8, 1, 256, kF32, kS32, kW32>);
    if (s.lanes == 16) return go(block_norm_grad_kernel<16, 1, 256, kF32, kS32, kW32>);
    if (s.lanes == 32) return go(block_norm_grad_kernel<32, 1, 256, kF32, kS32, kW32>);
    if (s.lanes == 64 && s.chunks == 1) return go(block_norm_grad_kernel<64, 1, 256, kF32, kS32, kW32>);
    if (s.lanes == 64) return go(block_norm_grad_kernel<64, 2, 256, kF32, kS32, kW32>);
    if (s.threads <= 512) return go(block_norm_grad_kernel<0, 1, 512, kF32, kS32, kW32>);
    if (s.chunks == 1) return go(block_norm_grad_kernel<0, 1, 1024, kF32, kS32, kW32>);
    return go(block_norm_grad_kernel<0, 2, 1024, kF32, kS32, kW32>);
  } else {
    if (s.lanes == 8) return go(block_norm_kernel<8, 1, kF32, kS32>);
    if (s.lanes == 16) return go(block_norm_kernel<16, 1, kF32, kS32>);
    if (s.lanes == 32) return go(block_norm_kernel<32, 1, kF32, kS32>);
    if (s.lanes == 64) return go(block_norm_kernel<64, 1, kF32, kS32>);
    if (s.chunks == 1) return go(block_norm_kernel<0, 1, kF32, kS32>);
    return go(block_norm_kernel<0, 2, kF32, kS32>);
  }
}
template <bool kGrad, bool kW32>
void launch_rows(const Shape& s, int64_t grid, bool f32, bool s32, const BlockNormParams& p, hipStream_t st) {
  if (f32 && s32)
    launch<kGrad, true, true, kW32>(s, grid, p, st);
  else if (f32)
    launch<kGrad, true, false, kW32>(s, grid, p, st);
  else if (s32)
    launch<kGrad, false, true, kW32>(s, grid, p, st);
  else
    launch<kGrad, false, false, kW32>(s, grid, p, st);
}
template <bool kGrad>
void launch_kinds(const Shape& s, int64_t grid, bool f32, bool s32, const BlockNormParams& p, hipStream_t st) {
  // (the forward pass reads weights of either kind as they come)
  if (kGrad && ((p.w_f32 && (p.post_w || p.pre_w)) || (p.gate_f32 && (p.gate_kind == kGateChannel || p.gate_kind == kGateFull))))
    launch_rows<kGrad, kGrad>(s, grid, f32, s32, p, st);
  else
    launch_rows<kGrad, false>(s, grid, f32, s32, p, st);
}

bool kind_ok(int k) { return k == HSMOE_OUT_F32 || k == HSMOE_OUT_BF16; }
int check_norm(const char* who, int64_t m, int64_t d, float eps, const hsmoe_block_norm_spec* n) {
  if (!n || m < 0 || d < 1 || !(eps >= 0.0f) || !kind_ok(n->row_kind) || !kind_ok(n->stream_kind) || !kind_ok(n->weight_kind) ||
      !kind_ok(n->gate_kind) || n->gate_form < kGateNone || n->gate_form > kGateFull ||
      (n->gate_form == kGateNone && n->gate_dev) || (n->gate_form != kGateNone && !n->gate_dev && m > 0))
    return fail(HSMOE_ERR_ARG, "%s: bad arguments", who);
  if (d % 8 != 0 || d > kMaxD) return fail(HSMOE_ERR_SHAPE, "%s: d must be a multiple of 8 and at most %d", who, kMaxD);
  if (m >= (1ll << 31)) return fail(HSMOE_ERR_SHAPE, "%s: m must be below 2^31", who);
  if (!aligned(n->post_w_dev, 16) || !aligned(n->pre_w_dev, 16) || !aligned(n->gate_dev, n->gate_form == kGateToken ? 4 : 16))
    return fail(HSMOE_ERR_SHAPE, "%s: weights and gates must be 16-byte aligned", who);
  return HSMOE_OK;
}
BlockNormParams params_of(int64_t m, int64_t d, float scale, float eps, const hsmoe_block_norm_spec* n) {
  BlockNormParams p{};
  p.post_w = n->post_w_dev, p.pre_w = n->pre_w_dev, p.gate = n->gate_dev;
  p.m = m, p.d = (int)d, p.gate_kind = n->gate_form;
  p.w_f32 = n->weight_kind == HSMOE_OUT_F32, p.gate_f32 = n->gate_kind == HSMOE_OUT_F32;
  p.scale = scale, p.eps = eps, p.per = 1.0f / (float)d;
  return p;
}

}  // namespace
}  // namespace hsmoe

using namespace hsmoe;

extern "C" int hsmoe_block_norm(const void* f, const void* h, int64_t m, int64_t d, const hsmoe_block_norm_spec* spec,
                                float scale, float eps, void* h_out, void* n_out, hsmoe_stream_t stream) {
  const char* who = "hsmoe_block_norm";
  if (int rc = check_norm(who, m, d, eps, spec)) return rc;
  if (m == 0) return HSMOE_OK;
  if (!f || !h || !h_out || (spec->pre_w_dev != nullptr) != (n_out != nullptr)) return fail(HSMOE_ERR_ARG, "%s: null pointer", who);
  if (!aligned(f, 16) || !aligned(h, 16) || !aligned(h_out, 16) || !aligned(n_out, 16))
    return fail(HSMOE_ERR_SHAPE, "%s: rows must be 16-byte aligned", who);
  BlockNormParams p = params_of(m, d, scale, eps, spec);
  p.f = f, p.h = h, p.h_out = h_out, p.n_out = n_out;
  const Shape s = shape_of(d, false);
  if (!grid_fits((m + s.rows - 1) / s.rows, s.threads)) return fail(HSMOE_ERR_SHAPE, "%s: too many rows of this width for one launch", who);
  launch_kinds<false>(s, (m + s.rows - 1) / s.rows, spec->row_kind == HSMOE_OUT_F32, spec->stream_kind == HSMOE_OUT_F32, p,
                      (hipStream_t)stream);
  return check_launch(who);
}

extern "C" size_t hsmoe_block_norm_grad_workspace_size(int64_t m, int64_t d) {
  if (m < 1 || d < 8 || d > kMaxD) return 0;
  return (size_t)grad_groups(m, shape_of(d, true), true, false) * 3 * d * sizeof(float);
}

extern "C" int hsmoe_block_norm_grad(const void* d_h, const void* d_n, const void* f, const void* h_out, int64_t m,
                                     int64_t d, const hsmoe_block_norm_spec* spec, float scale, float eps, void* d_f,
                                     void* d_x, float* d_post, void* d_gate, float* d_pre, void* workspace,
                                     size_t workspace_bytes, hsmoe_stream_t stream) {
  const char* who = "hsmoe_block_norm_grad";
  if (int rc = check_norm(who, m, d, eps, spec)) return rc;
  if ((d_post && !spec->post_w_dev) || (d_pre && !spec->pre_w_dev) || (d_gate && spec->gate_form == kGateNone) || (d_n && !spec->pre_w_dev))
    return fail(HSMOE_ERR_ARG, "%s: the gradient of what is not there", who);
  if (m > 0 && !d_h && !d_n) return fail(HSMOE_ERR_ARG, "%s: null pointer", who);
  const bool sum_gate = d_gate && spec->gate_form == kGateChannel;
  const bool sums = d_post || d_pre || sum_gate;
  if (m > 0 && (!f || (d_n && !h_out))) return fail(HSMOE_ERR_ARG, "%s: null pointer", who);
  const void* rows[] = {d_h, d_n, f, h_out, d_f, d_x};
  for (const void* q : rows)
    if (!aligned(q, 16)) return fail(HSMOE_ERR_SHAPE, "%s: rows must be 16-byte aligned", who);
  if (!aligned(d_gate, spec->gate_form == kGateFull ? 16 : 4) || !aligned(d_post, 4) || !aligned(d_pre, 4))
    return fail(HSMOE_ERR_SHAPE, "%s: misaligned gradients", who);
  const Shape s = shape_of(d, true);
  const int64_t groups = m > 0 ? grad_groups(m, s, sums, spec->row_kind == HSMOE_OUT_F32 || spec->stream_kind == HSMOE_OUT_F32) : 0;
  const size_t need = sums ? (size_t)groups * 3 * d * sizeof(float) : 0;
  if (need && (!workspace || workspace_bytes < need)) return fail(HSMOE_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", who, need);
  if (need && !aligned(workspace, 16)) return fail(HSMOE_ERR_SHAPE, "%s: misaligned workspace", who);
  BlockNormParams p = params_of(m, d, scale, eps, spec);
  p.d_h = d_h, p.d_n = d_n, p.f = f, p.h = h_out;
  p.d_f = d_f, p.d_x = d_x, p.d_gate = sum_gate ? nullptr : d_gate;
  p.part = sums ? (float*)workspace : nullptr;
  p.sum_pre = d_pre && d_n, p.sum_post = d_post, p.sum_gate = sum_gate;
  hipStream_t st = (hipStream_t)stream;
  if (groups)
    launch_kinds<true>(s, groups, spec->row_kind == HSMOE_OUT_F32, spec->stream_kind == HSMOE_OUT_F32, p, st);
  if (sums) {
    const int g = (int)groups;
    const JoinParams j{(const float*)workspace, {d_pre, d_post, sum_gate ? (float*)d_gate : nullptr}, {d_n ? g : 0, g, g}, (int)d};
    hipLaunchKernelGGL(block_norm_join_kernel, dim3((unsigned)((d + 63) / 64), 3), dim3(kJoinWaves * 64), 0, st, j);
  }
  return check_launch(who);
}

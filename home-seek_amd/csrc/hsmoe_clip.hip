// The norm of many tensors together, and all of them cut down to a limit on it:
//   norm = (sum of x^2 over all values of all tensors)^(1/2), or max |x|
//   out  = x * min(1, max_norm / (norm + 1e-6))
// Squares and their sums in 64 bits: no gradient is too large or too small for its
// square.  Two passes over the data, bound by HBM: one for the norm, of which every
// workgroup leaves its part, and one that adds up the parts (in every workgroup, in
// one order; once for all, by a launch between, where much data goes to other tensors),
// and multiplies.  The second goes through the data backwards, so that
// what the first read last comes out of the caches.  Tensors that are clipped in
// place and need no clipping are not touched.  Measured: 1.24 GB in 60 tensors, bf16 and
// fp32, the norm 211 us (5.9 TB/s; reads alone reach 6.5), with the clipped copy 640; 6
// tensors of 8064 values in all 7.6 us.  More workgroups, or fewer loads on their way,
// change nothing.
#include <algorithm>
#include <cmath>
#include <vector>

#include "hsmoe_common.h"
#include "hsmoe_internal.h"

namespace hsmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 16384;        // values that a workgroup takes at a time
constexpr int kPiece = 2048;         // .. or in piece_kernel, all in all
constexpr int kBlocks = 1024;        // workgroups of a pass that go through chunks, at most
constexpr int64_t kMuch = 1 << 24;   // values from which piece_kernel is worth the launch of norm_join_kernel
constexpr int kPer = 112;            // tensors per launch: their addresses are kernel arguments, so that a captured graph holds them
constexpr int64_t kSmall = 32768;    // values up to which one workgroup does it all
constexpr int kSmallThreads = 1024;
constexpr int kSmallChunk = 1024;    // values that one of its waves takes at a time

enum { kInF32 = 1, kOutF32 = 2, kInVec = 4, kOutVec = 8, kSame = 16 };

struct Batch {
  const void* in[kPer];
  void* out[kPer];
  int64_t count[kPer];
  uint32_t first[kPer + 1];  // chunks before the tensor's
  uint8_t flags[kPer];
  int n;
};

// A part of the norm: the sum of squares, or the largest magnitude's bits (those of a
// NaN are above all others').
template <bool kMax>
struct Part;
template <>
struct Part<false> {
  double v = 0.0;
  __device__ __forceinline__ void take(float x) { v = __builtin_fma((double)x, (double)x, v); }
  __device__ __forceinline__ void join(const Part& o) { v += o.v; }
  __device__ __forceinline__ Part lane(int x) const {
    Part o;
    o.v = __shfl_xor(v, x, 64);
    return o;
  }
  __device__ __forceinline__ double norm() const { return sqrt(v); }
};
template <>
struct Part<true> {
  unsigned long long v = 0;
  __device__ __forceinline__ void take(float x) {
    const unsigned long long b = __float_as_uint(x) & 0x7fffffffu;
    v = b > v ? b : v;
  }
  __device__ __forceinline__ void join(const Part& o) { v = o.v > v ? o.v : v; }
  __device__ __forceinline__ Part lane(int x) const {
    Part o;
    o.v = (unsigned long long)(unsigned)__shfl_xor((int)v, x, 64);
    return o;
  }
  __device__ __forceinline__ double norm() const { return (double)__uint_as_float((uint32_t)v); }
};

// The workgroup's threads' parts, joined in a fixed order, in every thread.
template <bool kMax, int kN>
__device__ __forceinline__ Part<kMax> join_block(Part<kMax> p) {
  __shared__ decltype(p.v) mem[kN / 64];
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) p.join(p.lane(off));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) mem[threadIdx.x >> 6] = p.v;
  __syncthreads();
  Part<kMax> all;
#pragma unroll
  for (int w = 0; w < kN / 64; ++w) {
    Part<kMax> o;
    o.v = mem[w];
    all.join(o);
  }
  return all;
}

// min(1, max_norm / (norm + 1e-6)) = a b; NaN stays NaN, and nothing is beyond an infinite
// limit, an infinite norm neither (inf / inf would make NaN of every value).  Where fp32 does not hold the
// factor with all its bits (a norm of 2^100 limits), two factors of half its exponent do.
struct Factor {
  float a, b;
};
__device__ __forceinline__ Factor factor(double norm, float max_norm) {
  const double c = (double)max_norm / (norm + 1e-6);
  if (c >= 1.0 || (isinf(max_norm) && !isnan(norm))) return {1.0f, 1.0f};
  if (!(c < 0x1p-100) || c == 0.0) return {1.0f, (float)c};
  const int e = ilogb(c) / 2;
  return {(float)ldexp(1.0, e), (float)ldexp(c, -e)};
}

struct Vals {
  float v[8];
};
// Eight values as they lie in memory.
template <bool kF32>
struct Raw {
  uint32_t w[kF32 ? 8 : 4] = {};
  __device__ __forceinline__ float at(int i) const {
    if (kF32) return __uint_as_float(w[i]);
    return i & 1 ? __uint_as_float(w[i >> 1] & 0xffff0000u) : __uint_as_float(w[i >> 1] << 16);
  }
};
template <bool kF32>
__device__ __forceinline__ Raw<kF32> read8(const void* base, int64_t at) {
  Raw<kF32> r;
  const char* p = (const char*)base + at * (kF32 ? 4 : 2);
#pragma unroll
  for (int i = 0; i < (kF32 ? 2 : 1); ++i) {
    const uint4 a = ldg<uint4>(p + 16 * i);
    r.w[4 * i] = a.x, r.w[4 * i + 1] = a.y, r.w[4 * i + 2] = a.z, r.w[4 * i + 3] = a.w;
  }
  return r;
}
template <bool kF32>
__device__ __forceinline__ float read1(const void* base, int64_t at) {
  return kF32 ? ((const float*)base)[at] : bf16_bits_to_f32(((const uint16_t*)base)[at]);
}
template <bool kF32>
__device__ __forceinline__ void write8(void* base, int64_t at, const Vals& r) {
  if (kF32) {
    float4* p = reinterpret_cast<float4*>((float*)base + at);
    p[0] = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
    p[1] = make_float4(r.v[4], r.v[5], r.v[6], r.v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = f32_to_bf16_bits(r.v[2 * i]) | f32_to_bf16_bits(r.v[2 * i + 1]) << 16;
    *reinterpret_cast<uint4*>((uint16_t*)base + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <bool kF32>
__device__ __forceinline__ void write1(void* base, int64_t at, float v) {
  if (kF32) ((float*)base)[at] = v;
  else ((uint16_t*)base)[at] = (uint16_t)f32_to_bf16_bits(v);
}

// Values a .. b of a tensor, kN threads.
template <bool kMax, bool kF32, int kN>
__device__ __forceinline__ void take_part(const void* in, int64_t a, int64_t b, bool vec, Part<kMax>& s) {
  int64_t done = a;
  if (vec) {
    constexpr int kAhead = (kF32 ? 2 : 4) * (kN == kThreads ? 2 : 1) / (kN == 64 ? 2 : 1);
    const int64_t whole = a + (b - a) / 8 * 8;
    for (int64_t i = a + (int64_t)(threadIdx.x % kN) * 8; i < whole; i += (int64_t)kAhead * kN * 8) {
      Raw<kF32> v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) v[j] = i + (int64_t)j * kN * 8 < whole ? read8<kF32>(in, i + (int64_t)j * kN * 8) : Raw<kF32>{};
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
#pragma unroll
        for (int k = 0; k < 8; ++k) s.take(v[j].at(k));
    }
    done = whole;
  }
  for (int64_t i = done + threadIdx.x % kN; i < b; i += kN) s.take(read1<kF32>(in, i));
}
template <bool kF32, bool kO32, int kN>
__device__ __forceinline__ void scale_part(const void* in, void* out, int64_t a, int64_t b, bool vec, Factor c) {
  int64_t done = a;
  if (vec) {
    constexpr int kAhead = (kF32 ? 2 : 4) * (kN == kThreads ? 2 : 1) / (kN == 64 ? 2 : 1);
    const int64_t whole = a + (b - a) / 8 * 8;
    for (int64_t i = a + (int64_t)(threadIdx.x % kN) * 8; i < whole; i += (int64_t)kAhead * kN * 8) {
      Raw<kF32> v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) v[j] = i + (int64_t)j * kN * 8 < whole ? read8<kF32>(in, i + (int64_t)j * kN * 8) : Raw<kF32>{};
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        Vals o;
#pragma unroll
        for (int k = 0; k < 8; ++k) o.v[k] = v[j].at(k) * c.a * c.b;
        if (i + (int64_t)j * kN * 8 < whole) write8<kO32>(out, i + (int64_t)j * kN * 8, o);
      }
    }
    done = whole;
  }
  for (int64_t i = done + threadIdx.x % kN; i < b; i += kN) write1<kO32>(out, i, read1<kF32>(in, i) * c.a * c.b);
}
template <bool kMax, int kN>
__device__ __forceinline__ void take_any(const Batch& t, int j, int64_t a, int64_t b, Part<kMax>& s) {
  const bool vec = t.flags[j] & kInVec;
  if (t.flags[j] & kInF32) take_part<kMax, true, kN>(t.in[j], a, b, vec, s);
  else take_part<kMax, false, kN>(t.in[j], a, b, vec, s);
}
template <int kN>
__device__ __forceinline__ void scale_any(const Batch& t, int j, int64_t a, int64_t b, Factor c) {
  if (c.a == 1.0f && c.b == 1.0f && (t.flags[j] & kSame)) return;
  const bool vec = (t.flags[j] & (kInVec | kOutVec)) == (kInVec | kOutVec);
  switch (t.flags[j] & (kInF32 | kOutF32)) {
    case 0: return scale_part<false, false, kN>(t.in[j], t.out[j], a, b, vec, c);
    case kInF32: return scale_part<true, false, kN>(t.in[j], t.out[j], a, b, vec, c);
    case kOutF32: return scale_part<false, true, kN>(t.in[j], t.out[j], a, b, vec, c);
    default: return scale_part<true, true, kN>(t.in[j], t.out[j], a, b, vec, c);
  }
}

// The tensor that chunk c belongs to (the chunks of t.n tensors, none of them empty).
__device__ __forceinline__ int tensor_of(const Batch& t, uint32_t c) {
  int lo = 0, hi = t.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <bool kMax>
__global__ void __launch_bounds__(kThreads) norm_part_kernel(Batch t, Part<kMax>* parts) {
  Part<kMax> s;
  for (uint32_t c = blockIdx.x; c < t.first[t.n]; c += gridDim.x) {
    const int j = tensor_of(t, c);
    const int64_t a = (int64_t)(c - t.first[j]) * kChunk, b = a + kChunk < t.count[j] ? a + kChunk : t.count[j];
    take_any<kMax, kThreads>(t, j, a, b, s);
  }
  s = join_block<kMax, kThreads>(s);
  if (threadIdx.x == 0) parts[blockIdx.x] = s;
}

template <bool kMax>
__device__ __forceinline__ double norm_of(const Part<kMax>* parts, int n) {
  Part<kMax> s;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += kThreads) s.join(parts[i]);
  return join_block<kMax, kThreads>(s).norm();
}

template <bool kMax>
__global__ void __launch_bounds__(kThreads) scale_kernel(Batch t, const Part<kMax>* parts, int n_parts, float max_norm, float* norm_out) {
  const double norm = norm_of<kMax>(parts, n_parts);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const Factor f = factor(norm, max_norm);
  const uint32_t chunks = t.first[t.n];
  for (uint32_t i = blockIdx.x; i < chunks; i += gridDim.x) {
    const uint32_t c = chunks - 1 - i;
    const int j = tensor_of(t, c);
    const int64_t a = (int64_t)(c - t.first[j]) * kChunk, b = a + kChunk < t.count[j] ? a + kChunk : t.count[j];
    scale_any<kThreads>(t, j, a, b, f);
  }
}

// The norm, and the factor for piece_kernel (NULL: the norm alone).
template <bool kMax>
__global__ void __launch_bounds__(kThreads) norm_join_kernel(const Part<kMax>* parts, int n_parts, float max_norm, float* norm_out, Factor* f) {
  const double norm = norm_of<kMax>(parts, n_parts);
  if (threadIdx.x) return;
  *norm_out = (float)norm;
  if (f) *f = factor(norm, max_norm);
}

// The second pass over much data: a workgroup takes 2048 values and ends, so that
// what is on its way is one narrow window that moves through the tensors (a copy runs
// at 6.2 TB/s this way, at 5.4 by workgroups that go through all of it side by side).
template <bool kF32, bool kO32>
__device__ __forceinline__ void scale_piece(const void* in, void* out, int64_t a, int64_t b, bool vec, Factor c) {
  if (vec && b - a == kPiece) {
    if constexpr (kF32 && kO32) {
      float4 v[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) v[i] = reinterpret_cast<const float4*>((const float*)in + a)[i * kThreads + threadIdx.x];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        reinterpret_cast<float4*>((float*)out + a)[i * kThreads + threadIdx.x] =
            make_float4(v[i].x * c.a * c.b, v[i].y * c.a * c.b, v[i].z * c.a * c.b, v[i].w * c.a * c.b);
    } else {
      const int64_t at = a + (int64_t)threadIdx.x * 8;
      const Raw<kF32> v = read8<kF32>(in, at);
      Vals o;
#pragma unroll
      for (int k = 0; k < 8; ++k) o.v[k] = v.at(k) * c.a * c.b;
      write8<kO32>(out, at, o);
    }
    return;
  }
  for (int64_t i = a + threadIdx.x; i < b; i += kThreads) write1<kO32>(out, i, read1<kF32>(in, i) * c.a * c.b);
}
__global__ void __launch_bounds__(kThreads) piece_kernel(Batch t, const Factor* factor) {
  const uint32_t piece = gridDim.x - 1 - blockIdx.x, chunk = piece / (kChunk / kPiece);
  const int j = tensor_of(t, chunk), flags = t.flags[j];
  const int64_t a = (int64_t)(chunk - t.first[j]) * kChunk + piece % (kChunk / kPiece) * kPiece;
  const int64_t b = a + kPiece < t.count[j] ? a + kPiece : t.count[j];
  const Factor c = *factor;
  if (a >= b || (c.a == 1.0f && c.b == 1.0f && (flags & kSame))) return;
  const bool vec = (flags & (kInVec | kOutVec)) == (kInVec | kOutVec);
  switch (flags & (kInF32 | kOutF32)) {
    case 0: return scale_piece<false, false>(t.in[j], t.out[j], a, b, vec, c);
    case kInF32: return scale_piece<true, false>(t.in[j], t.out[j], a, b, vec, c);
    case kOutF32: return scale_piece<false, true>(t.in[j], t.out[j], a, b, vec, c);
    default: return scale_piece<true, true>(t.in[j], t.out[j], a, b, vec, c);
  }
}

// Few values: one workgroup, one launch, whose waves take chunks of kSmallChunk (60 tensors
// of 10000 values in all 12 us; tensor after tensor by all waves 61).
template <bool kMax, bool kClip>
__global__ void __launch_bounds__(kSmallThreads) small_kernel(Batch t, float max_norm, float* norm_out) {
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), chunks = t.first[t.n];
  auto each = [&](auto f) {
    for (uint32_t c = wave; c < chunks; c += kSmallThreads / 64) {
      const int j = tensor_of(t, c);
      const int64_t a = (int64_t)(c - t.first[j]) * kSmallChunk;
      f(j, a, a + kSmallChunk < t.count[j] ? a + kSmallChunk : t.count[j]);
    }
  };
  Part<kMax> s;
  each([&](int j, int64_t a, int64_t b) { take_any<kMax, 64>(t, j, a, b, s); });
  const double norm = join_block<kMax, kSmallThreads>(s).norm();
  if (threadIdx.x == 0) *norm_out = (float)norm;
  if (!kClip) return;
  const Factor f = factor(norm, max_norm);
  each([&](int j, int64_t a, int64_t b) { scale_any<64>(t, j, a, b, f); });
}

// ---------------------------------------------------------------- host
struct Tensors {
  int64_t n;
  const void* const* in;
  void* const* out;  // NULL: the norm alone
  const int64_t* counts;
  const int32_t *kinds, *out_kinds;
};

int64_t bytes_of(int64_t count, int kind) { return count * (kind == HSMOE_OUT_F32 ? 4 : 2); }

int check_tensors(const char* who, const Tensors& t, double norm_type, float max_norm, const float* norm_out) {
  if (t.n < 0 || t.n > (1 << 20) || !norm_out || (t.n > 0 && (!t.in || !t.counts || !t.kinds))) return fail(HSMOE_ERR_ARG, "%s: bad arguments", who);
  if (norm_type != 2.0 && !(std::isinf(norm_type) && norm_type > 0)) return fail(HSMOE_ERR_ARG, "%s: a norm of type 2 or infinity", who);
  if (!(max_norm >= 0.0f)) return fail(HSMOE_ERR_ARG, "%s: the limit must not be negative", who);
  if (!aligned(norm_out, 4)) return fail(HSMOE_ERR_SHAPE, "%s: misaligned norm", who);
  struct Range {
    uintptr_t a, b;
    bool write;
  };
  std::vector<Range> ranges;
  for (int64_t i = 0; i < t.n; ++i) {
    const int k = t.kinds[i], o = t.out ? t.out_kinds[i] : k;
    if (t.counts[i] < 0 || (k != HSMOE_OUT_F32 && k != HSMOE_OUT_BF16) || (o != HSMOE_OUT_F32 && o != HSMOE_OUT_BF16))
      return fail(HSMOE_ERR_ARG, "%s: bad arguments", who);
    if (t.counts[i] == 0) continue;
    if (!t.in[i] || (t.out && !t.out[i])) return fail(HSMOE_ERR_ARG, "%s: null pointer", who);
    if (t.counts[i] >= (1ll << 38)) return fail(HSMOE_ERR_SHAPE, "%s: a tensor of 2^38 values and more", who);
    if (!aligned(t.in[i], k == HSMOE_OUT_F32 ? 4 : 2) || (t.out && !aligned(t.out[i], o == HSMOE_OUT_F32 ? 4 : 2)))
      return fail(HSMOE_ERR_SHAPE, "%s: misaligned tensor", who);
    if (!t.out) continue;
    const uintptr_t a = (uintptr_t)t.in[i], w = (uintptr_t)t.out[i];
    if (a != w || k != o) ranges.push_back({a, a + (uintptr_t)bytes_of(t.counts[i], k), false});
    ranges.push_back({w, w + (uintptr_t)bytes_of(t.counts[i], o), true});
  }
  // what is written overlaps nothing: a value that is read twice would be clipped twice, or not, as workgroups come
  std::sort(ranges.begin(), ranges.end(), [](const Range& x, const Range& y) { return x.a < y.a; });
  uintptr_t written = 0, seen = 0;
  for (const Range& r : ranges) {
    if (r.a < (r.write ? seen : written)) return fail(HSMOE_ERR_ARG, "%s: tensors overlap", who);
    seen = std::max(seen, r.b);
    if (r.write) written = std::max(written, r.b);
  }
  return HSMOE_OK;
}

// Tensors from `at` on that go into one launch; at: the first that does not.
Batch batch_of(const Tensors& t, int64_t& at, int chunk = kChunk) {
  Batch b{};
  uint64_t chunks = 0;
  for (; at < t.n && b.n < kPer; ++at) {
    const int64_t c = t.counts[at];
    if (c == 0) continue;
    const int j = b.n++;
    b.in[j] = t.in[at], b.out[j] = t.out ? t.out[at] : nullptr, b.count[j] = c;
    const bool f = t.kinds[at] == HSMOE_OUT_F32, o = t.out && t.out_kinds[at] == HSMOE_OUT_F32;
    b.flags[j] = (uint8_t)((f ? kInF32 : 0) | (o ? kOutF32 : 0) | (aligned(b.in[j], 16) ? kInVec : 0) | (aligned(b.out[j], 16) ? kOutVec : 0) |
                           (b.in[j] == b.out[j] && f == o ? kSame : 0));
    b.first[j] = (uint32_t)chunks;
    chunks += (uint64_t)((c + chunk - 1) / chunk);  // (kPer tensors of less than 2^38 values: below 2^31)
    b.first[b.n] = (uint32_t)chunks;
  }
  return b;
}

size_t parts_bytes(int64_t n) { return (size_t)((n + kPer - 1) / kPer) * kBlocks * sizeof(Part<false>); }

template <bool kMax>
int run_clip(const char* who, const Tensors& t, float max_norm, float* norm_out, void* workspace, hipStream_t st) {
  int64_t total = 0, live = 0, moved = 0;
  for (int64_t i = 0; i < t.n; ++i) {
    total += t.counts[i], live += t.counts[i] > 0;
    if (t.out && (t.out[i] != t.in[i] || t.out_kinds[i] != t.kinds[i])) moved += t.counts[i];
  }
  if (total <= kSmall && live <= kPer) {
    int64_t at = 0;
    const Batch b = batch_of(t, at, kSmallChunk);
    if (t.out) hipLaunchKernelGGL((small_kernel<kMax, true>), dim3(1), dim3(kSmallThreads), 0, st, b, max_norm, norm_out);
    else hipLaunchKernelGGL((small_kernel<kMax, false>), dim3(1), dim3(kSmallThreads), 0, st, b, max_norm, norm_out);
    return check_launch(who);
  }
  Part<kMax>* parts = (Part<kMax>*)workspace;
  int n_parts = 0;
  for (int64_t at = 0; at < t.n;) {
    const Batch b = batch_of(t, at);
    if (!b.n) continue;
    const int blocks = (int)std::min<uint32_t>(b.first[b.n], kBlocks);
    hipLaunchKernelGGL((norm_part_kernel<kMax>), dim3(blocks), dim3(kThreads), 0, st, b, parts + n_parts);
    n_parts += blocks;
  }
  // (what is clipped in place often needs no clipping: workgroups that only find that out
  // would cost 30 us for 1 GB, in 180, and gain 40 in 607 where it does)
  const bool much = moved >= kMuch;
  Factor* f = much ? (Factor*)((char*)workspace + parts_bytes(t.n)) : nullptr;
  if (!t.out || much)
    hipLaunchKernelGGL((norm_join_kernel<kMax>), dim3(1), dim3(kThreads), 0, st, parts, n_parts, max_norm, norm_out, f);
  if (!t.out) return check_launch(who);
  for (int64_t at = 0; at < t.n;) {
    const bool first = at == 0 && !much;
    const Batch b = batch_of(t, at);
    if (!b.n && !first) continue;
    const int64_t pieces = (int64_t)b.first[b.n] * (kChunk / kPiece);
    if (much && grid_fits(pieces, kThreads)) {
      hipLaunchKernelGGL(piece_kernel, dim3((unsigned)pieces), dim3(kThreads), 0, st, b, f);
      continue;
    }
    const int blocks = std::max(1, (int)std::min<uint32_t>(b.first[b.n], kBlocks));
    hipLaunchKernelGGL((scale_kernel<kMax>), dim3(blocks), dim3(kThreads), 0, st, b, parts, n_parts, max_norm, first ? norm_out : nullptr);
  }
  return check_launch(who);
}

int clip(const char* who, const Tensors& t, double norm_type, float max_norm, float* norm_out, void* workspace, size_t workspace_bytes,
         hsmoe_stream_t stream) {
  try {
    if (int rc = check_tensors(who, t, norm_type, max_norm, norm_out)) return rc;
  } catch (...) {
    return fail(HSMOE_ERR_WORKSPACE, "%s: out of host memory", who);
  }
  const size_t need = hsmoe_grad_norm_workspace_size(t.n);
  if (need && (!workspace || workspace_bytes < need)) return fail(HSMOE_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", who, need);
  if (need && !aligned(workspace, 8)) return fail(HSMOE_ERR_SHAPE, "%s: misaligned workspace", who);
  return norm_type == 2.0 ? run_clip<false>(who, t, max_norm, norm_out, workspace, (hipStream_t)stream)
                          : run_clip<true>(who, t, max_norm, norm_out, workspace, (hipStream_t)stream);
}

}  // namespace
}  // namespace hsmoe

using namespace hsmoe;

extern "C" size_t hsmoe_grad_norm_workspace_size(int64_t n) {
  return n < 1 ? 0 : parts_bytes(n) + sizeof(Factor);
}

extern "C" int hsmoe_grad_norm(int64_t n, const void* const* tensors, const int64_t* counts, const int32_t* kinds,
                               double norm_type, float* norm_out, void* workspace, size_t workspace_bytes,
                               hsmoe_stream_t stream) {
  return clip("hsmoe_grad_norm", Tensors{n, tensors, nullptr, counts, kinds, nullptr}, norm_type, 1.0f, norm_out, workspace, workspace_bytes, stream);
}

extern "C" int hsmoe_clip_grads(int64_t n, const void* const* tensors, const int64_t* counts, const int32_t* kinds,
                                void* const* outs, const int32_t* out_kinds, double norm_type, float max_norm,
                                float* norm_out, void* workspace, size_t workspace_bytes, hsmoe_stream_t stream) {
  if (n > 0 && (!outs || !out_kinds)) return fail(HSMOE_ERR_ARG, "hsmoe_clip_grads: bad arguments");
  static void* const none[1] = {nullptr};
  return clip("hsmoe_clip_grads", Tensors{n, tensors, n > 0 ? outs : none, counts, kinds, out_kinds}, norm_type, max_norm, norm_out, workspace,
              workspace_bytes, stream);
}

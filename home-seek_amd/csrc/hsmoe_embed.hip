// Embedding lookup with a scale, and its gradient.
//   out[t] = scale * table[ids[t]]               (a row of zeros for an id outside the table)
//   d_table[v] = scale * sum of d_out[t] over the tokens t with ids[t] = v
// The gradient sorts the tokens by id, stably, so that every row's terms are added
// in the order of the tokens, and cuts the sorted tokens into chunks of 32, so that
// a word that makes up much of a batch is summed by many workgroups: a run of equal
// ids inside a chunk is a row of the table; the ends of chunks that share a run leave
// fp32 sums, which a second launch adds in their order.  All of it is bound by HBM.
// Measured: 16381 tokens of 4096 bf16 looked up 37 us, with all of them different 44
// (6.1 TB/s); the gradient of a table of 129280 x 4096 216 us: sort and places beside
// 1.06 GB of zeros 165, sums 38, joins 8.  (Rows that no token names cleared beside the
// sums, by a flag each, instead of all before them, took 5 to 13 us longer.)
#include <algorithm>

#include "hsmoe_common.h"
#include "hsmoe_internal.h"

namespace hsmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kJoinThreads = 512;
constexpr int kChunk = 32;           // sorted tokens per chunk
constexpr int kUnit = 8;             // .. and per group of threads, where d_out has up to
constexpr int64_t kFew = 1 << 22;    // .. that many values
constexpr int kSortThreads = 1024;
constexpr int64_t kSortByRank = 65536;  // tokens up to which places are found by bisection
constexpr uint32_t kNoId = 1u << 30;    // an id outside the table, above all others

// The id of token t, -1 outside the table.
__device__ __forceinline__ int id_of(const void* ids, bool wide, int64_t t, int64_t vocab) {
  const int64_t v = wide ? ((const int64_t*)ids)[t] : (int64_t)((const int32_t*)ids)[t];
  return v >= 0 && v < vocab ? (int)v : -1;
}

template <bool kF32>
__device__ __forceinline__ float value(const void* p, int64_t at) {
  return kF32 ? ((const float*)p)[at] : bf16_bits_to_f32(((const uint16_t*)p)[at]);
}
template <bool kF32>
__device__ __forceinline__ void put(void* p, int64_t at, float v) {
  if (kF32) ((float*)p)[at] = v;
  else ((uint16_t*)p)[at] = (uint16_t)f32_to_bf16_bits(v);
}

// kVec values of a row at a time: 8 where rows are 16-byte aligned, else one.
template <int kVec>
struct Vals {
  float v[kVec];
};
template <int kVec, bool kF32>
__device__ __forceinline__ Vals<kVec> read(const void* base, int64_t at) {
  Vals<kVec> r;
  if constexpr (kVec == 1) {
    r.v[0] = value<kF32>(base, at);
  } else if constexpr (kF32) {
    const char* p = (const char*)base + at * 4;
    const uint4 a = ldg<uint4>(p), b = ldg<uint4>(p + 16);
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = __uint_as_float(w[i]);
  } else {
    const uint4 a = ldg<uint4>((const char*)base + at * 2);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[2 * i] = __uint_as_float(w[i] << 16), r.v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  return r;
}
// As they lie in memory.
template <int kVec, bool kF32>
struct Raw {
  uint32_t w[kVec == 1 ? 1 : kF32 ? 8 : 4];
  __device__ __forceinline__ float at(int i) const {
    if (kF32) return __uint_as_float(w[i]);
    if (kVec == 1) return __uint_as_float(w[0] << 16);
    return i & 1 ? __uint_as_float(w[i >> 1] & 0xffff0000u) : __uint_as_float(w[i >> 1] << 16);
  }
};
template <int kVec, bool kF32>
__device__ __forceinline__ Raw<kVec, kF32> fetch(const void* base, int64_t at) {
  Raw<kVec, kF32> r;
  const char* p = (const char*)base + at * (kF32 ? 4 : 2);
  if constexpr (kVec == 1) {
    r.w[0] = kF32 ? *(const uint32_t*)p : *(const uint16_t*)p;
  } else {
#pragma unroll
    for (int i = 0; i < (kF32 ? 2 : 1); ++i) {
      const uint4 a = ldg<uint4>(p + 16 * i);
      r.w[4 * i] = a.x, r.w[4 * i + 1] = a.y, r.w[4 * i + 2] = a.z, r.w[4 * i + 3] = a.w;
    }
  }
  return r;
}
template <int kVec, bool kF32>
__device__ __forceinline__ void write(void* base, int64_t at, const Vals<kVec>& r) {
  if constexpr (kVec == 1) {
    put<kF32>(base, at, r.v[0]);
  } else if constexpr (kF32) {
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

// ---------------------------------------------------------------- lookup
struct EmbedParams {
  const void* ids;
  const void* table;
  void* out;
  int64_t m, vocab, d, ld;  // ld: values between the table's rows
  bool wide;
  int shift;                // 2^shift threads per row ..
  uint32_t slabs;           // .. and that many workgroups
  float scale;
};
// Vectors of a row per thread at a time: 8 KB written by a workgroup (16381 rows of 4096
// bf16 to fp32, 16 KB by a workgroup 85 us, 8 KB 77; to bf16 8 KB 44, 4 KB 46).
constexpr int ahead(bool out_f32) { return out_f32 ? 1 : 2; }
template <int kVec, bool kF32, bool kOutF32>
__global__ void __launch_bounds__(kThreads) embed_kernel(EmbedParams p) {
  constexpr int kAhead = ahead(kOutF32);
  const int lanes = 1 << p.shift;
  const uint32_t slabs = kVec == 1 ? 1 : p.slabs, group = slabs == 1 ? blockIdx.x : blockIdx.x / slabs, slab = blockIdx.x - group * slabs;
  const int64_t row = (int64_t)group * (kThreads >> p.shift) + (threadIdx.x >> p.shift);
  if (row >= p.m) return;
  const int id = id_of(p.ids, p.wide, row, p.vocab);
  const int64_t from = (int64_t)(id < 0 ? 0 : id) * p.ld, to = row * p.d, step = (int64_t)kAhead * lanes * kVec;
  for (int64_t c = slab * step + (int64_t)(threadIdx.x & (lanes - 1)) * kVec; c < p.d; c += step * slabs) {
    Vals<kVec> v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t at = c + (int64_t)i * lanes * kVec;
      v[i] = id >= 0 && at < p.d ? read<kVec, kF32>(p.table, from + at) : Vals<kVec>{};
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t at = c + (int64_t)i * lanes * kVec;
#pragma unroll
      for (int j = 0; j < kVec; ++j) v[i].v[j] = id >= 0 ? v[i].v[j] * p.scale : 0.0f;
      if (at < p.d) write<kVec, kOutF32>(p.out, to + at, v[i]);
    }
  }
}

// ---------------------------------------------------------------- gradient
// The tokens by (id, t): sorted_id[r] and token[r], those with an id outside the
// table last with sorted_id -1.  First every 1024 tokens by themselves, by a workgroup
// each, while other workgroups clear the table's gradient (which is written once
// more than needed where a token falls, but waits for no order), the rest of which the
// next launch clears: 16381 tokens are sorted long before a gigabyte is cleared.  Then a token's place is its place in its own
// 1024 plus, for each of the others, the number of smaller ids there (or equal ones, if
// they come before it), found by bisection in LDS.
struct SortParams {
  const void* ids;
  int64_t m, vocab;
  bool wide;
  int sorters;
  int *sorted_id, *token;   // what is sorted in the end
  int *part_id, *part_token;  // by 1024
  char* clear;
  int64_t clear_bytes, early;  // early: pieces cleared beside the first launch
  int rankers;
};
// A workgroup clears 16 KB and ends, four pieces of 4 KB that are eight apart: what is
// written at a time is then one narrow window that moves through the table (129280 x
// 4096 bf16: 165 us, 175 by 16 KB in a row; 155 by workgroups of one piece each, which
// the sort's 1024 threads do not allow).
constexpr int64_t kClear = kSortThreads;  // 16-byte words
constexpr int64_t kPiece = 256;
__device__ __forceinline__ void clear_part(char* p, int64_t bytes, int64_t part) {
  typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
  const int64_t to_line = -(intptr_t)p & 15, head = bytes < to_line ? bytes : to_line, words = (bytes - head) / 16;
  if (part == 0) {
    for (int64_t i = threadIdx.x; i < head; i += kSortThreads) p[i] = 0;
    for (int64_t i = head + words * 16 + threadIdx.x; i < bytes; i += kSortThreads) p[i] = 0;
  }
  const int64_t piece = (part / 8 * (kClear / kPiece) + threadIdx.x / kPiece) * 8 + part % 8, i = piece * kPiece + threadIdx.x % kPiece;
  if (i < words) __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, reinterpret_cast<u32x4*>(p + head) + i);
}
__global__ void __launch_bounds__(kSortThreads) embed_sort_kernel(SortParams p) {
  if ((int)blockIdx.x >= p.sorters) {
    clear_part(p.clear, p.clear_bytes, (int64_t)blockIdx.x - p.sorters);
    return;
  }
  __shared__ unsigned long long mem[kSortThreads];
  const int i = threadIdx.x;
  const int64_t t = (int64_t)blockIdx.x * kSortThreads + i;
  const int id = t < p.m ? id_of(p.ids, p.wide, t, p.vocab) : -1;
  // bitonic, on (id, place): no two are the same, so the result is the stable sort's
  unsigned long long key = (unsigned long long)(id < 0 ? kNoId : (uint32_t)id) << 10 | (unsigned)i;
  // (no further than the tokens reach: what is behind them is sorted as it is)
  const int64_t there = p.m - (int64_t)blockIdx.x * kSortThreads;
  for (int size = 2; size <= kSortThreads && size / 2 < there; size *= 2)
    for (int step = size / 2; step > 0; step /= 2) {
      unsigned long long other;
      if (step >= 64) {
        __syncthreads();
        mem[i] = key;
        __syncthreads();
        other = mem[i ^ step];
      } else {
        other = (unsigned long long)__shfl_xor((long long)key, step, 64);
      }
      const bool up = !(i & size), low = !(i & step);
      key = (key < other) == (up == low) ? key : other;
    }
  const uint32_t v = (uint32_t)(key >> 10);
  const int64_t from = (int64_t)blockIdx.x * kSortThreads + (int)(key & 1023);
  if (t < p.m) {  // (places behind the last token sort behind all others)
    const bool one = p.sorters == 1;
    (one ? p.sorted_id : p.part_id)[t] = one && v == kNoId ? -1 : (int)v;
    (one ? p.token : p.part_token)[t] = (int)from;
  }
}

// 64 tokens per workgroup, a wave for each of 16 sorted parts at a time.
__global__ void __launch_bounds__(kSortThreads) embed_rank_kernel(SortParams p) {
  if ((int)blockIdx.x >= p.rankers) {
    clear_part(p.clear, p.clear_bytes, (int64_t)blockIdx.x - p.rankers + p.early);
    return;
  }
  __shared__ int ids[kSortThreads * 16];
  __shared__ int counts[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m = (int)p.m, parts = p.sorters, t = blockIdx.x * 64 + lane, own = t / kSortThreads;
  const int id = t < m ? p.part_id[t] : 0;
  int n = 0;
  for (int p0 = 0; p0 < parts; p0 += 16) {
    __syncthreads();
    for (int i = threadIdx.x; i < kSortThreads * 16; i += kSortThreads) {
      const int at = p0 * kSortThreads + i;
      ids[i] = at < m ? p.part_id[at] : (int)kNoId;
    }
    __syncthreads();
    const int part = p0 + wave;
    if (part < parts && part != own) {
      // the number of ids below id, or not above it in an earlier part
      const int limit = part < own ? id + 1 : id;  // (of kNoId: 2^30 + 1)
      int lo = 0;
#pragma unroll
      for (int step = kSortThreads / 2; step > 0; step /= 2)
        if (ids[wave * kSortThreads + lo + step - 1] < limit) lo += step;
      if (ids[wave * kSortThreads + lo] < limit) ++lo;  // (lo <= 1023 so far)
      const int there = m - part * kSortThreads;
      n += lo < there ? lo : there;
    }
  }
  counts[wave][lane] = n;
  __syncthreads();
  if (wave || t >= m) return;
  n = t % kSortThreads;
#pragma unroll
  for (int w = 0; w < 16; ++w) n += counts[w][lane];
  p.sorted_id[n] = (uint32_t)id == kNoId ? -1 : id;
  p.token[n] = p.part_token[t];
}
__global__ void __launch_bounds__(kSortThreads) embed_clear_kernel(char* p, int64_t bytes) {
  clear_part(p, bytes, blockIdx.x);
}

// More tokens: digits of ten bits, lowest first, each sorted by hsmoe_moe_sort.
// digit_kernel: the digit of what the pass before has put in row r (token r in the
// first pass), -1 where there is none.
__global__ void __launch_bounds__(kThreads) embed_digit_kernel(const void* ids, bool wide, int64_t m, int64_t vocab, const int* order,
                                                               int shift, int64_t* digit) {
  const int64_t r = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (r >= m) return;
  const int64_t t = order ? order[r] : r;
  const int id = t < 0 ? -1 : id_of(ids, wide, t, vocab);
  digit[r] = id < 0 ? -1 : (id >> shift) & 1023;
}
// order <- what this pass puts in row r
__global__ void __launch_bounds__(kThreads) embed_order_kernel(const int* pairs, const int* before, int64_t m, int* order) {
  const int64_t r = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (r >= m) return;
  const int q = pairs[r];
  order[r] = q < 0 ? -1 : before ? before[q] : q;
}
__global__ void __launch_bounds__(kThreads) embed_sorted_kernel(const void* ids, bool wide, int64_t m, int64_t vocab, const int* order,
                                                                int* sorted_id) {
  const int64_t r = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (r < m) sorted_id[r] = order[r] < 0 ? -1 : id_of(ids, wide, order[r], vocab);
}

struct SumParams {
  const void* d_out;
  const int *sorted_id, *token;
  void* d_table;
  float* part;          // fp32 [chunks][2][d]: a chunk's first run, if the chunk before has its beginning, and its last, if it goes on
  int64_t m, d, ld, ld_out;  // ld: values between the table's rows, ld_out: between d_out's
  int64_t chunks;
  int shift, slabs;     // 2^shift threads per chunk, `slabs` times that many vectors cover a row
  bool add;
  float scale;
};
template <int kVec, bool kOutF32>
__device__ __forceinline__ void finish(const SumParams& p, int id, int64_t col, const Vals<kVec>& s) {
  const int64_t at = (int64_t)id * p.ld + col;
  Vals<kVec> v;
  if (p.add) {
    const Vals<kVec> old = read<kVec, kOutF32>(p.d_table, at);
#pragma unroll
    for (int i = 0; i < kVec; ++i) v.v[i] = __fmaf_rn(p.scale, s.v[i], old.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) v.v[i] = p.scale * s.v[i];
  }
  write<kVec, kOutF32>(p.d_table, at, v);
}
template <int kVec>
__device__ __forceinline__ void leave(float* to, const Vals<kVec>& s) {
#pragma unroll
  for (int i = 0; i < kVec; ++i) to[i] = s.v[i];
}

// Sums of the runs of a chunk, for kVec columns per thread.  The chunk's ids and
// tokens are read once; then eight rows are on their way at a time.  Few tokens: kOwn of
// a chunk's rows are for a group of threads by itself, that takes the runs which begin
// there, to their ends (all of it captured: 100 tokens of 4096 22 us by whole chunks, 12.6
// so with a sort no longer than they need; 1000 24 and 20; 4096 30 and 34).
template <int kVec, bool kF32, bool kOutF32, int kOwn>
__global__ void __launch_bounds__(kThreads) embed_sum_kernel(SumParams p) {
  __shared__ int2 mem[kThreads / 8][kChunk + 1];  // (id, token) of the workgroup's chunks, and the id behind each
  __shared__ int before[kThreads / 8];
  constexpr int kParts = kChunk / kOwn;
  const int lanes = 1 << p.shift, per = kThreads >> p.shift, mine = threadIdx.x >> p.shift;
  const int64_t u0 = (int64_t)(blockIdx.x / p.slabs) * per;
  const int64_t chunk = (u0 + mine) / kParts;
  for (int i = threadIdx.x; i < per * (kChunk + 1); i += kThreads) {
    const int64_t r = (u0 + i / (kChunk + 1)) / kParts * kChunk + i % (kChunk + 1);
    mem[i / (kChunk + 1)][i % (kChunk + 1)] = r < p.m ? make_int2(p.sorted_id[r], p.token[r]) : make_int2(-1, 0);
  }
  for (int i = threadIdx.x; i < per; i += kThreads) {
    const int64_t r = (u0 + i) / kParts * kChunk - 1;
    before[i] = r >= 0 && r < p.m ? p.sorted_id[r] : -1;
  }
  __syncthreads();
  const int64_t col = ((int64_t)(blockIdx.x % p.slabs) * lanes + (threadIdx.x & (lanes - 1))) * kVec;
  if (chunk >= p.chunks || col >= p.d) return;
  const int begin = (int)((u0 + mine) % kParts) * kOwn;
  int id = mem[mine][begin].x;
  if (id < 0) return;
  bool open = begin == 0 && before[mine] == id;                            // the run began before the chunk
  bool others = kParts > 1 && begin > 0 && mem[mine][begin - 1].x == id;  // it began in another group's rows
  bool done = false;
  float* part = p.part + chunk * 2 * p.d + col;
  Vals<kVec> s = {};
  constexpr int kAhead = 8;
  for (int r = begin; r < kChunk; r += kAhead) {
    const int now = mem[mine][r].x;
    if (now < 0 || (kParts > 1 && r >= begin + kOwn && (done || others || now != id))) break;
    Raw<kVec, kF32> v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int2 e = mem[mine][r + i];
      v[i] = fetch<kVec, kF32>(p.d_out, (int64_t)(e.x < 0 ? mem[mine][r].y : e.y) * p.ld_out + col);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int next = mem[mine][r + i].x;
      if (next < 0 || (kParts > 1 && done)) continue;
      if (next != id) {  // the run before is done
        if (!(kParts > 1 && others)) {
          if (open) leave<kVec>(part, s);
          else finish<kVec, kOutF32>(p, id, col, s);
        }
        if (kParts > 1 && r + i >= begin + kOwn) {  // the next one is another group's
          done = true;
          continue;
        }
        open = others = false, id = next, s = Vals<kVec>{};
      }
#pragma unroll
      for (int j = 0; j < kVec; ++j) s.v[j] += v[i].at(j);
    }
  }
  if (kParts > 1 && (done || others)) return;
  // the last run: goes on in the next chunk, or ends here
  if (mem[mine][kChunk].x == id) leave<kVec>(part + (open ? 0 : p.d), s);
  else if (open) leave<kVec>(part, s);
  else finish<kVec, kOutF32>(p, id, col, s);
}

// Runs over several chunks: the chunk where one begins adds what the next ones left.
// A workgroup per chunk and 64 vectors of columns; its eight waves take an
// eighth of the run's chunks each (a word that is all of 16384 tokens: 512 of them; one
// wave by itself: 30 us), and are joined in their order.  Lanes look for the run's end 64 chunks at a time.
template <int kVec, bool kOutF32>
__global__ void __launch_bounds__(kJoinThreads) embed_join_kernel(SumParams p) {
  constexpr int kWaves = kJoinThreads / 64;
  __shared__ float mem[kWaves - 1][64 * kVec];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t chunk = blockIdx.x / p.slabs, r0 = chunk * kChunk, r1 = r0 + kChunk;
  const int64_t col = ((int64_t)(blockIdx.x % p.slabs) * 64 + lane) * kVec;
  if (r1 >= p.m) return;
  const int id = p.sorted_id[r1], last = p.sorted_id[r1 - 1], first = p.sorted_id[r0], before = r0 > 0 ? p.sorted_id[r0 - 1] : -1;
  if (id < 0 || last != id) return;         // nothing goes on
  if (first == id && before == id) return;  // it began earlier
  int64_t end = chunk + 1;                  // the first chunk that does not begin with the run
  for (bool on = true; on;) {
    const int64_t c = end + lane;
    const uint64_t other = __ballot(!(c < p.chunks && p.sorted_id[c * kChunk] == id));
    on = other == 0;
    end += on ? 64 : __builtin_ctzll(other);
  }
  const int64_t all = end - chunk, per = (all + kWaves - 1) / kWaves;  // chunk itself left its second sum, the others their first
  const int64_t c0 = chunk + wave * per, c1 = c0 + per < end ? c0 + per : end;
  Vals<kVec> s = {};
  if (col < p.d) {
    auto at = [&](int64_t c) { return (c * 2 + (c == chunk)) * p.d + col; };
    int64_t c = c0;
    constexpr int kAhead = 16;
    for (; c + kAhead <= c1; c += kAhead) {
      Raw<kVec, true> v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) v[i] = fetch<kVec, true>(p.part, at(c + i));
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int j = 0; j < kVec; ++j) s.v[j] += v[i].at(j);
    }
    for (; c < c1; ++c) {
      const Raw<kVec, true> v = fetch<kVec, true>(p.part, at(c));
#pragma unroll
      for (int j = 0; j < kVec; ++j) s.v[j] += v.at(j);
    }
  }
  if (wave > 0)
#pragma unroll
    for (int j = 0; j < kVec; ++j) mem[wave - 1][j * 64 + lane] = s.v[j];
  __syncthreads();
  if (wave > 0 || col >= p.d) return;
#pragma unroll
  for (int w = 0; w < kWaves - 1; ++w)
#pragma unroll
    for (int j = 0; j < kVec; ++j) s.v[j] += mem[w][j * 64 + lane];
  finish<kVec, kOutF32>(p, id, col, s);
}

// ---------------------------------------------------------------- host
int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// Threads per row: a power of two of them that covers d in vectors, up to a workgroup.
int shift_for(int64_t vectors) {
  int s = 0;
  while (s < 8 && (1ll << s) < vectors) ++s;
  return s;
}

struct GradSpace {
  int64_t ids, token, part_id, part_token, order, digit, offsets, pairs, rows, sort, sort_bytes, part, bytes;
};
GradSpace space_of(int64_t m, int64_t d) {
  GradSpace s{};
  const int64_t n = up(m * 4, 256);
  s.ids = 0, s.token = n, s.bytes = 2 * n;
  if (m > kSortThreads && m <= kSortByRank) {
    s.part_id = s.bytes, s.part_token = s.bytes + n, s.bytes += 2 * n;
  } else if (m > kSortByRank) {
    s.order = s.bytes, s.digit = s.order + n, s.offsets = s.digit + 2 * n, s.pairs = s.offsets + up(1025 * 4, 256);
    s.rows = s.pairs + n, s.sort = s.rows + n;
    s.sort_bytes = (int64_t)hsmoe_moe_sort_workspace_size(m, 1, 1024);
    s.bytes = s.sort + up(s.sort_bytes, 256);
  }
  s.part = s.bytes;
  s.bytes += (m + kChunk - 1) / kChunk * 2 * d * 4;
  return s;
}

bool kind_ok(int k) { return k == HSMOE_OUT_F32 || k == HSMOE_OUT_BF16; }
int check_embed(const char* who, const void* ids, int id_kind, int64_t m, int64_t vocab, int64_t d, int64_t ld, int a, int b) {
  if (m < 0 || vocab < 1 || d < 1 || ld < d || !kind_ok(a) || !kind_ok(b) || (id_kind != HSMOE_IDS_I32 && id_kind != HSMOE_IDS_I64))
    return fail(HSMOE_ERR_ARG, "%s: bad arguments", who);
  if (m >= (1ll << 31) || vocab >= (1ll << 30) || d >= (1 << 23) || ld >= (1ll << 31))
    return fail(HSMOE_ERR_SHAPE, "%s: sizes beyond 2^31 tokens, 2^30 rows or 2^23 columns", who);
  if (m > 0 && !ids) return fail(HSMOE_ERR_ARG, "%s: null pointer", who);
  if (!aligned(ids, id_kind == HSMOE_IDS_I64 ? 8 : 4)) return fail(HSMOE_ERR_SHAPE, "%s: misaligned ids", who);
  return HSMOE_OK;
}
int size_of(int kind) { return kind == HSMOE_OUT_F32 ? 4 : 2; }
bool rows16(const void* p, int64_t ld, int kind) { return aligned(p, 16) && ld * size_of(kind) % 16 == 0; }

template <bool kSum, int kVec, bool kF32, bool kOutF32>
void launch_grad(const SumParams& p, hipStream_t st) {
  const bool few = kSum && p.m * p.d <= kFew;
  const int64_t per = kSum ? kThreads >> p.shift : 1, units = few ? p.chunks * (kChunk / kUnit) : p.chunks;
  const dim3 grid((unsigned)((units + per - 1) / per * p.slabs)), block(kSum ? kThreads : kJoinThreads);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, p); };
  if constexpr (kSum) few ? go(embed_sum_kernel<kVec, kF32, kOutF32, kUnit>) : go(embed_sum_kernel<kVec, kF32, kOutF32, kChunk>);
  else go(embed_join_kernel<kVec, kOutF32>);
}
template <bool kSum, int kVec>
void launch_grad(const SumParams& p, bool f32, bool out_f32, hipStream_t st) {
  if (f32 && out_f32) launch_grad<kSum, kVec, true, true>(p, st);
  else if (f32) launch_grad<kSum, kVec, true, false>(p, st);
  else if (out_f32) launch_grad<kSum, kVec, false, true>(p, st);
  else launch_grad<kSum, kVec, false, false>(p, st);
}

}  // namespace
}  // namespace hsmoe

using namespace hsmoe;

extern "C" int hsmoe_embed(const void* ids, int id_kind, int64_t m, const void* table, int64_t table_row_stride,
                           int table_kind, int64_t vocab, int64_t d, float scale, int out_kind, void* out,
                           hsmoe_stream_t stream) {
  const char* who = "hsmoe_embed";
  if (int rc = check_embed(who, ids, id_kind, m, vocab, d, table_row_stride, table_kind, out_kind)) return rc;
  if (m == 0) return HSMOE_OK;
  if (!table || !out) return fail(HSMOE_ERR_ARG, "%s: null pointer", who);
  if (!aligned(table, size_of(table_kind)) || !aligned(out, size_of(out_kind))) return fail(HSMOE_ERR_SHAPE, "%s: misaligned rows", who);
  EmbedParams p{ids, table, out, m, vocab, d, table_row_stride, id_kind == HSMOE_IDS_I64, 0, 1, scale};
  const bool vec = d % 8 == 0 && rows16(table, table_row_stride, table_kind) && rows16(out, d, out_kind);
  const int64_t vectors = vec ? d / 8 : d, each = ahead(out_kind == HSMOE_OUT_F32);
  p.shift = shift_for((vectors + each - 1) / each);
  if (vec) p.slabs = (uint32_t)((vectors + each * kThreads - 1) / (each * kThreads));
  const int64_t per = kThreads >> p.shift, groups = (m + per - 1) / per * p.slabs;
  if (!grid_fits(groups, kThreads)) return fail(HSMOE_ERR_SHAPE, "%s: too many rows of this width for one launch", who);
  const dim3 grid((unsigned)groups), block(kThreads);
  hipStream_t st = (hipStream_t)stream;
  const bool f = table_kind == HSMOE_OUT_F32, o = out_kind == HSMOE_OUT_F32;
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, p); };
  if (vec) f ? (o ? go(embed_kernel<8, true, true>) : go(embed_kernel<8, true, false>))
             : (o ? go(embed_kernel<8, false, true>) : go(embed_kernel<8, false, false>));
  else f ? (o ? go(embed_kernel<1, true, true>) : go(embed_kernel<1, true, false>))
         : (o ? go(embed_kernel<1, false, true>) : go(embed_kernel<1, false, false>));
  return check_launch(who);
}

extern "C" size_t hsmoe_embed_grad_workspace_size(int64_t m, int64_t d) {
  return m < 1 || d < 1 ? 0 : (size_t)space_of(m, d).bytes;
}

extern "C" int hsmoe_embed_grad(const void* d_out, int64_t d_row_stride, int d_kind, const void* ids, int id_kind,
                                int64_t m, int64_t vocab, int64_t d, float scale, int add, void* d_table,
                                int64_t table_row_stride, int table_kind, void* workspace, size_t workspace_bytes,
                                hsmoe_stream_t stream) {
  const char* who = "hsmoe_embed_grad";
  if (int rc = check_embed(who, ids, id_kind, m, vocab, d, table_row_stride, table_kind, d_kind)) return rc;
  if (m >= (1 << 24)) return fail(HSMOE_ERR_SHAPE, "%s: 2^24 tokens and more", who);
  if (!d_table || (m > 0 && (!d_out || d_row_stride < d)) || (add != 0 && add != 1) || (!add && table_row_stride != d))
    return fail(HSMOE_ERR_ARG, "%s: bad arguments", who);
  if (!aligned(d_table, size_of(table_kind)) || !aligned(d_out, size_of(d_kind))) return fail(HSMOE_ERR_SHAPE, "%s: misaligned rows", who);
  const GradSpace sp = m > 0 ? space_of(m, d) : GradSpace{};
  if (m > 0 && (!workspace || workspace_bytes < (size_t)sp.bytes))
    return fail(HSMOE_ERR_WORKSPACE, "%s: workspace of %lld bytes needed", who, (long long)sp.bytes);
  if (!aligned(workspace, 16)) return fail(HSMOE_ERR_SHAPE, "%s: misaligned workspace", who);
  hipStream_t st = (hipStream_t)stream;
  char* mem = (char*)workspace;
  const bool wide = id_kind == HSMOE_IDS_I64;
  int *sorted_id = (int*)(mem + sp.ids), *token = (int*)(mem + sp.token);
  const int64_t bytes = add ? 0 : vocab * d * size_of(table_kind);
  const int64_t clears = (bytes + 8 * kClear * 16 - 1) / (8 * kClear * 16) * 8;  // (eight share out their pieces)
  SumParams p{};
  p.m = m, p.d = d, p.ld = table_row_stride, p.ld_out = d_row_stride, p.chunks = (m + kChunk - 1) / kChunk;
  p.add = add, p.scale = scale;
  const bool vec = d % 8 == 0 && rows16(d_out, d_row_stride, d_kind) && rows16(d_table, table_row_stride, table_kind);
  const int64_t vectors = vec ? d / 8 : d, join_slabs = (vectors + 63) / 64;
  p.shift = std::max(shift_for(vectors), 3);
  p.slabs = (int)((vectors + (1ll << p.shift) - 1) >> p.shift);
  // (all launches or none: those behind one that fails would take its places from what lies in the workspace)
  if (!grid_fits(clears + kSortByRank / 64, kSortThreads) || !grid_fits(p.chunks * p.slabs, kThreads) ||
      !grid_fits(p.chunks * join_slabs, kJoinThreads))
    return fail(HSMOE_ERR_SHAPE, "%s: a gradient of 64 GiB, or too many tokens of this width, for one launch", who);
  if (m == 0) {
    if (!clears) return HSMOE_OK;
    hipLaunchKernelGGL(embed_clear_kernel, dim3((unsigned)clears), dim3(kSortThreads), 0, st, (char*)d_table, bytes);
    return check_launch(who);
  }
  if (m <= kSortByRank) {
    SortParams s{ids, m, vocab, wide, (int)((m + kSortThreads - 1) / kSortThreads), sorted_id, token, (int*)(mem + sp.part_id),
                 (int*)(mem + sp.part_token), (char*)d_table, bytes, clears, (int)((m + 63) / 64)};
    if (s.sorters > 1) s.early = clears * 5 / 8;
    hipLaunchKernelGGL(embed_sort_kernel, dim3((unsigned)(s.sorters + s.early)), dim3(kSortThreads), 0, st, s);
    if (s.sorters > 1)
      hipLaunchKernelGGL(embed_rank_kernel, dim3((unsigned)(s.rankers + clears - s.early)), dim3(kSortThreads), 0, st, s);
  } else {
    if (clears) hipLaunchKernelGGL(embed_clear_kernel, dim3((unsigned)clears), dim3(kSortThreads), 0, st, (char*)d_table, bytes);
    const dim3 grid((unsigned)((m + kThreads - 1) / kThreads)), block(kThreads);
    int *order = (int*)(mem + sp.order), *pairs = (int*)(mem + sp.pairs);
    int64_t* digit = (int64_t*)(mem + sp.digit);
    const int* before = nullptr;
    int* after = token;  // passes write token and order in turn
    for (int shift = 0; shift == 0 || (vocab - 1) >> shift; shift += 10) {
      hipLaunchKernelGGL(embed_digit_kernel, grid, block, 0, st, ids, wide, m, vocab, before, shift, digit);
      if (int rc = hsmoe_moe_sort(digit, m, 1, 1024, (int32_t*)(mem + sp.offsets), pairs, (int32_t*)(mem + sp.rows), mem + sp.sort,
                                  (size_t)sp.sort_bytes, stream))
        return rc;
      hipLaunchKernelGGL(embed_order_kernel, grid, block, 0, st, pairs, before, m, after);
      before = after;
      after = after == token ? order : token;
    }
    hipLaunchKernelGGL(embed_sorted_kernel, grid, block, 0, st, ids, wide, m, vocab, before, sorted_id);
    token = const_cast<int*>(before);
  }
  p.d_out = d_out, p.sorted_id = sorted_id, p.token = token, p.d_table = d_table, p.part = (float*)(mem + sp.part);
  const bool f = d_kind == HSMOE_OUT_F32, o = table_kind == HSMOE_OUT_F32;
  if (vec) launch_grad<true, 8>(p, f, o, st);
  else launch_grad<true, 1>(p, f, o, st);
  if (p.chunks > 1) {
    p.slabs = (int)join_slabs;
    if (vec) launch_grad<false, 8>(p, f, o, st);
    else launch_grad<false, 1>(p, f, o, st);
  }
  return check_launch(who);
}

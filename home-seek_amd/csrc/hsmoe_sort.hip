// (token, slot) pairs sorted by expert, token rows copied to that order, and
// the way back: a token's rows summed with its weights, with the gradient of
// both.  Pair q = t * top_k + j is token t's slot j; its row r is its place
// among the pairs of valid ids, ordered by (expert, q).  All of it moves bytes:
// the bound is HBM, and latency where there are few tokens.
#include "hsmoe_common.h"
#include "hsmoe_internal.h"

namespace hsmoe {
namespace {

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kSortMaxExperts = 1024;  // = kSortThreads: one thread per expert in the scans
constexpr int kSortMaxBlocks = 256;

// Pairs per workgroup: 1024 while that gives at most 256 workgroups (each reads
// every workgroup's histogram), multiples of 1024 beyond.
int64_t sort_chunk(int64_t pairs) {
  const int64_t per = (pairs + kSortMaxBlocks - 1) / kSortMaxBlocks;
  return (per + kSortThreads - 1) / kSortThreads * kSortThreads;
}

// The expert of pair q, n_experts if its id is none.
__device__ __forceinline__ int pair_expert(const int64_t* idx, int64_t q, int n_experts) {
  const int64_t e = idx[q];
  return e >= 0 && e < n_experts ? (int)e : n_experts;
}

// Counts pairs [from, to) into rows 0-7 of cnt (those before `split`) or 8-15
// (integers: the order of the LDS atomics does not show), sixteen ids per thread
// on their way at a time.  Lane l counts in its row l % 8: a popular expert would
// have the lanes of a wave add to one word in turn.
constexpr int kCopies = kSortWaves / 2;
__device__ __forceinline__ void count_pairs(const int64_t* idx, int64_t from, int64_t split, int64_t to, int n_experts,
                                            int (&cnt)[kSortWaves][kSortMaxExperts]) {
  const int copy = threadIdx.x & (kCopies - 1);
  constexpr int kAhead = 16;
  for (int64_t q = from + threadIdx.x; q < to; q += kAhead * kSortThreads) {
    int e[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      e[i] = q + i * kSortThreads < to ? pair_expert(idx, q + i * kSortThreads, n_experts) : n_experts;
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (e[i] < n_experts) atomicAdd(&cnt[copy + (q + i * kSortThreads < split ? 0 : kCopies)][e[i]], 1);
  }
}

__device__ __forceinline__ void clear_counts(int n_experts, int (&cnt)[kSortWaves][kSortMaxExperts]) {
  for (int c = threadIdx.x & 63; c < n_experts; c += 64) cnt[threadIdx.x >> 6][c] = 0;
}
// Thread e: the pairs of expert e before and from `split` on (0 for other threads).
__device__ __forceinline__ void sum_counts(int n_experts, const int (&cnt)[kSortWaves][kSortMaxExperts], int& before,
                                           int& after) {
  before = after = 0;
  if ((int)threadIdx.x >= n_experts) return;
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    before += cnt[i][threadIdx.x];
    after += cnt[kCopies + i][threadIdx.x];
  }
}

// Histogram of a chunk's experts.
__global__ void __launch_bounds__(kSortThreads)
    sort_hist_kernel(const int64_t* __restrict__ idx, int64_t pairs, int n_experts, int64_t chunk,
                     int* __restrict__ hist) {
  __shared__ int cnt[kSortWaves][kSortMaxExperts];
  const int64_t q0 = blockIdx.x * chunk;
  clear_counts(n_experts, cnt);
  __syncthreads();
  count_pairs(idx, q0, q0, min(pairs, q0 + chunk), n_experts, cnt);
  __syncthreads();
  int before, after;
  sum_counts(n_experts, cnt, before, after);
  if ((int)threadIdx.x < n_experts) hist[(int64_t)blockIdx.x * n_experts + threadIdx.x] = after;
}

// Inclusive sum over the workgroup's threads of one value each.
__device__ __forceinline__ int block_scan(int v, int* s_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(v, off, 64);
    if (lane >= off) v += o;
  }
  if (lane == 63) s_wave[wave] = v;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) before += w < wave ? s_wave[w] : 0;
  return v + before;
}

// Places a chunk's pairs.  Thread e holds the next free row of expert e: the
// experts before it (a scan of the totals) and the earlier chunks' pairs of e.
// 1024 pairs at a time: a pair's rank within its wave is the number of lower
// lanes with its expert, found with one ballot per bit of the id; the waves'
// counts are then summed in wave order, so pairs of one expert keep their
// order and the result is the stable sort.
// hist == NULL: every workgroup counts all pairs for itself, which saves the
// launch that counts and its gap where there are few (kSortAlone).
__global__ void __launch_bounds__(kSortThreads)
    sort_place_kernel(const int64_t* __restrict__ idx, int64_t pairs, int n_experts, int64_t chunk,
                      const int* __restrict__ hist, int* __restrict__ offsets, int* __restrict__ pair_of,
                      int* __restrict__ row_of) {
  __shared__ int cnt[kSortWaves][kSortMaxExperts];  // pairs per wave and expert, then their first rows
  __shared__ int s_wave[kSortWaves];
  __shared__ int s_total;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t q0 = blockIdx.x * chunk, q1 = min(pairs, q0 + chunk);
  int total = 0, before = 0;  // pairs of expert tid: all, and those of earlier chunks
  int e = q0 + tid < q1 ? pair_expert(idx, q0 + tid, n_experts) : n_experts;  // of the first 1024 pairs
  if (hist) {
    if (tid < n_experts) {
      const int* h = hist + tid;
#pragma unroll 8
      for (int b = 0; b < (int)gridDim.x; ++b) {
        const int c = h[(int64_t)b * n_experts];
        before += b < (int)blockIdx.x ? c : 0;
        total += c;
      }
    }
  } else {
    clear_counts(n_experts, cnt);
    __syncthreads();
    count_pairs(idx, 0, q0, pairs, n_experts, cnt);
    __syncthreads();
    sum_counts(n_experts, cnt, before, total);
    total += before;
  }
  const int upto = block_scan(total, s_wave);
  int next = upto - total + before;
  if (tid == kSortThreads - 1) s_total = upto;
  if (blockIdx.x == 0) {
    if (tid < n_experts) offsets[tid + 1] = upto;
    if (tid == 0) offsets[0] = 0;
  }
  __syncthreads();
  for (int64_t q = max(q0, (int64_t)s_total) + tid; q < q1; q += kSortThreads) pair_of[q] = -1;  // rows behind the last
  const int bits = 32 - __clz(n_experts);
  for (int64_t base = q0; base < q1; base += kSortThreads) {
    const int64_t q = base + tid;
    if (base > q0) e = q < q1 ? pair_expert(idx, q, n_experts) : n_experts;
    clear_counts(n_experts, cnt);  // each wave its own row
    uint64_t same = ~0ull;
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((e >> b) & 1);
      same &= ((e >> b) & 1) ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    if (e < n_experts && rank == 0) cnt[wave][e] = __popcll(same);
    __syncthreads();
    if (tid < n_experts) {
      int c[kSortWaves];
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) c[w] = cnt[w][tid];
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) {
        cnt[w][tid] = next;
        next += c[w];
      }
    }
    __syncthreads();
    if (q < q1) {
      int row = -1;
      if (e < n_experts) {
        row = cnt[wave][e] + rank;
        pair_of[row] = (int)q;
      }
      row_of[q] = row;
    }
    if (base + kSortThreads < q1) __syncthreads();  // (which would wait for the stores)
  }
}

// ---------------------------------------------------------------- rows
// Rows are moved in vectors of T (16 bytes where every row is 16-byte aligned,
// else one element).
constexpr int kRowThreads = 256;

// A row number out of an order that a caller may have made: -1 unless it is one.
__device__ __forceinline__ int64_t checked_row(int r, int64_t n_rows) { return r >= 0 && r < n_rows ? r : -1; }

// One workgroup per token and 512 vectors of its row: the row is read once and
// written to the token's up to top_k rows (written once each: reading per sorted
// row instead would read every token top_k times).  The workgroup of token t
// also clears those of rows t * top_k ... that lie behind the last sorted one.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
    gather_kernel(const T* __restrict__ x, int64_t x_stride, int64_t n_vec, const int* __restrict__ row_of, int top_k,
                  const int* __restrict__ last, int64_t n_rows, T* __restrict__ out) {
  const int64_t t = blockIdx.x;
  const int64_t c0 = (int64_t)blockIdx.y * 2 * kRowThreads + threadIdx.x, c1 = c0 + kRowThreads;
  const T* src = x + t * x_stride;
  T a{}, b{};
  if (c0 < n_vec) a = src[c0];
  if (c1 < n_vec) b = src[c1];
  const int end = *last;
  for (int j = 0; j < top_k; ++j) {
    const int64_t q = t * top_k + j, r = checked_row(row_of[q], n_rows);
    if (r >= 0) {
      if (c0 < n_vec) out[r * n_vec + c0] = a;
      if (c1 < n_vec) out[r * n_vec + c1] = b;
    }
    if (q >= end) {
      if (c0 < n_vec) out[q * n_vec + c0] = T{};
      if (c1 < n_vec) out[q * n_vec + c1] = T{};
    }
  }
}

// kN consecutive values of a row as fp32, and back with one rounding.
template <typename S, int kN>
struct Vals {
  float v[kN];
};
template <typename S, int kN>
__device__ __forceinline__ Vals<S, kN> load_vals(const S* p);
template <>
__device__ __forceinline__ Vals<uint16_t, 8> load_vals<uint16_t, 8>(const uint16_t* p) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  Vals<uint16_t, 8> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r.v[2 * i] = bf16_bits_to_f32(w[i] & 0xffffu);
    r.v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  return r;
}
template <>
__device__ __forceinline__ Vals<float, 8> load_vals<float, 8>(const float* p) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
template <>
__device__ __forceinline__ Vals<uint16_t, 1> load_vals<uint16_t, 1>(const uint16_t* p) {
  return {{bf16_bits_to_f32(*p)}};
}
template <>
__device__ __forceinline__ Vals<float, 1> load_vals<float, 1>(const float* p) {
  return {{*p}};
}
__device__ __forceinline__ void store_vals(uint16_t* p, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = f32_to_bf16_bits(v[2 * i]) | f32_to_bf16_bits(v[2 * i + 1]) << 16;
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store_vals(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store_vals(uint16_t* p, const float (&v)[1]) { *p = (uint16_t)f32_to_bf16_bits(v[0]); }
__device__ __forceinline__ void store_vals(float* p, const float (&v)[1]) { *p = v[0]; }

// out[t] = sum_j w[t, j] rows[row_of[t, j]] (+ residual[t]), in slot order, in
// fp32.  A thread has kN columns and issues the loads of up to kK slots before
// it uses the first.
template <typename S, typename O, int kN, int kK>
__global__ void __launch_bounds__(kRowThreads)
    combine_kernel(const S* __restrict__ rows, int64_t n_rows, int64_t d, const int* __restrict__ row_of,
                   const float* __restrict__ w, int top_k, const O* __restrict__ residual, O* __restrict__ out) {
  const int64_t t = blockIdx.x;
  const int64_t col = ((int64_t)blockIdx.y * kRowThreads + threadIdx.x) * kN;
  if (col >= d) return;
  float acc[kN] = {};
  Vals<O, kN> res;
  if (residual) res = load_vals<O, kN>(residual + t * d + col);
  for (int j0 = 0; j0 < top_k; j0 += kK) {
    Vals<S, kN> v[kK];
    int64_t r[kK];
    float wj[kK];
#pragma unroll
    for (int j = 0; j < kK; ++j) {
      r[j] = j0 + j < top_k ? checked_row(row_of[t * top_k + j0 + j], n_rows) : -1;
      wj[j] = w && j0 + j < top_k ? w[t * top_k + j0 + j] : 1.0f;
      if (r[j] >= 0) v[j] = load_vals<S, kN>(rows + r[j] * d + col);
    }
#pragma unroll
    for (int j = 0; j < kK; ++j) {
      if (r[j] >= 0) {
#pragma unroll
        for (int i = 0; i < kN; ++i) acc[i] = __builtin_fmaf(wj[j], v[j].v[i], acc[i]);
      }
    }
  }
  if (residual) {
#pragma unroll
    for (int i = 0; i < kN; ++i) acc[i] += res.v[i];
  }
  store_vals(out + t * d + col, acc);
}

// d_rows[row_of[t, j]] = w[t, j] d_out[t] and d_w[t, j] = <d_out[t], rows[row_of[t, j]]>:
// one workgroup per token, so that d_out[t] is read once and the dots need no
// second pass; slots in groups of kK (their partial dots stay in registers).
// Rows behind the last sorted one are cleared as in gather_kernel.
template <typename S, typename O, int kN, int kK>
__global__ void __launch_bounds__(kRowThreads)
    combine_grad_kernel(const O* __restrict__ d_out, const S* __restrict__ rows, int64_t n_rows, int64_t d,
                        const int* __restrict__ row_of, const float* __restrict__ w, int top_k,
                        const int* __restrict__ last, S* __restrict__ d_rows, float* __restrict__ d_w) {
  __shared__ float s_dot[kRowThreads / 64][kK];
  const int64_t t = blockIdx.x;
  const int end = *last;
  const float zero[kN] = {};
  for (int j0 = 0; j0 < top_k; j0 += kK) {
    int64_t r[kK];
    float wj[kK], dot[kK] = {};
#pragma unroll
    for (int j = 0; j < kK; ++j) {
      r[j] = j0 + j < top_k ? checked_row(row_of[t * top_k + j0 + j], n_rows) : -1;
      wj[j] = w && j0 + j < top_k ? w[t * top_k + j0 + j] : 1.0f;
    }
    for (int64_t col = (int64_t)threadIdx.x * kN; col < d; col += kRowThreads * kN) {
      Vals<S, kN> v[kK];
      const Vals<O, kN> g = load_vals<O, kN>(d_out + t * d + col);
      if (d_w) {
#pragma unroll
        for (int j = 0; j < kK; ++j)
          if (r[j] >= 0) v[j] = load_vals<S, kN>(rows + r[j] * d + col);
      }
#pragma unroll
      for (int j = 0; j < kK; ++j) {
        if (r[j] >= 0) {
          float o[kN];
#pragma unroll
          for (int i = 0; i < kN; ++i) o[i] = wj[j] * g.v[i];
          if (d_rows) store_vals(d_rows + r[j] * d + col, o);
          if (d_w) {
#pragma unroll
            for (int i = 0; i < kN; ++i) dot[j] = __builtin_fmaf(g.v[i], v[j].v[i], dot[j]);
          }
        }
        const int64_t q = t * top_k + j0 + j;
        if (d_rows && j0 + j < top_k && q >= end) store_vals(d_rows + q * d + col, zero);
      }
    }
    if (!d_w) continue;
#pragma unroll
    for (int j = 0; j < kK; ++j) {
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) dot[j] += __shfl_xor(dot[j], off, 64);
      if ((threadIdx.x & 63) == 0) s_dot[threadIdx.x >> 6][j] = dot[j];
    }
    __syncthreads();
    if ((int)threadIdx.x < kK && j0 + (int)threadIdx.x < top_k) {
      float s = 0.0f;
#pragma unroll
      for (int v = 0; v < kRowThreads / 64; ++v) s += s_dot[v][threadIdx.x];
      d_w[t * top_k + j0 + threadIdx.x] = s;  // 0 for a slot without a row
    }
    __syncthreads();
  }
}

bool rows_aligned(const void* p, int64_t row_bytes) { return !p || (aligned(p, 16) && row_bytes % 16 == 0); }

int check_rows(const char* what, int64_t m, int top_k, int64_t d) {
  if (m < 0 || top_k < 1 || d < 1) return fail(HSMOE_ERR_ARG, "%s: bad counts", what);
  if (top_k > 16) return fail(HSMOE_ERR_SHAPE, "%s: top_k must be at most 16", what);
  // a launch's threads in one dimension stay below 2^32 (256 per token), its workgroups below 2^16 (256 columns each)
  if (m >= (1 << 24)) return fail(HSMOE_ERR_SHAPE, "%s: m must be below 2^24", what);
  if (d > (1 << 23)) return fail(HSMOE_ERR_SHAPE, "%s: rows of at most 2^23 values", what);
  return HSMOE_OK;
}

template <typename S, typename O, int kN>
void launch_combine(const void* rows, int64_t n_rows, int64_t d, const int* row_of, const float* w, int top_k,
                    const void* residual, void* out, int64_t m, hipStream_t st) {
  const dim3 grid((unsigned)m, (unsigned)((d + kRowThreads * kN - 1) / (kRowThreads * kN)));
  hipLaunchKernelGGL((combine_kernel<S, O, kN, 8>), grid, dim3(kRowThreads), 0, st, (const S*)rows, n_rows, d, row_of, w,
                     top_k, (const O*)residual, (O*)out);
}

template <typename S, typename O, int kN>
void launch_combine_grad(const void* d_out, const void* rows, int64_t n_rows, int64_t d, const int* row_of,
                         const float* w, int top_k, const int* last, void* d_rows, float* d_w, int64_t m,
                         hipStream_t st) {
  hipLaunchKernelGGL((combine_grad_kernel<S, O, kN, 8>), dim3((unsigned)m), dim3(kRowThreads), 0, st, (const O*)d_out,
                     (const S*)rows, n_rows, d, row_of, w, top_k, last, (S*)d_rows, d_w);
}

}  // namespace
}  // namespace hsmoe

using namespace hsmoe;

// Up to this many pairs every workgroup counts them all, and there is one launch.
// Sort and gather (rows of 4096 bf16, 256 experts), one launch / two: 6144 pairs
// 17.4 / 18.9 us, 12288 27.5 / 27.1, 16384 36.4 / 34.3, 24576 51.8 / 47.2.
static constexpr int64_t kSortAlone = 12288;

extern "C" size_t hsmoe_moe_sort_workspace_size(int64_t m, int top_k, int64_t n_experts) {
  if (m < 1 || top_k < 1 || n_experts < 1 || m >= (1 << 24) || top_k > 16) return 0;
  const int64_t pairs = m * top_k;
  if (pairs <= kSortAlone) return 0;
  const int64_t chunk = sort_chunk(pairs);
  return (size_t)((pairs + chunk - 1) / chunk * n_experts * 4);
}

extern "C" int hsmoe_moe_sort(const int64_t* topk_idx, int64_t m, int top_k, int64_t n_experts, int32_t* offsets,
                              int32_t* pair_of_row, int32_t* row_of_pair, void* workspace, size_t workspace_bytes,
                              hsmoe_stream_t stream) {
  if (int rc = check_rows("hsmoe_moe_sort", m, top_k, 1)) return rc;
  if (n_experts < 1 || n_experts > kSortMaxExperts)
    return fail(HSMOE_ERR_SHAPE, "hsmoe_moe_sort: 1 to %d experts", kSortMaxExperts);
  if (!offsets || (m > 0 && (!topk_idx || !pair_of_row || !row_of_pair)))
    return fail(HSMOE_ERR_ARG, "hsmoe_moe_sort: null pointer");
  if ((topk_idx && !aligned(topk_idx, 8)) || !aligned(offsets, 4) || (pair_of_row && !aligned(pair_of_row, 4)) ||
      (row_of_pair && !aligned(row_of_pair, 4)))
    return fail(HSMOE_ERR_SHAPE, "hsmoe_moe_sort: misaligned pointer");
  const int64_t pairs = m * top_k;
  const size_t need = hsmoe_moe_sort_workspace_size(m, top_k, n_experts);
  if (need && (!workspace || workspace_bytes < need))
    return fail(HSMOE_ERR_WORKSPACE, "hsmoe_moe_sort: workspace of %zu bytes needed", need);
  hipStream_t st = (hipStream_t)stream;
  const int64_t chunk = pairs > 0 ? sort_chunk(pairs) : 1, blocks = pairs > 0 ? (pairs + chunk - 1) / chunk : 1;
  if (need) {
    hipLaunchKernelGGL(sort_hist_kernel, dim3((unsigned)blocks), dim3(kSortThreads), 0, st, topk_idx, pairs,
                       (int)n_experts, chunk, (int*)workspace);
  }
  hipLaunchKernelGGL(sort_place_kernel, dim3((unsigned)blocks), dim3(kSortThreads), 0, st, topk_idx, pairs,
                     (int)n_experts, chunk, need ? (const int*)workspace : nullptr, offsets, pair_of_row, row_of_pair);
  return check_launch("hsmoe_moe_sort");
}

extern "C" int hsmoe_moe_gather(const void* x, int64_t x_row_stride, int64_t m, int64_t d, int row_kind,
                                const int32_t* offsets, int64_t n_experts, const int32_t* row_of_pair, int top_k,
                                void* rows_out, hsmoe_stream_t stream) {
  if (int rc = check_rows("hsmoe_moe_gather", m, top_k, d)) return rc;
  if (row_kind != HSMOE_OUT_F32 && row_kind != HSMOE_OUT_BF16)
    return fail(HSMOE_ERR_ARG, "hsmoe_moe_gather: bad row kind %d", row_kind);
  if (n_experts < 1 || x_row_stride < d) return fail(HSMOE_ERR_ARG, "hsmoe_moe_gather: bad counts");
  if (m == 0) return HSMOE_OK;
  if (!x || !offsets || !row_of_pair || !rows_out) return fail(HSMOE_ERR_ARG, "hsmoe_moe_gather: null pointer");
  const int64_t s = row_kind == HSMOE_OUT_F32 ? 4 : 2;
  const bool wide = rows_aligned(x, d * s) && rows_aligned(rows_out, d * s) && x_row_stride * s % 16 == 0;
  if (!aligned(x, s) || !aligned(rows_out, s)) return fail(HSMOE_ERR_SHAPE, "hsmoe_moe_gather: misaligned rows");
  const int64_t n_vec = wide ? d * s / 16 : d, stride = wide ? x_row_stride * s / 16 : x_row_stride;
  const dim3 grid((unsigned)m, (unsigned)((n_vec + 2 * kRowThreads - 1) / (2 * kRowThreads)));
  hipStream_t st = (hipStream_t)stream;
  const int* last = offsets + n_experts;
  const int64_t n_rows = m * top_k;
  if (wide)
    hipLaunchKernelGGL(gather_kernel<uint4>, grid, dim3(kRowThreads), 0, st, (const uint4*)x, stride, n_vec, row_of_pair,
                       top_k, last, n_rows, (uint4*)rows_out);
  else if (s == 4)
    hipLaunchKernelGGL(gather_kernel<uint32_t>, grid, dim3(kRowThreads), 0, st, (const uint32_t*)x, stride, n_vec,
                       row_of_pair, top_k, last, n_rows, (uint32_t*)rows_out);
  else
    hipLaunchKernelGGL(gather_kernel<uint16_t>, grid, dim3(kRowThreads), 0, st, (const uint16_t*)x, stride, n_vec,
                       row_of_pair, top_k, last, n_rows, (uint16_t*)rows_out);
  return check_launch("hsmoe_moe_gather");
}

// Calls launch<S, O, kN> for the row type, the output type and the vector width.
#define HSMOE_ROW_TYPES(launch, row_kind, out_kind, wide, ...)                       \
  do {                                                                               \
    if (row_kind == HSMOE_OUT_BF16 && out_kind == HSMOE_OUT_BF16) {                  \
      if (wide) launch<uint16_t, uint16_t, 8>(__VA_ARGS__);                          \
      else launch<uint16_t, uint16_t, 1>(__VA_ARGS__);                               \
    } else if (row_kind == HSMOE_OUT_BF16) {                                         \
      if (wide) launch<uint16_t, float, 8>(__VA_ARGS__);                             \
      else launch<uint16_t, float, 1>(__VA_ARGS__);                                  \
    } else if (out_kind == HSMOE_OUT_BF16) {                                         \
      if (wide) launch<float, uint16_t, 8>(__VA_ARGS__);                             \
      else launch<float, uint16_t, 1>(__VA_ARGS__);                                  \
    } else {                                                                         \
      if (wide) launch<float, float, 8>(__VA_ARGS__);                                \
      else launch<float, float, 1>(__VA_ARGS__);                                     \
    }                                                                                \
  } while (0)

static bool bad_kind(int kind) { return kind != HSMOE_OUT_F32 && kind != HSMOE_OUT_BF16; }

extern "C" int hsmoe_moe_combine(const void* rows, int row_kind, int64_t n_rows, int64_t m, int64_t d,
                                 const int32_t* row_of_pair, const float* topk_w, int top_k, const void* residual,
                                 int out_kind, void* out, hsmoe_stream_t stream) {
  if (int rc = check_rows("hsmoe_moe_combine", m, top_k, d)) return rc;
  if (bad_kind(row_kind) || bad_kind(out_kind)) return fail(HSMOE_ERR_ARG, "hsmoe_moe_combine: bad row or output kind");
  if (m == 0) return HSMOE_OK;
  if (n_rows < 0 || (n_rows > 0 && !rows) || !row_of_pair || !out)
    return fail(HSMOE_ERR_ARG, "hsmoe_moe_combine: null pointer");
  const int64_t rb = row_kind == HSMOE_OUT_F32 ? 4 : 2, ob = out_kind == HSMOE_OUT_F32 ? 4 : 2;
  if (!aligned(rows, rb) || !aligned(out, ob) || (residual && !aligned(residual, ob)))
    return fail(HSMOE_ERR_SHAPE, "hsmoe_moe_combine: misaligned rows");
  const bool wide = d % 8 == 0 && rows_aligned(rows, d * rb) && rows_aligned(out, d * ob) && rows_aligned(residual, d * ob);
  HSMOE_ROW_TYPES(launch_combine, row_kind, out_kind, wide, rows, n_rows, d, row_of_pair, topk_w, top_k, residual, out, m,
                  (hipStream_t)stream);
  return check_launch("hsmoe_moe_combine");
}

extern "C" int hsmoe_moe_combine_grad(const void* d_out, int out_kind, const void* rows, int row_kind, int64_t m,
                                      int64_t d, const int32_t* offsets, int64_t n_experts,
                                      const int32_t* row_of_pair, const float* topk_w, int top_k, void* d_rows,
                                      float* d_w, hsmoe_stream_t stream) {
  if (int rc = check_rows("hsmoe_moe_combine_grad", m, top_k, d)) return rc;
  if (bad_kind(row_kind) || bad_kind(out_kind))
    return fail(HSMOE_ERR_ARG, "hsmoe_moe_combine_grad: bad row or output kind");
  if (n_experts < 1) return fail(HSMOE_ERR_ARG, "hsmoe_moe_combine_grad: bad counts");
  if (m == 0 || (!d_rows && !d_w)) return HSMOE_OK;
  if (!d_out || !offsets || !row_of_pair || (d_w && !rows))
    return fail(HSMOE_ERR_ARG, "hsmoe_moe_combine_grad: null pointer");
  const int64_t rb = row_kind == HSMOE_OUT_F32 ? 4 : 2, ob = out_kind == HSMOE_OUT_F32 ? 4 : 2;
  if (!aligned(d_out, ob) || (rows && !aligned(rows, rb)) || (d_rows && !aligned(d_rows, rb)))
    return fail(HSMOE_ERR_SHAPE, "hsmoe_moe_combine_grad: misaligned rows");
  const bool wide =
      d % 8 == 0 && rows_aligned(rows, d * rb) && rows_aligned(d_rows, d * rb) && rows_aligned(d_out, d * ob);
  HSMOE_ROW_TYPES(launch_combine_grad, row_kind, out_kind, wide, d_out, rows, m * top_k, d, row_of_pair, topk_w, top_k,
                  offsets + n_experts, d_rows, d_w, m, (hipStream_t)stream);
  return check_launch("hsmoe_moe_combine_grad");
}

// What the tiled matrix products share (hsmoe_linear.hip, hsmoe_fp4.hip): loads
// from global memory to LDS, and the order in which the workgroups take tiles.
#pragma once
#include "hsmoe_common.h"

namespace hsmoe {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kFar = 0x7ffffff0u;      // an offset that no resource reaches: reads as zero

__device__ __forceinline__ int64_t imin64(int64_t a, int64_t b) { return a < b ? a : b; }

// kFar where step i is not below `left`, else 0.
__device__ __forceinline__ uint32_t past(int i, int left) { return (uint32_t)((left - 1 - i) >> 31) & kFar; }

// Values that are the same in every lane, in scalar registers.
__device__ __forceinline__ int64_t uniform64(int64_t v) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// 16 bytes per lane from global memory to LDS, lane l's to dst + 16 l.  Written
// out because the compiler waits for every such load it knows of before reads of
// LDS, whatever they read (each ds_read_b64_tr_b16 of the bf16 tiles); the waits are
// the kernels' own.  No register
// is written: the load takes its address when it is issued.  (s_nop 4: a vector
// instruction may have written the resource's scalar registers, v_readfirstlane
// for one; a memory instruction may read them five wait states later.)
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void lds_load16(i32x4 r, uint32_t off, const char* dst) {
  const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)dst;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(at), "v"(off), "s"(r)
               : "memory", "m0");
}
// A resource over `bytes` bytes from base on (both the same in every lane), as make_buf's.
__device__ __forceinline__ i32x4 lds_buf(const char* base, uint32_t bytes) {
  const uint64_t b = (uint64_t)base;
  return i32x4{__builtin_amdgcn_readfirstlane((int)b), __builtin_amdgcn_readfirstlane((int)(b >> 32) & 0xffff),
               __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}

// The workgroup's place among row_tiles x col_tiles.  Tiles are numbered so that
// four row tiles go through the column tiles together; workgroup b runs on XCD
// b % 8, and the XCDs take the numbers in chunks of up to 32, one tile for each
// of an XCD's CUs: its L2 serves a row tile to eight column tiles and a column
// tile to four row tiles, and experts of unequal size are spread over all XCDs
// (an eighth of all tiles in a row for each XCD: 1.4 times the time with 64
// experts whose rows fall as 1 / sqrt(rank)).  False: nothing left for it.
constexpr int kChunk = 32;
__device__ __forceinline__ bool place_tile(int b, int row_tiles, int col_tiles, int& rt, int& ct) {
  const int total = row_tiles * col_tiles, size = total >= 8 * kChunk ? kChunk : (total + 7) / 8;
  const int x = b & 7, at = b >> 3;
  if (size <= 0) return false;
  const int t = (at / size * 8 + x) * size + at % size;
  if (t >= total) return false;
  const int band = 4 * col_tiles, b0 = t / band, in = t % band;
  const int height = row_tiles - 4 * b0 < 4 ? row_tiles - 4 * b0 : 4;
  rt = 4 * b0 + in % height;
  ct = in / height;
  return true;
}

}  // namespace
}  // namespace hsmoe

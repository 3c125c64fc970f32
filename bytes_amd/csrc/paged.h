// Paged dense KV caches: what the append, decode and page-sparse kernels share.
//
// A cache is [num_blocks, Hk, block_size, D] bf16 or fp8 (OCP e4m3fn), any
// strides with unit stride along D.  Token p of sequence b is row p % block_size
// of block table[b, p / block_size].  Sequence b holds lens[b] tokens (clamped to
// what its table row can name); a token takes part if its block id lies in
// [0, num_blocks).
#pragma once
#include "dense_tile.h"

namespace bytes_amd {

struct PagedKv {
  const void* k;
  const void* v;
  int64_t k_sb, k_sh, k_ss;          // element strides: block, KV head, row
  int64_t v_sb, v_sh, v_ss;
  const int32_t* table;              // [B, width], row stride bt_sb
  int64_t bt_sb;
  const int32_t* lens;               // [B]
  int bs, nblocks, width;
  FastDiv dbs;                       // division by bs
};

// Tokens of sequence b: negative lengths count as 0, lengths past the table row as its capacity.
__device__ __forceinline__ int paged_len(const PagedKv& c, int b) {
  const int n = c.lens[b];
  return n < 0 ? 0 : min(n, c.width * c.bs);
}

// NaN-propagating minimum and maximum (the page metadata's rule).
__device__ __forceinline__ float nan_min(float a, float b) { return (a < b || a != a) ? a : b; }
__device__ __forceinline__ float nan_max(float a, float b) { return (a > b || a != a) ? a : b; }

// Host-side checks of a cache's shape; 0 or a hipError_t.
inline int paged_check(int block_size, int num_blocks, int width) {
  if (block_size <= 0 || num_blocks <= 0 || width < 0) return (int)hipErrorInvalidValue;
  if ((int64_t)width * block_size > 0x7FFFFFFF - 1024) return (int)hipErrorInvalidConfiguration;
  return 0;
}

}  // namespace bytes_amd

// Attention of several new tokens per sequence over a paged cache: what the kernel for
// many rows (paged_prompt.hip) and the one for few (paged_prompt_few.hip) share.
#pragma once
#include "paged.h"

namespace bytes_amd {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kSlack = 8.f;        // log2 of how far weights may pass 1

struct PromptArgs {
  PagedKv c;
  const uint16_t* q;
  int64_t q_st, q_sh;
  uint16_t* out;
  int64_t o_st, o_sh;
  const int32_t* cu;                 // [B + 1]
  const float *ks, *vs;              // [num_blocks, Hk], or null
  int64_t ks_sb, ks_sh, vs_sb, vs_sh;
  float* part_acc;                   // [unit][split][row][D]
  float* part_ml;                    // [unit][split][row][2]
  int T, B, Hk, G, D;
  int cap, window, sinks;            // no window: 2^30
  int nsplit, tiles;                 // parts of a unit's keys; row tiles at most
  int by_keys;                       // row tiles in the order of find_tile_by_keys
  int flip;                          // the scale is negative: queries change sign
  int nwg, span;                     // few rows: workgroups among which keys are dealt, or 0; tokens that 32 rows reach over, at most
  float scale_log2, v_scale;
  FastDiv dHk, dG, dsplit, dnwg;
};

// Row tile number r of the batch: rows r0 .. of sequence b, whose new tokens are rows
// t0 .. t0 + n - 1 of q (b = B: the rows past the last sequence).  False past the last.
struct RowTile {
  int b, t0, n, r0;
  int len;                           // of the sequence, as it is given
  int index;                         // of the tile, in the order of the sequences
};
template <int ROWS>
__device__ __forceinline__ bool find_tile(const PromptArgs& a, int r, int lane, RowTile& x) {
  x.index = r;
  for (int b0 = 0; b0 <= a.B; b0 += 64) {
    const int b = b0 + lane, bc = min(b, a.B);
    const int c0 = min(max(a.cu[bc], 0), a.T), c1 = b < a.B ? min(max(a.cu[bc + 1], 0), a.T) : a.T;
    const int len = a.c.lens[min(b, a.B - 1)];
    const int n = b <= a.B ? max(c1 - c0, 0) : 0;
    const uint32_t mine = (uint32_t)((n * a.G + ROWS - 1) / ROWS);
    const uint32_t incl = wave_prefix_sum(mine);
    const int total = __builtin_amdgcn_readlane((int)incl, 63);
    if (r < total) {
      const int l = __ffsll((unsigned long long)__ballot((int)incl > r)) - 1;
      x.b = b0 + l;
      x.t0 = __builtin_amdgcn_readlane(c0, l);
      x.n = __builtin_amdgcn_readlane(n, l);
      x.len = __builtin_amdgcn_readlane(len, l);
      x.r0 = (r - __builtin_amdgcn_readlane((int)(incl - mine), l)) * ROWS;
      return true;
    }
    r -= total;
  }
  return false;
}

// The same with the tiles of several sequences (below 64) in the order of the keys up to their last
// row, most first: those of sequence b that see more than x keys are its last ones, so their
// number over the batch is one wave sum, and x is found by halving.  (In the order of the sequences
// the CUs end further apart: 4 x 1024 after 476 each over e4m3, 32 heads over 8 of 128, 110.9 us and
// 94.5; 4 sequences of 1.2K to 16K with 1K to 3K new 858 and 758; equal 8K prompts 1200 and 1200.)
template <int ROWS>
__device__ __forceinline__ bool find_tile_by_keys(const PromptArgs& a, int r, int lane, RowTile& x) {
  const int b = min(lane, a.B);
  const int c0 = min(max(a.cu[b], 0), a.T), c1 = lane < a.B ? min(max(a.cu[min(b + 1, a.B)], 0), a.T) : a.T;
  const int len = a.c.lens[min(b, a.B - 1)], n = lane <= a.B ? max(c1 - c0, 0) : 0;
  const int tiles = (n * a.G + ROWS - 1) / ROWS, p0 = lane < a.B ? max(min(len, a.cap) - n, 0) : 0;
  auto over = [&](int k) {                                 // this lane's tiles that see more than k keys
    const int y = k - p0;                                  // their last row's token is y or later
    return y <= 0 ? tiles : y >= n ? 0 : tiles - (int)((uint32_t)(y * a.G) / (uint32_t)ROWS);
  };
  auto all_over = [&](int k) { return __builtin_amdgcn_readlane((int)wave_prefix_sum((uint32_t)over(k)), 63); };
  if (all_over(0) <= r) return false;
  int lo = 0, hi = max(a.cap, a.T);                        // over lo there are more than r, over hi none
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (all_over(mid) > r) lo = mid;
    else hi = mid;
  }
  const int mine = over(lo) - over(hi), left = r - all_over(hi);       // hi = lo + 1
  const int incl = (int)wave_prefix_sum((uint32_t)mine);
  const int l = __ffsll((unsigned long long)__ballot(incl > left)) - 1;
  x.b = l;
  x.t0 = __builtin_amdgcn_readlane(c0, l);
  x.n = __builtin_amdgcn_readlane(n, l);
  x.len = __builtin_amdgcn_readlane(len, l);
  const int at = __builtin_amdgcn_readlane(tiles - over(lo) - (incl - mine), l) + left;
  x.r0 = at * ROWS;
  x.index = __builtin_amdgcn_readlane((int)wave_prefix_sum((uint32_t)tiles) - tiles, l) + at;
  return true;
}

// The first n of 64 bits.
__device__ __forceinline__ uint64_t low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }

// Eight bf16 numbers with infinities and NaN made 0; odd: whether there were any.
__device__ __forceinline__ u32x4 finite_only(const u32x4& x, bool& odd) {
  u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool lo = (x[j] & 0x7F80u) == 0x7F80u, hi = (x[j] & 0x7F800000u) == 0x7F800000u;
    r[j] = x[j] & ((lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u));
    odd = odd | lo | hi;
  }
  return r;
}

__device__ __forceinline__ float half_max(float v) {   // of a lane and its partner lane ^ 32
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Four consecutive results; zeros where nothing was seen.
__device__ __forceinline__ void store_bf16x4(uint16_t* out, const f32x16& x, int at, float by) {
  typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
  bf16x4 r;
#pragma unroll
  for (int u = 0; u < 4; ++u) r[u] = (__bf16)(by == 0.f ? 0.f : x[at + u] * by);
  *reinterpret_cast<u32x2*>(out) = __builtin_bit_cast(u32x2, r);
}

// Tokens that `rows` consecutive rows can reach over.
constexpr int64_t row_span(int64_t rows, int64_t G) { return (rows - 1 + G - 1) / G + 1; }

// How a call is cut up.
struct PromptPlan {
  int waves, nsplit;                 // 32 rows each of a workgroup (1: the kernel for few); parts of a unit's keys
  int nwg;                           // few: workgroups among which all units' keys are dealt, or 0
  int64_t tiles, units;              // row tiles, and (row tile, KV head) pairs, at most
  int rows() const { return waves * 32; }
  size_t workspace(int D) const {
    const size_t parts = nwg ? (size_t)nwg * 2 : nsplit < 2 ? 0 : (size_t)units * nsplit;
    return parts * rows() * (D + 2) * 4;
  }
};

// Workgroups among which `granules` of few rows' keys are dealt.
int few_grid(int64_t granules);
// 32 rows to a workgroup, whose four waves take key tiles in turn; 0 or a hipError_t.
int launch_prompt_few(const PromptArgs& a, int kv_type, const PromptPlan& plan, hipStream_t st);

}  // namespace bytes_amd

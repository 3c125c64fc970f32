// Attention of several new tokens per sequence over a paged cache: what the kernel for
// many rows (paged_prompt.hip) and the one for few (paged_prompt_few.hip) share.
#pragma once
#include "paged.h"
#include "paged_prompt_tiles.h"

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
  FastDiv dHk, dG, dnwg;
};

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

// 32 rows to a workgroup, whose four waves take key tiles in turn; 0 or a hipError_t.
int launch_prompt_few(const PromptArgs& a, int kv_type, const PromptPlan& plan, hipStream_t st);

}  // namespace bytes_amd

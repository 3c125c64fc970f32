// Attention of one new token per sequence over a paged cache, within a sliding window
// and the first tokens (sinks), and over caches in 8 bits with a scale for each block
// and KV head.
//
//   out[b, h] = sum_t p_t vs_t v_t / sum_t p_t,  p_t = exp(scale * ks_t * (q . k_t) - max)
//
// over the tokens t < n of sequence b whose block exists and, with a window w and s
// sinks, t >= n - w or t < s.  ks_t, vs_t are the scales of token t's block (one for the
// tensor: in scale, and v_scale for the values).
//
// The split, tile loop and join of paged_split.h, over slots instead of tokens: the
// sinks' 32-token tiles, then those that the window reaches into, so that what lies
// between costs nothing.  A slot's scales travel with its tile (64 floats of LDS): the
// keys' multiply the fp32 scores, the values' the fp32 weights before these are split
// into bf16 parts, so codes enter the products exactly.
//
// Bound by memory: 29 sequences of 6.6K to 16K, 64 heads over 8 of 128, e4m3 with scales
// (685 MB) take 121 us, 5.7 TB/s (one scale for the tensor 116; without any arithmetic, not an answer,
// 115; int8, whose widening takes more instructions, 131), where streaming reads reach 7.1; a window of 4096 and 4 sinks in 16
// sequences of 12K to 32K, 8 heads of 128 in bf16 (269 MB), 50 us, 5.4 TB/s with its join of 4.6, in 8 bits 36 (one scale),
// 44 (e4m3) and 48 (int8).
#include "paged_split.h"

namespace bytes_amd {

struct PagedWindowArgs : PagedDecodeArgs {
  int window, sinks;                 // no window: 2^30
  const float *ks, *vs;              // [num_blocks, Hk], or null
  int64_t ks_sb, ks_sh, vs_sb, vs_sh;

  // Tokens below `near` and from `lo` on are seen; slots from `near_tiles` on are `gap` tokens further.
  struct View {
    FastDiv dbs;
    int sinks, lo, near_tiles, gap;
    __device__ __forceinline__ void operator()(int s, int& place, int& off, bool& ok) const {
      const int p = s < near_tiles ? s : s + gap;
      place = fast_div(p, dbs);
      off = p - place * (int)dbs.d;
      ok = p < sinks || p >= lo;
    }
  };
  __device__ __forceinline__ View view(int n) const {
    const int lo = max(n - window, 0), near_tiles = (min(sinks, n) + 31) & ~31;
    return View{c.dbs, sinks, lo, near_tiles, max((lo & ~31) - near_tiles, 0)};
  }
  __device__ __forceinline__ int slots(int n) const { return n - view(n).gap; }
  __device__ __forceinline__ PagedScales scales(int hk, float* lds) const {
    return PagedScales{ks + hk * ks_sh, vs + hk * vs_sh, ks_sb, vs_sb, lds};
  }
  // A tile of bytes takes as long as one of bf16 and more, read alone (int8, us from a graph, a workgroup per unit
  // and the even split: one sequence of 2 KV heads of 64, 500 tokens 6.7, 750 8.4 and 7.9, 1000 9.8 and 7.8,
  // 2000 16.3 and 7.9; of 4 heads of 128, 300 tokens 7.3 and 8.9, 500 8.8 and 8.9, 1000 13.5 and 8.9; 64
  // sequences of 2 heads of 64, 1500 tokens 14.4 and 15.3, 2000 17.6 and 17.9; eagerly, where the host's second launch
  // counts, 1000 tokens of 2 heads of 64 9.7 and 9.1 to 10.6).
  static constexpr int dim_cost(int type) { return type == kBf16Cache ? 4 : 5; }
};

// Slots that a table row of `cap` tokens can give.
static int64_t window_slots(int64_t cap, int window, int sinks) {
  const int64_t most = (int64_t)window + sinks + 2 * 32;
  return cap < most ? cap : most;
}

}  // namespace bytes_amd

using namespace bytes_amd;

extern "C" {

int bytes_paged_window_workspace_size(int B, int Hq, int Hk, int D, int kv_type, int block_size, int max_blocks,
                                      int window, int sinks, size_t* bytes) {
  if (!bytes || B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 || (D != 64 && D != 128) || window <= 0 || sinks < 0 ||
      kv_type < kBf16Cache || kv_type > kInt8Blocks)
    return (int)hipErrorInvalidValue;
  const int rc = paged_check(block_size, 1, max_blocks);
  if (rc) return rc;
  const int64_t cap = window_slots((int64_t)max_blocks * block_size, window, sinks);
  const DecodeShape s = decode_shape(B, Hq, Hk, cap);
  *bytes = short_waves(s.units, cap, D, PagedWindowArgs::dim_cost(kv_type)) ? 0 : decode_workspace(decode_grid(s.units, s.granules), D);
  return 0;
}

int bytes_paged_window_attn(const void* q, int64_t q_sb, int64_t q_sh, const void* k_paged, int64_t k_sb, int64_t k_sh,
                            int64_t k_ss, const void* v_paged, int64_t v_sb, int64_t v_sh, int64_t v_ss, int kv_type,
                            const void* k_scales, int64_t ks_sb, int64_t ks_sh, const void* v_scales, int64_t vs_sb,
                            int64_t vs_sh, const void* block_table, int64_t bt_sb, const void* context_lens, void* out,
                            int64_t o_sb, int64_t o_sh, int B, int Hq, int Hk, int D, int block_size, int num_blocks,
                            int max_blocks, int window, int sinks, float scale, float v_scale, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (!q || !k_paged || !v_paged || !block_table || !context_lens || !out || B <= 0 || Hk <= 0 || Hq <= 0 ||
      Hq % Hk != 0 || (D != 64 && D != 128) || max_blocks <= 0 || window <= 0 || sinks < 0 || kv_type < kBf16Cache ||
      kv_type > kInt8Blocks || (kv_type >= kE4m3Blocks && (!k_scales || !v_scales)))
    return (int)hipErrorInvalidValue;
  const int rc = paged_check(block_size, num_blocks, max_blocks);
  if (rc) return rc;
  const int64_t cap = window_slots((int64_t)max_blocks * block_size, window, sinks);
  const DecodeShape shape = decode_shape(B, Hq, Hk, cap);
  if (shape.granules > 0x7FFFFFFF || B > 65535) return (int)hipErrorInvalidConfiguration;
  PagedWindowArgs a;
  decode_args(a, q, q_sb, q_sh, k_paged, k_sb, k_sh, k_ss, v_paged, v_sb, v_sh, v_ss, block_table, bt_sb, context_lens,
              out, o_sb, o_sh, B, Hq, Hk, block_size, num_blocks, max_blocks, shape, workspace);
  a.window = window < (1 << 30) ? window : (1 << 30), a.sinks = sinks < (1 << 30) ? sinks : (1 << 30);
  a.ks = static_cast<const float*>(k_scales), a.ks_sb = ks_sb, a.ks_sh = ks_sh;
  a.vs = static_cast<const float*>(v_scales), a.vs_sb = vs_sb, a.vs_sh = vs_sh;
  a.scale_log2 = scale * kLog2e, a.v_scale = v_scale;
  if (!short_waves(shape.units, cap, D, PagedWindowArgs::dim_cost(kv_type)) &&
      (!workspace || workspace_bytes < decode_workspace(a.nwg, D)))
    return (int)hipErrorInvalidValue;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (kv_type) {
    case kBf16Cache: return launch_decode_of<PagedWindowArgs, kBf16Cache>(a, D, shape, cap, st);
    case kFp8Cache: return launch_decode_of<PagedWindowArgs, kFp8Cache>(a, D, shape, cap, st);
    case kE4m3Blocks: return launch_decode_of<PagedWindowArgs, kE4m3Blocks>(a, D, shape, cap, st);
    default: return launch_decode_of<PagedWindowArgs, kInt8Blocks>(a, D, shape, cap, st);
  }
}

}  // extern "C"

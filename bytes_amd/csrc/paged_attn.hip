// Attention of one new token per sequence over a paged KV cache.
//
//   out[b, h] = v_scale * softmax_p(scale * q[b, h] . k[b, h / G, p]) v[b, h / G, p]
//
// over the tokens p of sequence b that take part (paged.h); a row none of whose
// tokens does gets zeros.  Scores, softmax statistics and sums are fp32 (products
// of bf16 values are exact there).
//
// Split: the lengths are known on the device only, and may differ by any factor.
// A unit is up to 16 query heads of one KV head of one sequence; its tokens are
// cut into granules of 128 (one 32-token tile for each of a workgroup's four
// waves).  All granules of all units, in the order (sequence, KV head, head
// block, token), are dealt to the fixed grid in equal runs: every workgroup sums
// the granules of the batch (one load of lens per 64 sequences and a wave prefix
// sum) and finds its run.  A run covers parts of units; a part that is a whole
// unit is finished in place, others (at most two per workgroup: its first and its
// last) leave (max, sum, values) in fp32 for the second launch, which joins each
// unit's parts in token order.  So the work per workgroup differs by at most one
// granule whatever the lengths, and the result does not depend on timing.
// Tables that hold short contexts only take a workgroup per unit and no second
// launch (short_waves).
// Bound by memory: four sequences of 64K to 128K (8 KV heads of 128, 1.6 GB) take 245
// us, 6.6 TB/s, where streaming reads reach 7.1; 29 of 6.6K to 16K over an fp8 cache (0.68
// GB) 116, 5.9 TB/s.  Eight of 3.4K to 8K (95 MB) take 23, six tiles per wave between a
// start and an end that stream nothing, and the join.
#include "paged_split.h"

using namespace bytes_amd;

extern "C" {

int bytes_paged_decode_workspace_size(int B, int Hq, int Hk, int D, int kv_fp8, int block_size, int max_blocks,
                                      size_t* bytes) {
  if (!bytes || B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 || (D != 64 && D != 128)) return (int)hipErrorInvalidValue;
  const int rc = paged_check(block_size, 1, max_blocks);
  if (rc) return rc;
  const int64_t cap = (int64_t)max_blocks * block_size;
  const DecodeShape s = decode_shape(B, Hq, Hk, cap);
  *bytes = short_waves(s.units, cap, D, PagedDecodeArgs::dim_cost(kv_fp8)) ? 0 : decode_workspace(decode_grid(s.units, s.granules), D);
  return 0;
}

int bytes_paged_decode_attn(const void* q, int64_t q_sb, int64_t q_sh, const void* k_paged, int64_t k_sb, int64_t k_sh,
                            int64_t k_ss, const void* v_paged, int64_t v_sb, int64_t v_sh, int64_t v_ss, int kv_fp8,
                            const void* block_table, int64_t bt_sb, const void* context_lens, void* out, int64_t o_sb,
                            int64_t o_sh, int B, int Hq, int Hk, int D, int block_size, int num_blocks, int max_blocks,
                            float scale, float v_scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !k_paged || !v_paged || !block_table || !context_lens || !out || B <= 0 || Hk <= 0 || Hq <= 0 ||
      Hq % Hk != 0 || (D != 64 && D != 128) || max_blocks <= 0)
    return (int)hipErrorInvalidValue;
  const int rc = paged_check(block_size, num_blocks, max_blocks);
  if (rc) return rc;
  const int64_t cap = (int64_t)max_blocks * block_size;
  const DecodeShape shape = decode_shape(B, Hq, Hk, cap);
  if (shape.granules > 0x7FFFFFFF || B > 65535) return (int)hipErrorInvalidConfiguration;
  PagedDecodeArgs a;
  decode_args(a, q, q_sb, q_sh, k_paged, k_sb, k_sh, k_ss, v_paged, v_sb, v_sh, v_ss, block_table, bt_sb, context_lens,
              out, o_sb, o_sh, B, Hq, Hk, block_size, num_blocks, max_blocks, shape, workspace);
  a.scale_log2 = scale * kLog2e, a.v_scale = v_scale;
  if (!short_waves(shape.units, cap, D, PagedDecodeArgs::dim_cost(kv_fp8)) && (!workspace || workspace_bytes < decode_workspace(a.nwg, D)))
    return (int)hipErrorInvalidValue;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return kv_fp8 ? launch_decode_of<PagedDecodeArgs, kFp8Cache>(a, D, shape, cap, st)
                : launch_decode_of<PagedDecodeArgs, kBf16Cache>(a, D, shape, cap, st);
}

}  // extern "C"

// New tokens into a paged KV cache, with the position rotation on the way.
//
// Token i of sequence b's n new ones has position p = lens[b] - n + i (lens
// counts the new tokens).  Its key's (and query's) first R dims are rotated in
// pairs (x0, x1) -> (x0 c - x1 s, x1 c + x0 s) with row p of the cos / sin
// tables, pairs (j, j + R/2) or neighbours (2j, 2j + 1); the result, divided by the
// cache's scale in fp32, is rounded to the cache's type.  The
// blocks' elementwise min / max (of the values as stored) are kept for the
// page-sparse decode.
//
// A lane takes 16 elements of one head (an item): for pairs (j, j + R/2) two runs
// of 8, R/2 apart, so both of a pair are in its registers and its cos and sin are
// 8 consecutive floats.  D/16 lanes cover a row; a wave's 64 lanes are 64/(D/16)
// rows.
//  * One token per sequence: a wave's rows are heads (keys, values and queries in
//    one list) of one token.  3.9 us for a single token, 5.2 for 30 with min / max:
//    length, block id, rows and min / max follow one another.
//  * Prompts: a wave's rows are consecutive tokens of one sequence.  Values and
//    queries (and keys where no min / max is kept) go in spans of as many positions
//    as a wave has rows, keys with min / max in blocks: a wave has a whole block's
//    new tokens, so it folds their min / max in registers and across its lanes,
//    without atomics or a second read.  Spans are numbered over the batch; every
//    wave finds its own from a prefix sum over the sequences, rows past the last
//    sequence being one more.
//    Made for blocks of 8 to 64 rows where min / max are kept: of smaller ones a wave
//    has few rows, of larger ones many in turn (us, four chunks of 1 to 2K tokens of
//    28 + 2 x 4 heads of 128 and of 14 + 2 x 2 of 64, from a graph: without min / max 25
//    and 10 with any block; with them, blocks of 1 row 59 and 33, of 2 40 and 21, of 4
//    31 and 14, of 8 27 and 12, of 16 26 and 12, of 64 26 and 13, of 128 35 and 18, of
//    256 55 and 27, of 1024 172 and 86).
// Bound by memory: a 32K-token prompt of 32 query and 8 KV heads (0.4 GB read, 0.4
// GB written) takes 160 us, 5.1 TB/s; a plain copy of 2 GiB runs at 4.9.
#include "paged_append.h"

namespace bytes_amd {

// One token of one sequence per wave and up to 64 / LPR of its heads' rows.
template <int D, bool FP8>
__global__ __launch_bounds__(kAppendWaves * 64) void paged_append_one_kernel(AppendArgs a) {
  PREFETCH_ARGS(a);
  constexpr int LPR = D / 16, ROWS = 64 / LPR;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int gid = blockIdx.x * kAppendWaves + w;
  const int t = fast_div(gid, a.d_per_token);
  if (t >= a.T) return;
  const int len = a.c.lens[t];
  const AppendItem it(a, lane % LPR);
  const int r = (gid - t * a.per_token) * ROWS + lane / LPR, rows = 2 * a.Hk + a.Hq;
  const bool live = r < rows, key = r < a.Hk, value = !key && r < 2 * a.Hk;
  const int h = key ? r : value ? r - a.Hk : live ? r - 2 * a.Hk : 0;
  // the row, at once with the length; values are never rotated: their item is 16 dims in a row
  const int d0 = value ? 16 * it.c : it.d0, d1 = value ? 16 * it.c + 8 : it.d1;
  const uint16_t* src = key || !live ? a.k + t * a.k_st + h * a.k_sh : value ? a.v + t * a.v_st + h * a.v_sh
                                                                              : a.q + t * a.q_st + h * a.q_sh;
  const u32x4 x0 = ld16(src + d0), x1 = ld16(src + d1);
  const int p = len - 1;
  const bool placed = len > 0 && p < a.cap;
  const int ps = placed ? p : 0, blk = fast_div(ps, a.c.dbs), off = ps - blk * a.c.bs;
  const int id = a.c.table[(int64_t)t * a.c.bt_sb + blk];
  const bool held = placed && id >= 0 && id < a.c.nblocks;
  float x[16];
  widen8(x0, x);
  widen8(x1, x + 8);
  if (live && !value && it.turn && placed) {
    Turn tr;
    load_turn(a, it, ps, tr);
    if (key) turn_item<true>(a, tr, x);
    else turn_item<false>(a, tr, x);
  }
  if (!live) return;
  if (key) {
    if (!held) return;
    float mn[16], mx[16];
    uint16_t* pmn = a.kmin + ((int64_t)id * a.Hk + h) * D;
    uint16_t* pmx = a.kmax + ((int64_t)id * a.Hk + h) * D;
    if (a.kmin && off) {
      load_item(pmn, it, mn);
      load_item(pmx, it, mx);
    }
    store_cache<FP8>(cache_row<FP8>(a.c.k, a.c.k_sb, a.c.k_sh, a.c.k_ss, id, h, off), it, a.k_scale, x);
    if (!a.kmin) return;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      mn[j] = off ? lower(mn[j], x[j]) : x[j];
      mx[j] = off ? upper(mx[j], x[j]) : x[j];
    }
    store_item(pmn, it, mn);
    store_item(pmx, it, mx);
  } else if (value) {
    if (!held) return;
    char* to = cache_row<FP8>(a.c.v, a.c.v_sb, a.c.v_sh, a.c.v_ss, id, h, off);
    if constexpr (FP8) {
      AppendItem flat = it;
      flat.d0 = d0, flat.d1 = d1;
      store_cache<FP8>(to, flat, a.v_scale, x);
    } else {
      *reinterpret_cast<u32x4*>(to + 2 * d0) = x0;
      *reinterpret_cast<u32x4*>(to + 2 * d1) = x1;
    }
  } else {
    if (!placed) {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = 0.f;
    }
    store_item(a.q_out + t * a.qo_st + h * a.qo_sh, it, x);
  }
}

template <int D, bool FP8>
__global__ __launch_bounds__(kAppendWaves * 64) void paged_append_kernel(AppendArgs a) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Span s;
  if (blockIdx.x < a.k_grid) {
    const int r = fast_div((int)blockIdx.x, a.dk_wgs);
    const int h0 = (((int)blockIdx.x - r * a.k_wgs) * kAppendWaves + w) * kKeyHeads;
    if (h0 >= a.Hk || !find_span(a, r, a.k_span, a.dk_span, lane, s) || s.b == a.B) return;
    append_span<D, FP8, kKeys, kKeyHeads>(a, s, h0, min(kKeyHeads, a.Hk - h0), lane);
  } else {
    const int x = (int)((int64_t)blockIdx.x - a.k_grid), r = fast_div(x, a.do_wgs);
    const int g = (x - r * a.o_wgs) * kAppendWaves + w, gv = (a.Hk + kRowHeads - 1) / kRowHeads;
    const bool values = g < gv;
    const int h0 = (values ? g : g - gv) * kRowHeads, heads = values ? a.Hk : a.Hq;
    if (h0 >= heads || !find_span(a, r, row_span<D>(), FastDiv{1u, (uint32_t)__builtin_ctz(row_span<D>()), (uint32_t)row_span<D>()}, lane, s)) return;
    if (values) {
      if (s.b < a.B) append_span<D, FP8, kValues, kRowHeads>(a, s, h0, min(kRowHeads, heads - h0), lane);
    } else {
      append_span<D, FP8, kQueries, kRowHeads>(a, s, h0, min(kRowHeads, heads - h0), lane);
    }
  }
}

}  // namespace bytes_amd

using namespace bytes_amd;

extern "C" {

int bytes_paged_kv_append(const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh,
                          const void* q, int64_t q_st, int64_t q_sh, void* q_out, int64_t qo_st, int64_t qo_sh,
                          void* k_paged, int64_t kp_sb, int64_t kp_sh, int64_t kp_ss, void* v_paged, int64_t vp_sb,
                          int64_t vp_sh, int64_t vp_ss, int kv_fp8, void* kmin, void* kmax, const void* block_table,
                          int64_t bt_sb, const void* context_lens, const void* cu_seqlens, const void* cos,
                          int64_t cos_st, const void* sin, int64_t sin_st, int positions, int rot, int interleaved,
                          float k_scale, float v_scale, int T, int B, int Hq, int Hk, int D, int block_size,
                          int num_blocks, int max_blocks, void* stream) {
  if (!k || !v || !k_paged || !v_paged || !block_table || !context_lens || T < 0 || B <= 0 || Hk <= 0 || Hq < 0 ||
      max_blocks <= 0)                             // (a table's first column is read for every token)
    return (int)hipErrorInvalidValue;
  if ((D != 64 && D != 128) || rot < 0 || rot > D || rot % 16 != 0 || (!cu_seqlens && T != B))
    return (int)hipErrorInvalidValue;
  if ((q == nullptr) != (q_out == nullptr) || (q == nullptr) != (Hq == 0) || (kmin == nullptr) != (kmax == nullptr))
    return (int)hipErrorInvalidValue;
  int rc = paged_check(block_size, num_blocks, max_blocks);
  if (rc) return rc;
  if (rot && (!cos || !sin || (int64_t)positions < (int64_t)max_blocks * block_size)) return (int)hipErrorInvalidValue;
  if (T == 0) return 0;
  AppendArgs a = {};
  a.c.k = k_paged;
  a.c.v = v_paged;
  a.c.k_sb = kp_sb, a.c.k_sh = kp_sh, a.c.k_ss = kp_ss;
  a.c.v_sb = vp_sb, a.c.v_sh = vp_sh, a.c.v_ss = vp_ss;
  a.c.table = static_cast<const int32_t*>(block_table);
  a.c.bt_sb = bt_sb;
  a.c.lens = static_cast<const int32_t*>(context_lens);
  a.c.bs = block_size, a.c.nblocks = num_blocks, a.c.width = max_blocks;
  a.c.dbs = make_fastdiv((uint32_t)block_size);
  a.k = static_cast<const uint16_t*>(k), a.k_st = k_st, a.k_sh = k_sh;
  a.v = static_cast<const uint16_t*>(v), a.v_st = v_st, a.v_sh = v_sh;
  a.q = static_cast<const uint16_t*>(q), a.q_st = q_st, a.q_sh = q_sh;
  a.q_out = static_cast<uint16_t*>(q_out), a.qo_st = qo_st, a.qo_sh = qo_sh;
  a.kmin = static_cast<uint16_t*>(kmin), a.kmax = static_cast<uint16_t*>(kmax);
  a.cu = static_cast<const int32_t*>(cu_seqlens);
  a.cos = static_cast<const float*>(cos), a.sin = static_cast<const float*>(sin);
  a.cos_st = cos_st, a.sin_st = sin_st;
  a.rot = rot, a.interleaved = interleaved ? 1 : 0;
  a.k_scale = k_scale, a.v_scale = v_scale;
  a.T = T, a.B = B, a.Hq = Hq, a.Hk = Hk;
  a.cap = max_blocks * block_size;
  int64_t grid;
  if (!cu_seqlens) {
    const int rows_per_wave = 64 / (D / 16);
    a.per_token = (2 * Hk + Hq + rows_per_wave - 1) / rows_per_wave;
    a.d_per_token = make_fastdiv((uint32_t)a.per_token);
    if ((int64_t)T * a.per_token > 0x7FFFFFF0) return (int)hipErrorInvalidConfiguration;
    grid = ((int64_t)T * a.per_token + kAppendWaves - 1) / kAppendWaves;
  } else {
    // a sequence's n tokens lie in at most n / span + 2 spans, and in at most n
    auto spans = [&](int len) {
      const int64_t n = (int64_t)T / len + 2 * ((int64_t)B + 1);
      return n < T ? n : (int64_t)T;
    };
    const int per_key = kAppendWaves * kKeyHeads;
    const int span = D == 128 ? row_span<128>() : row_span<64>();
    a.k_span = kmin ? block_size : span;
    a.dk_span = make_fastdiv((uint32_t)a.k_span);
    a.k_wgs = (Hk + per_key - 1) / per_key;
    a.k_grid = spans(a.k_span) * a.k_wgs;
    a.dk_wgs = make_fastdiv((uint32_t)a.k_wgs);
    const int groups = (Hk + kRowHeads - 1) / kRowHeads + (Hq + kRowHeads - 1) / kRowHeads;
    a.o_wgs = (groups + kAppendWaves - 1) / kAppendWaves;
    a.do_wgs = make_fastdiv((uint32_t)a.o_wgs);
    grid = a.k_grid + spans(span) * a.o_wgs;
  }
  if (grid > 0x7FFFFFFF) return (int)hipErrorInvalidConfiguration;
  const dim3 g((unsigned)grid), block(kAppendWaves * 64);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define PA(DD, F8)                                                                   \
  if (cu_seqlens) hipLaunchKernelGGL((paged_append_kernel<DD, F8>), g, block, 0, st, a); \
  else hipLaunchKernelGGL((paged_append_one_kernel<DD, F8>), g, block, 0, st, a)
  if (D == 128) {
    if (kv_fp8) { PA(128, true); }
    else { PA(128, false); }
  } else {
    if (kv_fp8) { PA(64, true); }
    else { PA(64, false); }
  }
#undef PA
  return (int)hipGetLastError();
}

}  // extern "C"

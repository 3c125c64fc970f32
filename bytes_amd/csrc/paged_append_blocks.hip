// New tokens into a paged KV cache held in 8 bits with a scale for each block and
// KV head, keys and values apart: a row's code stands for code * scale[block, head].
//
// Rows x are the rotated keys (rounded to fp32 from their exact products) and the
// values, infinities held to the largest bf16 number.  For every block that receives
// rows, and every head:
//   a  = max |x| over the new rows of the block (NaN is not counted)
//   c  = a / 127 (int8), or the smallest power of two of at least a / 448 (e4m3)
//   s' = c where the sequence enters the block at its first row, else max(s, c)
//   where s' > s, the rows before the new ones: code = round(code * (s / s'))
//   new rows: code = round(x / s'), to nearest even (NaN: 0 in int8, NaN in e4m3)
// e4m3 keeps its relative step over its range, so a power of two costs it nothing and
// rows are rescaled without a rounding (but for the format's subnormals); int8 takes
// the scale that uses its range, and a row that is rescaled is off by another half of
// the new step each time (a block of 16 rows that arrive one by one has its largest
// value replaced about 3 times).
//
// Waves as in paged_append.hip: a wave takes up to 64 / (D / 16) heads' rows of one
// token each, or one head's new rows of one block.  It finds their maximum in
// registers, folds it across lanes, and stores them; no atomics, one writer to a scale.
// Rows of blocks that fit the wave's registers are read once.
// Bound by memory for prompts: 6656 tokens of 28 query and 4 KV heads of 128 to int8 (119 MB) take
// 28.6 us, 4.2 TB/s, where a large copy reaches 4.9; the steps of a batch by what follows one
// another (lengths, block id, scale, row): 30 sequences' tokens of 64 and 8 heads, e4m3, 4.7 us.  A scale that grows
// adds its block's earlier rows, which the head's own D / 16 lanes take four at a time: 32 sequences' tokens of 64 and 8
// heads in the second half of their blocks, N(0, 1), median and longest, of 16, 64 and 128 rows: e4m3 10.7 and 13, 22
// and 28, 5.2 and 38 us, int8, whose scales grow more often, 11.4 and 14, 23 and 33, 38 and 67.
#include "paged_append.h"

namespace bytes_amd {

struct BlockAppendArgs : AppendArgs {
  float *ks, *vs;                    // [num_blocks, Hk]
  int64_t ks_sb, ks_sh, vs_sb, vs_sh;
};

constexpr float kBf16Max = 3.3895313892515355e38f;

__device__ __forceinline__ float held_finite(float x) { return x > kBf16Max ? kBf16Max : (x < -kBf16Max ? -kBf16Max : x); }

template <bool INT8>
__device__ __forceinline__ float fit_scale(float a) {
  if constexpr (INT8) return a / 127.f;
  if (!(a > 0.f)) return 0.f;
  // 448 = 1.75 * 2^8: a's exponent less 8, one more where its significand is above 1.75
  const uint32_t u = __float_as_uint(a);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)max(e, 1) << 23);
}

// A stored scale as it counts: what no append leaves (negative, NaN, infinite) as 0.
__device__ __forceinline__ float stored_scale(float s) { return s > 0.f && s <= 3.4028234663852886e38f ? s : 0.f; }

// Eight values / s as codes.  s > 0.
__device__ __forceinline__ uint32_t int8_bits(float y) {
  y = y == y ? fminf(fmaxf(y, -127.f), 127.f) : 0.f;
  return __float_as_uint(y + 12582912.f) & 0xFFu;  // 1.5 * 2^23: the sum's last bits are the nearest whole number
}
template <bool INT8>
__device__ __forceinline__ u32x2 codes8(const float* x) {
  if constexpr (!INT8) return narrow8_fp8(x);
  u32x2 r;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    r[j] = int8_bits(x[4 * j]) | int8_bits(x[4 * j + 1]) << 8 | int8_bits(x[4 * j + 2]) << 16 | int8_bits(x[4 * j + 3]) << 24;
  return r;
}
template <bool INT8>
__device__ __forceinline__ void widen_codes8(const u32x2& r, float* x) {
  if constexpr (!INT8) {
    widen8_fp8(r, x);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)(int8_t)(r[j >> 2] >> (8 * (j & 3)));
  }
}

// One row's two runs of 8 as codes of scale s.
template <bool INT8>
__device__ __forceinline__ void store_codes(char* to, int d0, int d1, float s, const float* x) {
  float y[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) y[j] = s > 0.f ? x[j] / s : (INT8 || x[j] == x[j] ? 0.f : x[j]);
  *reinterpret_cast<u32x2*>(to + d0) = codes8<INT8>(y);
  *reinterpret_cast<u32x2*>(to + d1) = codes8<INT8>(y + 8);
}

// Rows r0, r0 + step, .. < n of a block and head at `row0`, this lane's 16 codes of each
// (at 16 c), times r.
template <bool INT8>
__device__ __forceinline__ void rescale_rows(char* row0, int64_t ss, int c, int r0, int step, int n, float ratio) {
  constexpr int U = 4;                             // rows in flight
  for (int i = r0; i < n; i += U * step) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = ld16(row0 + (int64_t)min(i + u * step, n - 1) * ss + 16 * c);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * step >= n) break;
      float x[16];
      widen_codes8<INT8>(u32x2{raw[u][0], raw[u][1]}, x);
      widen_codes8<INT8>(u32x2{raw[u][2], raw[u][3]}, x + 8);
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] *= ratio;
      const u32x2 a = codes8<INT8>(x), b = codes8<INT8>(x + 8);
      *reinterpret_cast<u32x4*>(row0 + (int64_t)(i + u * step) * ss + 16 * c) = u32x4{a[0], a[1], b[0], b[1]};
    }
  }
}

__device__ __forceinline__ float max_abs16(const float* x) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) m = fmaxf(m, fabsf(x[j]));
  return m;
}
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), CTRL, 0xF, 0xF, false));
}
// The largest over the LPR neighbouring lanes of a row (4 or 8 of them), every one receiving it.
template <int LPR>
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, dpp_f32<0xB1>(v));                  // lanes 1, 0, 3, 2
  v = fmaxf(v, dpp_f32<0x4E>(v));                  // lanes 2, 3, 0, 1
  if (LPR == 8) v = fmaxf(v, dpp_f32<0x141>(v));   // the other four of eight
  return v;
}

// One token of one sequence per wave and up to 64 / LPR of its heads' rows.
template <int D, bool INT8>
__global__ __launch_bounds__(kAppendWaves * 64) void paged_append_block_one_kernel(BlockAppendArgs a) {
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
  const int d0 = value ? 16 * it.c : it.d0, d1 = value ? 16 * it.c + 8 : it.d1;
  const uint16_t* src = key || !live ? a.k + t * a.k_st + h * a.k_sh : value ? a.v + t * a.v_st + h * a.v_sh
                                                                              : a.q + t * a.q_st + h * a.q_sh;
  const u32x4 x0 = ld16(src + d0), x1 = ld16(src + d1);
  const int p = len - 1;
  const bool placed = len > 0 && p < a.cap;
  const int ps = placed ? p : 0, blk = fast_div(ps, a.c.dbs), off = ps - blk * a.c.bs;
  const int id = a.c.table[(int64_t)t * a.c.bt_sb + blk];
  const bool held = placed && id >= 0 && id < a.c.nblocks;
  const bool cached = held && live && (key || value);
  float* sp = key ? a.ks + id * a.ks_sb + h * a.ks_sh : a.vs + id * a.vs_sb + h * a.vs_sh;
  const float was = cached && off ? stored_scale(*sp) : 0.f;
  float x[16];
  widen8(x0, x);
  widen8(x1, x + 8);
  if (live && !value && it.turn && placed) {
    Turn tr;
    load_turn(a, it, ps, tr);
    if (key) turn_item<true>(a, tr, x);
    else turn_item<false>(a, tr, x);
  }
  if (live && !key && !value) {
    if (!placed) {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = 0.f;
    }
    store_item(a.q_out + t * a.qo_st + h * a.qo_sh, it, x);
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) x[j] = held_finite(x[j]);
  const float s = fmaxf(was, fit_scale<INT8>(row_max<LPR>(max_abs16(x))));
  if (!cached) return;
  char* row0 = key ? cache_row<true>(a.c.k, a.c.k_sb, a.c.k_sh, a.c.k_ss, id, h, 0)
                   : cache_row<true>(a.c.v, a.c.v_sb, a.c.v_sh, a.c.v_ss, id, h, 0);
  const int64_t ss = key ? a.c.k_ss : a.c.v_ss;
  store_codes<INT8>(row0 + off * ss, d0, d1, s, x);
  if (off && s > was) rescale_rows<INT8>(row0, ss, it.c, 0, 1, off, was / s);
  if (it.c == 0) *sp = s;
}

// The new rows of one block and one key or value head, by one wave.
template <int D, bool INT8, bool KEY>
__device__ __forceinline__ void append_block(const BlockAppendArgs& a, const Span& s, int h, int lane) {
  constexpr int LPR = D / 16, ROWS = 64 / LPR, HOLD = 2;
  AppendItem it(a, lane % LPR);
  if (!KEY) it.d0 = 16 * it.c, it.d1 = 16 * it.c + 8;
  const uint16_t* src = (KEY ? a.k + h * a.k_sh : a.v + h * a.v_sh);
  const int64_t st = KEY ? a.k_st : a.v_st;
  // rows with a position in the table: p1 .. p2 - 1, all in one block
  const int p1 = max(s.p0, 0), p2 = min(s.p0 + s.n, a.cap);
  if (p1 >= p2) return;
  const int blk = fast_div(p1, a.c.dbs), off = p1 - blk * a.c.bs, n = p2 - p1;
  const int id = a.c.table[(int64_t)s.b * a.c.bt_sb + blk];
  if (id < 0 || id >= a.c.nblocks) return;
  float* sp = KEY ? a.ks + id * a.ks_sb + h * a.ks_sh : a.vs + id * a.vs_sb + h * a.vs_sh;
  const float was = off ? stored_scale(*sp) : 0.f;
  src += (int64_t)(s.t0 + (p1 - s.p0)) * st;
  auto load = [&](int i, float* x) {               // row i of the new ones, rotated
    widen8(ld16(src + i * st + it.d0), x);
    widen8(ld16(src + i * st + it.d1), x + 8);
    if (KEY && it.turn) {
      Turn tr;
      load_turn(a, it, p1 + i, tr);
      turn_item<true>(a, tr, x);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = held_finite(x[j]);
  };
  const int i0 = lane / LPR;
  float x[HOLD][16], m = 0.f;
#pragma unroll
  for (int u = 0; u < HOLD; ++u) {
    load(min(i0 + u * ROWS, n - 1), x[u]);         // (rows past the last: its values again)
    m = fmaxf(m, max_abs16(x[u]));
  }
  for (int i = i0 + HOLD * ROWS; i < n; i += ROWS) {
    float y[16];
    load(i, y);
    m = fmaxf(m, max_abs16(y));
  }
  const float now = fmaxf(was, fit_scale<INT8>(wave_max_f32(m)));
  char* row0 = KEY ? cache_row<true>(a.c.k, a.c.k_sb, a.c.k_sh, a.c.k_ss, id, h, 0)
                   : cache_row<true>(a.c.v, a.c.v_sb, a.c.v_sh, a.c.v_ss, id, h, 0);
  const int64_t ss = KEY ? a.c.k_ss : a.c.v_ss;
#pragma unroll
  for (int u = 0; u < HOLD; ++u) {
    const int i = i0 + u * ROWS;
    if (i < n) store_codes<INT8>(row0 + (int64_t)(off + i) * ss, it.d0, it.d1, now, x[u]);
  }
  for (int i = i0 + HOLD * ROWS; i < n; i += ROWS) {
    float y[16];
    load(i, y);
    store_codes<INT8>(row0 + (int64_t)(off + i) * ss, it.d0, it.d1, now, y);
  }
  if (off && now > was) rescale_rows<INT8>(row0, ss, it.c, i0, ROWS, off, was / now);
  if (lane == 0) *sp = now;
}

template <int D, bool INT8>
__global__ __launch_bounds__(kAppendWaves * 64) void paged_append_block_kernel(BlockAppendArgs a) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Span s;
  if (blockIdx.x < a.k_grid) {
    const int r = fast_div((int)blockIdx.x, a.dk_wgs);
    const int h = ((int)blockIdx.x - r * a.k_wgs) * kAppendWaves + w;
    if (h >= 2 * a.Hk || !find_span(a, r, a.k_span, a.dk_span, lane, s) || s.b == a.B) return;
    if (h < a.Hk) append_block<D, INT8, true>(a, s, h, lane);
    else append_block<D, INT8, false>(a, s, h - a.Hk, lane);
  } else {
    const int x = (int)((int64_t)blockIdx.x - a.k_grid), r = fast_div(x, a.do_wgs);
    const int h0 = ((x - r * a.o_wgs) * kAppendWaves + w) * kRowHeads;
    if (h0 >= a.Hq || !find_span(a, r, row_span<D>(), FastDiv{1u, (uint32_t)__builtin_ctz(row_span<D>()), (uint32_t)row_span<D>()}, lane, s)) return;
    append_span<D, true, kQueries, kRowHeads>(a, s, h0, min(kRowHeads, a.Hq - h0), lane);
  }
}

}  // namespace bytes_amd

using namespace bytes_amd;

extern "C" {

int bytes_paged_kv_append_blocks(const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh,
                                 const void* q, int64_t q_st, int64_t q_sh, void* q_out, int64_t qo_st, int64_t qo_sh,
                                 void* k_paged, int64_t kp_sb, int64_t kp_sh, int64_t kp_ss, void* v_paged, int64_t vp_sb,
                                 int64_t vp_sh, int64_t vp_ss, int kv_type, void* k_scales, int64_t ks_sb, int64_t ks_sh,
                                 void* v_scales, int64_t vs_sb, int64_t vs_sh, const void* block_table, int64_t bt_sb,
                                 const void* context_lens, const void* cu_seqlens, const void* cos, int64_t cos_st,
                                 const void* sin, int64_t sin_st, int positions, int rot, int interleaved, int T, int B,
                                 int Hq, int Hk, int D, int block_size, int num_blocks, int max_blocks, void* stream) {
  if (!k || !v || !k_paged || !v_paged || !k_scales || !v_scales || !block_table || !context_lens || T < 0 || B <= 0 ||
      Hk <= 0 || Hq < 0 || max_blocks <= 0 || (kv_type != kE4m3Blocks && kv_type != kInt8Blocks))
    return (int)hipErrorInvalidValue;
  if ((D != 64 && D != 128) || rot < 0 || rot > D || rot % 16 != 0 || (!cu_seqlens && T != B))
    return (int)hipErrorInvalidValue;
  if ((q == nullptr) != (q_out == nullptr) || (q == nullptr) != (Hq == 0)) return (int)hipErrorInvalidValue;
  int rc = paged_check(block_size, num_blocks, max_blocks);
  if (rc) return rc;
  if (rot && (!cos || !sin || (int64_t)positions < (int64_t)max_blocks * block_size)) return (int)hipErrorInvalidValue;
  if (T == 0) return 0;
  BlockAppendArgs a = {};
  a.c.k = k_paged;
  a.c.v = v_paged;
  a.c.k_sb = kp_sb, a.c.k_sh = kp_sh, a.c.k_ss = kp_ss;
  a.c.v_sb = vp_sb, a.c.v_sh = vp_sh, a.c.v_ss = vp_ss;
  a.ks = static_cast<float*>(k_scales), a.ks_sb = ks_sb, a.ks_sh = ks_sh;
  a.vs = static_cast<float*>(v_scales), a.vs_sb = vs_sb, a.vs_sh = vs_sh;
  a.c.table = static_cast<const int32_t*>(block_table);
  a.c.bt_sb = bt_sb;
  a.c.lens = static_cast<const int32_t*>(context_lens);
  a.c.bs = block_size, a.c.nblocks = num_blocks, a.c.width = max_blocks;
  a.c.dbs = make_fastdiv((uint32_t)block_size);
  a.k = static_cast<const uint16_t*>(k), a.k_st = k_st, a.k_sh = k_sh;
  a.v = static_cast<const uint16_t*>(v), a.v_st = v_st, a.v_sh = v_sh;
  a.q = static_cast<const uint16_t*>(q), a.q_st = q_st, a.q_sh = q_sh;
  a.q_out = static_cast<uint16_t*>(q_out), a.qo_st = qo_st, a.qo_sh = qo_sh;
  a.cu = static_cast<const int32_t*>(cu_seqlens);
  a.cos = static_cast<const float*>(cos), a.sin = static_cast<const float*>(sin);
  a.cos_st = cos_st, a.sin_st = sin_st;
  a.rot = rot, a.interleaved = interleaved ? 1 : 0;
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
    const int span = D == 128 ? row_span<128>() : row_span<64>();
    a.k_span = block_size;
    a.dk_span = make_fastdiv((uint32_t)a.k_span);
    a.k_wgs = (2 * Hk + kAppendWaves - 1) / kAppendWaves;
    a.k_grid = spans(a.k_span) * a.k_wgs;
    a.dk_wgs = make_fastdiv((uint32_t)a.k_wgs);
    const int groups = (Hq + kRowHeads - 1) / kRowHeads;
    a.o_wgs = (groups + kAppendWaves - 1) / kAppendWaves;
    a.do_wgs = make_fastdiv((uint32_t)a.o_wgs);
    grid = a.k_grid + spans(span) * a.o_wgs;
  }
  if (grid > 0x7FFFFFFF) return (int)hipErrorInvalidConfiguration;
  const dim3 g((unsigned)grid), block(kAppendWaves * 64);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define PB(DD, I8)                                                                             \
  if (cu_seqlens) hipLaunchKernelGGL((paged_append_block_kernel<DD, I8>), g, block, 0, st, a); \
  else hipLaunchKernelGGL((paged_append_block_one_kernel<DD, I8>), g, block, 0, st, a)
  if (D == 128) {
    if (kv_type == kInt8Blocks) { PB(128, true); }
    else { PB(128, false); }
  } else {
    if (kv_type == kInt8Blocks) { PB(64, true); }
    else { PB(64, false); }
  }
#undef PB
  return (int)hipGetLastError();
}

}  // extern "C"

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
#include "paged.h"

namespace bytes_amd {

struct AppendArgs {
  PagedKv c;
  const uint16_t *k, *v, *q;         // new rows [T, heads, D]
  int64_t k_st, k_sh, v_st, v_sh, q_st, q_sh;
  uint16_t* q_out;                   // [T, Hq, D]
  int64_t qo_st, qo_sh;
  uint16_t *kmin, *kmax;             // [num_blocks, Hk, D], or null
  const int32_t* cu;                 // [B + 1], or null: one token per sequence
  const float *cos, *sin;            // rows of R / 2
  int64_t cos_st, sin_st;
  int rot, interleaved;
  float k_scale, v_scale;
  int T, B, Hq, Hk;
  int cap;                           // positions a table row holds
  // prompts: workgroups of the key spans come first; per span, the waves' head groups
  int k_span, k_wgs, o_wgs;          // key span length; workgroups per key span, per other span
  int64_t k_grid;                    // workgroups of all key spans
  FastDiv dk_span, dk_wgs, do_wgs;
  int per_token;                     // one token each: waves per token
  FastDiv d_per_token;
};

constexpr int kAppendWaves = 4;
// A wave's share of a prompt: the rows it holds at once, of one key head or of
// two value or query heads.  Short waves in large numbers keep the memory busy
// while others look up their span (us for 32K tokens of 32 + 2 x 8 heads in blocks
// of 64, four chunks of 1 to 2K tokens of 28 + 2 x 4 heads in blocks of 16): one
// key and two other heads 160 and 28; spans twice as long 164 and 28, four times
// 179 and 34; one other head 195 and 33, four 160 and 29; two key heads 166 and 32.
constexpr int kKeyHeads = 1, kRowHeads = 2;
template <int D>
constexpr int row_span() { return 64 / (D / 16); }

__device__ __forceinline__ void widen8(const u32x4& r, float* x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = __uint_as_float(r[j] << 16);
    x[2 * j + 1] = __uint_as_float(r[j] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ u32x4 narrow8(const float* x) {
  u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    r[j] = (uint32_t)f32_to_bf16_bits(x[2 * j]) | ((uint32_t)f32_to_bf16_bits(x[2 * j + 1]) << 16);
  return r;
}

// fp32 -> e4m3, to nearest even; beyond the largest finite value that value, NaN stays NaN.
__device__ __forceinline__ float clamp_e4m3(float x) { return x > 448.f ? 448.f : (x < -448.f ? -448.f : x); }
__device__ __forceinline__ u32x2 narrow8_fp8(const float* x) {
  u32x2 r;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(x[4 * j]), clamp_e4m3(x[4 * j + 1]), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(x[4 * j + 2]), clamp_e4m3(x[4 * j + 3]), w, true);
    r[j] = (uint32_t)w;
  }
  return r;
}
__device__ __forceinline__ void widen8_fp8(const u32x2& r, float* x) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(r[j], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(r[j], true);
    x[4 * j] = a[0], x[4 * j + 1] = a[1], x[4 * j + 2] = b[0], x[4 * j + 3] = b[1];
  }
}


// What a lane does with each row: its item's two runs, and whether it is rotated.
struct AppendItem {
  int c, d0, d1;
  bool turn;
  __device__ __forceinline__ AppendItem(const AppendArgs& a, int c_) : c(c_) {
    turn = 16 * c < a.rot;
    const bool halves = turn && !a.interleaved;
    d0 = halves ? 8 * c : 16 * c;
    d1 = halves ? 8 * c + a.rot / 2 : 16 * c + 8;
  }
};

struct Turn {                        // cos and sin of an item's 8 pairs
  float c[8], s[8];
};
__device__ __forceinline__ void load_turn(const AppendArgs& a, const AppendItem& it, int64_t p, Turn& r) {
  const float* cp = a.cos + p * a.cos_st + 8 * it.c;
  const float* sp = a.sin + p * a.sin_st + 8 * it.c;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(cp + 4 * j), y = *reinterpret_cast<const f32x4*>(sp + 4 * j);
#pragma unroll
    for (int e = 0; e < 4; ++e) r.c[4 * j + e] = x[e], r.s[4 * j + e] = y[e];
  }
}
// x0 c - x1 s from its exact products (8 by 24 bits), rounded to fp32.
__device__ __forceinline__ float turned_exact(double x0, double c, double x1, double s) {
  return (float)__builtin_fma(x0, c, -(x1 * s));
}
// EXACT for keys, which stay in the cache and in its min / max.  The second rounding,
// to bf16, takes one in some 2^17 of them to the other side of a bf16 step than one
// rounding of the exact value would (those within half an fp32 step of a midpoint);
// with the products rounded to fp32 too it is one in some 2^15.  Queries, most of a
// prompt's rows, take fp32.
template <bool EXACT>
__device__ __forceinline__ void turn_item(const AppendArgs& a, const Turn& r, float* x) {
  float y[16];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x0 = a.interleaved ? x[2 * j] : x[j], x1 = a.interleaved ? x[2 * j + 1] : x[j + 8];
    if constexpr (EXACT) {
      y[j] = turned_exact(x0, r.c[j], x1, r.s[j]);
      y[j + 8] = turned_exact(x1, r.c[j], -x0, r.s[j]);
    } else {
      y[j] = x0 * r.c[j] - x1 * r.s[j];
      y[j + 8] = x1 * r.c[j] + x0 * r.s[j];
    }
  }
  if (a.interleaved) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[2 * j] = y[j], x[2 * j + 1] = y[j + 8];
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = y[j];
  }
}

// Stores the item in its cache row (`to` the row's start); x becomes what the cache then holds.
template <bool FP8>
__device__ __forceinline__ void store_cache(char* to, const AppendItem& it, float scale, float* x) {
  if constexpr (FP8) {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = x[j] / scale;
    const u32x2 r0 = narrow8_fp8(x), r1 = narrow8_fp8(x + 8);
    *reinterpret_cast<u32x2*>(to + it.d0) = r0;
    *reinterpret_cast<u32x2*>(to + it.d1) = r1;
    widen8_fp8(r0, x);
    widen8_fp8(r1, x + 8);
  } else {
    const u32x4 r0 = narrow8(x), r1 = narrow8(x + 8);
    *reinterpret_cast<u32x4*>(to + 2 * it.d0) = r0;
    *reinterpret_cast<u32x4*>(to + 2 * it.d1) = r1;
    widen8(r0, x);
    widen8(r1, x + 8);
  }
}
__device__ __forceinline__ void store_item(uint16_t* row, const AppendItem& it, const float* x) {
  *reinterpret_cast<u32x4*>(row + it.d0) = narrow8(x);
  *reinterpret_cast<u32x4*>(row + it.d1) = narrow8(x + 8);
}
__device__ __forceinline__ void load_item(const uint16_t* row, const AppendItem& it, float* x) {
  widen8(ld16(row + it.d0), x);
  widen8(ld16(row + it.d1), x + 8);
}
template <bool FP8>
__device__ __forceinline__ char* cache_row(const void* base, int64_t sb, int64_t sh, int64_t ss, int id, int h, int off) {
  return static_cast<char*>(const_cast<void*>(base)) + (id * sb + h * sh + off * ss) * (FP8 ? 1 : 2);
}

// IEEE minimum / maximum: a NaN stays, and the order of the values does not matter.
__device__ __forceinline__ float lower(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ float upper(float a, float b) { return __builtin_elementwise_maximum(a, b); }

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

// A span of new tokens: rows t0 .. t0 + n - 1 of sequence b (b = B: rows past the
// last sequence), the first at position p0 (negative: no position).
struct Span {
  int b, t0, n, p0;
};

__device__ __forceinline__ int floor_div(int p, const FastDiv& d) { return p >= 0 ? fast_div(p, d) : -1 - fast_div(-1 - p, d); }

// Span number r of the batch, spans being aligned to multiples of `len`
// positions; false past the last.  Lane l looks at sequence 64 i + l.
__device__ __forceinline__ bool find_span(const AppendArgs& a, int r, int len, const FastDiv& dlen, int lane, Span& s) {
  for (int b0 = 0; b0 <= a.B; b0 += 64) {
    const int b = b0 + lane, bc = min(b, a.B);
    const int c0 = min(max(a.cu[bc], 0), a.T), c1 = b < a.B ? min(max(a.cu[bc + 1], 0), a.T) : a.T;
    const int n = b <= a.B ? max(c1 - c0, 0) : 0;
    const int end = b < a.B ? max(a.c.lens[min(b, a.B - 1)], 0) : 0, first = end - n;
    const int f0 = floor_div(first, dlen);
    const uint32_t mine = n > 0 ? (uint32_t)(floor_div(end - 1, dlen) - f0 + 1) : 0u;
    const uint32_t incl = wave_prefix_sum(mine);
    const int total = __builtin_amdgcn_readlane((int)incl, 63);
    if (r < total) {
      const int l = __ffsll((unsigned long long)__ballot((int)incl > r)) - 1;
      const int j = r - __builtin_amdgcn_readlane((int)(incl - mine), l);
      const int sn = __builtin_amdgcn_readlane(n, l), sc = __builtin_amdgcn_readlane(c0, l);
      const int sf = __builtin_amdgcn_readlane(first, l), s0 = __builtin_amdgcn_readlane(f0, l) + j;
      const int64_t lo = max((int64_t)s0 * len, (int64_t)sf), hi = min(((int64_t)s0 + 1) * len, (int64_t)sf + sn);
      s.b = b0 + l;
      s.p0 = (int)lo;
      s.t0 = sc + (int)(lo - sf);
      s.n = (int)(hi - lo);
      if (s.b == a.B) s.p0 = -0x40000000;          // no sequence: no position
      return true;
    }
    r -= total;
  }
  return false;
}

enum : int { kKeys = 0, kValues = 1, kQueries = 2 };

// The span's rows of NH heads from h0 (nh of them exist), ROWS tokens at a time.
template <int D, bool FP8, int KIND, int NH>
__device__ __forceinline__ void append_span(const AppendArgs& a, const Span& s, int h0, int nh, int lane) {
  constexpr int LPR = D / 16, ROWS = 64 / LPR;
  AppendItem it(a, lane % LPR);
  if (KIND == kValues) it.d0 = 16 * it.c, it.d1 = 16 * it.c + 8;
  const bool fold = KIND == kKeys && a.kmin != nullptr;
  float mn[NH][16], mx[NH][16];
  if (fold) {
#pragma unroll
    for (int u = 0; u < NH; ++u)
#pragma unroll
      for (int j = 0; j < 16; ++j) mn[u][j] = __builtin_inff(), mx[u][j] = kNegInf;
  }
  const uint16_t* src = KIND == kKeys ? a.k : KIND == kValues ? a.v : a.q;
  const int64_t st = KIND == kKeys ? a.k_st : KIND == kValues ? a.v_st : a.q_st;
  const int64_t sh = KIND == kKeys ? a.k_sh : KIND == kValues ? a.v_sh : a.q_sh;
  const int32_t* table = a.c.table + (int64_t)min(s.b, a.B - 1) * a.c.bt_sb;
  int block = -1;                                  // (one block per span where min / max are folded)
  for (int i0 = 0; i0 < s.n; i0 += ROWS) {
    const int i = i0 + lane / LPR;
    const bool row = i < s.n;
    const int t = s.t0 + (row ? i : 0), p = s.p0 + (row ? i : 0);
    const bool placed = row && p >= 0 && p < a.cap;
    const int ps = placed ? p : 0;
    u32x4 raw[NH][2];
#pragma unroll
    for (int u = 0; u < NH; ++u) {
      const uint16_t* x = src + t * st + (h0 + min(u, nh - 1)) * sh;
      raw[u][0] = ld16(x + it.d0);
      raw[u][1] = ld16(x + it.d1);
    }
    int id = -1, off = 0;
    if (KIND != kQueries) {
      const int blk = fast_div(ps, a.c.dbs);
      off = ps - blk * a.c.bs;
      id = table[blk];
    }
    const bool held = placed && id >= 0 && id < a.c.nblocks;
    Turn tr;
    if (KIND != kValues && it.turn) load_turn(a, it, ps, tr);
#pragma unroll
    for (int u = 0; u < NH; ++u) {
      if (u >= nh) break;
      float x[16];
      widen8(raw[u][0], x);
      widen8(raw[u][1], x + 8);
      if (KIND != kValues && it.turn) turn_item<KIND == kKeys>(a, tr, x);
      if (KIND == kQueries) {
        if (!placed) {
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j] = 0.f;
        }
        if (row) store_item(a.q_out + t * a.qo_st + (h0 + u) * a.qo_sh, it, x);
      } else if (held) {
        char* to = KIND == kKeys ? cache_row<FP8>(a.c.k, a.c.k_sb, a.c.k_sh, a.c.k_ss, id, h0 + u, off)
                                 : cache_row<FP8>(a.c.v, a.c.v_sb, a.c.v_sh, a.c.v_ss, id, h0 + u, off);
        if constexpr (KIND == kValues && !FP8) {
          *reinterpret_cast<u32x4*>(to + 2 * it.d0) = raw[u][0];
          *reinterpret_cast<u32x4*>(to + 2 * it.d1) = raw[u][1];
        } else {
          store_cache<FP8>(to, it, KIND == kKeys ? a.k_scale : a.v_scale, x);
        }
        if (fold) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            mn[u][j] = lower(mn[u][j], x[j]);
            mx[u][j] = upper(mx[u][j], x[j]);
          }
        }
      }
    }
    if (fold) {
      const unsigned long long m = __ballot(held);
      if (m) block = __builtin_amdgcn_readlane(id, __ffsll(m) - 1);
    }
  }
  if (!fold || block < 0) return;
  const int p1 = max(s.p0, 0);
  const bool entered = p1 - fast_div(p1, a.c.dbs) * a.c.bs == 0;         // at the block's first row
#pragma unroll
  for (int u = 0; u < NH; ++u) {
    if (u >= nh) break;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      mn[u][j] = fold_rows<LPR>(mn[u][j], lower);
      mx[u][j] = fold_rows<LPR>(mx[u][j], upper);
    }
    if (lane >= LPR) continue;
    uint16_t* pmn = a.kmin + ((int64_t)block * a.Hk + h0 + u) * D;
    uint16_t* pmx = a.kmax + ((int64_t)block * a.Hk + h0 + u) * D;
    if (!entered) {
      float o[16];
      load_item(pmn, it, o);
#pragma unroll
      for (int j = 0; j < 16; ++j) mn[u][j] = lower(mn[u][j], o[j]);
      load_item(pmx, it, o);
#pragma unroll
      for (int j = 0; j < 16; ++j) mx[u][j] = upper(mx[u][j], o[j]);
    }
    store_item(pmn, it, mn[u]);
    store_item(pmx, it, mx[u]);
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

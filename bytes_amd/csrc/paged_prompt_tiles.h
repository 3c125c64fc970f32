// Attention of several new tokens per sequence: which rows a workgroup has, and how a call is
// cut up.  The arithmetic alone, for arguments ARGS with T, B, G, cap, tiles, cu and c.lens (and
// the wave's operations, declared before this): a program on the host can run a wave's 64 lanes
// through it, and a test does.
#pragma once
#include <stdint.h>

namespace bytes_amd {

constexpr int kPromptKeys = 64;      // of a tile of the kernel for many rows

// Row tile number r of the batch: rows r0 .. of sequence b, whose new tokens are rows
// t0 .. t0 + n - 1 of q (b = B: the rows past the last sequence).  False past the last.
struct RowTile {
  int b, t0, n, r0;
  int len;                           // of the sequence, as it is given
  int index;                         // of the tile, in the order of the sequences
};
// The position of the first of the n new tokens of a sequence of `len`; none of them has one where
// `len` is below 0.
__device__ __forceinline__ int first_position(int len, int n) { return max(len, 0) - n; }
template <int ROWS, class ARGS>
__device__ __forceinline__ bool find_tile(const ARGS& a, int r, int lane, RowTile& x) {
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
template <int ROWS, class ARGS>
__device__ __forceinline__ bool find_tile_by_keys(const ARGS& a, int r, int lane, RowTile& x) {
  const int b = min(lane, a.B);
  const int c0 = min(max(a.cu[b], 0), a.T), c1 = lane < a.B ? min(max(a.cu[min(b + 1, a.B)], 0), a.T) : a.T;
  const int len = a.c.lens[min(b, a.B - 1)], n = lane <= a.B ? max(c1 - c0, 0) : 0;
  const int tiles = (n * a.G + ROWS - 1) / ROWS, p0 = lane < a.B ? max(min(max(len, 0), a.cap) - n, 0) : 0;
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
  return x.index < a.tiles;                                // (offsets that overlap have more: no room for their parts)
}

// Row t of q with head g of its group: the row tile that has it, and its row there.  False if
// it is of no sequence, or of a tile past the last that there is room for (offsets that overlap).
template <int ROWS, class ARGS>
__device__ __forceinline__ bool find_row(const ARGS& a, int t, int g, int lane, int& tile, int& row) {
  int tiles = 0;                                           // of the sequences before
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane, bc = min(b, a.B - 1);
    const int c0 = min(max(a.cu[bc], 0), a.T), c1 = min(max(a.cu[bc + 1], 0), a.T);
    const int n = b < a.B ? max(c1 - c0, 0) : 0;
    const uint32_t mine = (uint32_t)((n * a.G + ROWS - 1) / ROWS);
    const uint32_t incl = wave_prefix_sum(mine);
    const unsigned long long in = __ballot(n > 0 && t >= c0 && t < c0 + n);
    if (in) {
      const int l = __ffsll(in) - 1, at = (t - __builtin_amdgcn_readlane(c0, l)) * a.G + g;
      tile = tiles + __builtin_amdgcn_readlane((int)(incl - mine), l) + at / ROWS;
      row = at % ROWS;
      return tile < a.tiles;
    }
    tiles += __builtin_amdgcn_readlane((int)incl, 63);
  }
  return false;
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

// cus: compute units; cap: positions that a table row holds.
inline PromptPlan prompt_plan(int64_t cus, int64_t T, int64_t B, int64_t Hk, int64_t G, int D, int64_t cap, int window,
                              int sinks) {
  PromptPlan p;
  p.nwg = 0, p.nsplit = 1;
  int64_t slots;                                   // that a row tile can see
  // whole row tiles, and one that is not full per sequence (and of the rows past the
  // last); none without rows
  auto cut = [&](int waves) {
    p.waves = waves;
    const int64_t n = T * G / p.rows() + B + 1, most = T * ((G + p.rows() - 1) / p.rows());
    p.tiles = n < most ? n : most;
    p.units = p.tiles * Hk;
    const int64_t see = (int64_t)window + sinks + row_span(p.rows(), G) + 2 * kPromptKeys;
    slots = cap < see ? cap : see;
  };
  cut(1);
  // Up to 32 rows of a sequence read its cache once as one tile (eight sequences of 27K to 64K,
  // 8 KV heads of 128, 24 rows: 248 us, 289 in tiles of 128; 33 rows, two tiles: 472 and 348).
  // (Rows that are read once stream past the caches: with plain loads 276 and not 248.)
  // Where contexts are short, and as many tiles of 32 rows as the CUs hold at once, they take
  // fewer steps one after another (32 heads over 8 of 128: 500 tokens 19.2 and 19.7 us, 500 after 500 28.5 and 38.5,
  // 300 after 930 33.9 and 35.8, 300 after 1200 38.1 and 33.8, 300 after 1700 46.5 and 37.1; 28 over 4, 307 after
  // 975 32.0 and 33.4; 24 over 8, whose units are few, 25 after 1500 16.8 and 21.6, 100 after 1850 29.4 and 29.5;
  // 14 over 2 of 64: 1500 tokens 22.4 and 31.6, 1000 after 1000 27.5 and 32.6).
  const bool lone = T * G <= 32 * B, idle = 2 * p.units < cus;
  const bool fits = T * G * Hk / 32 <= cus * (D == 64 ? 4 : 2) && slots <= (D == 64 || idle ? 2048 : 1280);
  if (lone || fits) {
    // Dealt by the bytes of what a tile sees, which one workgroup reads alone: over 128 KB (one
    // sequence, 8 heads of 128, 256 tokens: whole units 11.4 us, dealt 12.4; 512 tokens 14.7 and
    // 12.3), over 512 KB where the units keep half the CUs busy anyway (16 sequences, 1000 tokens:
    // 22.5 and 24.0; 2000: 38.3 and 36.9), over 2 MB where there are enough for all (60 sequences
    // of 1200 to 2400 tokens: 81 and 91; 30 of 800 to 8000: 118 and 105).
    const int64_t granules = p.units * ((slots + 127) / 128), bytes = slots * D * 4;
    // Several tiles to a sequence: only where the units are few and see over 256 KB (25 tokens after 802, 8
    // heads of 128: 19.9 and 13.6; 100 after 1900, 14 heads over 2 of 64: 21.9 and 15.2; but 100 after 900
    // of 8 heads of 64, 256 KB: 14.2 and 16.3; 307 after 975, 28 heads over 4 of 128: 28.8 and 41.7).
    const int64_t alone = lone ? (p.units >= cus ? 2 << 20 : idle ? 128 << 10 : 512 << 10) : 256 << 10;
    if ((lone || idle) && bytes > alone && granules <= 1 << 24) p.nwg = (int)(granules < cus ? granules : cus);
    return p;
  }
  // (Sequences of hardly 256 rows leave most of such a tile empty: 63 single tokens and a chunk of 512,
  // 8K to 16K of context, 962 us and 845; 31 and a chunk of 2048, 4K to 8K, 391 and 370.)
  const int64_t room = D == 64 ? 2 * cus : cus;    // eight waves of D = 64 are half a CU's
  cut(8);
  if (p.units < room || T * G < 512 * B) cut(4);
  if (p.units >= room) return p;
  // Tiles of D = 64 that hardly differ in their keys fill the CUs from 1.4 to each on (4 x 1000 after 2000, 14
  // heads over 2: 68 us, 84 in two parts); whole prompts leave the CUs to the longest (4000 tokens 86 and
  // 79; 1000 after 15000, 32 heads over 8: 318 and 184).
  if (D == 64 && p.units * (2 * B * cap - (T < B * cap ? T : B * cap)) / (2 * B * cap) >= cus * 7 / 5) return p;
  // parts: as many as the CUs hold at once, by the tiles that there are (half of a sequence's last one),
  // none of fewer than 8 key tiles
  const int64_t units = ((T * G + p.rows() - 1) / p.rows() + (B - 1) / 2) * Hk;
  const int64_t want = 2 * room / units, most = slots / (8 * kPromptKeys);
  const int64_t n = want < most ? want : most;
  p.nsplit = (int)(n < 1 ? 1 : n > 128 ? 128 : n);
  return p;
}

}  // namespace bytes_amd

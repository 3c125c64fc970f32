// Causal attention of several new tokens per sequence over a paged cache, whole or
// within a sliding window and the first tokens (sinks).
//
//   out[i, h] = sum_t p_t vs_t v_t / sum_t p_t,  p_t = exp(scale * ks_t * (q . k_t) - max)
//
// for the query at position p = n - m + i of a sequence of n tokens, m of them new, over
// the tokens t <= p whose block exists and, with a window w and s sinks, t > p - w or
// t < s.  ks_t, vs_t: the scales of token t's block (or one for the tensor).
//
// Rows: the G query heads of a KV head read the same keys, so a workgroup's rows are
// (token, head of the group) pairs, token major: 32 to a wave.  Keys come in tiles of 64,
// staged through LDS for the workgroup.
//   S^T[t][row] = K[t][:] . Q[row][:]   32x32x16 MFMA; A = K rows from LDS, B = Q in registers
//   softmax per row: a lane has half of a row's keys, its partner lane + 32 the others
//   O^T[d][row] += V^T[d][t] P^T[t][row]  A = V read transposed (ds_read_b64_tr_b16)
// The output registers of S^T hold, for lane half e, the keys 8 g + 4 e .. + 3: the second
// product takes its keys in that order, so P goes from one to the other without leaving
// the lane.  P is rounded to bf16 (nearest even, 2^-8 of a weight at most, as much as the
// result's own rounding: error against 64 bits 0.0023 of the norm, 0.0017 of it the
// result's rounding; with a second bf16 part, which makes three products of two, 0.0017, and a 16K prompt takes
// 3100 us for 2150, a window of 32K 808 for 581, 3K chunks over e4m3 265 for 205); its sum stays in fp32.
// The running maximum moves only where a score passes it by 2^8, so most tiles leave the
// accumulators as they are; weights are then up to 2^8, which changes no relative error.
//
// Bound by products and softmax one after the other: a 16K prompt of 32 heads over 8 of 128 takes 2080 to 2250
// us by card, 980 to 1060 TFLOP/s, where a 16384^3 bf16 product of the library reaches 1400 and products alone,
// nothing loaded or stored, 2060.  A wave's tile is 32 matrix instructions (1024 clocks) and 207 others (some 1200,
// an exponential counted as four), and takes 2290 of its SIMD: the two waves there hardly work beside each
// other.  The matrix units are busy for 45%, LDS is read in 34% and in conflict for 11%, the clock falls to 1.9 GHz.
// Left out one at a time, of 2240 then (not answers): loads to LDS 1870 us, exponentials 2080, reads of K
// 1870, of V 2060, the second product 1630, the first 1600; none of reads and loads 1370.  No faster:
// products of one tile among the softmax of the other in one wave 2330, 64 rows per wave 3840
// (registers), raised wave priority, dot products for the sums, one tile more on its way.  Over e4m3 with
// scales 2260 (over e4m3 with one scale 2090): 64 multiplications more per lane and tile; folding the
// keys' into the exponent's multiply-add takes 3% longer.
//
// A workgroup has 256 rows, eight waves, one to a CU, where that makes units for all CUs, and else
// 128, two to a CU: 16K prompt 2050 and 2090, last 4096 of 16K 889 and 944, a 4096 prompt 147 and 161;
// 4 x 1024 after 476 each, which is two rounds of the larger tiles, 98 and 93 (when a batch's
// tiles started in the order of its sequences; see find_tile_by_keys).
#include "paged_prompt.h"

namespace bytes_amd {

constexpr int kKeys = kPromptKeys;

// NW waves of 32 rows.
template <int D, int TYPE, bool HALVES, int NW>
__global__ __launch_bounds__(NW * 64, NW == 4 && D == 128 && TYPE == kBf16Cache && !HALVES ? 1 : 2) void paged_prompt_kernel(PromptArgs a) {
  constexpr bool BYTES = TYPE != kBf16Cache, SCALED = TYPE >= kE4m3Blocks;
  using Elem = typename std::conditional<BYTES, uint8_t, uint16_t>::type;
  constexpr int EPC = 16 / (int)sizeof(Elem), CPR = D / EPC;         // elements per chunk, chunks per row
  constexpr int RPW = 64 / CPR, RPI = NW * RPW, NI = RPI < kKeys ? kKeys / RPI : 1;
  static_assert(RPW <= 16, "a wave's rows of one instruction lie in 16 of a block");
  constexpr int KK = D / 16, DB = D / 32, VT = kKeys * D * 2;
  __shared__ __attribute__((aligned(16))) char smem[2][2 * VT];      // [buffer][K, V]
  // scales of a tile's tokens: in scalar registers where 16 of them share a block, else in LDS
  constexpr bool SCALES_LDS = SCALED && !HALVES;
  __shared__ float sc[2][SCALES_LDS ? 128 : 1];
  __shared__ int odd_tiles;                        // some had an infinity or NaN left out

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, e = lane >> 5;
  const int per = a.Hk * a.nsplit;
  const int tile = a.tiles - 1 - (int)blockIdx.x / per;              // the last rows, which see most, first
  const int rest = (int)blockIdx.x % per, split = fast_div(rest, a.dHk), hk = rest - split * a.Hk;
  RowTile x;
  if (a.by_keys) {
    if (!find_tile_by_keys<NW * 32>(a, a.tiles - 1 - tile, lane, x)) return;
  } else if (!find_tile<NW * 32>(a, tile, lane, x)) return;
  const int row = x.r0 + w * 32 + l32, rows = x.n * a.G;
  const bool exists = row < rows;
  const int i = fast_div(exists ? row : 0, a.dG), h = hk * a.G + (exists ? row : 0) - i * a.G;
  uint16_t* out = a.out + (int64_t)(x.t0 + i) * a.o_st + (int64_t)h * a.o_sh;
  if (x.b == a.B) {                                // rows of no sequence
    if (exists && split == 0) {
      for (int d = e * (D / 2); d < (e + 1) * (D / 2); d += 8) *reinterpret_cast<u32x4*>(out + d) = u32x4{0, 0, 0, 0};
    }
    return;
  }
  // (what all lanes share goes to scalar registers)
  auto same = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  const int p0 = same(first_position(x.len, x.n));
  const int p = p0 + i;
  const bool placed = exists && p >= 0 && p < a.cap;
  const int first = fast_div(x.r0, a.dG), last = min(fast_div(x.r0 + NW * 32 - 1, a.dG), x.n - 1);
  const int p_lo = same(max(p0 + first, 0)), p_hi = same(min(p0 + last, a.cap - 1));
  // this wave's positions
  const int wl = fast_div(min(x.r0 + w * 32, rows - 1), a.dG), wh = fast_div(min(x.r0 + w * 32 + 31, rows - 1), a.dG);
  const bool wave_any = x.r0 + w * 32 < rows;
  const int w_lo = same(max(p0 + wl, 0)), w_hi = same(wave_any ? min(p0 + wh, a.cap - 1) : -1);
  // keys: tiles of the sinks, then from the window's first one on
  const int end = max(p_hi + 1, 0), lo_key = max(p_lo - a.window + 1, 0);
  const int near_tiles = (min(a.sinks, end) + kKeys - 1) & -kKeys;
  const int gap = max((lo_key & -kKeys) - near_tiles, 0);
  const int ntiles = p_lo > p_hi ? 0 : (end - gap + kKeys - 1) / kKeys;
  const int j0 = same((int)((int64_t)ntiles * split / a.nsplit)), j1 = same((int)((int64_t)ntiles * (split + 1) / a.nsplit));

  bf16x8 qb[KK];
  {
    const uint16_t* qp = a.q + (int64_t)(x.t0 + i) * a.q_st + (int64_t)h * a.q_sh + e * 8;
    const uint32_t sign = a.flip ? 0x80008000u : 0u;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      u32x4 raw = ld16_live(qp + kk * 16, placed);
      raw ^= u32x4{sign, sign, sign, sign};
      qb[kk] = __builtin_bit_cast(bf16x8, raw);
    }
  }
  float m_run = kNegInf, l_run = 0.f;
  f32x16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int u = 0; u < 16; ++u) acc[db][u] = 0.f;

  const int32_t* table = a.c.table + (int64_t)x.b * a.c.bt_sb;
  const Elem* kb = static_cast<const Elem*>(a.c.k) + hk * a.c.k_sh;
  const Elem* vb = static_cast<const Elem*>(a.c.v) + hk * a.c.v_sh;
  const int r_in = lane / CPR, col = lane % CPR;
  // HALVES: this lane's row among the 16 that its wave's instructions read of, and its column
  const int row16 = (w * RPW & 15) + r_in;
  const int kcol = BYTES ? col : kswz<D>(w * RPW + r_in, col), vcol = BYTES ? col : vswz<D>(w * RPW + r_in, col);
  const uint32_t ko = row16 * (int)a.c.k_ss + kcol * EPC, vo = row16 * (int)a.c.v_ss + vcol * EPC;
  static_assert(RPI % 8 == 0 && (D / 8) % 8 == 0 && (RPI % (D / 8) == 0 || BYTES), "the swizzle is that of the instruction's first row");
  auto start = [&](int j) { return j * kKeys < near_tiles ? j * kKeys : j * kKeys + gap; };
  // tile j's table entries: lane l's token is start(j) + l
  auto fetch = [&](int j) {
    PagedIds t;
    const int s = start(j) + lane, sc_ = min(s, end - 1);
    const int place = fast_div(max(sc_, 0), a.c.dbs);
    t.ok = j < j1 && s < end;
    t.off = t.ok ? s - place * a.c.bs : 0;
    t.id = table[place];
    return t;
  };
  auto settle = [&](PagedIds& t) {
    const bool in = t.id >= 0 && t.id < a.c.nblocks;
    t.ok = t.ok && in;
    t.id = in ? t.id : 0;
  };
  // Tile j's rows: bf16 ones go to LDS on their own (lane l's 16 bytes to the wave's place + 16 l,
  // so the swizzle is in the column that it reads), bytes to registers first.
  constexpr bool DMA = !BYTES && HALVES;
  constexpr int NR = DMA ? 1 : NI;
  u32x4 kr[NR], vr[NR];
  auto issue = [&](const PagedIds& t, int to) {
    // every lane its own token's place: 64-bit products once a tile
    const int64_t ka = t.id * a.c.k_sb + t.off * a.c.k_ss, va = t.id * a.c.v_sb + t.off * a.c.v_ss;
    auto at = [](int64_t x, int l) {
      return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32 |
                       (uint32_t)__builtin_amdgcn_readlane((int)x, l));
    };
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      const int base = u * RPI + w * RPW;          // this wave's rows of the instruction
      if (RPI > kKeys && base >= kKeys) break;
      if constexpr (HALVES) {                      // all in one block: one scalar base
        const Elem *kp = kb + at(ka, base & ~15), *vp = vb + at(va, base & ~15);
        if constexpr (DMA) {
          char* to_k = smem[to] + base * (D * 2);
          lds_dma16<false>(buf_rsrc(kp, 0xFFFFFFFFu), to_k, 2 * ko);
          lds_dma16<false>(buf_rsrc(vp, 0xFFFFFFFFu), to_k + VT, 2 * vo);
        } else {
          kr[u] = ld16(kp + ko);
          vr[u] = ld16(vp + vo);
        }
      } else {
        kr[u] = ld16(kb + __shfl(ka, base + r_in, 64) + col * EPC);
        vr[u] = ld16(vb + __shfl(va, base + r_in, 64) + col * EPC);
        asm volatile("" ::: "memory");             // (one row's addresses in registers at a time)
      }
    }
  };
  float kscale = 0.f, vscale = 0.f, kg[4], vg[4];
  auto scales = [&](const PagedIds& t) {
    if constexpr (SCALED) {
      const float x = a.ks[t.id * a.ks_sb + hk * a.ks_sh], y = a.vs[t.id * a.vs_sb + hk * a.vs_sh];
      kscale = t.ok ? x : 0.f;
      vscale = t.ok ? y : 0.f;
    }
  };
  // They are in buffer `to` after this and a barrier.  CHECK, tiles that some rows do not see
  // whole: values of slots that are no token become 0, as do infinities and NaN, which no
  // weight of 0 would take away; returns whether this lane met any.
  auto finish = [&](int to, uint64_t named, auto check) {
    constexpr bool CHECK = decltype(check)::value;
    char *kst = smem[to], *vst = kst + VT;
    bool odd = false;
    if constexpr (DMA) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if constexpr (CHECK) {
#pragma unroll
        for (int u = 0; u < NI; ++u) {
          const int rr = u * RPI + w * RPW + r_in;
          if (RPI > kKeys && rr >= kKeys) break;
          u32x4* at = reinterpret_cast<u32x4*>(vst + (u * RPI + w * RPW) * (D * 2) + lane * 16);
          const u32x4 v = *at;
          *at = (named >> rr) & 1 ? finite_only(v, odd) : u32x4{0, 0, 0, 0};
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < NI; ++u) {
        const int rr = u * RPI + w * RPW + r_in;
        if (RPI > kKeys && rr >= kKeys) break;
        if constexpr (CHECK) {
          const uint32_t keep = (named >> rr) & 1 ? ~0u : 0u;
          vr[u] &= u32x4{keep, keep, keep, keep};
        }
        if constexpr (BYTES) {
          u32x4 k0, k1, v0, v1;
          bytes16_to_bf16<TYPE == kInt8Blocks>(kr[u], k0, k1);
          bytes16_to_bf16<TYPE == kInt8Blocks>(vr[u], v0, v1);
          if constexpr (CHECK && TYPE != kInt8Blocks) v0 = finite_only(v0, odd), v1 = finite_only(v1, odd);
          *reinterpret_cast<u32x4*>(kst + rr * (D * 2) + kswz<D>(rr, 2 * col) * 16) = k0;
          *reinterpret_cast<u32x4*>(kst + rr * (D * 2) + kswz<D>(rr, 2 * col + 1) * 16) = k1;
          *reinterpret_cast<u32x4*>(vst + rr * (D * 2) + vswz<D>(rr, 2 * col) * 16) = v0;
          *reinterpret_cast<u32x4*>(vst + rr * (D * 2) + vswz<D>(rr, 2 * col + 1) * 16) = v1;
        } else {
          *reinterpret_cast<u32x4*>(kst + rr * (D * 2) + kswz<D>(rr, col) * 16) = kr[u];
          *reinterpret_cast<u32x4*>(vst + rr * (D * 2) + vswz<D>(rr, col) * 16) = CHECK ? finite_only(vr[u], odd) : vr[u];
        }
        asm volatile("" ::: "memory");             // (one row's conversion in registers at a time)
      }
    }
    if constexpr (SCALES_LDS) {
      if (w == 0) sc[to][lane] = kscale, sc[to][64 + lane] = vscale;
    }
    if constexpr (SCALED && HALVES) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        kg[g] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(kscale), 16 * g));
        vg[g] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vscale), 16 * g));
      }
    }
    return odd;
  };
  // Whether all rows at positions lo .. hi see all of the tile at t0.
  auto all_see = [&](int t0, int lo, int hi) {
    return t0 + kKeys - 1 <= lo && (t0 > hi - a.window || t0 + kKeys <= a.sinks);
  };

  // The tile's keys that this lane's row sees.
  auto seen = [&](int t0, uint64_t named) {
    return placed ? named & low_bits(p - t0 + 1) & (~low_bits(p - a.window + 1 - t0) | low_bits(a.sinks - t0)) : 0ull;
  };
  // One staged tile.
  auto compute = [&](int from, int t0, uint64_t named) {
    const char *kst = smem[from], *vst = kst + VT;
    // keys that all of the wave's rows see
    const bool whole = named == ~0ull && all_see(t0, w_lo, w_hi);
    f32x16 s[2];
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int u = 0; u < 16; ++u) s[blk][u] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const int rr = blk * 32 + l32;
        const bf16x8 ka = __builtin_bit_cast(
            bf16x8, *reinterpret_cast<const u32x4*>(kst + rr * (D * 2) + kswz<D>(rr, kk * 2 + e) * 16));
        s[blk] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka, qb[kk], s[blk], 0, 0, 0);
      }
    // four reads of K ahead of the products that take them
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int z = 0; z < 2 * KK - 4; ++z) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
    if constexpr (SCALED) {
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int u = 0; u < 16; ++u)
          s[blk][u] *= SCALES_LDS ? sc[from][blk * 32 + (u >> 2) * 8 + e * 4 + (u & 3)] : kg[2 * blk + (u >> 3)];
    }
    if (!whole) {
      const uint64_t see = seen(t0, named);
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const uint32_t m = (uint32_t)(see >> (32 * blk)) >> (4 * e);
#pragma unroll
        for (int u = 0; u < 16; ++u)
          if (!((m >> (8 * (u >> 2) + (u & 3))) & 1u)) s[blk][u] = kNegInf;
      }
    }
    float mx = kNegInf;
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int u = 0; u < 16; ++u) mx = __builtin_elementwise_maximum(mx, s[blk][u]);
    mx = half_max(mx);
    if (__any((mx - m_run) * a.scale_log2 > kSlack)) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = m_new == kNegInf ? 0.f : fast_exp2((m_run - m_new) * a.scale_log2);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int u = 0; u < 16; ++u) acc[db][u] *= alpha;
    }
    const float mc = m_run == kNegInf ? 0.f : m_run * a.scale_log2;
    auto weight = [&](float x) { return fast_exp2(__builtin_fmaf(x, a.scale_log2, -mc)); };
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      bf16x8 pb;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        float pk = weight(s[kk >> 1][(kk & 1) * 8 + u]);
        l_run += pk;
        if constexpr (SCALES_LDS) pk *= sc[from][64 + kk * 16 + (u >> 2) * 8 + e * 4 + (u & 3)];
        else if constexpr (SCALED) pk *= vg[kk];
        pb[u] = (__bf16)pk;
      }
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        u32x2 t[2];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int rr = kk * 16 + hf * 8 + e * 4 + ((lane >> 2) & 3), d = db * 32 + (lane & 16) + (lane & 3) * 4;
          t[hf] = tr16(vst + rr * (D * 2) + vswz<D>(rr, d >> 3) * 16 + (d & 7) * 2);
        }
        acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8, u32x4{t[0][0], t[0][1], t[1][0], t[1][1]}), pb, acc[db], 0, 0, 0);
      }
    }
  };

  if (j0 < j1) {
    if (threadIdx.x == 0) odd_tiles = 0;
    PagedIds next = fetch(j0);
    settle(next);
    uint64_t named = 0, named_next = __ballot(next.ok);
    scales(next);
    issue(next, j0 & 1);
    next = fetch(j0 + 1);
    __syncthreads();
    auto done = [&](int j) {                       // tile j is in LDS
      const int t0 = start(j);
      if (named_next == ~0ull && all_see(t0, p_lo, p_hi)) finish(j & 1, named_next, std::false_type{});
      else if (__any(finish(j & 1, named_next, std::true_type{})) && lane == 0) odd_tiles = 1;
      named = named_next;
      lds_barrier();
    };
    done(j0);
    for (int j = j0; j < j1; ++j) {
      const bool more = j + 1 < j1;
      if (more) {                                  // (the other buffer was last read before the barrier)
        settle(next);
        named_next = __ballot(next.ok);
        scales(next);
        issue(next, (j + 1) & 1);
        next = fetch(j + 2);
      }
      const int t0 = start(j);
      if (t0 <= w_hi) compute(j & 1, t0, named);
      if (more) done(j + 1);
    }
    if (TYPE != kInt8Blocks && odd_tiles) {
      // Infinities and NaN that were left out: rows that see them take them, others do not.
      // Again through the tiles that some row does not see whole, without weights: any
      // above 0 gives the same.
      for (int j = j0; j < j1; ++j) {
        PagedIds t = fetch(j);
        settle(t);
        const uint64_t there = __ballot(t.ok);
        const int t0 = start(j);
        if (there == ~0ull && all_see(t0, p_lo, p_hi)) continue;
        const uint64_t see = seen(t0, there);
        for (int k = 0; k < kKeys; ++k) {
          if (!((there >> k) & 1)) continue;
          const int id = __builtin_amdgcn_readlane(t.id, k), off = __builtin_amdgcn_readlane(t.off, k);
          const Elem* vp = vb + (int64_t)id * a.c.v_sb + (int64_t)off * a.c.v_ss;
          const bool mine = (see >> k) & 1;
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int u = 0; u < 16; ++u) {
              const int d = db * 32 + 8 * (u >> 2) + 4 * e + (u & 3);
              const uint32_t raw = vp[d];
              const float v = BYTES ? ((raw & 0x7Fu) == 0x7Fu ? __builtin_nanf("") : 0.f) : __uint_as_float(raw << 16);
              if (mine && (__float_as_uint(v) & 0x7F800000u) == 0x7F800000u) acc[db][u] += v;
              asm volatile("" ::: "memory");       // (few registers for a path that is hardly taken)
            }
        }
      }
    }
  }

  l_run = half_sum(l_run);
  if (!placed) l_run = 0.f;                        // a row without a position gets zeros
  if (a.nsplit > 1) {
    const size_t slot = (((size_t)x.index * a.Hk + hk) * a.nsplit + split) * (NW * 32) + w * 32 + l32;
    if (!exists) return;
    float* pa = a.part_acc + slot * D;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(pa + db * 32 + 8 * g + 4 * e) =
            f32x4{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
    if (e == 0)
      reinterpret_cast<float2*>(a.part_ml)[slot] = make_float2(m_run == kNegInf ? kNegInf : m_run * a.scale_log2, l_run);
    return;
  }
  if (!exists) return;
  const float by = l_run == 0.f ? 0.f : a.v_scale / l_run;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) store_bf16x4(out + db * 32 + 8 * g + 4 * e, acc[db], 4 * g, by);
}

// Joins the parts of a row's keys: one wave per (row of q, query head, 64 dims).
template <int D, int NW>
__global__ __launch_bounds__(64) void paged_prompt_join_kernel(PromptArgs a) {
  constexpr int ROWS = NW * 32;
  constexpr int NSL = D / 64;
  const int lane = threadIdx.x, item = lane & 15, grp = lane >> 4;
  const int slice = blockIdx.y % NSL, h = blockIdx.y / NSL, t = blockIdx.x;
  const int hk = fast_div(h, a.dG);
  int tile, row;
  if (!find_row<ROWS>(a, t, h - hk * a.G, lane, tile, row)) return;
  const size_t base = ((size_t)tile * a.Hk + hk) * a.nsplit * ROWS + row;
  auto slot = [&](int u) { return base + (size_t)u * ROWS; };
  paged_join<4>(a.nsplit, lane, slot, reinterpret_cast<const float2*>(a.part_ml),
                reinterpret_cast<const f32x4*>(a.part_acc) + slice * 16 + item, D / 4, [&](const f32x4& A, float L) {
                  if (grp == 0)
                    paged_store(a.out + (int64_t)t * a.o_st + (int64_t)h * a.o_sh + slice * 64 + item * 4, A, L, a.v_scale);
                });
}

template <int D, int TYPE, bool HALVES>
static int launch_prompt(const PromptArgs& a, const PromptPlan& plan, hipStream_t st) {
  const dim3 grid((unsigned)(plan.units * plan.nsplit)), block(plan.waves * 64);
  if (plan.waves == 8) hipLaunchKernelGGL((paged_prompt_kernel<D, TYPE, HALVES, 8>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((paged_prompt_kernel<D, TYPE, HALVES, 4>), grid, block, 0, st, a);
  int rc = (int)hipGetLastError();
  if (rc || plan.nsplit < 2) return rc;
  const dim3 jgrid((unsigned)a.T, (unsigned)(a.Hk * a.G * (D / 64)));
  if (plan.waves == 8) hipLaunchKernelGGL((paged_prompt_join_kernel<D, 8>), jgrid, dim3(64), 0, st, a);
  else hipLaunchKernelGGL((paged_prompt_join_kernel<D, 4>), jgrid, dim3(64), 0, st, a);
  return (int)hipGetLastError();
}
template <int TYPE>
static int launch_prompt_of(const PromptArgs& a, int D, const PromptPlan& plan, hipStream_t st) {
  const bool halves = paged_halves(a.c);
  if (D == 128) return halves ? launch_prompt<128, TYPE, true>(a, plan, st) : launch_prompt<128, TYPE, false>(a, plan, st);
  return halves ? launch_prompt<64, TYPE, true>(a, plan, st) : launch_prompt<64, TYPE, false>(a, plan, st);
}

}  // namespace bytes_amd

using namespace bytes_amd;

extern "C" {

int bytes_paged_prompt_workspace_size(int T, int B, int Hq, int Hk, int D, int block_size, int max_blocks, int window,
                                      int sinks, size_t* bytes) {
  if (!bytes || T < 0 || B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 || (D != 64 && D != 128) || window <= 0 || sinks < 0)
    return (int)hipErrorInvalidValue;
  const int rc = paged_check(block_size, 1, max_blocks);
  if (rc) return rc;
  if (T == 0) {
    *bytes = 0;
    return 0;
  }
  *bytes = prompt_plan(device_cu_count(), T, B, Hk, Hq / Hk, D, (int64_t)max_blocks * block_size, window, sinks).workspace(D);
  return 0;
}

int bytes_paged_prompt_attn(const void* q, int64_t q_st, int64_t q_sh, const void* k_paged, int64_t k_sb, int64_t k_sh,
                            int64_t k_ss, const void* v_paged, int64_t v_sb, int64_t v_sh, int64_t v_ss, int kv_type,
                            const void* k_scales, int64_t ks_sb, int64_t ks_sh, const void* v_scales, int64_t vs_sb,
                            int64_t vs_sh, const void* block_table, int64_t bt_sb, const void* context_lens,
                            const void* cu_seqlens, void* out, int64_t o_st, int64_t o_sh, int T, int B, int Hq, int Hk,
                            int D, int block_size, int num_blocks, int max_blocks, int window, int sinks, float scale,
                            float v_scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !k_paged || !v_paged || !block_table || !context_lens || !cu_seqlens || !out || T < 0 || B <= 0 || Hk <= 0 ||
      Hq <= 0 || Hq % Hk != 0 || (D != 64 && D != 128) || max_blocks <= 0 || window <= 0 || sinks < 0 ||
      kv_type < kBf16Cache || kv_type > kInt8Blocks || (kv_type >= kE4m3Blocks && (!k_scales || !v_scales)))
    return (int)hipErrorInvalidValue;
  const int rc0 = paged_check(block_size, num_blocks, max_blocks);
  if (rc0) return rc0;
  if (T == 0) return 0;
  const int64_t G = Hq / Hk;
  const PromptPlan plan = prompt_plan(device_cu_count(), T, B, Hk, G, D, (int64_t)max_blocks * block_size, window, sinks);
  PromptArgs a = {};
  a.window = window < (1 << 30) ? window : (1 << 30), a.sinks = sinks < (1 << 30) ? sinks : (1 << 30);
  a.nsplit = plan.nsplit;
  if ((int64_t)T * G + plan.rows() > 0x7FFFFFFF || plan.units * plan.nsplit > 0x7FFFFFFF || T > (1 << 30) ||
      (int64_t)Hq * (D / 64) > 65535)
    return (int)hipErrorInvalidConfiguration;
  if (plan.workspace(D) && (!workspace || workspace_bytes < plan.workspace(D))) return (int)hipErrorInvalidValue;
  a.c.k = k_paged, a.c.k_sb = k_sb, a.c.k_sh = k_sh, a.c.k_ss = k_ss;
  a.c.v = v_paged, a.c.v_sb = v_sb, a.c.v_sh = v_sh, a.c.v_ss = v_ss;
  a.c.table = static_cast<const int32_t*>(block_table), a.c.bt_sb = bt_sb;
  a.c.lens = static_cast<const int32_t*>(context_lens);
  a.c.bs = block_size, a.c.nblocks = num_blocks, a.c.width = max_blocks;
  a.c.dbs = make_fastdiv((uint32_t)block_size);
  a.q = static_cast<const uint16_t*>(q), a.q_st = q_st, a.q_sh = q_sh;
  a.out = static_cast<uint16_t*>(out), a.o_st = o_st, a.o_sh = o_sh;
  a.cu = static_cast<const int32_t*>(cu_seqlens);
  a.ks = static_cast<const float*>(k_scales), a.ks_sb = ks_sb, a.ks_sh = ks_sh;
  a.vs = static_cast<const float*>(v_scales), a.vs_sb = vs_sb, a.vs_sh = vs_sh;
  a.part_ml = static_cast<float*>(workspace);
  a.part_acc = a.part_ml + (plan.nwg ? (size_t)plan.nwg * 2 : (size_t)plan.units * plan.nsplit) * plan.rows() * 2;
  a.by_keys = B > 1 && B < 64;
  a.nwg = plan.nwg, a.span = (int)row_span(32, G);
  a.T = T, a.B = B, a.Hk = Hk, a.G = (int)G, a.D = D;
  a.cap = max_blocks * block_size;
  a.tiles = (int)plan.tiles;
  a.flip = scale < 0.f ? 1 : 0;
  // (at least the smallest normal number: times -inf, a masked score, it is -inf)
  a.scale_log2 = fmaxf(fabsf(scale) * kLog2e, 1.17549435e-38f);
  a.v_scale = scale == scale ? v_scale : scale;    // (no number: NaN in every row that sees a token)
  a.dHk = make_fastdiv((uint32_t)Hk), a.dG = make_fastdiv((uint32_t)G);
  a.dnwg = make_fastdiv((uint32_t)(a.nwg ? a.nwg : 1));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (plan.waves == 1) return launch_prompt_few(a, kv_type, plan, st);
  switch (kv_type) {
    case kBf16Cache: return launch_prompt_of<kBf16Cache>(a, D, plan, st);
    case kFp8Cache: return launch_prompt_of<kFp8Cache>(a, D, plan, st);
    case kE4m3Blocks: return launch_prompt_of<kE4m3Blocks>(a, D, plan, st);
    default: return launch_prompt_of<kInt8Blocks>(a, D, plan, st);
  }
}

}  // extern "C"

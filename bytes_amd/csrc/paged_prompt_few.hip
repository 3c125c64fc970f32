// paged_prompt.hip's attention where rows are few: draft tokens over long contexts, and
// prompts too short to fill the chip with row tiles.
//
// A workgroup has 32 rows of one KV head, and its four waves take the key tiles, 32 keys
// each, in turn, with rows and tiles in registers and LDS of their own (paged_wave_tiles), so
// that there are four times as many tiles on their way as rows in work, and no barrier
// until the waves' sums are merged through LDS in wave order.  The products, the softmax and
// what infinite values do are those of paged_prompt.hip.
//
// Short contexts: a workgroup for each unit, 32 rows of a KV head.  Long ones: a sequence's
// units have as many granules of 128 keys as its last rows see, and those of all units, in
// the order (sequence, row tile, KV head, key), are dealt to a fixed grid in equal runs, as
// paged_split.h does for single tokens (with an equal number of workgroups for each, eight
// sequences of 27K to 64K wait for the longest: 24 rows of 8 heads of 128, 322 us and 243).  A
// run's parts of units leave (max, sum, values) in fp32 for a second launch that joins them in
// key order.
// Bound by memory there over bf16: 1.52 GB in those 243 us, 6.3 TB/s, where streaming reads reach 7.1.  Over 8 bits half the
// bytes take 182 to 210 us (e4m3 with one scale 182, with block scales 191, int8 208): loads, conversion, LDS, products and
// softmax of a tile follow one another in its wave, with two waves to a SIMD (vector instructions 29%, matrix 15%,
// LDS 44% of the time).
// Short contexts are bound by what follows one another: row tile, table, keys, products (three
// prompts of 200 to 300, 14 heads over 2 of 64, window 128: 9.6 us; tiles of 128 rows 13.6).
#include "paged_prompt.h"

namespace bytes_amd {

constexpr int kFewWaves = 4;

// The codes of four e4m3 numbers with NaN made 0; odd: whether there were any.
__device__ __forceinline__ uint32_t numbers_only(uint32_t x, bool& odd) {
  const uint32_t nan = (((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;       // 1 in the bytes that are
  odd = odd | (nan != 0);
  return x & ~(nan * 0xFFu);
}

// A weight as the sum of two bf16 numbers, off by at most 2^-16 of it, so that a draft's row is as near its definition
// as the same token's decode (0.0017 of the norm, the result's own rounding; 0.0023 with one).  INF as in
// paged_tile: both positive wherever the weight is.  Weights in one, two and all three parts, us: eight drafts over
// 27K to 64K, 24 heads over 8 of 128, bf16 248, 248 and 255, e4m3 with scales 187, 203 and 221, int8 204, 219
// and 231; one prompt of 500 tokens, 32 heads over 8 of 128, 17.5, 18.3 and 19.3, 300 after 1200 34.2, 37.2 and 40.1.
struct WeightParts {
  uint32_t hi;
  float lo;
};
// Weight number j of eight into its pairs w; even: the one before, of which it is the second.
template <bool INF>
__device__ __forceinline__ void put_weight(float p, int j, WeightParts& even, u32x4 (&w)[2]) {
  const uint32_t hi = leading8<INF>(p);
  const float lo = p - __uint_as_float(hi);                // (exact)
  if (j & 1) {
    w[0][j >> 1] = upper16(even.hi, hi);
    w[1][j >> 1] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)even.lo, (__bf16)lo});
  } else {
    even = {hi, lo};
  }
}

constexpr int kFewGranule = kFewWaves * 32;        // keys

// Sequence b: its new tokens are rows t0 .. t0 + n - 1 of q.
struct FewSeq {
  int t0, n, len;
  int tiles, gran;                   // row tiles; granules of each, at most what its rows see
  __device__ __forceinline__ uint32_t work() const { return (uint32_t)tiles * (uint32_t)gran; }
};
__device__ __forceinline__ void few_count(const PromptArgs& a, FewSeq& x) {
  const uint32_t held = (uint32_t)min(max(x.len, 0), a.cap);
  const uint32_t near_tiles = (min((uint32_t)a.sinks, held) + 31u) & ~31u;
  const uint32_t slots = min(held, near_tiles + (uint32_t)a.window + (uint32_t)a.span + 31u);
  x.tiles = (x.n * a.G + 31) / 32;
  x.gran = (int)max(1u, (slots + kFewGranule - 1) / kFewGranule);
}
__device__ __forceinline__ FewSeq few_seq(const PromptArgs& a, int b) {
  FewSeq x;
  x.t0 = min(max(a.cu[b], 0), a.T);
  x.n = max(min(max(a.cu[b + 1], 0), a.T) - x.t0, 0);
  x.len = a.c.lens[b];
  few_count(a, x);
  return x;
}

// All units' granules, dealt in equal runs.  Lane l sums those of sequences l * per .. + per - 1 (of one
// KV head); offsets that overlap count no more than kMostWork in each.
constexpr uint32_t kMostWork = 1u << 24;           // (the host deals no more than that)
struct FewDeal {
  uint32_t mine, incl;
  int per, total;                    // granules of the batch
  FewSeq own;                        // of the lane: its only sequence where per == 1

  __device__ __forceinline__ FewDeal(const PromptArgs& a, int lane) {
    per = (a.B + 63) / 64;
    mine = 0u;
    for (int i = 0; i < per; ++i) {
      const int b = lane * per + i;
      own = few_seq(a, min(b, a.B - 1));
      if (b < a.B) mine = min(mine + min(own.work(), kMostWork), kMostWork);
    }
    incl = wave_prefix_sum(mine);
    total = (int)min((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)incl, 63) * (uint32_t)a.Hk, (uint64_t)0x7FFFFFFF);
  }
  __device__ __forceinline__ FewSeq seq(const PromptArgs& a, int b) const {
    if (per != 1) return few_seq(a, b);
    FewSeq x;
    x.t0 = __builtin_amdgcn_readlane(own.t0, b);
    x.n = __builtin_amdgcn_readlane(own.n, b);
    x.len = __builtin_amdgcn_readlane(own.len, b);
    x.tiles = __builtin_amdgcn_readlane(own.tiles, b);
    x.gran = __builtin_amdgcn_readlane(own.gran, b);
    return x;
  }
  // Granules (of one KV head) of the sequences before lane l's.
  __device__ __forceinline__ uint32_t before_lane(int l) const { return (uint32_t)__builtin_amdgcn_readlane((int)(incl - mine), l); }
  // The sequence that granule g lies in and its first granule; false where there is none.
  __device__ __forceinline__ bool find(const PromptArgs& a, int g, int& b, FewSeq& x, int& first) const {
    const unsigned long long past = __ballot((uint64_t)incl * (uint32_t)a.Hk > (uint64_t)g);
    if (!past) return false;
    const int l = __ffsll(past) - 1;
    first = (int)(before_lane(l) * (uint32_t)a.Hk);
    for (b = l * per; b < a.B; ++b) {
      x = seq(a, b);
      const int64_t n = (int64_t)x.work() * a.Hk;
      if (g < first + n) return true;
      first += (int)n;
    }
    return false;
  }
  // Runs: workgroup w has granules [start(w), start(w + 1)).
  __device__ __forceinline__ int start(const PromptArgs& a, int w) const {
    const int q = fast_div(total, a.dnwg), r = total - q * a.nwg;
    return w * q + min(w, r);
  }
  __device__ __forceinline__ int owner(const PromptArgs& a, int g) const {
    const int q = fast_div(total, a.dnwg), r = total - q * a.nwg, big = r * (q + 1);
    return min(g < big ? g / (q + 1) : q ? r + (g - big) / q : 0, a.nwg - 1);
  }
};

template <int D, int TYPE, bool HALVES>
__global__ __launch_bounds__(kFewWaves * 64, 2) void paged_prompt_few_kernel(PromptArgs a) {
  constexpr bool BYTES = TYPE != kBf16Cache, SCALED = TYPE >= kE4m3Blocks;
  using Elem = typename std::conditional<BYTES, uint8_t, uint16_t>::type;
  using C = DenseCfg<D>;
  constexpr int KK = D / 16, DB = D / 32, PITCH = D + 4;   // (of the merge: rows off each other's banks)
  constexpr int MERGE = kFewWaves * 32 * PITCH * 4;
  __shared__ __attribute__((aligned(16))) char smem[MERGE > kFewWaves * C::WAVE ? MERGE : kFewWaves * C::WAVE];
  __shared__ float sc[SCALED ? kFewWaves * 64 : 1], wm[kFewWaves * 32], wl[kFewWaves * 32];

  const int same_lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  auto same = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  auto zeros = [&](int t, int h0, int nh) {                // heads h0 .. of row t
    for (int j = threadIdx.x; j < nh * (D / 8); j += kFewWaves * 64)
      *reinterpret_cast<u32x4*>(a.out + (int64_t)t * a.o_st + (int64_t)(h0 + j / (D / 8)) * a.o_sh + j % (D / 8) * 8) =
          u32x4{0, 0, 0, 0};
  };
  int b, tile, hk, t = 0, g = 0, g0 = 0, g1;               // granules t .. of the unit, g .. of the batch
  FewSeq x;
  if (a.nwg) {
    const FewDeal all(a, same_lane);
    for (int r = min(max(a.cu[a.B], 0), a.T) + (int)blockIdx.x; r < a.T; r += a.nwg) zeros(r, 0, a.Hk * a.G);
    g = g0 = same(all.start(a, blockIdx.x)), g1 = same(all.start(a, blockIdx.x + 1));
    int first;
    if (g0 >= g1 || !all.find(a, g0, b, x, first)) return;
    const int unit = (g0 - first) / x.gran;
    t = g0 - first - unit * x.gran;
    tile = fast_div(unit, a.dHk), hk = unit - tile * a.Hk;
  } else {
    const int r = a.tiles - 1 - fast_div((int)blockIdx.x, a.dHk);       // the last rows, which see most, first
    hk = (int)blockIdx.x - (a.tiles - 1 - r) * a.Hk;
    RowTile y;
    if (!find_tile<32>(a, r, same_lane, y)) return;
    b = y.b, x.t0 = y.t0, x.n = y.n, x.len = y.len, tile = y.r0 / 32;
    if (b == a.B) {                                        // rows of no sequence
      for (int i = y.r0; i < min(y.r0 + 32, y.n * a.G); ++i) zeros(y.t0 + fast_div(i, a.dG), hk * a.G + i - fast_div(i, a.dG) * a.G, 1);
      return;
    }
    few_count(a, x);
    g1 = x.gran;
  }
  for (;;) {
    int lane = same_lane;
    asm volatile("" : "+v"(lane));                         // (addresses are not kept from one part for the next)
    const int l32 = lane & 31, e = lane >> 5;
    const int m = min(x.gran - t, g1 - g);                   // granules of this part
    const int r0 = tile * 32, rows = x.n * a.G;
    // row r of the tile: its token and head
    auto place_of = [&](int r, int& i, int& h) {
      const int row = min(r0 + r, rows - 1);
      i = fast_div(row, a.dG);
      h = hk * a.G + row - i * a.G;
    };
    int i, h;
    place_of(l32, i, h);
    const bool exists = r0 + l32 < rows;
    const int p0 = same(first_position(x.len, x.n)), p = p0 + i;
    const bool placed = exists && p >= 0 && p < a.cap;
    const int first = fast_div(r0, a.dG), last = fast_div(min(r0 + 31, rows - 1), a.dG);
    const int p_lo = same(max(p0 + first, 0)), p_hi = same(min(p0 + last, a.cap - 1));
    // slots: the sinks' tiles, then those from the window's first on
    const int end = max(p_hi + 1, 0), lo_key = max(p_lo - a.window + 1, 0);
    const int near_tiles = (min(a.sinks, end) + 31) & -32;
    const int gap = max((lo_key & -32) - near_tiles, 0);
    const int slots = p_lo > p_hi ? 0 : end - gap;

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

    auto token = [&](int s) { return s < near_tiles ? s : s + gap; };
    auto find = [&](int s, int& place, int& off, bool& ok) {
      const int t = token(s);
      place = fast_div(t, a.c.dbs);
      off = t - place * a.c.bs;
      ok = true;
    };
    // Whether all rows see all of the 32 tokens from t0 on.
    auto all_see = [&](int t0) { return t0 + 31 <= p_lo && (t0 > p_hi - a.window || t0 + 32 <= a.sinks); };
    auto seen = [&](int t0, uint32_t named) {
      return placed ? named & (uint32_t)(low_bits(p - t0 + 1) & (~low_bits(p - a.window + 1 - t0) | low_bits(a.sinks - t0))) : 0u;
    };
    bool odd = false;                                        // an infinity or NaN was left out
    char* wbuf = smem + w * C::WAVE;
    const PagedScales scales{a.ks + hk * a.ks_sh, a.vs + hk * a.vs_sh, a.ks_sb, a.vs_sb, sc + w * 64};
    // Tiles that some row does not see whole: no weight of 0 would take infinities and NaN away.
    auto ready = [&](int s, PagedRows<D, TYPE, HALVES>& rows_) {
      if (TYPE == kInt8Blocks || all_see(token(s))) return;
#pragma unroll
      for (int u = 0; u < PagedRows<D, TYPE, HALVES>::CPL; ++u) {
        u32x4& v = rows_.r.v[u];
        if constexpr (BYTES) {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = numbers_only(v[k], odd);
        } else {
          v = finite_only(v, odd);
        }
      }
    };
    auto compute = [&](int s0, uint32_t vmask) {
      const char *kst = wbuf, *vst = wbuf + C::VT;
      const int t0 = token(s0);
      int l = lane;
      asm volatile("" : "+v"(l));                          // (addresses in LDS are not kept in registers)
      const int l32 = l & 31, e = l >> 5;
      f32x16 s;
#pragma unroll
      for (int u = 0; u < 16; ++u) s[u] = 0.f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const bf16x8 ka = __builtin_bit_cast(
            bf16x8, *reinterpret_cast<const u32x4*>(kst + l32 * (D * 2) + kswz<D>(l32, kk * 2 + e) * 16));
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka, qb[kk], s, 0, 0, 0);
      }
      f32x4 vs[4];
      if constexpr (SCALED) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 k4 = *reinterpret_cast<const f32x4*>(scales.lds + 8 * g + 4 * e);
          vs[g] = *reinterpret_cast<const f32x4*>(scales.lds + 32 + 8 * g + 4 * e);
#pragma unroll
          for (int u = 0; u < 4; ++u) s[4 * g + u] *= k4[u];
        }
      }
      if (!(vmask == ~0u && all_see(t0))) {
        const uint32_t m = seen(t0, vmask) >> (4 * e);
#pragma unroll
        for (int u = 0; u < 16; ++u)
          if (!((m >> (8 * (u >> 2) + (u & 3))) & 1u)) s[u] = kNegInf;
      }
      float mx = kNegInf;
#pragma unroll
      for (int u = 0; u < 16; ++u) mx = __builtin_elementwise_maximum(mx, s[u]);
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
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        u32x4 w[2];
        WeightParts even;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          float pk = fast_exp2(__builtin_fmaf(s[8 * kk + u], a.scale_log2, -mc));
          l_run += pk;
          if constexpr (SCALED) pk *= vs[2 * kk + (u >> 2)][u & 3];
          put_weight<TYPE == kBf16Cache>(pk, u, even, w);
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          u32x2 t[2];
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const int rr = kk * 16 + hf * 8 + e * 4 + ((l >> 2) & 3), d = db * 32 + (l & 16) + (l & 3) * 4;
            t[hf] = tr16(vst + rr * (D * 2) + vswz<D>(rr, d >> 3) * 16 + (d & 7) * 2);
          }
          const bf16x8 v = __builtin_bit_cast(bf16x8, u32x4{t[0][0], t[0][1], t[1][0], t[1][1]});
#pragma unroll
          for (int i = 0; i < 2; ++i)
            acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, __builtin_bit_cast(bf16x8, w[i]), acc[db], 0, 0, 0);
        }
      }
    };
    const int32_t* table = a.c.table + (int64_t)b * a.c.bt_sb;
    const int s_begin = t * kFewGranule + w * 32, s_end = min((t + m) * kFewGranule, slots);
    paged_wave_tiles<D, TYPE, HALVES>(a.c, table, hk, s_begin, s_end, kFewWaves * 32, lane, wbuf, find, scales, ready, compute);
    if (TYPE != kInt8Blocks && __any(odd)) {
      // What was left out, added without weights (any above 0 gives the same) to the rows that see it.
      const Elem* vb = static_cast<const Elem*>(a.c.v) + hk * a.c.v_sh;
      for (int s = s_begin; s < s_end; s += kFewWaves * 32) {
        const int t0 = token(s);
        if (all_see(t0)) continue;
        for (int k = 0; k < 32 && s + k < s_end; ++k) {
          const int place = fast_div(t0 + k, a.c.dbs), id = table[place];
          if (id < 0 || id >= a.c.nblocks) continue;
          const Elem* vp = vb + (int64_t)id * a.c.v_sb + (int64_t)(t0 + k - place * a.c.bs) * a.c.v_ss;
          const bool mine = (seen(t0, ~0u) >> k) & 1;
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int u = 0; u < 16; ++u) {
              const uint32_t raw = vp[db * 32 + 8 * (u >> 2) + 4 * e + (u & 3)];
              const float v = BYTES ? ((raw & 0x7Fu) == 0x7Fu ? __builtin_nanf("") : 0.f) : __uint_as_float(raw << 16);
              if (mine && (__float_as_uint(v) & 0x7F800000u) == 0x7F800000u) acc[db][u] += v;
              asm volatile("" ::: "memory");                 // (few registers for a path that is hardly taken)
            }
        }
      }
    }

    // The waves' sums, in wave order.
    l_run = half_sum(l_run);
    float* wacc = reinterpret_cast<float*>(smem);
    __syncthreads();
    if (e == 0) {
      wm[w * 32 + l32] = m_run == kNegInf ? kNegInf : m_run * a.scale_log2;
      wl[w * 32 + l32] = placed ? l_run : 0.f;
    }
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(wacc + (w * 32 + l32) * PITCH + db * 32 + 8 * g + 4 * e) =
            f32x4{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
    __syncthreads();
    const bool whole = m == x.gran;
    const size_t base = ((size_t)blockIdx.x * 2 + (g == g0 ? 0 : 1)) * 32;
    int item = threadIdx.x;
    asm volatile("" : "+v"(item));                         // (nor are the places of sums)
    for (; item < 32 * (D / 4); item += kFewWaves * 64) {
      const int r = item / (D / 4), d4 = item % (D / 4);
      if (r0 + r >= rows) break;                           // (rows ascend with the item)
      float M = kNegInf;
#pragma unroll
      for (int u = 0; u < kFewWaves; ++u) M = fmaxf(M, wm[u * 32 + r]);
      const float Ms = M == kNegInf ? 0.f : M;
      float L = 0.f;
      f32x4 A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < kFewWaves; ++u) {
        const float f = fast_exp2(wm[u * 32 + r] - Ms);
        L += f * wl[u * 32 + r];
        A += f * *reinterpret_cast<const f32x4*>(wacc + (u * 32 + r) * PITCH + 4 * d4);
      }
      if (!whole) {
        reinterpret_cast<f32x4*>(a.part_acc + (base + r) * D)[d4] = A;
        if (d4 == 0) reinterpret_cast<float2*>(a.part_ml)[base + r] = make_float2(M, L);
      } else {
        int ri, rh;
        place_of(r, ri, rh);
        paged_store(a.out + (int64_t)(x.t0 + ri) * a.o_st + (int64_t)rh * a.o_sh + 4 * d4, A, L, a.v_scale);
      }
    }
    g += m;
    if (g >= g1) return;
    __syncthreads();
    t = 0;
    if (++hk == a.Hk) {
      hk = 0;
      if (++tile == x.tiles) {
        tile = 0;
        do {
          if (++b >= a.B) return;
          x = few_seq(a, b);                       // (the lanes' counts are not kept in registers)
        } while (x.tiles == 0);
      }
    }
  }
}

// Joins the parts of each unit that more than one workgroup had: one wave per (row of q, query
// head, 64 dims).
template <int D>
__global__ __launch_bounds__(64) void paged_prompt_few_join_kernel(PromptArgs a) {
  constexpr int NSL = D / 64;
  const int lane = threadIdx.x, item = lane & 15, grp = lane >> 4;
  const int slice = blockIdx.y % NSL, h = blockIdx.y / NSL, row_q = blockIdx.x;
  const FewDeal all(a, lane);
  // the sequence whose rows those are, and its granules' first
  int b = -1;
  for (int i = 0; i < all.per && b < 0; ++i) {
    const int at = lane * all.per + i;
    const FewSeq x = all.per == 1 ? all.own : few_seq(a, min(at, a.B - 1));
    if (at < a.B && row_q >= x.t0 && row_q < x.t0 + x.n) b = at;
  }
  const unsigned long long in = __ballot(b >= 0);
  if (!in) return;                                         // a row of no sequence
  const int l = __ffsll(in) - 1;
  b = __builtin_amdgcn_readlane(b, l);
  uint32_t before = all.before_lane(l);
  for (int i = l * all.per; i < b; ++i) before += all.seq(a, i).work();
  const FewSeq x = all.seq(a, b);
  const int hk = fast_div(h, a.dG), row = (row_q - x.t0) * a.G + h - hk * a.G, tile = row / 32;
  const int64_t s = (int64_t)before * a.Hk + ((int64_t)tile * a.Hk + hk) * x.gran;
  if (s + x.gran > all.total) return;                      // (offsets that overlap)
  const int w0 = all.owner(a, (int)s), w1 = all.owner(a, (int)s + x.gran - 1);
  if (w0 >= w1) return;                                    // finished in place
  const int slot0 = all.start(a, w0) == (int)s ? 0 : 1;
  auto slot = [&](int u) { return ((size_t)(w0 + u) * 2 + (u == 0 ? slot0 : 0)) * 32 + (row & 31); };
  paged_join<4>(w1 - w0 + 1, lane, slot, reinterpret_cast<const float2*>(a.part_ml),
                reinterpret_cast<const f32x4*>(a.part_acc) + slice * 16 + item, D / 4, [&](const f32x4& A, float L) {
                  if (grp == 0)
                    paged_store(a.out + (int64_t)row_q * a.o_st + (int64_t)h * a.o_sh + slice * 64 + item * 4, A, L, a.v_scale);
                });
}

template <int D, int TYPE>
static void launch(const PromptArgs& a, dim3 grid, hipStream_t st) {
  if (paged_halves(a.c)) hipLaunchKernelGGL((paged_prompt_few_kernel<D, TYPE, true>), grid, dim3(kFewWaves * 64), 0, st, a);
  else hipLaunchKernelGGL((paged_prompt_few_kernel<D, TYPE, false>), grid, dim3(kFewWaves * 64), 0, st, a);
}
template <int TYPE>
static int launch_of(const PromptArgs& a, dim3 grid, hipStream_t st) {
  if (a.D == 128) launch<128, TYPE>(a, grid, st);
  else launch<64, TYPE>(a, grid, st);
  const int rc = (int)hipGetLastError();
  if (rc || !a.nwg) return rc;
  const dim3 jgrid((unsigned)a.T, (unsigned)(a.Hk * a.G * (a.D / 64)));
  if (a.D == 128) hipLaunchKernelGGL((paged_prompt_few_join_kernel<128>), jgrid, dim3(64), 0, st, a);
  else hipLaunchKernelGGL((paged_prompt_few_join_kernel<64>), jgrid, dim3(64), 0, st, a);
  return (int)hipGetLastError();
}
int launch_prompt_few(const PromptArgs& a, int kv_type, const PromptPlan& plan, hipStream_t st) {
  const dim3 grid((unsigned)(plan.nwg ? plan.nwg : plan.units));
  switch (kv_type) {
    case kBf16Cache: return launch_of<kBf16Cache>(a, grid, st);
    case kFp8Cache: return launch_of<kFp8Cache>(a, grid, st);
    case kE4m3Blocks: return launch_of<kE4m3Blocks>(a, grid, st);
    default: return launch_of<kInt8Blocks>(a, grid, st);
  }
}

}  // namespace bytes_amd

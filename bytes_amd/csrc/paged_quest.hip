// Page-sparse decode over a paged KV cache: block bounds, and attention over
// the blocks that they select.
//
//   bound[b, h, j] = scale * sum_d q_d * (q_d >= 0 ? kmax_d : kmin_d)
//
// over the min / max of block table[b, j], the largest score that any of its
// keys can have.  The products of bf16 values are exact in fp32 and their sum is
// taken in fp64, where (but for products 2^37 apart) it is exact too: its order
// does not move a selection.  It is scaled there and rounded to fp32 once.  Blocks
// that hold no token that takes part (paged.h) get -inf, blocks that reach into
// the sequence's last local_w tokens +inf.
//
// Attention over the selection: a workgroup serves one query head and a run of
// its selected blocks' rows.  It selects the npick best of the head's bounds
// itself (the order of bytes_topk: bound descending, lowest place first on equal
// bounds; wave_select.h), or takes a list of places.  Heads of one KV head sit on
// one XCD, whose L2 then serves the blocks that several of them select.
#include "paged.h"
#include "wave_select.h"

namespace bytes_amd {

struct PageBoundArgs {
  PagedKv c;
  const uint16_t *q, *kmin, *kmax;
  int64_t q_sb, q_sh;
  float* bound;
  int64_t b_sb, b_sh;
  int Hk, G, local_w, skip;          // skip: sequences of at most that many blocks need no bounds
  FastDiv dHk;
  double scale;
};

constexpr int kBoundWaves = 4, kBoundTile = 16;    // blocks per tile, one tile per wave

// The literal sum, for tiles with a non-finite entry: lane l's block is l % 16 of
// the tile, its head h0 + l / 16.
__device__ __forceinline__ double bound_literal(const uint16_t* q, const uint16_t* lo, const uint16_t* hi, int D) {
  double s = 0.0;
  for (int d = 0; d < D; ++d) {
    const float x = bf16_bits_to_f32(q[d]);
    s += (double)x * (double)bf16_bits_to_f32(x >= 0.f ? hi[d] : lo[d]);
  }
  return s;
}

// Bounds of 16 blocks per wave for the heads of one KV head: with q split into its
// positive and negative parts, q+ . kmax + q- . kmin on the fp64 matrix
// instruction of four 4x4x4 products: A = q parts of four heads (lane: head l % 4,
// the same for each product), B = entries of 4 x 4 blocks (lane: block l % 16 of
// the tile), dims by l / 16.  A lane reads its block's 16-byte chunks l / 16, + 4,
// .. straight into registers (which dims a step takes does not matter, as long as
// A and B agree); q's parts are widened once per workgroup, in LDS.  The result is
// at lane: head l / 16, block l % 16.  A tile with an infinite or NaN entry, where
// the part of q that is 0 would give NaN, takes the literal sum.
// Bound by its loads and then its products for large batches: 44 MB of min / max (seven
// sequences of 32K to 64K, 8 KV heads of 128, blocks of 32) take 16.5 us from a graph,
// 12.4 of them the loads alone (3.5 TB/s, in pieces of 256 bytes: the heads of a block
// are different workgroups'); with the sums on the vector unit 24.  One sequence of
// 32K (4.2 MB): 5.2, launch and round trips; two tiles per wave, half the waves, 7.7
// (and 17.2 for the 44 MB).
template <int D, int NG>
__global__ __launch_bounds__(kBoundWaves * 64, 4) void page_bound_kernel(PageBoundArgs a) {
  PREFETCH_ARGS(a);
  constexpr int NCH = D / 32;                      // chunks per lane and row
  __shared__ __attribute__((aligned(16))) double parts[NG][D][4][2];    // [group][step, l / 16][head][q+, q-]
  __shared__ int odd_q;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.y, k = lane >> 4;
  const int chunk = fast_div((int)blockIdx.x, a.dHk), hk = (int)blockIdx.x - chunk * a.Hk;
  const int tile = chunk * kBoundWaves + w, j = tile * kBoundTile + (lane & 15);
  const int len = __builtin_amdgcn_readfirstlane(paged_len(a.c, b));
  const int id = a.c.table[(int64_t)b * a.c.bt_sb + min(j, a.c.width - 1)];
  const int full = fast_div(len + a.c.bs - 1, a.c.dbs);        // blocks that hold tokens
  if (full <= a.skip) return;
  const int recent = a.local_w > 0 ? fast_div(max(len - a.local_w, 0), a.c.dbs) : 0x7FFFFFFF;
  const bool held = j < full && id >= 0 && id < a.c.nblocks;
  const int64_t row = ((int64_t)(held ? id : 0) * a.Hk + hk) * D;
  u32x4 lo[NCH], hi[NCH];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    lo[c] = ld16(a.kmin + row + (k + 4 * c) * 8);
    hi[c] = ld16(a.kmax + row + (k + 4 * c) * 8);
  }
  auto nonfinite = [](const u32x4& x) {            // a bf16 exponent of all ones
    uint32_t e = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) e |= (x[i] & 0x7F807F80u) + 0x00800080u;
    return (e & 0x80008000u) != 0u;
  };
  auto value = [](const u32x4& x, int e) {         // element e of a chunk
    const uint32_t y = x[e >> 1];
    return __uint_as_float(e & 1 ? y & 0xFFFF0000u : y << 16);
  };
  const uint16_t* qh = a.q + b * a.q_sb + (int64_t)hk * a.G * a.q_sh;
  for (int g0 = 0; g0 < a.G; g0 += 4 * NG) {
    if (g0) __syncthreads();
    if (threadIdx.x == 0) odd_q = 0;
    __syncthreads();
    // one chunk of one head per thread: dims 8 c' .. + 7 with c' = k + 4 c are step (c, e) of lanes k
    for (int x = threadIdx.x; x < 4 * NG * (D / 8); x += kBoundWaves * 64) {
      const int h = x / (D / 8), cc = x - h * (D / 8);
      const u32x4 r = ld16(qh + (int64_t)min(g0 + h, a.G - 1) * a.q_sh + cc * 8);
      if (nonfinite(r)) odd_q = 1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = value(r, e);
        double* to = parts[h >> 2][(cc >> 2) * 32 + e * 4 + (cc & 3)][h & 3];
        to[0] = fmaxf(y, 0.f);
        to[1] = fminf(y, 0.f);
      }
    }
    __syncthreads();
    bool odd = odd_q != 0;
#pragma unroll
    for (int c = 0; c < NCH; ++c) odd = odd || nonfinite(lo[c]) || nonfinite(hi[c]);
    double s[NG];
    if (!__any(odd)) {
      double up[NG], down[NG];
#pragma unroll
      for (int n = 0; n < NG; ++n) up[n] = down[n] = 0.0;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        // widened for every group of heads anew: kept across the groups, the 2 D / 4
        // registers of them spill
        u32x4 l = lo[c], h = hi[c];
        asm volatile("" : "+v"(l), "+v"(h));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const double kmx = value(h, e), kmn = value(l, e);
#pragma unroll
          for (int n = 0; n < NG; ++n) {
            const double* q = parts[n][c * 32 + e * 4 + k][lane & 3];
            up[n] = __builtin_amdgcn_mfma_f64_4x4x4f64(q[0], kmx, up[n], 0, 0, 0);
            down[n] = __builtin_amdgcn_mfma_f64_4x4x4f64(q[1], kmn, down[n], 0, 0, 0);
          }
          if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // (keeps the LDS reads from piling up)
        }
      }
#pragma unroll
      for (int n = 0; n < NG; ++n) s[n] = up[n] + down[n];
    } else {
#pragma unroll
      for (int n = 0; n < NG; ++n)
        s[n] = bound_literal(qh + (int64_t)min(g0 + 4 * n + k, a.G - 1) * a.q_sh, a.kmin + row, a.kmax + row, D);
    }
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int g = g0 + 4 * n + k;
      float v = (float)(s[n] * a.scale);
      if (j >= recent) v = __builtin_inff();
      if (!held) v = kNegInf;
      if (g < a.G && j < a.c.width) a.bound[b * a.b_sb + (int64_t)(hk * a.G + g) * a.b_sh + j] = v;
    }
  }
}

struct PagedQuestArgs {
  PagedKv c;
  const uint16_t* q;
  int64_t q_sb, q_sh;
  const float* bound;                // [B, Hq, width], row strides b_sb, b_sh; or null:
  int64_t b_sb, b_sh;
  const int32_t* pages;              // [B, Hq, npick], row strides p_sb, p_sh
  int64_t p_sb, p_sh;
  uint16_t* out;
  int64_t o_sb, o_sh;
  float* part_acc;                   // [B * Hq][nsplit][D]
  float* part_ml;                    // [B * Hq][nsplit][2]
  int Hq, G, npick, chunk, nsplit, nwg;
  int b_vec;                         // bound rows are whole 16-byte chunks
  FastDiv dsplit, dHq, dG;
  float scale_log2, v_scale;
};

constexpr int kPickMax = 4096;       // blocks of a sequence that a workgroup selects from; blocks of a run
constexpr int kSelectThreads = 1024, kSelectMax = 16 * kSelectThreads;     // the same of the selection launch
constexpr int kPickWaves = 4, kPickThreads = kPickWaves * 64;

// A wave's tile: 16-byte chunks, LPR lanes to a row, RPI rows to an instruction, NB
// instructions of K and as many of V in flight.
template <int D, bool FP8>
struct PickCfg {
  static constexpr int EPC = FP8 ? 16 : 8;         // dims per lane
  static constexpr int LPR = D / EPC, RPI = 64 / LPR;
  static constexpr int NB = RPI == 16 ? 4 : 8;
  static constexpr int TILE = NB * RPI;            // rows
};

// Selection of the k best of n bounds (k < n <= NT * PER): put(rank in ascending place order, place).
// vec: the row starts on a 16-byte boundary and its storage ends on one.
template <int NT, int PER, class PUT>
__device__ __forceinline__ void pick_blocks(const float* bound, bool vec, int n, int k, uint32_t* ws, const PUT& put) {
  uint32_t key[PER];
  if (vec) {
    u32x4 v[PER / 4];
#pragma unroll
    for (int u = 0; u < PER / 4; ++u) v[u] = ld16(bound + 4 * min(PER / 4 * (int)threadIdx.x + u, (n - 1) / 4));
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const uint32_t x = v[u / 4][u % 4];
      key[u] = score_order_key(__uint_as_float(x));
    }
  } else {
    float v[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) v[u] = bound[min(PER * (int)threadIdx.x + u, n - 1)];
#pragma unroll
    for (int u = 0; u < PER; ++u) key[u] = score_order_key(v[u]);
  }
  const BlockSel sel = block_select<NT, PER>(key, n, k, ws);
  block_select_emit<NT, PER>(key, n, sel, ws, [&](uint32_t pos, int idx, uint32_t) { put((int)pos, idx); });
}

// Dot product of the lane's dims of a K row with its q (bf16 pairs), fp32 sums.
template <bool FP8>
__device__ __forceinline__ float dot_chunk(const u32x4& k, const uint32_t (&q)[FP8 ? 8 : 4]) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t x = k[j];                       // (a cast of the vector's element itself reads its first one)
    if constexpr (FP8) {
      s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false),
                                          __builtin_bit_cast(bf16x2, q[2 * j]), s, false);
      s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true),
                                          __builtin_bit_cast(bf16x2, q[2 * j + 1]), s, false);
    } else {
      s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x), __builtin_bit_cast(bf16x2, q[j]), s, false);
    }
  }
  return s;
}
// acc += p * the lane's dims of a V row.
template <bool FP8>
__device__ __forceinline__ void add_chunk(const u32x4& v, float p, float (&acc)[FP8 ? 16 : 8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (FP8) {
      const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(v[j], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(v[j], true);
      acc[4 * j] = __builtin_fmaf(p, a[0], acc[4 * j]);
      acc[4 * j + 1] = __builtin_fmaf(p, a[1], acc[4 * j + 1]);
      acc[4 * j + 2] = __builtin_fmaf(p, b[0], acc[4 * j + 2]);
      acc[4 * j + 3] = __builtin_fmaf(p, b[1], acc[4 * j + 3]);
    } else {
      acc[2 * j] = __builtin_fmaf(p, __uint_as_float(v[j] << 16), acc[2 * j]);
      acc[2 * j + 1] = __builtin_fmaf(p, __uint_as_float(v[j] & 0xFFFF0000u), acc[2 * j + 1]);
    }
  }
}

// One query head and one run of its slots (slot s: row s % block_size of pick s /
// block_size).  A head alone would use one column in 16 of a matrix instruction,
// so rows are multiplied on the vector unit as they arrive: LPR lanes hold a row,
// each group of them keeps its own maximum, denominator and sums (fp32
// throughout), and groups and waves are merged at the end.  No LDS stage, so
// registers alone bound the waves in flight.  RUNS: block sizes that are multiples of
// RPI, whose instructions' rows lie in one block and start at a scalar address.
// Bound by what a run does besides streaming: every run of a head begins with the
// selection, while no row is in flight, and has few tiles per wave, each issued when
// the one before is done.  2048 of 32K to 64K fp8 tokens of 7 x 24 heads (84 MB of
// distinct rows) take 24 us, 3.5 TB/s, 4 of them the selection; 2048 of 32K bf16 tokens
// of 28 heads (24 MB) 10.5.  (That blocks lie anywhere is not it: the decode reads
// blocks of 16 rows in the same order at 6.6.)  With two tiles in flight per wave a
// whole call takes 53 for 46.5 and 22 for 20.
template <int D, bool FP8, bool RUNS>
__global__ __launch_bounds__(kPickThreads, 4) void paged_quest_kernel(PagedQuestArgs a) {
  using P = PickCfg<D, FP8>;
  using Elem = typename std::conditional<FP8, uint8_t, uint16_t>::type;
  constexpr int EPC = P::EPC, LPR = P::LPR, RPI = P::RPI, NB = P::NB;
  __shared__ int32_t list[kPickMax];               // block ids of the run's picks, -1: none
  __shared__ __attribute__((aligned(16))) uint32_t work[block_select_words<kPickThreads>()];
  __shared__ int tail;                             // the pick that is the sequence's last block, which may be short
  static_assert(sizeof(work) >= kPickWaves * (D + 2) * 4, "the merge fits");
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int idx = xcd_run(blockIdx.x, a.nwg), unit = fast_div(idx, a.dsplit), split = idx - unit * a.nsplit;
  const int b = fast_div(unit, a.dHq), h = unit - b * a.Hq, hk = fast_div(h, a.dG);
  const int len = __builtin_amdgcn_readfirstlane(paged_len(a.c, b));
  const int full = fast_div(len + a.c.bs - 1, a.c.dbs);
  const int picks = a.bound ? min(a.npick, full) : a.npick;
  const int s0 = split * a.chunk, s1 = min(s0 + a.chunk, picks * a.c.bs);
  if (split > 0 && s0 >= s1) return;               // (split 0 of an empty sequence writes its zeros)
  const int c = lane % LPR, grp = lane / LPR;
  uint32_t q[EPC / 2];
  {
    const uint16_t* qp = a.q + (int64_t)b * a.q_sb + (int64_t)h * a.q_sh + c * EPC;
#pragma unroll
    for (int j = 0; j < EPC / 8; ++j) {
      const u32x4 r = ld16(qp + 8 * j);
#pragma unroll
      for (int e = 0; e < 4; ++e) q[4 * j + e] = r[e];
    }
  }
  // the run's blocks
  const int32_t* table = a.c.table + (int64_t)b * a.c.bt_sb;
  const int i0 = fast_div(s0, a.c.dbs), i1 = s1 > s0 ? fast_div(s1 - 1, a.c.dbs) + 1 : i0;
  if (threadIdx.x == 0) tail = -1;
  __syncthreads();
  auto put = [&](int i, int place) {
    if (i < i0 || i >= i1) return;
    const bool in = place >= 0 && place < full;
    const int id = table[in ? place : 0];
    list[i - i0] = in && id >= 0 && id < a.c.nblocks ? id : -1;
    if (place == full - 1) tail = i;
  };
  if (a.bound && full > a.npick) {
    const float* bound = a.bound + (int64_t)b * a.b_sb + (int64_t)h * a.b_sh;
    const bool vec = a.b_vec != 0;
    if (full <= 4 * kPickThreads) pick_blocks<kPickThreads, 4>(bound, vec, full, a.npick, work, put);
    else if (full <= 8 * kPickThreads) pick_blocks<kPickThreads, 8>(bound, vec, full, a.npick, work, put);
    else pick_blocks<kPickThreads, 16>(bound, vec, full, a.npick, work, put);
  } else {
    const int32_t* pages = a.pages + b * a.p_sb + h * a.p_sh;
    for (int i = i0 + threadIdx.x; i < i1; i += kPickThreads) put(i, a.bound ? i : pages[i]);
  }
  __syncthreads();
  const int short_at = tail, short_rows = len - (full - 1) * a.c.bs;      // rows of the sequence's last block

  const Elem* kb = static_cast<const Elem*>(a.c.k) + hk * a.c.k_sh;
  const Elem* vb = static_cast<const Elem*>(a.c.v) + hk * a.c.v_sh;
  float m_run = kNegInf, l_run = 0.f, acc[EPC];
#pragma unroll
  for (int j = 0; j < EPC; ++j) acc[j] = 0.f;
  const uint32_t k_lane = (uint32_t)(grp * (int)a.c.k_ss + c * EPC), v_lane = (uint32_t)(grp * (int)a.c.v_ss + c * EPC);
  for (int t = s0 + w * P::TILE; t < s1; t += kPickWaves * P::TILE) {
    u32x4 k[NB], v[NB];
    bool ok[NB];
    bool all = true;
    int first_id = 0, first_off = 0, first_i = 0;  // RUNS: lane u's instruction u
    if (RUNS) {
      const int s = min(t + (lane & (NB - 1)) * RPI, s1 - 1);
      first_i = fast_div(s, a.c.dbs);
      first_off = s - first_i * a.c.bs;
      first_off -= first_off % RPI;                // (s1 - 1 need not start an instruction's rows)
      first_id = list[first_i - i0];
    }
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      const int s = t + u * RPI + grp;
      if (RUNS) {
        const int id = __builtin_amdgcn_readlane(first_id, u), off = __builtin_amdgcn_readlane(first_off, u);
        const int i = __builtin_amdgcn_readlane(first_i, u);
        ok[u] = s < s1 && id >= 0 && !(i == short_at && off + grp >= short_rows);
        const int64_t ids = id < 0 ? 0 : id;
        k[u] = ld16(kb + ids * a.c.k_sb + off * a.c.k_ss + k_lane);
        v[u] = ld16(vb + ids * a.c.v_sb + off * a.c.v_ss + v_lane);
      } else {
        const int sc = min(s, s1 - 1), i = fast_div(sc, a.c.dbs), off = sc - i * a.c.bs, id = list[i - i0];
        ok[u] = s < s1 && id >= 0 && !(i == short_at && off >= short_rows);
        const int64_t ids = id < 0 ? 0 : id;
        k[u] = ld16(kb + ids * a.c.k_sb + off * a.c.k_ss + c * EPC);
        v[u] = ld16(vb + ids * a.c.v_sb + off * a.c.v_ss + c * EPC);
      }
      all = all && ok[u];
    }
    float s[NB], mx = kNegInf;
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      float x = dot_chunk<FP8>(k[u], q);
      // over the row's lanes, every lane receiving the sum
      if (LPR == 16) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xF, 0xF, false));
      if (LPR >= 8) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x141, 0xF, 0xF, false));
      x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xF, 0xF, false));
      x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xF, 0xF, false));
      s[u] = ok[u] ? x * a.scale_log2 : kNegInf;
      mx = __builtin_elementwise_maximum(mx, s[u]);
    }
    if (!__all(all)) {                             // weight 0 times what an unused row holds need not be 0
#pragma unroll
      for (int u = 0; u < NB; ++u)
        if (!ok[u]) v[u] = u32x4{0, 0, 0, 0};
    }
    const float m_new = __builtin_elementwise_maximum(m_run, mx), m_use = m_new == kNegInf ? 0.f : m_new;
    const float alpha = fast_exp2(m_run - m_use);
    m_run = m_new;
    l_run *= alpha;
#pragma unroll
    for (int j = 0; j < EPC; ++j) acc[j] *= alpha;
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      const float p = fast_exp2(s[u] - m_use);
      l_run += p;
      add_chunk<FP8>(v[u], p, acc);
    }
  }
  // groups of the wave, then the waves in order
  {
    const float m = fold_rows<LPR>(m_run, [](float x, float y) { return __builtin_elementwise_maximum(x, y); });
    const float f = fast_exp2(m_run - (m == kNegInf ? 0.f : m));
    auto add = [](float x, float y) { return x + y; };
    m_run = m;
    l_run = fold_rows<LPR>(l_run * f, add);
#pragma unroll
    for (int j = 0; j < EPC; ++j) acc[j] = fold_rows<LPR>(acc[j] * f, add);
  }
  float* wacc = reinterpret_cast<float*>(work);    // [wave][D], then (m, l) per wave
  float* wml = wacc + kPickWaves * D;
  if (grp == 0) {
#pragma unroll
    for (int j = 0; j < EPC / 4; ++j)
      reinterpret_cast<f32x4*>(wacc + w * D + c * EPC)[j] = f32x4{acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]};
    if (c == 0) wml[2 * w] = m_run, wml[2 * w + 1] = l_run;
  }
  __syncthreads();
  if ((int)threadIdx.x >= D / 4) return;
  float M = kNegInf, L = 0.f;
#pragma unroll
  for (int u = 0; u < kPickWaves; ++u) M = __builtin_elementwise_maximum(M, wml[2 * u]);
  const float Ms = M == kNegInf ? 0.f : M;
  f32x4 A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < kPickWaves; ++u) {
    const float f = fast_exp2(wml[2 * u] - Ms);
    L += f * wml[2 * u + 1];
    A += f * reinterpret_cast<const f32x4*>(wacc + u * D)[threadIdx.x];
  }
  if (picks * a.c.bs <= a.chunk) {
    paged_store(a.out + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + 4 * threadIdx.x, A, L, a.v_scale);
  } else {
    const size_t r = (size_t)unit * a.nsplit + split;
    reinterpret_cast<f32x4*>(a.part_acc + r * D)[threadIdx.x] = A;
    if (threadIdx.x == 0) reinterpret_cast<float2*>(a.part_ml)[r] = make_float2(M, L);
  }
}

// The selection as a launch of its own, for sequences of more blocks than a
// workgroup of the attention selects from: one workgroup per query head, its
// places ascending, -1 past a short sequence's.  Below that it costs more than the
// selection that every run of a head repeats (us of a call, in the kernel and as a
// launch: one sequence of 32K, 28 heads, 2048 blocks 19.3 and 22.9; one of 60000, 8
// heads, 3750 blocks 16.4 and 17.6; 16 of 8K, 64 heads, 512 blocks 49 and 69).
__global__ __launch_bounds__(kSelectThreads) void paged_select_kernel(PagedQuestArgs a, int32_t* pages) {
  __shared__ __attribute__((aligned(16))) uint32_t work[block_select_words<kSelectThreads>()];
  const int b = fast_div((int)blockIdx.x, a.dHq), h = (int)blockIdx.x - b * a.Hq;
  const int full = fast_div(paged_len(a.c, b) + a.c.bs - 1, a.c.dbs);
  int32_t* to = pages + (int64_t)blockIdx.x * a.npick;
  if (full <= a.npick) {
    for (int i = threadIdx.x; i < a.npick; i += kSelectThreads) to[i] = i < full ? i : -1;
    return;
  }
  const float* bound = a.bound + (int64_t)b * a.b_sb + (int64_t)h * a.b_sh;
  auto put = [&](int i, int place) { to[i] = place; };
  if (full <= 8 * kSelectThreads) pick_blocks<kSelectThreads, 8>(bound, a.b_vec != 0, full, a.npick, work, put);
  else pick_blocks<kSelectThreads, 16>(bound, a.b_vec != 0, full, a.npick, work, put);
}

// Joins the runs of each head that has several, in order: one wave per (sequence,
// head, 64 dims), four runs at a time, as the decode's join.
template <int D>
__global__ __launch_bounds__(64) void paged_quest_join_kernel(PagedQuestArgs a) {
  constexpr int NSL = D / 64;
  const int lane = threadIdx.x, item = lane & 15, grp = lane >> 4;
  const int slice = blockIdx.x % NSL, unit = blockIdx.x / NSL, b = fast_div(unit, a.dHq), h = unit - b * a.Hq;
  const int full = fast_div(paged_len(a.c, b) + a.c.bs - 1, a.c.dbs);
  const int slots = (a.bound ? min(a.npick, full) : a.npick) * a.c.bs;
  if (slots <= a.chunk) return;                    // finished in place
  const int parts = (slots + a.chunk - 1) / a.chunk;
  paged_join<8>(parts, lane, [&](int i) { return (size_t)unit * a.nsplit + i; },
                reinterpret_cast<const float2*>(a.part_ml),
                reinterpret_cast<const f32x4*>(a.part_acc) + slice * 16 + item, D / 4, [&](const f32x4& A, float L) {
                  if (grp == 0) paged_store(a.out + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + slice * 64 + item * 4, A, L,
                                            a.v_scale);
                });
}

// Runs of a head's slots: as many as make about four workgroups per CU, whole
// rounds of the four waves' tiles, and no more blocks than a run's list holds.
// Four are what fit a CU's registers (us of a call, 2048 of 32K to 64K fp8 tokens of
// 7 x 24 heads: 47; one per CU 54, two 49, eight 56; one sequence of 32K, 28 heads:
// 19.3 with any of them).
static int pick_step(int D, int fp8) {
  if (D == 128) return kPickWaves * (fp8 ? PickCfg<128, true>::TILE : PickCfg<128, false>::TILE);
  return kPickWaves * (fp8 ? PickCfg<64, true>::TILE : PickCfg<64, false>::TILE);
}
static void quest_plan(int64_t units, int64_t slots, int bs, int step, int* chunk, int* nsplit) {
  const int64_t target = 4 * (int64_t)device_cu_count();
  int64_t c = (slots * units + target - 1) / target;
  c = (c + step - 1) / step * step;
  const int64_t most = (int64_t)(kPickMax - 1) * bs / step * step;       // a run may start within a block
  const int64_t whole = (slots + step - 1) / step * step;
  if (c > whole) c = whole;
  if (c > most) c = most;
  if (c < step) c = step;
  *chunk = (int)c;
  *nsplit = (int)((slots + c - 1) / c);
}
// The selection launch's lists.
static size_t selected_bytes(int64_t units, int max_blocks, int npick) {
  return max_blocks <= kPickMax || max_blocks > kSelectMax ? 0 : (size_t)units * npick * 4;
}
static size_t quest_workspace(int64_t units, int nsplit, int D) {
  return nsplit <= 1 ? 0 : (size_t)units * nsplit * (D + 2) * 4;
}

}  // namespace bytes_amd

using namespace bytes_amd;

extern "C" {

int bytes_paged_page_scores(const void* q, int64_t q_sb, int64_t q_sh, const void* kmin, const void* kmax,
                            const void* block_table, int64_t bt_sb, const void* context_lens, void* bound, int64_t b_sb,
                            int64_t b_sh, int B, int Hq, int Hk, int D, int block_size, int num_blocks, int max_blocks,
                            int local_w, int skip, double scale, void* stream) {
  if (!q || !kmin || !kmax || !block_table || !context_lens || !bound || B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 ||
      (D != 64 && D != 128) || local_w < 0 || max_blocks <= 0)
    return (int)hipErrorInvalidValue;
  int rc = paged_check(block_size, num_blocks, max_blocks);
  if (rc) return rc;
  if (B > 65535 || Hk > 65535) return (int)hipErrorInvalidConfiguration;
  PageBoundArgs a = {};
  a.c.table = static_cast<const int32_t*>(block_table), a.c.bt_sb = bt_sb;
  a.c.lens = static_cast<const int32_t*>(context_lens);
  a.c.bs = block_size, a.c.nblocks = num_blocks, a.c.width = max_blocks;
  a.c.dbs = make_fastdiv((uint32_t)block_size);
  a.q = static_cast<const uint16_t*>(q), a.q_sb = q_sb, a.q_sh = q_sh;
  a.kmin = static_cast<const uint16_t*>(kmin), a.kmax = static_cast<const uint16_t*>(kmax);
  a.bound = static_cast<float*>(bound), a.b_sb = b_sb, a.b_sh = b_sh;
  a.Hk = Hk, a.G = Hq / Hk, a.local_w = local_w, a.skip = skip < 0 ? -1 : skip, a.scale = scale;
  const int64_t chunks = (max_blocks + kBoundTile * kBoundWaves - 1) / (kBoundTile * kBoundWaves);
  if (chunks * Hk > 0x7FFFFFFF) return (int)hipErrorInvalidConfiguration;
  a.dHk = make_fastdiv((uint32_t)Hk);
  const dim3 grid((unsigned)(chunks * Hk), (unsigned)B), block(kBoundWaves * 64);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define PB(DD, N) hipLaunchKernelGGL((page_bound_kernel<DD, N>), grid, block, 0, st, a)
  if (D == 128) {
    if (a.G <= 4) PB(128, 1);
    else PB(128, 2);
  } else {
    if (a.G <= 4) PB(64, 1);
    else PB(64, 2);
  }
#undef PB
  return (int)hipGetLastError();
}

int bytes_paged_quest_workspace_size(int B, int Hq, int Hk, int D, int kv_fp8, int block_size, int max_blocks, int npick,
                                     size_t* bytes) {
  if (!bytes || B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 || (D != 64 && D != 128) || npick <= 0)
    return (int)hipErrorInvalidValue;
  const int rc = paged_check(block_size, 1, max_blocks > npick ? max_blocks : npick);
  if (rc) return rc;
  int chunk, ns;
  quest_plan((int64_t)B * Hq, (int64_t)npick * block_size, block_size, pick_step(D, kv_fp8), &chunk, &ns);
  *bytes = quest_workspace((int64_t)B * Hq, ns, D) + selected_bytes((int64_t)B * Hq, max_blocks, npick);
  return 0;
}

int bytes_paged_quest_attn(const void* q, int64_t q_sb, int64_t q_sh, const void* k_paged, int64_t k_sb, int64_t k_sh,
                           int64_t k_ss, const void* v_paged, int64_t v_sb, int64_t v_sh, int64_t v_ss, int kv_fp8,
                           const void* bound, int64_t b_sb, int64_t b_sh, const void* pages, int64_t p_sb, int64_t p_sh,
                           int npick, const void* block_table, int64_t bt_sb, const void* context_lens, void* out,
                           int64_t o_sb, int64_t o_sh, int B, int Hq, int Hk, int D, int block_size, int num_blocks,
                           int max_blocks, float scale, float v_scale, void* workspace, size_t workspace_bytes,
                           void* stream) {
  if (!q || !k_paged || !v_paged || (!bound && !pages) || !block_table || !context_lens || !out || B <= 0 || Hk <= 0 ||
      Hq <= 0 || Hq % Hk != 0 || (D != 64 && D != 128) || npick <= 0 || npick > max_blocks)
    return (int)hipErrorInvalidValue;
  int rc = paged_check(block_size, num_blocks, max_blocks);
  if (rc) return rc;
  if (bound && max_blocks > kSelectMax) return (int)hipErrorNotSupported;
  PagedQuestArgs a = {};
  a.c.k = k_paged, a.c.k_sb = k_sb, a.c.k_sh = k_sh, a.c.k_ss = k_ss;
  a.c.v = v_paged, a.c.v_sb = v_sb, a.c.v_sh = v_sh, a.c.v_ss = v_ss;
  a.c.table = static_cast<const int32_t*>(block_table), a.c.bt_sb = bt_sb;
  a.c.lens = static_cast<const int32_t*>(context_lens);
  a.c.bs = block_size, a.c.nblocks = num_blocks, a.c.width = max_blocks;
  a.c.dbs = make_fastdiv((uint32_t)block_size);
  a.q = static_cast<const uint16_t*>(q), a.q_sb = q_sb, a.q_sh = q_sh;
  a.bound = static_cast<const float*>(bound), a.b_sb = b_sb, a.b_sh = b_sh;
  a.b_vec = reinterpret_cast<uintptr_t>(bound) % 16 == 0 && b_sb % 4 == 0 && b_sh % 4 == 0 && b_sh >= (max_blocks + 3) / 4 * 4;
  a.pages = static_cast<const int32_t*>(pages), a.p_sb = p_sb, a.p_sh = p_sh;
  a.out = static_cast<uint16_t*>(out), a.o_sb = o_sb, a.o_sh = o_sh;
  a.Hq = Hq, a.G = Hq / Hk, a.npick = npick;
  a.dHq = make_fastdiv((uint32_t)Hq), a.dG = make_fastdiv((uint32_t)a.G);
  a.scale_log2 = scale * kLog2e, a.v_scale = v_scale;
  const int64_t units = (int64_t)B * Hq;
  quest_plan(units, (int64_t)npick * block_size, block_size, pick_step(D, kv_fp8), &a.chunk, &a.nsplit);
  if (units * a.nsplit > 0x7FFFFFFF || units * (D / 64) > 0x7FFFFFFF) return (int)hipErrorInvalidConfiguration;
  a.nwg = (int)(units * a.nsplit);
  a.dsplit = make_fastdiv((uint32_t)a.nsplit);
  const size_t parts = quest_workspace(units, a.nsplit, D);
  const size_t need = parts + (bound ? selected_bytes(units, max_blocks, npick) : 0);
  if (need && (!workspace || workspace_bytes < need)) return (int)hipErrorInvalidValue;
  if (parts) {
    a.part_acc = static_cast<float*>(workspace);
    a.part_ml = a.part_acc + (size_t)units * a.nsplit * D;
  }
  const bool small = k_ss >= 0 && k_ss <= (1 << 24) && v_ss >= 0 && v_ss <= (1 << 24);      // 32-bit lane offsets
  const dim3 grid((unsigned)a.nwg), block(kPickThreads);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (bound && max_blocks > kPickMax) {
    int32_t* list = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + parts);
    hipLaunchKernelGGL(paged_select_kernel, dim3((unsigned)units), dim3(kSelectThreads), 0, st, a, list);
    rc = (int)hipGetLastError();
    if (rc) return rc;
    a.bound = nullptr;
    a.pages = list, a.p_sh = npick, a.p_sb = (int64_t)Hq * npick;
  }
#define PS(DD, F8)                                                                                                 \
  if (small && block_size % PickCfg<DD, F8>::RPI == 0)                                                             \
    hipLaunchKernelGGL((paged_quest_kernel<DD, F8, true>), grid, block, 0, st, a);                                 \
  else hipLaunchKernelGGL((paged_quest_kernel<DD, F8, false>), grid, block, 0, st, a)
  if (D == 128) {
    if (kv_fp8) { PS(128, true); }
    else { PS(128, false); }
  } else {
    if (kv_fp8) { PS(64, true); }
    else { PS(64, false); }
  }
#undef PS
  rc = (int)hipGetLastError();
  if (rc || a.nsplit <= 1) return rc;
  const dim3 jgrid((unsigned)(units * (D / 64)));
  if (D == 128) hipLaunchKernelGGL(paged_quest_join_kernel<128>, jgrid, dim3(64), 0, st, a);
  else hipLaunchKernelGGL(paged_quest_join_kernel<64>, jgrid, dim3(64), 0, st, a);
  return (int)hipGetLastError();
}

}  // extern "C"

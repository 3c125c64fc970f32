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
// bounds; wave_select.h), or takes a list of places, and walks their rows through
// the paged tile loop; heads of one KV head sit on one XCD, whose L2 then serves
// the blocks that several of them select.
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
  int tiles, rounds;                 // waves' tiles of blocks per (b, KV head); tiles per wave
  double scale;
};

constexpr int kBoundWaves = 4;

// D/8 lanes hold a block's min / max (8 dims each); a wave takes 64 / (D/8) blocks
// at a time for NH query heads of one KV head, whose q stays in registers.
template <int D, int NH>
__global__ __launch_bounds__(kBoundWaves * 64) void page_bound_kernel(PageBoundArgs a) {
  PREFETCH_ARGS(a);
  constexpr int LPR = D / 8, ROWS = 64 / LPR;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane % LPR, grp = lane / LPR;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int len = __builtin_amdgcn_readfirstlane(paged_len(a.c, b));
  const int full = fast_div(len + a.c.bs - 1, a.c.dbs);        // blocks that hold tokens
  if (full <= a.skip) return;
  const int recent = a.local_w > 0 ? fast_div(max(len - a.local_w, 0), a.c.dbs) : 0x7FFFFFFF;
  const int32_t* table = a.c.table + (int64_t)b * a.c.bt_sb;
  const int t0 = (blockIdx.x * kBoundWaves + w) * a.rounds;
  if (t0 >= a.tiles) return;
  for (int g0 = 0; g0 < a.G; g0 += NH) {
    const int nh = min(NH, a.G - g0);
    // q of the lane's dims, -0 as 0, and its sign masks (both halves of a word)
    float q[NH][8];
    uint32_t sign[NH][4];
#pragma unroll
    for (int g = 0; g < NH; ++g) {
      const u32x4 r = ld16(a.q + b * a.q_sb + (int64_t)(hk * a.G + g0 + min(g, nh - 1)) * a.q_sh + c * 8);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = __uint_as_float(r[j] << 16) + 0.f, y = __uint_as_float(r[j] & 0xFFFF0000u) + 0.f;
        q[g][2 * j] = x, q[g][2 * j + 1] = y;
        sign[g][j] = (x < 0.f ? 0xFFFFu : 0u) | (y < 0.f ? 0xFFFF0000u : 0u);
      }
    }
    for (int r = 0; r < a.rounds && t0 + r < a.tiles; ++r) {
      const int j = (t0 + r) * ROWS + grp, jc = min(j, a.c.width - 1);
      const int id = table[jc];
      const bool held = j < full && id >= 0 && id < a.c.nblocks;
      const int64_t m = ((int64_t)(held ? id : 0) * a.Hk + hk) * D + c * 8;
      const u32x4 lo = ld16(a.kmin + m), hi = ld16(a.kmax + m);
      float mine = 0.f;                            // of head c (and c + LPR) of the lane's block
      float mine2 = 0.f;
#pragma unroll
      for (int g = 0; g < NH; ++g) {
        double s = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t k = (lo[e] & sign[g][e]) | (hi[e] & ~sign[g][e]);
          s += (double)(q[g][2 * e] * __uint_as_float(k << 16));
          s += (double)(q[g][2 * e + 1] * __uint_as_float(k & 0xFFFF0000u));
        }
        // over the block's lanes: rotations within each row of LPR lanes
#define BYTES_ADD(CTRL)                                                                                   \
  {                                                                                                       \
    const uint64_t u = __builtin_bit_cast(uint64_t, s);                                                   \
    const uint32_t l32 = (uint32_t)__builtin_amdgcn_update_dpp((int)u, (int)u, CTRL, 0xF, 0xF, false);    \
    const uint32_t h32 = (uint32_t)__builtin_amdgcn_update_dpp((int)(u >> 32), (int)(u >> 32), CTRL, 0xF, 0xF, false); \
    s += __builtin_bit_cast(double, ((uint64_t)h32 << 32) | l32);                                         \
  }
        if (LPR == 16) BYTES_ADD(0x128)            // row_ror:8
        BYTES_ADD(0x141)                           // row_half_mirror: lane i of 8 and lane 7 - i
        BYTES_ADD(0x4E)                            // quad_perm 2,3,0,1
        BYTES_ADD(0xB1)                            // quad_perm 1,0,3,2
#undef BYTES_ADD
        float v = (float)(s * a.scale);
        if (j >= recent) v = __builtin_inff();
        if (!held) v = kNegInf;
        if (g < LPR) mine = c == g ? v : mine;
        else mine2 = c == g - LPR ? v : mine2;
      }
      if (j < a.c.width) {
        float* to = a.bound + b * a.b_sb + (int64_t)(hk * a.G + g0) * a.b_sh + j;
        if (c < nh) to[(int64_t)c * a.b_sh] = mine;
        if (NH > LPR && c + LPR < nh) to[(int64_t)(c + LPR) * a.b_sh] = mine2;
      }
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
  FastDiv dsplit, dHq, dG;
  float scale_log2, v_scale;
};

constexpr int kPickMax = 4096;       // blocks of a sequence that a workgroup selects from
constexpr int kPickThreads = kDenseWaves * 64;

// Selection of the k best of n bounds (k < n <= 256 * PER) into list, ascending.
template <int PER>
__device__ __forceinline__ void pick_blocks(const float* bound, int n, int k, uint32_t* ws, int32_t* list) {
  uint32_t key[PER];
  float v[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) v[u] = bound[min(PER * (int)threadIdx.x + u, n - 1)];
#pragma unroll
  for (int u = 0; u < PER; ++u) key[u] = score_order_key(v[u]);
  const BlockSel sel = block_select<kPickThreads, PER>(key, n, k, ws);
  block_select_emit<kPickThreads, PER>(key, n, sel, ws, [&](uint32_t pos, int idx, uint32_t) { list[pos] = idx; });
}

template <int D, bool FP8, bool HALVES>
__global__ __launch_bounds__(kPickThreads, 2) void paged_quest_kernel(PagedQuestArgs a) {
  using C = DenseCfg<D>;
  PREFETCH_ARGS(a);
  __shared__ __attribute__((aligned(16))) char smem[C::kSmem];
  __shared__ int32_t list[kPickMax];
  static_assert(block_select_words<kPickThreads>() * 4 <= C::kSmem, "the selection's words fit the tile buffers");
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int idx = xcd_run(blockIdx.x, a.nwg), unit = fast_div(idx, a.dsplit), split = idx - unit * a.nsplit;
  const int b = fast_div(unit, a.dHq), h = unit - b * a.Hq, hk = fast_div(h, a.dG);
  const int len = __builtin_amdgcn_readfirstlane(paged_len(a.c, b));
  const int full = fast_div(len + a.c.bs - 1, a.c.dbs);
  const int picks = a.bound ? min(a.npick, full) : a.npick;
  const int s0 = split * a.chunk, s1 = min(s0 + a.chunk, picks * a.c.bs);
  if (split > 0 && s0 >= s1) return;               // (split 0 of an empty sequence writes its zeros)
  bf16x8 qb[C::KK];
  load_q_bf16<D>(a.q + (int64_t)b * a.q_sb + (int64_t)h * a.q_sh, a.q_sh, 1, lane, qb);
  const bool select = a.bound && full > a.npick;
  if (select) {
    const float* bound = a.bound + (int64_t)b * a.b_sb + (int64_t)h * a.b_sh;
    uint32_t* ws = reinterpret_cast<uint32_t*>(smem);
    if (full <= 4 * kPickThreads) pick_blocks<4>(bound, full, a.npick, ws, list);
    else if (full <= 8 * kPickThreads) pick_blocks<8>(bound, full, a.npick, ws, list);
    else pick_blocks<16>(bound, full, a.npick, ws, list);
    __syncthreads();
  }
  const int32_t* pages = a.pages + b * a.p_sb + h * a.p_sh;
  auto find = [&](int s, int& place, int& off, bool& ok) {
    const int i = fast_div(s, a.c.dbs);
    off = s - i * a.c.bs;
    const int j = select ? list[i] : a.bound ? i : pages[i];
    ok = j >= 0 && j < full && j * a.c.bs + off < len;
    place = ok ? j : 0;
  };
  float m_run = kNegInf, l_run = 0.f;
  f32x4 acc[C::DB];
#pragma unroll
  for (int db = 0; db < C::DB; ++db) acc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  paged_wave_loop<D, FP8, HALVES>(a.c, a.c.table + (int64_t)b * a.c.bt_sb, hk, s0 + w * kTile, s1, kDenseWaves * kTile,
                                  lane, a.scale_log2, qb, smem + w * C::WAVE, find, m_run, l_run, acc);
  const bool whole = picks * a.c.bs <= a.chunk;
  uint16_t* out = a.out + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh;
  const size_t r = (size_t)unit * a.nsplit + split;
  paged_merge_waves<D>(m_run, l_run, acc, reinterpret_cast<float*>(smem), 1,
                       [&](int, int d4, const f32x4& A, float M, float L) {
                         if (whole) {
                           paged_store(out + 4 * d4, A, L, a.v_scale);
                         } else {
                           reinterpret_cast<f32x4*>(a.part_acc + r * D)[d4] = A;
                           if (d4 == 0) reinterpret_cast<float2*>(a.part_ml)[r] = make_float2(M, L);
                         }
                       });
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

// Runs of a head's slots: as many as make about two workgroups per CU, a multiple
// of 128 slots (one tile per wave), at least that.
static void quest_plan(int64_t units, int64_t slots, int* chunk, int* nsplit) {
  const int step = kDenseWaves * kTile;
  const int64_t target = 2 * device_cu_count();
  int64_t c = (slots * units + target - 1) / target;
  c = (c + step - 1) / step * step;
  if (c < step) c = step;
  *chunk = (int)(c < 0x7FFFFF80 ? c : 0x7FFFFF80);
  *nsplit = (int)((slots + *chunk - 1) / *chunk);
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
  // tiles of blocks: one per wave until that makes 16 waves per CU, then several
  const int rows = 64 / (D / 8);
  a.tiles = (max_blocks + rows - 1) / rows;
  const int64_t waves = (int64_t)a.tiles * Hk * B, most = 16 * (int64_t)device_cu_count();
  a.rounds = (int)((waves + most - 1) / most);
  const int per_wg = a.rounds * kBoundWaves;
  const dim3 grid((unsigned)((a.tiles + per_wg - 1) / per_wg), (unsigned)Hk, (unsigned)B), block(kBoundWaves * 64);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define PB(DD, N) hipLaunchKernelGGL((page_bound_kernel<DD, N>), grid, block, 0, st, a)
  if (D == 128) {
    if (a.G <= 4) PB(128, 4);
    else PB(128, 8);
  } else {
    if (a.G <= 4) PB(64, 4);
    else PB(64, 8);
  }
#undef PB
  return (int)hipGetLastError();
}

int bytes_paged_quest_workspace_size(int B, int Hq, int Hk, int D, int block_size, int npick, size_t* bytes) {
  if (!bytes || B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 || (D != 64 && D != 128) || npick <= 0)
    return (int)hipErrorInvalidValue;
  const int rc = paged_check(block_size, 1, npick);
  if (rc) return rc;
  int chunk, ns;
  quest_plan((int64_t)B * Hq, (int64_t)npick * block_size, &chunk, &ns);
  *bytes = quest_workspace((int64_t)B * Hq, ns, D);
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
  if (bound && max_blocks > kPickMax) return (int)hipErrorNotSupported;
  PagedQuestArgs a = {};
  a.c.k = k_paged, a.c.k_sb = k_sb, a.c.k_sh = k_sh, a.c.k_ss = k_ss;
  a.c.v = v_paged, a.c.v_sb = v_sb, a.c.v_sh = v_sh, a.c.v_ss = v_ss;
  a.c.table = static_cast<const int32_t*>(block_table), a.c.bt_sb = bt_sb;
  a.c.lens = static_cast<const int32_t*>(context_lens);
  a.c.bs = block_size, a.c.nblocks = num_blocks, a.c.width = max_blocks;
  a.c.dbs = make_fastdiv((uint32_t)block_size);
  a.q = static_cast<const uint16_t*>(q), a.q_sb = q_sb, a.q_sh = q_sh;
  a.bound = static_cast<const float*>(bound), a.b_sb = b_sb, a.b_sh = b_sh;
  a.pages = static_cast<const int32_t*>(pages), a.p_sb = p_sb, a.p_sh = p_sh;
  a.out = static_cast<uint16_t*>(out), a.o_sb = o_sb, a.o_sh = o_sh;
  a.Hq = Hq, a.G = Hq / Hk, a.npick = npick;
  a.dHq = make_fastdiv((uint32_t)Hq), a.dG = make_fastdiv((uint32_t)a.G);
  a.scale_log2 = scale * kLog2e, a.v_scale = v_scale;
  const int64_t units = (int64_t)B * Hq;
  quest_plan(units, (int64_t)npick * block_size, &a.chunk, &a.nsplit);
  if (units * a.nsplit > 0x7FFFFFFF || units * (D / 64) > 0x7FFFFFFF) return (int)hipErrorInvalidConfiguration;
  a.nwg = (int)(units * a.nsplit);
  a.dsplit = make_fastdiv((uint32_t)a.nsplit);
  const size_t need = quest_workspace(units, a.nsplit, D);
  if (need && (!workspace || workspace_bytes < need)) return (int)hipErrorInvalidValue;
  if (need) {
    a.part_acc = static_cast<float*>(workspace);
    a.part_ml = a.part_acc + (size_t)units * a.nsplit * D;
  }
  const bool halves = paged_halves(a.c);
  const dim3 grid((unsigned)a.nwg), block(kPickThreads);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define PS(DD, F8, H) hipLaunchKernelGGL((paged_quest_kernel<DD, F8, H>), grid, block, 0, st, a)
#define PS_H(DD, F8)            \
  if (halves) PS(DD, F8, true); \
  else PS(DD, F8, false)
  if (D == 128) {
    if (kv_fp8) { PS_H(128, true); }
    else { PS_H(128, false); }
  } else {
    if (kv_fp8) { PS_H(64, true); }
    else { PS_H(64, false); }
  }
#undef PS_H
#undef PS
  rc = (int)hipGetLastError();
  if (rc || a.nsplit <= 1) return rc;
  const dim3 jgrid((unsigned)(units * (D / 64)));
  if (D == 128) hipLaunchKernelGGL(paged_quest_join_kernel<128>, jgrid, dim3(64), 0, st, a);
  else hipLaunchKernelGGL(paged_quest_join_kernel<64>, jgrid, dim3(64), 0, st, a);
  return (int)hipGetLastError();
}

}  // extern "C"

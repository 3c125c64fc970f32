// Attention of one new token per sequence over a paged cache: the even split of a
// batch's tokens over the grid, the kernel for short contexts and the join, for
// arguments ARGS whose slots() and view() say which tokens a sequence's query sees
// (paged_attn.hip: all of them).
#pragma once
#include "paged.h"

namespace bytes_amd {

constexpr int kGranule = kDenseWaves * kTile;      // tokens

struct PagedDecodeArgs {
  PagedKv c;
  const uint16_t* q;
  int64_t q_sb, q_sh;
  uint16_t* out;
  int64_t o_sb, o_sh;
  float* part_acc;                   // [workgroup][2][16][D]
  float* part_ml;                    // [workgroup][2][16][2]
  int B, Hk, HB, G, U;               // U = Hk * HB units per sequence
  int nwg;
  FastDiv dnwg, dhb, dG, dU;
  float scale_log2, v_scale;

  // The slots that a unit of a sequence of n tokens walks, and what a slot stands for
  // (paged_wave_loop's find): here every token.
  struct View {
    FastDiv dbs;
    __device__ __forceinline__ void operator()(int p, int& place, int& off, bool& ok) const {
      place = fast_div(p, dbs);
      off = p - place * (int)dbs.d;
      ok = true;
    }
  };
  __device__ __forceinline__ View view(int) const { return View{c.dbs}; }
  __device__ __forceinline__ int slots(int n) const { return n; }
  __device__ __forceinline__ PagedScales scales(int, float*) const { return PagedScales{}; }
  // What a token's dim counts in the choice of short_waves: the bytes of a key and a value.
  static constexpr int dim_cost(int type) { return type == kBf16Cache ? 4 : 2; }
};

// Granules of a sequence of n tokens: an empty one has one too, whose output is written like any other.
__device__ __forceinline__ int granules(int n) { return max(1, (n + kGranule - 1) / kGranule); }

// The batch's granules: lane l sums those of sequences l * per .. + per - 1.
template <class ARGS>
struct BatchGranules {
  uint32_t mine, incl;
  int per, total;                    // sequences per lane; granules of the batch, all units
  int len0;                          // length of the lane's last sequence: its only one where per == 1

  __device__ __forceinline__ BatchGranules(const ARGS& a, int lane) {
    per = (a.B + 63) / 64;
    mine = 0u;
    len0 = 0;
    for (int i = 0; i < per; ++i) {
      const int b = lane * per + i;
      len0 = paged_len(a.c, min(b, a.B - 1));
      mine += b < a.B ? (uint32_t)granules(a.slots(len0)) : 0u;
    }
    incl = wave_prefix_sum(mine);
    total = __builtin_amdgcn_readlane((int)incl, 63) * a.U;
  }
  // Length of sequence b, from the lane that holds it where there are at most 64.
  __device__ __forceinline__ int length(const ARGS& a, int b) const {
    return per == 1 ? __builtin_amdgcn_readlane(len0, b) : __builtin_amdgcn_readfirstlane(paged_len(a.c, b));
  }
  // Granules of one unit of each sequence before b.
  __device__ __forceinline__ int before(const ARGS& a, int b) const {
    const int l = b / per;
    int n = __builtin_amdgcn_readlane((int)(incl - mine), l);
    for (int i = l * per; i < b; ++i) n += granules(a.slots(length(a, i)));
    return n;
  }
  // The sequence that granule g lies in, its length, and its first granule.
  __device__ __forceinline__ void find(const ARGS& a, int g, int& b, int& len, int& first) const {
    const int l = __ffsll((unsigned long long)__ballot((int)incl * a.U > g)) - 1;
    first = __builtin_amdgcn_readlane((int)(incl - mine), l) * a.U;
    for (b = l * per;; ++b) {
      len = length(a, b);
      const int n = granules(a.slots(len)) * a.U;
      if (g < first + n || b == a.B - 1) return;
      first += n;
    }
  }
  // Runs: workgroup w has granules [start(w), start(w + 1)).
  __device__ __forceinline__ int start(const ARGS& a, int w) const {
    const int q = fast_div(total, a.dnwg), r = total - q * a.nwg;
    return w * q + min(w, r);
  }
  __device__ __forceinline__ int owner(const ARGS& a, int g) const {
    const int q = fast_div(total, a.dnwg), r = total - q * a.nwg, big = r * (q + 1);
    return g < big ? g / (q + 1) : r + (g - big) / q;
  }
};

template <class ARGS, int D, int TYPE, bool HALVES>
__global__ __launch_bounds__(kDenseWaves * 64, 2) void paged_decode_kernel(ARGS a) {
  using C = DenseCfg<D>;
  __shared__ __attribute__((aligned(16))) char smem[C::kSmem];
  __shared__ float sc[TYPE >= kE4m3Blocks ? kDenseWaves * 64 : 1];
  PREFETCH_ARGS(a);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const BatchGranules<ARGS> all(a, lane);
  const int g0 = all.start(a, blockIdx.x), g1 = all.start(a, blockIdx.x + 1);
  if (g0 >= g1) return;
  int b, len, first;
  all.find(a, g0, b, len, first);
  int n = granules(a.slots(len));                  // of one unit of the sequence
  int u = (g0 - first) / n, t = g0 - first - u * n;
  for (int g = g0;;) {
    const int m = min(n - t, g1 - g);              // granules of this part
    const int hk = fast_div(u, a.dhb), hb = u - hk * a.HB;
    const int hq0 = hk * a.G + hb * 16, nh = min(16, a.G - hb * 16);
    bf16x8 qb[C::KK];
    load_q_bf16<D>(a.q + (int64_t)b * a.q_sb + (int64_t)hq0 * a.q_sh, a.q_sh, nh, lane, qb);
    float m_run = kNegInf, l_run = 0.f;
    f32x4 acc[C::DB];
#pragma unroll
    for (int db = 0; db < C::DB; ++db) acc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    paged_wave_loop<D, TYPE, HALVES>(a.c, a.c.table + (int64_t)b * a.c.bt_sb, hk, t * kGranule + w * kTile,
                                     min(a.slots(len), (t + m) * kGranule), kGranule, lane, a.scale_log2, qb,
                                     smem + w * C::WAVE, a.view(len), m_run, l_run, acc, a.scales(hk, sc + w * 64));
    const bool whole = m == n;
    uint16_t* out = a.out + (int64_t)b * a.o_sb + (int64_t)hq0 * a.o_sh;
    const size_t slot = ((size_t)blockIdx.x * 2 + (g == g0 ? 0 : 1)) * 16;
    paged_merge_waves<D, kDenseWaves>(m_run, l_run, acc, reinterpret_cast<float*>(smem), nh,
                         [&](int h, int d4, const f32x4& A, float M, float L) {
                           if (whole) {
                             paged_store(out + (int64_t)h * a.o_sh + 4 * d4, A, L, a.v_scale);
                           } else {
                             reinterpret_cast<f32x4*>(a.part_acc + (slot + h) * D)[d4] = A;
                             if (d4 == 0) reinterpret_cast<float2*>(a.part_ml)[slot + h] = make_float2(M, L);
                           }
                         });
    g += m;
    if (g >= g1) return;
    t = 0;
    if (++u == a.U) {
      u = 0;
      ++b;
      len = all.length(a, b);
      n = granules(a.slots(len));
    }
  }
}

// Short contexts: a workgroup of NW waves per unit, which it finishes itself.
template <class ARGS, int D, int TYPE, bool HALVES, int NW>
__global__ __launch_bounds__(NW * 64) void paged_decode_short_kernel(ARGS a) {
  using C = DenseCfg<D>;
  static_assert(NW * C::WAVE >= splitk_smem_floats<D, NW>() * 4, "the merge fits the tile buffers");
  __shared__ __attribute__((aligned(16))) char smem[NW * C::WAVE];
  __shared__ float sc[TYPE >= kE4m3Blocks ? NW * 64 : 1];
  PREFETCH_ARGS(a);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = fast_div((int)blockIdx.x, a.dU), u = (int)blockIdx.x - b * a.U, hk = fast_div(u, a.dhb), hb = u - hk * a.HB;
  const int hq0 = hk * a.G + hb * 16, nh = min(16, a.G - hb * 16);
  const int len = __builtin_amdgcn_readfirstlane(paged_len(a.c, b));
  bf16x8 qb[C::KK];
  load_q_bf16<D>(a.q + (int64_t)b * a.q_sb + (int64_t)hq0 * a.q_sh, a.q_sh, nh, lane, qb);
  float m_run = kNegInf, l_run = 0.f;
  f32x4 acc[C::DB];
#pragma unroll
  for (int db = 0; db < C::DB; ++db) acc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  paged_wave_loop<D, TYPE, HALVES>(a.c, a.c.table + (int64_t)b * a.c.bt_sb, hk, w * kTile, a.slots(len), NW * kTile,
                                   lane, a.scale_log2, qb, smem + w * C::WAVE, a.view(len), m_run, l_run, acc,
                                   a.scales(hk, sc + w * 64));
  uint16_t* out = a.out + (int64_t)b * a.o_sb + (int64_t)hq0 * a.o_sh;
  paged_merge_waves<D, NW>(m_run, l_run, acc, reinterpret_cast<float*>(smem), nh,
                           [&](int h, int d4, const f32x4& A, float, float L) {
                             paged_store(out + (int64_t)h * a.o_sh + 4 * d4, A, L, a.v_scale);
                           });
}

// Joins the parts of each unit that more than one workgroup had: one wave per
// (sequence, query head, 64 dims).  3 to 6 us, a launch and its round trips; a join
// by the last workgroup to end would need counters that start every call at zero.
template <class ARGS, int D>
__global__ __launch_bounds__(64) void paged_join_kernel(ARGS a) {
  constexpr int NSL = D / 64;
  const int lane = threadIdx.x, item = lane & 15, grp = lane >> 4;
  const int slice = blockIdx.x % NSL, h = blockIdx.x / NSL, b = blockIdx.y;     // h: query head
  const BatchGranules<ARGS> all(a, lane);
  const int hk = fast_div(h, a.dG), hb = (h - hk * a.G) / 16, hl = h - hk * a.G - hb * 16;
  const int n = granules(a.slots(all.length(a, b)));
  const int s = all.before(a, b) * a.U + (hk * a.HB + hb) * n;
  const int w0 = all.owner(a, s), w1 = all.owner(a, s + n - 1);
  if (w0 == w1) return;                            // finished in place
  const int parts = w1 - w0 + 1;
  const int slot0 = all.start(a, w0) == s ? 0 : 1;
  auto slot = [&](int i) { return ((size_t)(w0 + i) * 2 + (i == 0 ? slot0 : 0)) * 16 + hl; };
  paged_join<8>(parts, lane, slot, reinterpret_cast<const float2*>(a.part_ml),
                reinterpret_cast<const f32x4*>(a.part_acc) + slice * 16 + item, D / 4, [&](const f32x4& A, float L) {
                  if (grp == 0) paged_store(a.out + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + slice * 64 + item * 4, A, L,
                                            a.v_scale);
                });
}

// Workgroups of the decode grid: one per CU, whose four waves' tiles in flight
// are what a CU's share of the memory system takes (eight sequences of up to 8K:
// 24.3 us, 25.3 with two per CU, whose parts are twice as many to join; four of
// 128K: 248 with either); two where the units are as many as the CUs, so that one
// starts and ends its units while the other streams (64 sequences of up to 500
// tokens: 14.4 with one, 13.2 with two; 32 of 16K: 228 and 229).  Never more than
// the batch's granules.
static int decode_grid(int64_t units, int64_t granules_max) {
  const int64_t cus = device_cu_count(), n = units >= cus ? 2 * cus : cus;
  return (int)(granules_max < n ? granules_max : n);
}

// Waves of a workgroup that does a whole unit by itself (one launch, no parts to
// join), or 0 for the even split.  By the bytes of a full table row, which one CU
// reads at about 50 GB/s: up to 256 KB (us from a graph, so without what a second
// launch costs the host; whole unit and split: one sequence of
// 2 KV heads of 64, 500 tokens 5.7 and 7.1, 1000 tokens 8.0 and 7.1; of 4 heads of
// 128, 500 tokens 7.8 and 8.3, 1000 tokens 13.4 and 8.9), twice that where the
// units keep half the CUs busy anyway (64 sequences of 4 heads of 128, 500 tokens
// 10.7 and 13.3, 1000 tokens 17.2 and 20.8).  Four waves where a tile each
// covers the row, or where two workgroups to a CU have units enough (200 sequences
// of 4 heads, 100 tokens: 15.8 with eight, 9.1 with four; split 18.0).
static int short_waves(int64_t units, int64_t cap, int D, int dim_cost) {
  const int64_t cus = device_cu_count(), bytes = cap * D * dim_cost;
  if (bytes > (2 * units >= cus ? 512 << 10 : 256 << 10)) return 0;
  return cap <= 4 * kTile || units >= 2 * cus ? 4 : 8;
}

struct DecodeShape {
  int64_t units, granules;           // of the batch, at most
};
static DecodeShape decode_shape(int B, int Hq, int Hk, int64_t cap) {
  const int G = Hq / Hk, HB = (G + 15) / 16;
  const int64_t per = (cap + kGranule - 1) / kGranule, units = (int64_t)B * Hk * HB;
  return {units, units * (per < 1 ? 1 : per)};
}

static size_t decode_workspace(int nwg, int D) { return (size_t)nwg * 2 * 16 * (D + 2) * 4; }

// The kernels of arguments a, whose tables hold `cap` slots at most; 0 or a hipError_t.
template <class ARGS, int D, int TYPE, bool HALVES>
int launch_decode(const ARGS& a, const DecodeShape& shape, int64_t cap, hipStream_t st) {
  const int waves = short_waves(shape.units, cap, D, ARGS::dim_cost(TYPE));
  if (waves) {
    const dim3 grid((unsigned)shape.units);
    if (waves == 4) hipLaunchKernelGGL((paged_decode_short_kernel<ARGS, D, TYPE, HALVES, 4>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_decode_short_kernel<ARGS, D, TYPE, HALVES, 8>), grid, dim3(512), 0, st, a);
    return (int)hipGetLastError();
  }
  hipLaunchKernelGGL((paged_decode_kernel<ARGS, D, TYPE, HALVES>), dim3((unsigned)a.nwg), dim3(kDenseWaves * 64), 0, st, a);
  const int rc = (int)hipGetLastError();
  if (rc) return rc;
  hipLaunchKernelGGL((paged_join_kernel<ARGS, D>), dim3((unsigned)(a.Hk * a.G * (D / 64)), (unsigned)a.B), dim3(64), 0, st, a);
  return (int)hipGetLastError();
}
template <class ARGS, int TYPE>
int launch_decode_of(const ARGS& a, int D, const DecodeShape& shape, int64_t cap, hipStream_t st) {
  const bool halves = paged_halves(a.c);
  if (D == 128)
    return halves ? launch_decode<ARGS, 128, TYPE, true>(a, shape, cap, st) : launch_decode<ARGS, 128, TYPE, false>(a, shape, cap, st);
  return halves ? launch_decode<ARGS, 64, TYPE, true>(a, shape, cap, st) : launch_decode<ARGS, 64, TYPE, false>(a, shape, cap, st);
}

// The arguments that every form shares, from a C entry's; the workspace for the parts.
inline void decode_args(PagedDecodeArgs& a, const void* q, int64_t q_sb, int64_t q_sh, const void* k, int64_t k_sb,
                        int64_t k_sh, int64_t k_ss, const void* v, int64_t v_sb, int64_t v_sh, int64_t v_ss,
                        const void* table, int64_t bt_sb, const void* lens, void* out, int64_t o_sb, int64_t o_sh, int B,
                        int Hq, int Hk, int block_size, int num_blocks, int max_blocks, const DecodeShape& shape,
                        void* workspace) {
  a.c.k = k, a.c.k_sb = k_sb, a.c.k_sh = k_sh, a.c.k_ss = k_ss;
  a.c.v = v, a.c.v_sb = v_sb, a.c.v_sh = v_sh, a.c.v_ss = v_ss;
  a.c.table = static_cast<const int32_t*>(table), a.c.bt_sb = bt_sb;
  a.c.lens = static_cast<const int32_t*>(lens);
  a.c.bs = block_size, a.c.nblocks = num_blocks, a.c.width = max_blocks;
  a.c.dbs = make_fastdiv((uint32_t)block_size);
  a.q = static_cast<const uint16_t*>(q), a.q_sb = q_sb, a.q_sh = q_sh;
  a.out = static_cast<uint16_t*>(out), a.o_sb = o_sb, a.o_sh = o_sh;
  a.B = B, a.Hk = Hk, a.G = Hq / Hk, a.HB = (a.G + 15) / 16, a.U = Hk * a.HB;
  a.nwg = decode_grid(shape.units, shape.granules);
  a.dnwg = make_fastdiv((uint32_t)a.nwg), a.dhb = make_fastdiv((uint32_t)a.HB), a.dG = make_fastdiv((uint32_t)a.G);
  a.dU = make_fastdiv((uint32_t)a.U);
  a.part_ml = static_cast<float*>(workspace);
  a.part_acc = a.part_ml + (size_t)a.nwg * 2 * 16 * 2;
}

}  // namespace bytes_amd

// Page-sparse decode over a paged KV cache: block bounds, and attention over
// the blocks that they select.
//
//   bound[b, h, j] = scale * sum_d q_d * (q_d >= 0 ? kmax_d : kmin_d)
//
// over the min / max of block table[b, j], the largest score that any of its
// keys can have.  The products of bf16 values are exact in fp64 and are summed
// there, so the order of the sum does not move a selection; the result is
// rounded to fp32 once.  Blocks that hold no token that takes part (paged.h) get
// -inf, blocks that reach into the sequence's last local_w tokens +inf.
#include "paged.h"

namespace bytes_amd {

struct PageBoundArgs {
  PagedKv c;
  const uint16_t *q, *kmin, *kmax;
  int64_t q_sb, q_sh;
  float* bound;
  int64_t b_sb, b_sh;
  int Hk, G, D, local_w;
  double scale;
};

// One thread per (block, query head).
__global__ __launch_bounds__(256) void page_bound_kernel(PageBoundArgs a) {
  const int j = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y, b = blockIdx.z;
  if (j >= a.c.width) return;
  const int len = paged_len(a.c, b), id = a.c.table[(int64_t)b * a.c.bt_sb + j];
  float r = kNegInf;
  if (j * a.c.bs < len && id >= 0 && id < a.c.nblocks) {
    if (a.local_w > 0 && j >= fast_div(max(len - a.local_w, 0), a.c.dbs)) {
      r = __builtin_inff();
    } else {
      const int64_t m = ((int64_t)id * a.Hk + h / a.G) * a.D;
      const uint16_t* q = a.q + b * a.q_sb + h * a.q_sh;
      double s = 0.0;
      for (int d = 0; d < a.D; ++d) {
        const float x = bf16_bits_to_f32(q[d]);
        s += (double)x * (double)bf16_bits_to_f32(x >= 0.f ? a.kmax[m + d] : a.kmin[m + d]);
      }
      r = (float)(s * a.scale);
    }
  }
  a.bound[b * a.b_sb + h * a.b_sh + j] = r;
}

struct PagedQuestArgs {
  PagedKv c;
  const uint16_t* q;
  int64_t q_sb, q_sh;
  const int32_t* pages;              // [B, Hq, npick], row strides p_sb, p_sh
  int64_t p_sb, p_sh;
  uint16_t* out;
  int64_t o_sb, o_sh;
  int Hq, G, npick;
  float scale_log2, v_scale;
};

// One workgroup per query head.
template <int D, bool FP8>
__global__ __launch_bounds__(kDenseWaves * 64, 2) void paged_pick_attn_kernel(PagedQuestArgs a) {
  using C = DenseCfg<D>;
  __shared__ __attribute__((aligned(16))) char smem[C::kSmem];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15, lg = lane >> 4;
  const int h = blockIdx.x % a.Hq, b = blockIdx.x / a.Hq, hk = h / a.G;
  bf16x8 qb[C::KK];
  load_q_bf16<D>(a.q + (int64_t)b * a.q_sb + (int64_t)h * a.q_sh, a.q_sh, 1, lane, qb);
  const int len = paged_len(a.c, b), n = a.npick * a.c.bs;
  const int32_t* table = a.c.table + (int64_t)b * a.c.bt_sb;
  const int32_t* pages = a.pages + b * a.p_sb + h * a.p_sh;
  char* kst = smem + w * C::WAVE;
  char* vst = kst + C::VT;
  float m_run = kNegInf, l_run = 0.f;
  f32x4 acc[C::DB];
#pragma unroll
  for (int db = 0; db < C::DB; ++db) acc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  using Regs = typename std::conditional<FP8, DenseRegs8<D>, DenseRegs<D>>::type;
  using Elem = typename std::conditional<FP8, uint8_t, uint16_t>::type;
  constexpr int CPR = FP8 ? D / 16 : D / 8, CPL = kTile * CPR / 64, EPC = FP8 ? 16 : 8;
  const Elem* kb = static_cast<const Elem*>(a.c.k) + hk * a.c.k_sh;
  const Elem* vb = static_cast<const Elem*>(a.c.v) + hk * a.c.v_sh;
  auto row = [&](int s, int& id, int& off, bool& ok) {
    const int ss = min(s, n - 1), i = fast_div(ss, a.c.dbs);
    const int j = pages[i];
    off = ss - i * a.c.bs;
    ok = s < n && j >= 0 && j < a.c.width && (int64_t)j * a.c.bs + off < len;
    id = table[ok ? j : 0];
    ok = ok && id >= 0 && id < a.c.nblocks;
    id = ok ? id : 0;
  };
  for (int t = w * kTile; t < n; t += kDenseWaves * kTile) {
    int id, off;
    bool ok;
    row(t + (lane & 31), id, off, ok);
    const uint32_t vmask = (uint32_t)__ballot(ok);
    Regs r;
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      const int pl = lane + 64 * i, rr = pl / CPR, col = (pl - rr * CPR) * EPC;
      row(t + rr, id, off, ok);
      r.k[i] = ld16(kb + id * a.c.k_sb + off * a.c.k_ss + col);
      r.v[i] = ld16_live(vb + id * a.c.v_sb + off * a.c.v_ss + col, ok);
    }
    wave_lds_sync();
    if constexpr (FP8) dense_stage_fp8<D>(lane, r, kst, vst);
    else dense_stage<D>(lane, r, kst, vst);
    wave_lds_sync();
    dense_compute<D>(vmask, a.scale_log2, lane, qb, kst, vst, m_run, l_run, acc);
  }
  constexpr int P = acc_pitch<D>();
  l_run = col_sum4(l_run);
  float* wm = reinterpret_cast<float*>(smem);
  float* wl = wm + kDenseWaves * 16;
  float* wacc = wl + kDenseWaves * 16;
  __syncthreads();
  if (lg == 0) {
    wm[w * 16 + l16] = m_run;
    wl[w * 16 + l16] = l_run;
  }
  f32x4* arow = reinterpret_cast<f32x4*>(wacc + (w * 16 + l16) * P);
#pragma unroll
  for (int db = 0; db < C::DB; ++db) arow[4 * db + lg] = acc[db];
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kDenseWaves * 64) {
    float M = kNegInf, L = 0.f, A = 0.f;
#pragma unroll
    for (int u = 0; u < kDenseWaves; ++u) M = fmaxf(M, wm[u * 16]);
    const float Ms = M == kNegInf ? 0.f : M;
#pragma unroll
    for (int u = 0; u < kDenseWaves; ++u) {
      const float f = fast_exp2(wm[u * 16] - Ms);
      L += f * wl[u * 16];
      A += f * wacc[u * 16 * P + d];
    }
    a.out[(int64_t)b * a.o_sb + (int64_t)h * a.o_sh + d] = f32_to_bf16_bits(L == 0.f ? 0.f : A / L * a.v_scale);
  }
}

}  // namespace bytes_amd

using namespace bytes_amd;

extern "C" {

int bytes_paged_page_scores(const void* q, int64_t q_sb, int64_t q_sh, const void* kmin, const void* kmax,
                            const void* block_table, int64_t bt_sb, const void* context_lens, void* bound, int64_t b_sb,
                            int64_t b_sh, int B, int Hq, int Hk, int D, int block_size, int num_blocks, int max_blocks,
                            int local_w, double scale, void* stream) {
  if (!q || !kmin || !kmax || !block_table || !context_lens || !bound || B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 ||
      (D != 64 && D != 128) || local_w < 0 || max_blocks <= 0)
    return (int)hipErrorInvalidValue;
  int rc = paged_check(block_size, num_blocks, max_blocks);
  if (rc) return rc;
  if (B > 65535 || Hq > 65535) return (int)hipErrorInvalidConfiguration;
  PageBoundArgs a;
  a.c = PagedKv{};
  a.c.table = static_cast<const int32_t*>(block_table), a.c.bt_sb = bt_sb;
  a.c.lens = static_cast<const int32_t*>(context_lens);
  a.c.bs = block_size, a.c.nblocks = num_blocks, a.c.width = max_blocks;
  a.c.dbs = make_fastdiv((uint32_t)block_size);
  a.q = static_cast<const uint16_t*>(q), a.q_sb = q_sb, a.q_sh = q_sh;
  a.kmin = static_cast<const uint16_t*>(kmin), a.kmax = static_cast<const uint16_t*>(kmax);
  a.bound = static_cast<float*>(bound), a.b_sb = b_sb, a.b_sh = b_sh;
  a.Hk = Hk, a.G = Hq / Hk, a.D = D, a.local_w = local_w, a.scale = scale;
  const dim3 grid((unsigned)((max_blocks + 255) / 256), (unsigned)Hq, (unsigned)B);
  hipLaunchKernelGGL(page_bound_kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
  return (int)hipGetLastError();
}

int bytes_paged_pick_attn(const void* q, int64_t q_sb, int64_t q_sh, const void* k_paged, int64_t k_sb, int64_t k_sh,
                          int64_t k_ss, const void* v_paged, int64_t v_sb, int64_t v_sh, int64_t v_ss, int kv_fp8,
                          const void* pages, int64_t p_sb, int64_t p_sh, int npick, const void* block_table,
                          int64_t bt_sb, const void* context_lens, void* out, int64_t o_sb, int64_t o_sh, int B, int Hq,
                          int Hk, int D, int block_size, int num_blocks, int max_blocks, float scale, float v_scale,
                          void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !k_paged || !v_paged || !pages || !block_table || !context_lens || !out || B <= 0 || Hk <= 0 || Hq <= 0 ||
      Hq % Hk != 0 || (D != 64 && D != 128) || npick <= 0 || npick > max_blocks)
    return (int)hipErrorInvalidValue;
  int rc = paged_check(block_size, num_blocks, max_blocks);
  if (rc) return rc;
  PagedQuestArgs a;
  a.c.k = k_paged, a.c.k_sb = k_sb, a.c.k_sh = k_sh, a.c.k_ss = k_ss;
  a.c.v = v_paged, a.c.v_sb = v_sb, a.c.v_sh = v_sh, a.c.v_ss = v_ss;
  a.c.table = static_cast<const int32_t*>(block_table), a.c.bt_sb = bt_sb;
  a.c.lens = static_cast<const int32_t*>(context_lens);
  a.c.bs = block_size, a.c.nblocks = num_blocks, a.c.width = max_blocks;
  a.c.dbs = make_fastdiv((uint32_t)block_size);
  a.q = static_cast<const uint16_t*>(q), a.q_sb = q_sb, a.q_sh = q_sh;
  a.pages = static_cast<const int32_t*>(pages), a.p_sb = p_sb, a.p_sh = p_sh;
  a.out = static_cast<uint16_t*>(out), a.o_sb = o_sb, a.o_sh = o_sh;
  a.Hq = Hq, a.G = Hq / Hk, a.npick = npick;
  a.scale_log2 = scale * kLog2e, a.v_scale = v_scale;
  if ((int64_t)B * Hq > 0x7FFFFFFF) return (int)hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)(B * Hq)), block(kDenseWaves * 64);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define PQ_(DD, F8) hipLaunchKernelGGL((paged_pick_attn_kernel<DD, F8>), grid, block, 0, st, a)
  if (D == 128) {
    if (kv_fp8) PQ_(128, true);
    else PQ_(128, false);
  } else {
    if (kv_fp8) PQ_(64, true);
    else PQ_(64, false);
  }
#undef PQ_
  return (int)hipGetLastError();
}

}  // extern "C"

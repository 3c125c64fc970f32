// Attention of one new token per sequence over a paged KV cache.
//
//   out[b, h] = v_scale * softmax_p(scale * q[b, h] . k[b, h / G, p]) v[b, h / G, p]
//
// over the tokens p of sequence b that take part (paged.h); a row none of whose
// tokens does gets zeros.  Scores, softmax statistics and sums are fp32 (K, V
// and Q products on MFMA are exact in fp32; the weights go to bf16 for the
// value product).
//
// A workgroup serves up to 16 query heads of one KV head; its waves take
// 32-token tiles in turn through the dense decode's tile (dense_tile.h).
#include "paged.h"

namespace bytes_amd {

struct PagedDecodeArgs {
  PagedKv c;
  const uint16_t* q;
  int64_t q_sb, q_sh;
  uint16_t* out;
  int64_t o_sb, o_sh;
  int Hk, HB, G;
  float scale_log2, v_scale;
};

template <int D, bool FP8>
__global__ __launch_bounds__(kDenseWaves * 64, 2) void paged_decode_kernel(PagedDecodeArgs a) {
  using C = DenseCfg<D>;
  __shared__ __attribute__((aligned(16))) char smem[C::kSmem];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15, lg = lane >> 4;
  const int hb = blockIdx.x % a.HB, hk = blockIdx.x / a.HB % a.Hk, b = blockIdx.x / (a.HB * a.Hk);
  const int hq0 = hk * a.G + hb * 16, nh = min(16, a.G - hb * 16);
  bf16x8 qb[C::KK];
  load_q_bf16<D>(a.q + (int64_t)b * a.q_sb + (int64_t)hq0 * a.q_sh, a.q_sh, nh, lane, qb);
  const int len = paged_len(a.c, b);
  const int32_t* table = a.c.table + (int64_t)b * a.c.bt_sb;
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
  // row of token j, clamped into the sequence; ok: the token takes part
  auto row = [&](int j, int& id, int& off, bool& ok) {
    const int jj = min(j, len - 1), blk = fast_div(jj, a.c.dbs);
    id = table[blk];
    off = jj - blk * a.c.bs;
    ok = j < len && id >= 0 && id < a.c.nblocks;
    id = ok ? id : 0;
  };
  for (int t = w * kTile; t < len; t += kDenseWaves * kTile) {
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
  // merge of the waves, in wave order
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
  for (int e = threadIdx.x; e < nh * D; e += kDenseWaves * 64) {
    const int h = e / D, d = e - h * D;
    float M = kNegInf, L = 0.f, A = 0.f;
#pragma unroll
    for (int u = 0; u < kDenseWaves; ++u) M = fmaxf(M, wm[u * 16 + h]);
    const float Ms = M == kNegInf ? 0.f : M;
#pragma unroll
    for (int u = 0; u < kDenseWaves; ++u) {
      const float f = fast_exp2(wm[u * 16 + h] - Ms);
      L += f * wl[u * 16 + h];
      A += f * wacc[(u * 16 + h) * P + d];
    }
    a.out[(int64_t)b * a.o_sb + (int64_t)(hq0 + h) * a.o_sh + d] = f32_to_bf16_bits(L == 0.f ? 0.f : A / L * a.v_scale);
  }
}

}  // namespace bytes_amd

using namespace bytes_amd;

extern "C" {

int bytes_paged_decode_workspace_size(int B, int Hq, int Hk, int D, int block_size, int max_blocks, size_t* bytes) {
  if (!bytes || B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 || (D != 64 && D != 128)) return (int)hipErrorInvalidValue;
  const int rc = paged_check(block_size, 1, max_blocks);
  if (rc) return rc;
  *bytes = 0;
  return 0;
}

int bytes_paged_decode_attn(const void* q, int64_t q_sb, int64_t q_sh, const void* k_paged, int64_t k_sb, int64_t k_sh,
                            int64_t k_ss, const void* v_paged, int64_t v_sb, int64_t v_sh, int64_t v_ss, int kv_fp8,
                            const void* block_table, int64_t bt_sb, const void* context_lens, void* out, int64_t o_sb,
                            int64_t o_sh, int B, int Hq, int Hk, int D, int block_size, int num_blocks, int max_blocks,
                            float scale, float v_scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !k_paged || !v_paged || !block_table || !context_lens || !out || B <= 0 || Hk <= 0 || Hq <= 0 ||
      Hq % Hk != 0 || (D != 64 && D != 128))
    return (int)hipErrorInvalidValue;
  int rc = paged_check(block_size, num_blocks, max_blocks);
  if (rc) return rc;
  PagedDecodeArgs a;
  a.c.k = k_paged, a.c.k_sb = k_sb, a.c.k_sh = k_sh, a.c.k_ss = k_ss;
  a.c.v = v_paged, a.c.v_sb = v_sb, a.c.v_sh = v_sh, a.c.v_ss = v_ss;
  a.c.table = static_cast<const int32_t*>(block_table), a.c.bt_sb = bt_sb;
  a.c.lens = static_cast<const int32_t*>(context_lens);
  a.c.bs = block_size, a.c.nblocks = num_blocks, a.c.width = max_blocks;
  a.c.dbs = make_fastdiv((uint32_t)block_size);
  a.q = static_cast<const uint16_t*>(q), a.q_sb = q_sb, a.q_sh = q_sh;
  a.out = static_cast<uint16_t*>(out), a.o_sb = o_sb, a.o_sh = o_sh;
  a.Hk = Hk, a.G = Hq / Hk, a.HB = (a.G + 15) / 16;
  a.scale_log2 = scale * kLog2e, a.v_scale = v_scale;
  const int64_t units = (int64_t)B * Hk * a.HB;
  if (units > 0x7FFFFFFF) return (int)hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)units), block(kDenseWaves * 64);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define PD(DD, F8) hipLaunchKernelGGL((paged_decode_kernel<DD, F8>), grid, block, 0, st, a)
  if (D == 128) {
    if (kv_fp8) PD(128, true);
    else PD(128, false);
  } else {
    if (kv_fp8) PD(64, true);
    else PD(64, false);
  }
#undef PD
  return (int)hipGetLastError();
}

}  // extern "C"

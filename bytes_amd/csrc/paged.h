// Paged dense KV caches: what the append, decode and page-sparse kernels share.
//
// A cache is [num_blocks, Hk, block_size, D] bf16 or fp8 (OCP e4m3fn), any
// strides with unit stride along D.  Token p of sequence b is row p % block_size
// of block table[b, p / block_size].  Sequence b holds lens[b] tokens (clamped to
// what its table row can name); a token takes part if its block id lies in
// [0, num_blocks).
#pragma once
#include "dense_tile.h"

namespace bytes_amd {

struct PagedKv {
  const void* k;
  const void* v;
  int64_t k_sb, k_sh, k_ss;          // element strides: block, KV head, row
  int64_t v_sb, v_sh, v_ss;
  const int32_t* table;              // [B, width], row stride bt_sb
  int64_t bt_sb;
  const int32_t* lens;               // [B]
  int bs, nblocks, width;
  FastDiv dbs;                       // division by bs
};

// Tokens of sequence b: negative lengths count as 0, lengths past the table row as its capacity.
__device__ __forceinline__ int paged_len(const PagedKv& c, int b) {
  const int n = c.lens[b];
  return n < 0 ? 0 : min(n, c.width * c.bs);
}

// Folds v over the lanes that hold the same part of other rows, LPR lanes to a row:
// rotations within the rows of 16, then the row and half swaps.  Every lane of the
// wave takes part and receives the result.
template <int LPR, class OP>
__device__ __forceinline__ float fold_rows(float v, OP op) {
  if (LPR <= 8)
    v = op(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), 0x128, 0xF, 0xF, false)));
  if (LPR <= 4)
    v = op(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), 0x124, 0xF, 0xF, false)));
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Host-side checks of a cache's shape; 0 or a hipError_t.  (Positions up to 2^30:
// sums of two stay in 32 bits.)
inline int paged_check(int block_size, int num_blocks, int width) {
  if (block_size <= 0 || num_blocks <= 0 || width < 0) return (int)hipErrorInvalidValue;
  if (block_size > (1 << 30) || (int64_t)width * block_size > (1 << 30)) return (int)hipErrorInvalidConfiguration;
  return 0;
}

// Whether 16-row halves of a tile can be addressed from one scalar base each:
// tiles start on multiples of 32 tokens, so with block sizes that are multiples
// of 16 a half never crosses a block, and 32-bit lane offsets hold its rows.
inline bool paged_halves(const PagedKv& c) {
  return c.bs % 16 == 0 && c.k_ss >= 0 && c.k_ss <= (1 << 24) && c.v_ss >= 0 && c.v_ss <= (1 << 24);
}

// ---- one wave's attention over the tokens of some slots ----
// A slot range is walked in 32-slot tiles through the dense tile (dense_tile.h).
// What a slot stands for is the caller's: find(s) gives (place in the table row,
// row in the block, whether it is a token).

// One tile's table entries: lane l's slot is s0 + l % 32.
struct PagedIds {
  int id, off;
  bool ok;
};

// fp8 rows of a tile into its bf16 LDS tile, as dense_stage_fp8 places them, two
// values an instruction (exact: every e4m3 value is a bf16 value).  A batch of 32
// sequences of up to 16K: 138 us with fp32 in between, 114 so.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void fp8x16_to_bf16_direct(const u32x4& in, u32x4& lo, u32x4& hi) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    lo[2 * j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(in[j], 1.0f, false));
    lo[2 * j + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(in[j], 1.0f, true));
    hi[2 * j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(in[2 + j], 1.0f, false));
    hi[2 * j + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(in[2 + j], 1.0f, true));
  }
}
template <int D>
__device__ __forceinline__ void paged_stage_fp8(int lane, const DenseRegs8<D>& r, char* kst, char* vst) {
  using R = DenseRegs8<D>;
#pragma unroll
  for (int i = 0; i < R::CPL8; ++i) {
    const int p = lane + 64 * i, rr = p / R::CPR8, pos = p - rr * R::CPR8;
    u32x4 k0, k1, v0, v1;
    fp8x16_to_bf16_direct(r.k[i], k0, k1);
    fp8x16_to_bf16_direct(r.v[i], v0, v1);
    *reinterpret_cast<u32x4*>(kst + rr * (D * 2) + kswz<D>(rr, 2 * pos) * 16) = k0;
    *reinterpret_cast<u32x4*>(kst + rr * (D * 2) + kswz<D>(rr, 2 * pos + 1) * 16) = k1;
    *reinterpret_cast<u32x4*>(vst + rr * (D * 2) + vswz<D>(rr, 2 * pos) * 16) = v0;
    *reinterpret_cast<u32x4*>(vst + rr * (D * 2) + vswz<D>(rr, 2 * pos + 1) * 16) = v1;
  }
}

// The tile's rows in flight: K and V of 32 tokens in registers.  HALVES: two
// scalar bases per tile (see paged_halves), else every lane's row number comes
// from the lane that holds it.  A tile past the end (live false) reads the first
// bytes of the cache, the same on every lane, so that every iteration issues the
// same instructions.
template <int D, bool FP8, bool HALVES>
struct PagedRows {
  using Elem = typename std::conditional<FP8, uint8_t, uint16_t>::type;
  using Regs = typename std::conditional<FP8, DenseRegs8<D>, DenseRegs<D>>::type;
  static constexpr int EPC = 16 / (int)sizeof(Elem);      // elements per 16-byte chunk
  static constexpr int CPR = D / EPC;                     // chunks per row
  static constexpr int CPL = kTile * CPR / 64;            // chunks per lane per tile
  static constexpr int RPI = 64 / CPR;                    // rows per instruction
  static_assert(RPI <= 16, "an instruction's rows lie in one half");

  const Elem *kb, *vb;               // the KV head's first row
  int64_t k_sb, k_ss, v_sb, v_ss;
  int lane, r0, col;                 // this lane's row within an instruction's rows, and its first dim
  Regs r;

  __device__ __forceinline__ PagedRows(const PagedKv& c, int hk, int lane_)
      : kb(static_cast<const Elem*>(c.k) + hk * c.k_sh), vb(static_cast<const Elem*>(c.v) + hk * c.v_sh), k_sb(c.k_sb),
        k_ss(c.k_ss), v_sb(c.v_sb), v_ss(c.v_ss), lane(lane_), r0(lane_ / CPR), col(lane_ % CPR * EPC) {}

  __device__ __forceinline__ void issue(const PagedIds& t, bool live) {
    if constexpr (HALVES) {
      const uint32_t ko = live ? (uint32_t)(r0 * (int)k_ss + col) : 0u, vo = live ? (uint32_t)(r0 * (int)v_ss + col) : 0u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int id = live ? __builtin_amdgcn_readlane(t.id, 16 * h) : 0;
        const int off = live ? __builtin_amdgcn_readlane(t.off, 16 * h) : 0;
        const Elem* kp = kb + (int64_t)id * k_sb + (int64_t)off * k_ss;
        const Elem* vp = vb + (int64_t)id * v_sb + (int64_t)off * v_ss;
#pragma unroll
        for (int i = h * CPL / 2; i < (h + 1) * CPL / 2; ++i) {
          const int row = live ? i * RPI - 16 * h : 0;
          r.k[i] = ld16_nt(kp + (int64_t)row * k_ss + ko);
          r.v[i] = ld16_nt(vp + (int64_t)row * v_ss + vo);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < CPL; ++i) {
        const int src = r0 + i * RPI;
        const int id = live ? __shfl(t.id, src, 64) : 0, off = live ? __shfl(t.off, src, 64) : 0;
        const int c = live ? col : 0;
        r.k[i] = ld16_nt(kb + (int64_t)id * k_sb + (int64_t)off * k_ss + c);
        r.v[i] = ld16_nt(vb + (int64_t)id * v_sb + (int64_t)off * v_ss + c);
      }
    }
  }

  // Into the wave's LDS tile; values of slots that are no token become 0 (their
  // weight is 0, and 0 times what an unused row holds need not be).
  __device__ __forceinline__ void stage(uint32_t vmask, char* kst, char* vst) {
    if (vmask != 0xFFFFFFFFu) {
#pragma unroll
      for (int i = 0; i < CPL; ++i)
        if (!((vmask >> (r0 + i * RPI)) & 1u)) r.v[i] = u32x4{0, 0, 0, 0};
    }
    if constexpr (FP8) paged_stage_fp8<D>(lane, r, kst, vst);
    else dense_stage<D>(lane, r, kst, vst);
  }
};

// The number of 8 significant bits that x >= 0 starts with, as fp32 bits (a bf16
// number's, 16 zeros below); BELOW: the largest that is less than x (0 for 0).
template <bool BELOW>
__device__ __forceinline__ uint32_t leading8(float x) {
  const uint32_t u = __float_as_uint(x);
  return (BELOW ? __builtin_elementwise_sub_sat(u, 1u) : u) & 0xFFFF0000u;
}
// bf16 pair of the upper halves of two fp32 numbers' bits.
__device__ __forceinline__ uint32_t upper16(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }

// One staged tile: scores, online softmax and values, as dense_compute, with each
// weight as the sum of three bf16 numbers, which hold its 24 bits: three products
// per value block, whose matrix instructions have time to spare here (two, which lose
// up to 2^-16 of a weight, and three, us: eight sequences of up to 8K 22.7 and 22.8,
// four of 128K 245.8 and 246.3, 29 of up to 16K over an fp8 cache 116.9 and 117.2).
// INF, values that can be infinite: the first two are the numbers next below what
// they stand for, so that all three are positive wherever the weight is, and an
// infinite value that takes part gives that infinity and not the NaN that 0 or a
// negative number times it would add.  (What the first leaves is at most a whole step
// of it, 2^16 units of the weight's last place, the second's remainder then one of
// 2^8: either fits.)  That holds down to weights of 2^-100 of the row's largest; where
// one underflows fp32, here or as the factor of a rescaled or joined part, 0 times the
// infinity is NaN, as in any fp32 evaluation.  Caches of e4m3, which has no infinities,
// need no such care.
template <int D, bool INF>
__device__ __forceinline__ void paged_tile(uint32_t vmask, float scale_log2, int lane, const bf16x8 (&qb)[D / 32],
                                           const char* kst, const char* vst, float& m_run, float& l_run,
                                           f32x4 (&acc)[D / 16]) {
  using C = DenseCfg<D>;
  const int l16 = lane & 15, lg = lane >> 4;
  f32x4 s[2];
#pragma unroll
  for (int blk = 0; blk < 2; ++blk) {
    s[blk] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int row = blk * 16 + l16;
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) {
      const bf16x8 ka = __builtin_bit_cast(
          bf16x8, *reinterpret_cast<const u32x4*>(kst + row * (D * 2) + kswz<D>(row, kk * 4 + lg) * 16));
      s[blk] = mfma_bf16(ka, qb[kk], s[blk]);
    }
  }
  float x[8], mx = kNegInf;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = ((vmask >> ((j >> 2) * 16 + lg * 4 + (j & 3))) & 1u) ? s[j >> 2][j & 3] * scale_log2 : kNegInf;
    mx = __builtin_elementwise_maximum(mx, x[j]);
  }
  mx = col_max4(mx);
  const float m_new = fmaxf(m_run, mx);
  const float m_use = (m_new == kNegInf) ? 0.f : m_new;
  const float alpha = fast_exp2(m_run - m_use);
  float psum = 0.f;
  u32x4 w[3];                                      // the weights' parts, in pairs
  uint32_t even[3];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float p = fast_exp2(x[j] - m_use);
    psum += p;
    uint32_t u[3];
    u[0] = leading8<INF>(p);
    const float r1 = p - __uint_as_float(u[0]);    // (exact, as is the next)
    u[1] = leading8<INF>(r1);
    u[2] = __float_as_uint(r1 - __uint_as_float(u[1]));
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if (j & 1) w[i][j >> 1] = upper16(even[i], u[i]);
      else even[i] = u[i];
    }
  }
  l_run = l_run * alpha + psum;
  m_run = m_new;
  // V^T through two transposed reads per block of 16 dims (tile_softmax_pv_at's
  // layout), half of the blocks at a time: their products of one part do not wait for
  // each other (eight sequences of up to 8K: 22.8 us, 23.2 with a block at a time)
  constexpr int HALF = C::DB / 2;
  const StagedV<D> vaddr{vst};
#pragma unroll
  for (int d0 = 0; d0 < C::DB; d0 += HALF) {
    bf16x8 v[HALF];
#pragma unroll
    for (int u = 0; u < HALF; ++u) {
      u32x2 h[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
        h[hf] = tr16(vaddr(hf, hf * 16 + lg * 4 + (l16 >> 2), (d0 + u) * 16 + (l16 & 3) * 4));
      v[u] = __builtin_bit_cast(bf16x8, u32x4{h[0][0], h[0][1], h[1][0], h[1][1]});
      acc[d0 + u] *= alpha;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
      for (int u = 0; u < HALF; ++u) acc[d0 + u] = mfma_bf16(v[u], __builtin_bit_cast(bf16x8, w[i]), acc[d0 + u]);
  }
}

// Slots [s, s_end) in steps of `step` (s a multiple of 32 from the first slot):
// online softmax over them into m_run, l_run, acc.
template <int D, bool FP8, bool HALVES, class FIND>
__device__ __forceinline__ void paged_wave_loop(const PagedKv& c, const int32_t* table, int hk, int s, int s_end,
                                                int step, int lane, float scale_log2, const bf16x8 (&qb)[D / 32],
                                                char* wbuf, const FIND& find, float& m_run, float& l_run,
                                                f32x4 (&acc)[D / 16]) {
  if (s >= s_end) return;
  char* kst = wbuf;
  char* vst = wbuf + DenseCfg<D>::VT;
  PagedRows<D, FP8, HALVES> rows(c, hk, lane);
  // entries of the tile at s0: loaded well before they are used
  auto fetch = [&](int s0) {
    PagedIds t;
    int place;
    const int sl = s0 + (lane & 31);
    find(min(sl, s_end - 1), place, t.off, t.ok);
    t.ok = t.ok && sl < s_end;
    t.off = sl < s_end ? t.off : 0;  // (16 rows from there are read in HALVES: they have to be the block's)
    t.id = table[place];
    return t;
  };
  auto settle = [&](PagedIds& t) {   // ids that name a block; other slots read block 0
    const bool in = t.id >= 0 && t.id < c.nblocks;
    t.ok = t.ok && in;
    t.id = in ? t.id : 0;
  };
  PagedIds now = fetch(s), next = fetch(s + step);
  settle(now);
  rows.issue(now, true);
  for (; s < s_end; s += step) {
    const uint32_t vmask = (uint32_t)__ballot(now.ok);
    wave_lds_sync();
    rows.stage(vmask, kst, vst);
    settle(next);
    now = next;
    next = fetch(s + 2 * step);
    rows.issue(now, s + step < s_end);
    wave_lds_sync();
    paged_tile<D, !FP8>(vmask, scale_log2, lane, qb, kst, vst, m_run, l_run, acc);
  }
}

// Merge of the workgroup's waves through LDS, in wave order: put(h, d4, A, M, L)
// with four consecutive dims 4 * d4 .. of head h < nh, the maximum (log2 domain)
// and the denominator.  All threads of the workgroup call this; smem is free
// again when it returns.
template <int D, int NW, class PUT>
__device__ __forceinline__ void paged_merge_waves(float m_run, float l_run, f32x4 (&acc)[D / 16], float* smem, int nh,
                                                  const PUT& put) {
  constexpr int P = acc_pitch<D>(), D4 = D / 4;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15, lg = lane >> 4;
  l_run = col_sum4(l_run);
  float* wm = smem;
  float* wl = wm + NW * 16;
  float* wacc = wl + NW * 16;
  __syncthreads();
  if (lg == 0) {
    wm[w * 16 + l16] = m_run;
    wl[w * 16 + l16] = l_run;
  }
  f32x4* row = reinterpret_cast<f32x4*>(wacc + (w * 16 + l16) * P);
  if (l16 < nh) {
#pragma unroll
    for (int db = 0; db < D / 16; ++db) row[4 * db + lg] = acc[db];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < nh * D4; e += NW * 64) {
    const int h = e / D4, d4 = e - h * D4;
    float M = kNegInf;
#pragma unroll
    for (int u = 0; u < NW; ++u) M = fmaxf(M, wm[u * 16 + h]);
    const float Ms = (M == kNegInf) ? 0.f : M;
    float L = 0.f;
    f32x4 A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < NW; ++u) {
      const float f = fast_exp2(wm[u * 16 + h] - Ms);
      L += f * wl[u * 16 + h];
      A += f * reinterpret_cast<const f32x4*>(wacc + (u * 16 + h) * P)[d4];
    }
    put(h, d4, A, M, L);
  }
  __syncthreads();
}

// Four consecutive results; a row with nothing to attend to is 0.
__device__ __forceinline__ void paged_store(uint16_t* out, const f32x4& A, float L, float v_scale) {
  const float il = L == 0.f ? 0.f : v_scale / L;
  u32x2 r;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    r[j] = (uint32_t)f32_to_bf16_bits(L == 0.f ? 0.f : A[2 * j] * il) |
           ((uint32_t)f32_to_bf16_bits(L == 0.f ? 0.f : A[2 * j + 1] * il) << 16);
  *reinterpret_cast<u32x2*>(out) = r;
}

// Join of a row's parts by one wave: 16 lanes hold a part's dims (64 of them), the
// four lane groups take the parts in turn, each in order, and are folded by fixed
// row swaps.  slot(i): part i's place; pml: (maximum, denominator) by place; pacc:
// the lane's four values of place 0, places `pitch` apart.  The first 4 * PF parts
// and their statistics are loaded together, one round trip; a lane group past the
// last part adds zeros (0 times the last part's values again would not be 0 where
// those are infinite).
template <int PF, class SLOT, class PUT>
__device__ __forceinline__ void paged_join(int parts, int lane, const SLOT& slot, const float2* pml, const f32x4* pacc,
                                           int pitch, const PUT& put) {
  const int grp = lane >> 4;
  float2 ml[PF];
  f32x4 acc[PF];
#pragma unroll
  for (int u = 0; u < PF; ++u) {                   // parts past the last: its values again, not used
    const size_t r = slot(min(grp + 4 * u, parts - 1));
    ml[u] = pml[r];
    acc[u] = pacc[r * pitch];
  }
  float M = kNegInf;
#pragma unroll
  for (int u = 0; u < PF; ++u) M = fmaxf(M, ml[u].x);
  for (int i = 4 * PF + lane; i < parts; i += 64) M = fmaxf(M, pml[slot(i)].x);
  M = wave_max_f32(M);
  if (M == kNegInf) M = 0.f;
  float L = 0.f;
  f32x4 A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < PF; ++u) {
    const bool part = grp + 4 * u < parts;
    const float f = part ? fast_exp2(ml[u].x - M) : 0.f;
    L += f * ml[u].y;
    A += f * (part ? acc[u] : f32x4{0.f, 0.f, 0.f, 0.f});
  }
  for (int i = 4 * PF + grp; i < parts; i += 4) {
    const size_t r = slot(i);
    const float2 m = pml[r];
    const float f = fast_exp2(m.x - M);
    L += f * m.y;
    A += f * pacc[r * pitch];
  }
  L = col_sum4(L);
#pragma unroll
  for (int j = 0; j < 4; ++j) A[j] = col_sum4(A[j]);
  put(A, L);
}

}  // namespace bytes_amd

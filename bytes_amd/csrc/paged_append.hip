// New tokens into a paged KV cache, with the position rotation on the way.
//
// Token i of sequence b's n new ones has position p = lens[b] - n + i (lens
// counts the new tokens).  Its key's (and query's) first R dims are rotated in
// pairs (x0, x1) -> (x0 c - x1 s, x1 c + x0 s) with row p of the cos / sin
// tables, pairs (j, j + R/2) or neighbours (2j, 2j + 1), in fp32; the result,
// divided by the cache's scale, is rounded once to the cache's type.  The
// blocks' elementwise min / max (of the values as stored) are kept for the
// page-sparse decode.
//
// One workgroup per token; a thread takes 16 elements of one head: for pairs
// (j, j + R/2) two runs of 8, R/2 apart.  The workgroup of the first new token
// of each block also folds the block's min / max.
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
  int T, B, Hq, Hk, D;
};

// Row t's sequence, position and number of earlier new tokens of that sequence; false: no position.
__device__ __forceinline__ bool append_locate(const AppendArgs& a, int t, int& b, int64_t& p, int64_t& i) {
  if (!a.cu) {
    b = t;
    i = 0;
    p = (int64_t)a.c.lens[b] - 1;
  } else {
    int lo = 0, hi = a.B;              // first b with cu[b + 1] > t
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (a.cu[mid + 1] <= t) lo = mid + 1;
      else hi = mid;
    }
    b = lo;
    if (b >= a.B) return false;
    i = (int64_t)t - a.cu[b];
    p = (int64_t)a.c.lens[b] - ((int64_t)a.cu[b + 1] - t);
  }
  return i >= 0 && p >= 0 && p < (int64_t)a.c.width * a.c.bs;
}

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

// Where the two runs of 8 of item c start in a head of D dims.
__device__ __forceinline__ void item_runs(const AppendArgs& a, int c, int& d0, int& d1) {
  const bool halves = !a.interleaved && 16 * c < a.rot;
  d0 = halves ? 8 * c : 16 * c;
  d1 = halves ? 8 * c + a.rot / 2 : 16 * c + 8;
}

// Item c of a row at position p, rotated: x[0..7] and x[8..15] are its two runs.
__device__ __forceinline__ void load_rotated(const AppendArgs& a, const uint16_t* row, int c, int64_t p, float* x) {
  int d0, d1;
  item_runs(a, c, d0, d1);
  widen8(ld16(row + d0), x);
  widen8(ld16(row + d1), x + 8);
  if (16 * c >= a.rot) return;
  const float* cp = a.cos + p * a.cos_st + 8 * c;
  const float* sp = a.sin + p * a.sin_st + 8 * c;
  float y[16];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int e0 = a.interleaved ? 2 * j : j, e1 = a.interleaved ? 2 * j + 1 : j + 8;
    const float cs = cp[j], sn = sp[j];
    y[e0] = x[e0] * cs - x[e1] * sn;
    y[e1] = x[e1] * cs + x[e0] * sn;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) x[j] = y[j];
}

// Stores the item in the cache row; x becomes what the cache then holds.
template <bool FP8>
__device__ __forceinline__ void store_cache(void* row, int d0, int d1, float scale, float* x) {
  if constexpr (FP8) {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = x[j] / scale;
    const u32x2 r0 = narrow8_fp8(x), r1 = narrow8_fp8(x + 8);
    if (row) {
      *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(row) + d0) = r0;
      *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(row) + d1) = r1;
    }
    widen8_fp8(r0, x);
    widen8_fp8(r1, x + 8);
  } else {
    const u32x4 r0 = narrow8(x), r1 = narrow8(x + 8);
    if (row) {
      *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(row) + d0) = r0;
      *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(row) + d1) = r1;
    }
    widen8(r0, x);
    widen8(r1, x + 8);
  }
}

template <bool FP8>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
  const int t = blockIdx.x;
  const int items = a.D / 16;
  int b = 0;
  int64_t p = 0, i = 0;
  const bool placed = append_locate(a, t, b, p, i);
  const int blk = placed ? fast_div((int)p, a.c.dbs) : 0, off = placed ? (int)p - blk * a.c.bs : 0;
  const int id = placed ? a.c.table[(int64_t)b * a.c.bt_sb + blk] : -1;
  const bool held = id >= 0 && id < a.c.nblocks;
  constexpr int ES = FP8 ? 1 : 2;
  char* kc = static_cast<char*>(const_cast<void*>(a.c.k)) + ((int64_t)(held ? id : 0) * a.c.k_sb + off * a.c.k_ss) * ES;
  char* vc = static_cast<char*>(const_cast<void*>(a.c.v)) + ((int64_t)(held ? id : 0) * a.c.v_sb + off * a.c.v_ss) * ES;
  float x[16];
  for (int e = threadIdx.x; e < (2 * a.Hk + a.Hq) * items; e += blockDim.x) {
    const int h = e / items, c = e - h * items;
    if (h < a.Hk) {
      if (!held) continue;
      int d0, d1;
      item_runs(a, c, d0, d1);
      load_rotated(a, a.k + t * a.k_st + h * a.k_sh, c, p, x);
      store_cache<FP8>(kc + h * a.c.k_sh * ES, d0, d1, a.k_scale, x);
    } else if (h < 2 * a.Hk) {
      if (!held) continue;
      const int hh = h - a.Hk;
      const uint16_t* row = a.v + t * a.v_st + hh * a.v_sh + 16 * c;
      widen8(ld16(row), x);
      widen8(ld16(row + 8), x + 8);
      store_cache<FP8>(vc + hh * a.c.v_sh * ES, 16 * c, 16 * c + 8, a.v_scale, x);
    } else {
      const int hh = h - 2 * a.Hk;
      int d0, d1;
      item_runs(a, c, d0, d1);
      if (placed) {
        load_rotated(a, a.q + t * a.q_st + hh * a.q_sh, c, p, x);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = 0.f;
      }
      uint16_t* row = a.q_out + t * a.qo_st + hh * a.qo_sh;
      *reinterpret_cast<u32x4*>(row + d0) = narrow8(x);
      *reinterpret_cast<u32x4*>(row + d1) = narrow8(x + 8);
    }
  }
  // first new token of its block: the block's min / max over the run
  if (!a.kmin || !held || (off != 0 && i != 0)) return;
  const int64_t left = (int64_t)(a.cu ? min(a.cu[b + 1], a.T) : t + 1) - t;
  const int n = (int)(left < a.c.bs - off ? left : a.c.bs - off);
  for (int e = threadIdx.x; e < a.Hk * items; e += blockDim.x) {
    const int h = e / items, c = e - h * items;
    int d0, d1;
    item_runs(a, c, d0, d1);
    float mn[16], mx[16];
    uint16_t* pmn = a.kmin + ((int64_t)id * a.Hk + h) * a.D;
    uint16_t* pmx = a.kmax + ((int64_t)id * a.Hk + h) * a.D;
    if (off) {
      widen8(ld16(pmn + d0), mn);
      widen8(ld16(pmn + d1), mn + 8);
      widen8(ld16(pmx + d0), mx);
      widen8(ld16(pmx + d1), mx + 8);
    }
    for (int j = 0; j < n; ++j) {
      load_rotated(a, a.k + (t + j) * a.k_st + h * a.k_sh, c, p + j, x);
      store_cache<FP8>(nullptr, d0, d1, a.k_scale, x);
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        mn[u] = j == 0 && !off ? x[u] : nan_min(mn[u], x[u]);
        mx[u] = j == 0 && !off ? x[u] : nan_max(mx[u], x[u]);
      }
    }
    *reinterpret_cast<u32x4*>(pmn + d0) = narrow8(mn);
    *reinterpret_cast<u32x4*>(pmn + d1) = narrow8(mn + 8);
    *reinterpret_cast<u32x4*>(pmx + d0) = narrow8(mx);
    *reinterpret_cast<u32x4*>(pmx + d1) = narrow8(mx + 8);
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
  if (!k || !v || !k_paged || !v_paged || !block_table || !context_lens || T < 0 || B <= 0 || Hk <= 0 || Hq < 0)
    return (int)hipErrorInvalidValue;
  if ((D != 64 && D != 128) || rot < 0 || rot > D || rot % 16 != 0 || (!cu_seqlens && T != B))
    return (int)hipErrorInvalidValue;
  if ((q == nullptr) != (q_out == nullptr) || (q == nullptr) != (Hq == 0) || (kmin == nullptr) != (kmax == nullptr))
    return (int)hipErrorInvalidValue;
  int rc = paged_check(block_size, num_blocks, max_blocks);
  if (rc) return rc;
  if (rot && (!cos || !sin || (int64_t)positions < (int64_t)max_blocks * block_size)) return (int)hipErrorInvalidValue;
  if (T == 0) return 0;
  AppendArgs a;
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
  a.T = T, a.B = B, a.Hq = Hq, a.Hk = Hk, a.D = D;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (kv_fp8)
    hipLaunchKernelGGL(paged_append_kernel<true>, dim3((unsigned)T), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(paged_append_kernel<false>, dim3((unsigned)T), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

}  // extern "C"

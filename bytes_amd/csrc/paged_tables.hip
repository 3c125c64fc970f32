// Block tables, lengths and slot maps of a serving batch, from request lengths.
//
// State: a table [B, W] of block ids, lens [B], and the free blocks as a ring
// ring[N] with range = (head, count): free are ring[(head + i) % N], i < count.
// One step, for every sequence b in order (c: inclusive sums over the sequences):
//   n0 = lens held to 0 .. W bs; kept = min(n0, max(keep, 0))
//   back: the places ceil(kept / bs) <= j < ceil(n0 / bs) that name a block; with a
//     window of w tokens and s sinks also the run of places that name one, going
//     down from (kept - w + 1) / bs - 1 to ceil(s / bs): no position from kept on
//     sees their tokens
//   m = new if 0 < new <= W bs - kept, else 0; need = the places that m tokens enter
//   granted = m if (need == 0 or c_need <= count) and c_m <= T, else 0
// Blocks that are given back join the ring's end in (sequence, place) order and can
// be had from the next step on; new ones leave its start in that order.  So what is
// read of the ring and what is written to it are different parts, the result does
// not depend on timing, and no atomics are needed.
//
// Plan (one workgroup): a thread per sequence counts the blocks that come back
// (waves take those with many), four prefix sums with a carry, the lengths.
// Fill: a wave per sequence moves its blocks, a thread per token finds its sequence
// in cu.  Small steps run both in one launch.
// Bound by latency and launches: nothing here is read or written twice. A step of 32
// sequences that moves 3 KB takes 5.3 us in one launch (lengths, entries, two rounds of
// sums, the ring and the outputs follow one another), one of 256 with 34K new tokens 7.6
// and 3.6 in two (states that no cache holds: 10.2 and 5.4).  Without rows that end that plan takes 4.7; rows with more
// blocks to count than a thread takes alone go to the waves, one after another: 32 of them, as there, 5.5 more, 128 16.5,
// 256 33.  (Sixteen waves to the plan: 5.8, and 7.5 and 3.6.)
#include "common.h"

namespace bytes_amd {

struct TablesArgs {
  int32_t* table;
  int64_t bt_sb;
  int32_t *lens, *ring, *range;
  const int32_t *keep, *fresh;       // keep may be null: all
  int32_t *cu, *granted, *seqs, *positions;
  int64_t* slots;
  int32_t* plan;                     // [8][B]: see Plan; then head, count as they were
  int B, W, N, T, bs, cap, window, sinks;
  FastDiv dbs;
};

// A sequence's share of a step, kept in the workspace between the two parts.
enum : int { kKept = 0, kLast, kNeed, kStart, kBack, kRunLo, kRunHi, kPlanRows };

constexpr int kPlanWaves = 8, kPlanThreads = kPlanWaves * 64;
constexpr int kFillThreads = 256;
constexpr int kBySelf = 4;           // places that a thread counts alone
constexpr int kCuLds = 4096;         // sequences whose cu fits the fill's LDS
// A step that one workgroup takes in one launch (us, eager, one launch and two: 32 sequences and
// 32 rows of tokens 6.1 and 9.4, 1024 rows 6.5 and 9.4; 64 and 1024: 8.7 and 9.2; 128 and 128: 7.4 and
// 9.2; 128 and 1024: 10.4 and 9.2).
constexpr int kSmallB = 128;
constexpr bool small_step(int B, int T) { return B <= kSmallB && T <= 1536 - 8 * B; }

__device__ __forceinline__ bool names(int id, int N) { return id >= 0 && id < N; }
__device__ __forceinline__ int places(const TablesArgs& a, int n) { return fast_div(n + a.bs - 1, a.dbs); }

// Sums that stay at the largest number once they reach it: what is asked for may be more
// than 32 bits hold, and then is more than there is.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
// wave_prefix_sum with such sums.
__device__ __forceinline__ uint32_t wave_prefix_sat(uint32_t x) {
  x = add_sat(x, dpp_u32<0x111>(x));
  x = add_sat(x, dpp_u32<0x112>(x));
  x = add_sat(x, dpp_u32<0x114>(x));
  x = add_sat(x, dpp_u32<0x118>(x));
  x = add_sat(x, dpp_u32<0x142, 0xA>(x));
  return add_sat(x, dpp_u32<0x143, 0xC>(x));
}
// Inclusive prefix sums of N numbers over the workgroup's threads, and their totals.
template <int N>
__device__ __forceinline__ void group_scan(uint32_t (&v)[N], uint32_t (*sums)[N], uint32_t (&total)[N]) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = wave_prefix_sat(v[k]);
  __syncthreads();
  if (lane == 63) {
#pragma unroll
    for (int k = 0; k < N; ++k) sums[w][k] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    uint32_t before = 0;
    total[k] = 0;
    for (int i = 0; i < kPlanWaves; ++i) {
      if (i < w) before = add_sat(before, sums[i][k]);
      total[k] = add_sat(total[k], sums[i][k]);
    }
    v[k] = add_sat(v[k], before);
  }
}

// Places of [lo, hi) of a row that name a block.
__device__ __forceinline__ int count_named(const int32_t* row, int lo, int hi, int N, int lane) {
  constexpr int U = 4;                             // loads in flight
  int n = 0;
  for (int j0 = lo; j0 < hi; j0 += U * 64) {
    int id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = row[min(j0 + u * 64 + lane, hi - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) n += __popcll(__ballot(j0 + u * 64 + lane < hi && names(id[u], N)));
  }
  return n;
}
// The lowest place of the run that names blocks, going down from hi - 1 to lo.
__device__ __forceinline__ int run_down(const int32_t* row, int lo, int hi, int N, int lane) {
  while (hi > lo) {
    const int j = hi - 1 - lane;                   // lane 0 the highest
    const unsigned long long miss = __ballot(j < lo || !names(row[max(j, lo)], N));
    const int n = miss ? __ffsll(miss) - 1 : 64;
    hi -= n;
    if (n < 64) break;
  }
  return hi;
}

struct PlanShared {
  uint32_t asked[kPlanWaves][3], given[kPlanWaves][2];
  int big[kPlanThreads];
  int back[kPlanThreads], run[kPlanThreads];
  int nbig;
};

// cu and plan: in memory, or the workgroup's own.
__device__ __forceinline__ void make_plan(const TablesArgs& a, PlanShared& sh, int32_t* cu, int32_t* plan) {
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int count = min(max(a.range[1], 0), a.N);
  int head = a.range[0];
  head = head >= 0 && head < a.N ? head : 0;
  const int s_lo = fast_div(min(a.sinks, a.cap) + a.bs - 1, a.dbs);
  uint32_t asked_blocks = 0, asked_tokens = 0;     // of the sequences before these
  int blocks = 0, tokens = 0, given = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    const bool live = b < a.B;
    const int bc = min(b, a.B - 1);
    const int n0 = min(max(a.lens[bc], 0), a.cap);
    const int kept = a.keep ? min(n0, max(a.keep[bc], 0)) : n0;
    const int fresh = a.fresh[bc];
    const int m = live && fresh > 0 && fresh <= a.cap - kept ? fresh : 0;
    const int first = places(a, kept), last = places(a, n0);
    const int need = places(a, kept + m) - first;
    const int edge = kept - a.window + 1;          // a window keeps the tokens from there on
    const int r_hi = a.window && edge > 0 ? fast_div(edge, a.dbs) : 0;
    const int r_lo0 = min(s_lo, r_hi);
    // the blocks that come back
    const int32_t* row = a.table + (int64_t)bc * a.bt_sb;
    int back = 0, r_lo = r_hi;
    bool big = false;
    {                                              // (loads of a place that is there, all at once)
      int ends[kBySelf], run[kBySelf];
#pragma unroll
      for (int i = 0; i < kBySelf; ++i) {
        ends[i] = row[min(first + i, a.W - 1)];
        run[i] = row[max(r_hi - 1 - i, 0)];
      }
      bool on = live;
#pragma unroll
      for (int i = 0; i < kBySelf; ++i) {
        back += live && first + i < last && names(ends[i], a.N) ? 1 : 0;
        on = on && r_hi - 1 - i >= r_lo0 && names(run[i], a.N);
        r_lo -= on ? 1 : 0;
      }
      big = live && (last - first > kBySelf || (on && r_lo > r_lo0));
    }
    __syncthreads();
    if (tid == 0) sh.nbig = 0;
    __syncthreads();
    sh.back[tid] = back;
    sh.run[tid] = r_lo;
    if (big) sh.big[atomicAdd(&sh.nbig, 1)] = tid; // (in any order: each is counted by itself)
    __syncthreads();
    for (int i = w; i < sh.nbig; i += kPlanWaves) {
      const int u = sh.big[i], bb = b0 + u;
      const int bn0 = min(max(a.lens[bb], 0), a.cap), bk = a.keep ? min(bn0, max(a.keep[bb], 0)) : bn0;
      const int32_t* brow = a.table + (int64_t)bb * a.bt_sb;
      const int n = count_named(brow, places(a, bk), places(a, bn0), a.N, lane);
      const int lo = run_down(brow, s_lo, sh.run[u], a.N, lane);
      if (lane == 0) sh.back[u] = n, sh.run[u] = lo;
    }
    __syncthreads();
    r_lo = sh.run[tid];
    back = live ? sh.back[tid] + (r_hi - r_lo) : 0;
    // what fits
    uint32_t c[3] = {(uint32_t)need, (uint32_t)m, (uint32_t)back}, t[3];
    group_scan(c, sh.asked, t);
    const bool ok = (need == 0 || add_sat(asked_blocks, c[0]) <= (uint32_t)count) && add_sat(asked_tokens, c[1]) <= (uint32_t)a.T;
    asked_blocks = add_sat(asked_blocks, t[0]);
    asked_tokens = add_sat(asked_tokens, t[1]);
    const int got = ok ? m : 0, gneed = ok ? need : 0;
    uint32_t g[2] = {(uint32_t)gneed, (uint32_t)got}, tg[2];
    group_scan(g, sh.given, tg);
    if (live) {
      int32_t* p = plan + b;
      const int64_t B = a.B;
      p[kKept * B] = kept;
      p[kLast * B] = last;
      p[kNeed * B] = gneed;
      p[kStart * B] = blocks + (int)g[0] - gneed;
      p[kBack * B] = given + (int)c[2] - back;
      p[kRunLo * B] = r_lo;
      p[kRunHi * B] = r_hi;
      a.granted[b] = got;
      a.lens[b] = kept + got;
      cu[b] = a.cu[b] = tokens + (int)g[1] - got;
    }
    blocks += (int)tg[0];
    tokens += (int)tg[1];
    given += (int)t[2];
  }
  __syncthreads();                                 // (range has been read by all)
  if (tid == 0) {
    cu[a.B] = a.cu[a.B] = tokens;
    int32_t* was = plan + (int64_t)kPlanRows * a.B;
    was[0] = head;
    was[1] = count;
    int next = head + blocks;                      // (below 2 N, held to 31 bits by the host's check)
    a.range[0] = next >= a.N ? next - a.N : next;
    a.range[1] = min(count - blocks + given, a.N);
  }
}

__device__ __forceinline__ int ring_at(const TablesArgs& a, int head, int64_t i) {
  const uint64_t x = (uint64_t)(head + i), N = (uint64_t)a.N;      // below 2 N in a pool that is one
  return (int)(x < N ? x : x < 2 * N ? x - N : x % N);
}

// One wave: the blocks of sequence b that go back and come.
__device__ __forceinline__ void move_blocks(const TablesArgs& a, const int32_t* plan, int b, int lane) {
  const int32_t* p = plan + b;
  const int64_t B = a.B;
  const int kept = p[kKept * B], last = p[kLast * B], need = p[kNeed * B], start = p[kStart * B];
  const int r_lo = p[kRunLo * B], r_hi = p[kRunHi * B];
  const int head = plan[kPlanRows * B], count = plan[kPlanRows * B + 1];
  int64_t to = (int64_t)count + p[kBack * B];
  int32_t* row = a.table + (int64_t)b * a.bt_sb;
  for (int j = r_lo + lane; j < r_hi; j += 64) {
    a.ring[ring_at(a, head, to + (j - r_lo))] = row[j];
    row[j] = -1;
  }
  to += r_hi - r_lo;
  const int first = places(a, kept), end = max(last, first + need);
  for (int j0 = first; j0 < end; j0 += 64) {
    const int j = j0 + lane;
    const int id = j < last ? row[j] : -1;
    const bool goes = names(id, a.N);
    const unsigned long long m = __ballot(goes);
    if (goes) a.ring[ring_at(a, head, to + __popcll(m & ((1ull << lane) - 1)))] = id;
    to += __popcll(m);
    if (j < first + need) row[j] = a.ring[ring_at(a, head, start + (j - first))];
    else if (goes) row[j] = -1;
  }
}

// Token t of the step: its sequence (the one whose cu range holds it), position and slot.
__device__ __forceinline__ void place_token(const TablesArgs& a, const int32_t* plan, int t, const int32_t* cu) {
  int b = -1, p = -1;
  int64_t slot = -1;
  if (t < cu[a.B]) {
    int lo = 0, hi = a.B - 1;                      // the last b with cu[b] <= t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cu[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    const int64_t B = a.B;
    const int kept = plan[kKept * B + b];
    p = kept + t - cu[b];
    const int j = fast_div(p, a.dbs), first = places(a, kept);
    const int id = j < first ? a.table[b * a.bt_sb + j]
                             : a.ring[ring_at(a, plan[kPlanRows * B], plan[kStart * B + b] + (j - first))];
    if (names(id, a.N)) slot = (int64_t)id * a.bs + (p - j * a.bs);
  }
  a.seqs[t] = b;
  a.positions[t] = p;
  a.slots[t] = slot;
}

__global__ __launch_bounds__(kPlanThreads) void paged_tables_plan_kernel(TablesArgs a) {
  __shared__ PlanShared sh;
  make_plan(a, sh, a.cu, a.plan);
}

// A step of few sequences and tokens, by one workgroup that keeps the plan to itself.
__global__ __launch_bounds__(kPlanThreads) void paged_tables_small_kernel(TablesArgs a) {
  __shared__ PlanShared sh;
  __shared__ int32_t cu[kSmallB + 1], plan[kPlanRows * kSmallB + 2];
  make_plan(a, sh, cu, plan);
  __syncthreads();
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int t = threadIdx.x; t < a.T; t += kPlanThreads) place_token(a, plan, t, cu);
  for (int b = w; b < a.B; b += kPlanWaves) move_blocks(a, plan, b, lane);
}

__global__ __launch_bounds__(kFillThreads) void paged_tables_fill_kernel(TablesArgs a, int seq_wgs) {
  __shared__ int32_t lcu[kCuLds + 1];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  if ((int)blockIdx.x < seq_wgs) {
    const int b = blockIdx.x * (kFillThreads / 64) + w;
    if (b < a.B) move_blocks(a, a.plan, b, lane);
    return;
  }
  const int64_t t = ((int64_t)blockIdx.x - seq_wgs) * kFillThreads + tid;
  if (a.B <= kCuLds) {
    for (int i = tid; i <= a.B; i += kFillThreads) lcu[i] = a.cu[i];
    __syncthreads();
    if (t < a.T) place_token(a, a.plan, (int)t, lcu);
  } else if (t < a.T) {
    place_token(a, a.plan, (int)t, a.cu);
  }
}

static size_t tables_workspace(int64_t B) { return (size_t)(kPlanRows * B + 2) * 4; }

}  // namespace bytes_amd

using namespace bytes_amd;

extern "C" {

int bytes_paged_resize_workspace_size(int B, size_t* bytes) {
  if (!bytes || B <= 0) return (int)hipErrorInvalidValue;
  *bytes = tables_workspace(B);
  return 0;
}

int bytes_paged_resize(void* block_table, int64_t bt_sb, void* context_lens, void* free_blocks, void* free_range,
                       const void* keep, const void* new_lens, void* cu_seqlens, void* granted, void* seqs,
                       void* positions, void* slots, int B, int max_blocks, int num_blocks, int T, int block_size,
                       int window, int sinks, void* workspace, size_t workspace_bytes, void* stream) {
  if (!block_table || !context_lens || !free_blocks || !free_range || !new_lens || !cu_seqlens || !granted || !workspace ||
      (T > 0 && (!seqs || !positions || !slots)) || B <= 0 || max_blocks <= 0 || num_blocks <= 0 || T < 0 ||
      block_size <= 0 || window < 0 || sinks < 0 || (window == 0 && sinks != 0) || workspace_bytes < tables_workspace(B))
    return (int)hipErrorInvalidValue;
  if (block_size > (1 << 30) || (int64_t)max_blocks * block_size > (1 << 30) || num_blocks > (1 << 30) || T > (1 << 30) ||
      B > (1 << 24))
    return (int)hipErrorInvalidConfiguration;
  TablesArgs a = {};
  a.table = static_cast<int32_t*>(block_table), a.bt_sb = bt_sb;
  a.lens = static_cast<int32_t*>(context_lens);
  a.ring = static_cast<int32_t*>(free_blocks), a.range = static_cast<int32_t*>(free_range);
  a.keep = static_cast<const int32_t*>(keep), a.fresh = static_cast<const int32_t*>(new_lens);
  a.cu = static_cast<int32_t*>(cu_seqlens), a.granted = static_cast<int32_t*>(granted);
  a.seqs = static_cast<int32_t*>(seqs), a.positions = static_cast<int32_t*>(positions);
  a.slots = static_cast<int64_t*>(slots);
  a.plan = static_cast<int32_t*>(workspace);
  a.B = B, a.W = max_blocks, a.N = num_blocks, a.T = T, a.bs = block_size, a.cap = max_blocks * block_size;
  a.window = window < (1 << 30) ? window : (1 << 30), a.sinks = sinks;
  a.dbs = make_fastdiv((uint32_t)block_size);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (small_step(B, T)) {
    hipLaunchKernelGGL(paged_tables_small_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
    return (int)hipGetLastError();
  }
  hipLaunchKernelGGL(paged_tables_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
  const int rc = (int)hipGetLastError();
  if (rc) return rc;
  const int seq_wgs = (B + kFillThreads / 64 - 1) / (kFillThreads / 64);
  const int tok_wgs = (T + kFillThreads - 1) / kFillThreads;
  hipLaunchKernelGGL(paged_tables_fill_kernel, dim3((unsigned)(seq_wgs + tok_wgs)), dim3(kFillThreads), 0, st, a, seq_wgs);
  return (int)hipGetLastError();
}

}  // extern "C"

// A wave's 64 lanes on the host: each a context of its own, which all reach the same operations
// across lanes in the same order.  For index arithmetic of the kernels that uses nothing else.
#pragma once
#include <setjmp.h>
#include <stdint.h>
#include <stdlib.h>
#include <ucontext.h>

#include <algorithm>
#include <functional>
#include <vector>

#define __device__
#define __forceinline__ inline
using std::max;
using std::min;

namespace wave {
constexpr int kLanes = 64;
struct State {
  jmp_buf main, lane[kLanes];        // (a ucontext only to start a lane: its switches are system calls)
  int at = 0;                        // the lane that runs
  bool done[kLanes] = {};
  uint64_t slot[2][kLanes];          // of this operation and the last one
  int turn[kLanes] = {};
  std::function<void(int)> body;
};
inline State* s = nullptr;

// Hands x to the other lanes; returns all lanes' values once every one has come here.
inline const uint64_t* share(uint64_t x) {
  State& w = *s;
  const int l = w.at, t = w.turn[l]++ & 1;
  w.slot[t][l] = x;
  if (!_setjmp(w.lane[l])) _longjmp(w.main, 1);
  return w.slot[t];
}
inline void enter() {
  const int l = s->at;
  s->body(l);
  s->done[l] = true;
  _longjmp(s->main, 1);
}
// Runs f(lane) on all lanes, each up to its next operation in turn.
inline void run(const std::function<void(int)>& f) {
  constexpr size_t kStack = 64 << 10;
  static std::vector<char> stacks(kLanes * kStack);
  State w;
  s = &w;
  w.body = f;
  static volatile int left, l;       // (they outlive the jumps)
  for (left = kLanes; left;) {
    left = 0;
    for (l = 0; l < kLanes; l = l + 1) {
      if (w.done[l]) continue;
      w.at = l;
      if (!_setjmp(w.main)) {
        if (w.turn[l]) _longjmp(w.lane[l], 1);
        ucontext_t c;
        getcontext(&c);
        c.uc_stack.ss_sp = stacks.data() + l * kStack;
        c.uc_stack.ss_size = kStack;
        c.uc_link = nullptr;
        makecontext(&c, (void (*)())enter, 0);
        setcontext(&c);
      }
      left = left + !w.done[l];
    }
    if (left && left != kLanes) abort();             // lanes parted
  }
}
}  // namespace wave

inline int __ffsll(unsigned long long x) { return __builtin_ffsll((long long)x); }
inline unsigned long long __ballot(bool x) {
  const uint64_t* v = wave::share(x);
  unsigned long long m = 0;
  for (int l = 0; l < wave::kLanes; ++l) m |= (unsigned long long)(v[l] != 0) << l;
  return m;
}
inline int host_readlane(int x, int l) { return (int)(uint32_t)wave::share((uint32_t)x)[l & 63]; }
#define __builtin_amdgcn_readlane host_readlane
inline uint32_t wave_prefix_sum(uint32_t x) {
  const int me = wave::s->at;
  const uint64_t* v = wave::share(x);
  uint32_t sum = 0;
  for (int l = 0; l <= me; ++l) sum += (uint32_t)v[l];
  return sum;
}

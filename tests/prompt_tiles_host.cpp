// paged_prompt_attn's plan and a wave's search for its row tile, as the kernels run them, on
// the host.  stdin: calls of cus T B Hk G D cap window sinks, cu[B + 1], lens[B]; stdout for each:
// waves tiles nsplit nwg, the number of row tiles that were found and those (b t0 n r0 index, and the
// first row's position), then the tile and row of some rows of q (every `step`-th) with head 0 of its group (-1 -1: none).
#include "wave_host.h"
#include "../bytes_amd/csrc/paged_prompt_tiles.h"

#include <cstdio>

using namespace bytes_amd;

struct Args {
  int T, B, G, cap, tiles;
  const int32_t* cu;
  struct { const int32_t* lens; } c;
};

template <int ROWS>
static void tiles_of(const Args& a) {
  std::vector<RowTile> found;
  for (int r = 0; r < a.tiles; ++r) {
    RowTile x[wave::kLanes];
    bool ok[wave::kLanes];
    wave::run([&](int lane) {
      ok[lane] = a.B > 1 && a.B < 64 && ROWS > 32 ? find_tile_by_keys<ROWS>(a, r, lane, x[lane]) : find_tile<ROWS>(a, r, lane, x[lane]);
    });
    for (int l = 1; l < wave::kLanes; ++l)
      if (ok[l] != ok[0] || (ok[0] && (x[l].b != x[0].b || x[l].r0 != x[0].r0 || x[l].index != x[0].index))) abort();
    if (ok[0]) found.push_back(x[0]);
  }
  printf("%zu\n", found.size());
  for (const RowTile& x : found) printf("%d %d %d %d %d %d\n", x.b, x.t0, x.n, x.r0, x.index, first_position(x.len, x.n));
  const int step = a.T / 24 + 1;
  for (int t = 0; t < a.T; t += step) {
    int tile = -1, row = -1;
    wave::run([&](int lane) {
      int i = -1, j = -1;
      if (find_row<ROWS>(a, t, 0, lane, i, j) && lane == 0) tile = i, row = j;
    });
    printf("%d %d\n", tile, row);
  }
}

int main() {
  long long cus, T, B, Hk, G, D, cap, window, sinks;
  while (scanf("%lld%lld%lld%lld%lld%lld%lld%lld%lld", &cus, &T, &B, &Hk, &G, &D, &cap, &window, &sinks) == 9) {
    std::vector<int32_t> cu(B + 1), lens(B);
    for (int32_t& x : cu) if (scanf("%d", &x) != 1) return 1;
    for (int32_t& x : lens) if (scanf("%d", &x) != 1) return 1;
    const PromptPlan p = prompt_plan(cus, T, B, Hk, G, (int)D, cap, (int)window, (int)sinks);
    printf("%d %lld %d %d\n", p.waves, (long long)p.tiles, p.nsplit, p.nwg);
    const Args a{(int)T, (int)B, (int)G, (int)cap, (int)p.tiles, cu.data(), {lens.data()}};
    if (p.waves == 8) tiles_of<256>(a);
    else if (p.waves == 4) tiles_of<128>(a);
    else tiles_of<32>(a);
  }
  return 0;
}

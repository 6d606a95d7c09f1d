// bsattn_tree_plan.cpp -- how a tree attention's tokens are cut into the parts
// that its workgroups take (bsattn_tree.hip), and where their partials lie.
#include <algorithm>

#include "bsattn_internal.h"

namespace bsattn {

int64_t tree_plan(const Geometry& g, TreeBatch& tb) {
  const int cols = tb.max_tokens * g.group;
  tb.tiles = cols <= 16 ? 1 : cols <= 32 ? 2 : cols <= 64 ? 4 : cols <= 128 ? 8 : 16;
  tb.groups = (cols + 16 * tb.tiles - 1) / (16 * tb.tiles);
  int64_t all = 0;
  int most = 1;
  for (int i = 0; i < tb.n; ++i) {
    all += tb.units[i];
    most = std::max(most, tb.units[i]);
  }
  // One round of workgroups: eight waves of 256 registers fill a CU, of four two fit.
  // Two rounds cost starts, ends and partials: 64 columns over 8 x 32k bf16 tokens 188
  // us in one, 200 in two, 220 in three; 256 350, 369, 448; 100 over 4 x 131k int4 499,
  // 512, 523; 192 in windows of ragged trees 160, 187, 223.  (Ragged lengths would gain
  // from two, 96 columns over 32 requests: the step 541 and 524.)
  const int64_t want = (tb.tiles > 2 ? 1 : 2) * (int64_t)std::max(g.cus, 1), each = (int64_t)g.hkv * tb.groups;
  auto parts = [&](int i, int cu) { return std::max(1, (tb.units[i] + cu - 1) / cu); };
  auto fits = [&](int cu) {
    int64_t n = 0;
    for (int i = 0; i < tb.n; ++i) n += parts(i, cu);
    return n * each <= want;
  };
  auto cut = [&](int64_t workgroups) {
    const int64_t cu = std::max<int64_t>(4, (all * each + workgroups - 1) / workgroups);
    return ((int)std::min<int64_t>(cu, most) + 3) & ~3;
  };
  tb.cu = cut(want);
  int lo = tb.cu / 4, hi = (most + 3) / 4;  // in fours: the smallest that fits
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (fits(4 * mid)) hi = mid;
    else lo = mid + 1;
  }
  const bool even = 4 * lo <= 32 || 2 * (int64_t)4 * lo * want <= 3 * all * each;
  tb.cu = !fits(4 * lo) ? cut(want) : even ? 4 * lo : cut(3 * want);
  // With few units a workgroup's time is its ends: waves of one column tile leave half
  // as many teams' sums to join.  One request, 64 columns over 4k bf16 tokens (4 units
  // a workgroup) 18.4 us, 20.0 with waves of two, 8k (8) 19.6 and 21.2, 16k (16) 25.4
  // and 25.9, 32k 34.2 and 34.0; 128 columns over 8k 25.5 and 26.5, 16k 33.3 and 32.6,
  // 64k 74.5 and 66.5.
  tb.narrow = (tb.tiles == 4 || tb.tiles == 8) && tb.cu <= 12;
  // (it ends: a request of one part has no partials)
  while (true) {
    int64_t n = 0, blocks = 0;
    for (int i = 0; i < tb.n; ++i) {
      const int p = parts(i, tb.cu);
      tb.part0[i] = (int32_t)n;
      tb.row0[i] = (int32_t)blocks;
      n += p;
      if (p > 1) blocks += (int64_t)p * tb.max_tokens;
    }
    tb.part0[tb.n] = (int32_t)n;
    if (blocks * g.hq <= kPrefillRows) return blocks * g.hq;
    tb.cu *= 2;
  }
}

}  // namespace bsattn

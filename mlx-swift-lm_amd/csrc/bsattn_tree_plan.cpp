// bsattn_tree_plan.cpp -- how a tree attention's tokens are cut into the parts
// that its workgroups take (bsattn_tree.hip), and where their partials lie.
#include <algorithm>
#include <cstdint>

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
  // Workgroups of one round: eight waves of 256 registers fill a CU, of four two fit.
  // Further rounds cost starts, ends and partials, about the time of 12 units a
  // workgroup: 64 columns over 8 x 32k bf16 tokens 188 us in one round, 201 in two, 224
  // in three; 256 403, 428, 507; 100 over 4 x 131k int4 497, 511, 526; 192 in windows
  // of ragged trees 160, 190, 226.  Where the longest request's part would outlast the
  // others by far, more are shorter all the same: 96 columns over 32 requests of 300 to
  // 20000 tokens, bf16 300 us in two or three rounds, int4 342 in three, 382 in two; 64
  // over 40 x 9k bf16 tokens 334 with a part each, one round and a quarter, 296 in four.
  // By little they are not (what the others leave of the memory's rate falls to the
  // longest): 64 over 9 x 13k tokens, a seventh more units in the longest part, 96 us,
  // cut for two rounds 107.  One round more is not among the tries: it is at once good
  // enough for what three leave behind it (those int4 requests 382 for 342 us, 40 x 9k
  // int4 tokens 273 for 259) and gains 4% elsewhere at most.
  const int64_t want = (tb.tiles > 2 ? 1 : 2) * (int64_t)std::max(g.cus, 1), each = (int64_t)g.hkv * tb.groups;
  constexpr int64_t kEnds = 12;
  auto parts = [&](int i, int cu) { return std::max(1, (tb.units[i] + cu - 1) / cu); };
  auto workgroups = [&](int cu) {
    int64_t n = 0;
    for (int i = 0; i < tb.n; ++i) n += parts(i, cu);
    return n * each;
  };
  // (in units: all rounds as long as the longest part, or the work spread evenly and a part)
  auto time = [&](int cu) {
    const int64_t n = workgroups(cu), part = cu + kEnds;
    return std::min((n + want - 1) / want * part, (all * each + n * kEnds) / want + part);
  };
  const int64_t least = (tb.n * each + want - 1) / want, bound = all * each / want + kEnds;
  int64_t best = INT64_MAX;
  for (int64_t more : {0, 2, 3}) {
    if (best <= bound + bound / 8) break;
    const int64_t rounds = least + more;
    // in fours: the smallest that fits
    int lo = (int)std::max<int64_t>(1, all * each / (4 * rounds * want)), hi = std::max(lo, (most + 3) / 4);
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      if (workgroups(4 * mid) <= rounds * want) hi = mid;
      else lo = mid + 1;
    }
    const int64_t t = time(4 * lo);
    if (best == INT64_MAX || t < best - best / 8) {
      best = t;
      tb.cu = 4 * lo;
    }
  }
  // With few units a workgroup's time is its ends: waves of one column tile leave half
  // as many teams' sums to join.  One request, 64 columns over 4k bf16 tokens (4 units
  // a workgroup) 17.8 us, 19.3 with waves of two, 8k (8) 19.1 and 20.7, 16k (16) 24.4
  // and 25.2, 32k 33.0 and 33.5; 128 columns over 8k 25.9 and 26.1, 16k 33.9 and 32.4,
  // 64k 75.4 and 69.7.
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

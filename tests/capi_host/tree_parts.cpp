// tree_parts.cpp -- the parts of tree attentions over random batches, as the
// workgroups of the launch see them: every unit with a token that a node may see
// is taken once per column group, whole units first and no more than seven
// others in a part; every partial has a row of its own inside the workspace, and
// the join finds those that were written; also where a launch replays over
// requests of other lengths and counts.
#include <algorithm>
#include <random>
#include <set>

#include "stubs.h"

using namespace bsattn;

namespace {

struct Request {
  int T, N;  // tokens with the step's, the step's
};

// the launch over requests as they are now
void launch(const Geometry& g, const TreeBatch& tb, int64_t rows, const std::vector<Request>& now) {
  CHECK(rows % g.hq == 0 && rows <= kPrefillRows);
  const int64_t blocks = rows / g.hq;
  const int parts = tb.groups > 1 ? (tb.part0[tb.n] + 7) & ~7 : tb.part0[tb.n];
  std::set<int64_t> used;
  for (int i = 0; i < tb.n; ++i) CHECK(tb.part0[i + 1] > tb.part0[i]);
  std::vector<std::vector<int>> taken(tb.n);
  std::vector<std::set<int>> wrote(tb.n);  // parts
  for (int at = 0; at < parts; ++at) {
    int i = -1;
    for (int k = 0; k < tb.n; ++k) i += tb.part0[k] <= at;
    if (at >= tb.part0[tb.n]) continue;
    const int T = now[i].T, N = std::min({now[i].N, tb.max_tokens, T}), P = T - N;
    const int lo = tb.window > 0 ? std::max(0, P - tb.window + 1) : 0, u0 = lo >> 5;
    const int units = N > 0 ? ((T - 1) >> 5) - u0 + 1 : 0, most = tb.part0[i + 1] - tb.part0[i], part = at - tb.part0[i];
    int cu = tb.cu;
    if (units > tb.units[i]) cu = std::max(cu, ((units + most - 1) / most + 3) & ~3);
    CHECK((units + cu - 1) / cu <= most);
    if (part == 0) taken[i].assign(units, 0);
    if (N > 0) CHECK(tb.groups * 16 * tb.tiles >= N * g.group);
    if (part * (int64_t)cu >= units) continue;
    const int ua = u0 + part * cu, ub = std::min(ua + cu, u0 + units);
    const int whole0 = tb.window > 0 ? (std::max(0, P + N - tb.window) + 31) >> 5 : 0, whole1 = P >> 5;
    const int fa = std::min(std::max(ua, whole0), ub), full = std::max(std::min(ub, whole1) - fa, 0), places = ub - ua;
    CHECK(places >= 1 && places - full <= 7);
    for (int at_place = 0; at_place < places + 8; ++at_place) {
      const int p = std::min(at_place, places - 1), k = ua + p - full;
      const int unit = p < full ? fa + p : k < fa ? k : k + full;
      CHECK(unit >= ua && unit < ub);
      if (at_place >= places) continue;
      ++taken[i][unit - u0];
      // whole: every node sees every token (its window begins at its position)
      if (p < full) CHECK(32 * unit + 31 < P && (tb.window == 0 || 32 * unit > P + N - 1 - tb.window));
    }
    wrote[i].insert(part);
    if (most > 1)
      for (int node = 0; node < N; ++node) {
        const int64_t row = (int64_t)tb.row0[i] + (int64_t)part * tb.max_tokens + node;
        CHECK(row >= 0 && row < blocks && used.insert(row).second);
      }
  }
  for (int i = 0; i < tb.n; ++i) {
    for (int u : taken[i]) CHECK(u == 1);
    const int units = (int)taken[i].size(), most = tb.part0[i + 1] - tb.part0[i];
    int cu = tb.cu;
    if (units > tb.units[i]) cu = std::max(cu, ((units + most - 1) / most + 3) & ~3);
    CHECK((int)wrote[i].size() == (units + cu - 1) / cu);
  }
}

}  // namespace

int main() {
  std::mt19937 rng(11);
  auto pick = [&](int n) { return (int)(rng() % (unsigned)n); };
  const int heads[] = {1, 2, 4, 8, 16}, lengths[] = {1, 33, 64, 500, 5000, 24576};
  for (int tries = 0; tries < 3000; ++tries) {
    Geometry g{};
    g.hkv = heads[pick(5)];
    g.group = heads[pick(5)];
    g.hq = g.hkv * g.group;
    g.cus = pick(4) ? 256 : pick(300);
    g.tb = pick(2) ? 64 : 32;
    const int longest = lengths[pick(6)];  // units
    TreeBatch tb{};
    tb.n = 1 + pick(tries % 10 ? 12 : kMaxBatch);
    tb.max_tokens = 1 + pick(kMaxNodes);
    tb.window = pick(3) ? 0 : 1 + pick(pick(2) ? 70 : 3000);
    std::vector<int> held(tb.n);
    for (int i = 0; i < tb.n; ++i) {
      held[i] = pick(8) ? 1 + pick(pick(2) ? longest : std::min(longest, 40)) : 0;
      int64_t units = held[i];
      if (tb.window > 0) units = std::min<int64_t>(units, ((int64_t)tb.window + tb.max_tokens + 62) / 32);
      tb.units[i] = (int)units;
    }
    const int64_t rows = tree_plan(g, tb);
    CHECK(tb.cu >= 4 && tb.cu % 4 == 0);
    auto requests = [&](bool grown) {
      std::vector<Request> now(tb.n);
      for (int i = 0; i < tb.n; ++i) {
        const int most = grown && pick(2) ? 32 * 24576 : 32 * held[i];
        now[i].T = most ? (pick(3) ? most - pick(std::min(most, 40)) : pick(most + 1)) : 0;
        now[i].N = pick(6) ? std::min(1 + pick(tb.max_tokens), now[i].T) : 0;
      }
      return now;
    };
    launch(g, tb, rows, requests(false));
    launch(g, tb, rows, requests(false));
    launch(g, tb, rows, requests(true));
    // without a workspace: one part a request
    TreeBatch whole = tb;
    whole.cu = INT32_MAX / 32;
    for (int i = 0; i <= whole.n; ++i) whole.part0[i] = i;
    launch(g, whole, 0, requests(true));
  }
  std::puts("ok");
  return 0;
}

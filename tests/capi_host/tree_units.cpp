// tree_units.cpp -- the kernels' own integer code (bsattn_tree_parts.h) over
// random batches and what is left of it in the plan: every unit with a token
// that a node may see is taken once, whole units first; a part's places past its
// last unit repeat it; partials have rows of their own; requests that grew or
// shrank since the plan are covered; and the sets are those of a walk over the
// tokens.
#include <algorithm>
#include <random>
#include <set>

#include "../../mlx-swift-lm_amd/csrc/bsattn_tree_parts.h"
#include "stubs.h"

using namespace bsattn;

namespace {

// by the definition: whether some node of N behind P may see token t, and whether every one does
bool may_see(const TreeBatch& tb, int P, int N, int t) {
  // (a root's position is P, the deepest node's P + N - 1; a node's own path lies behind P)
  return t < P + N && (tb.window == 0 || t > P - tb.window);
}
bool all_see(const TreeBatch& tb, int P, int N, int t) { return t < P && (tb.window == 0 || t > P + N - 1 - tb.window); }

void request(const Geometry& g, const TreeBatch& tb, int64_t rows, int i, int T, int taken, std::set<int64_t>& used) {
  const TreeRange r = tree_range(tb, i, T, taken, g.group);
  const int most = tb.part0[i + 1] - tb.part0[i], parts = tree_parts(r);
  CHECK(r.T == T && r.N == std::min({taken, tb.max_tokens, T}) && r.P + r.N == T && (1 << r.lg) == g.group);
  CHECK(most >= 1 && parts <= most && (parts == 0) == (r.N == 0) && tree_direct(tb, i) == (most == 1));
  CHECK(tb.groups * 16 * tb.tiles >= r.N * g.group);
  std::set<int> seen;
  for (int part = 0; part < parts; ++part) {
    const TreePart p(tb, r, part);
    CHECK(p.places >= 1 && p.places <= r.cu && p.full >= 0 && p.places - p.full <= 7);
    for (int at = 0; at < p.places; ++at) {
      const int unit = p.unit(at);
      CHECK(seen.insert(unit).second);
      bool whole = true, any = false;
      for (int t = 32 * unit; t < 32 * unit + 32; ++t) {
        whole = whole && all_see(tb, r.P, r.N, t);
        any = any || may_see(tb, r.P, r.N, t);
      }
      CHECK(any && (at >= p.full || whole));
    }
    for (int at = p.places; at < p.places + 10; ++at) CHECK(p.unit(at) == p.unit(p.places - 1));
    for (int node = 0; most > 1 && node < r.N; ++node) {
      const int64_t row = tree_row(tb, i, part, node);
      CHECK(row >= 0 && row < rows / g.hq && used.insert(row).second);
    }
  }
  // no unit with a token that is seen is missing (the ends decide: the units are a run)
  if (r.N > 0) {
    const int first = tb.window > 0 ? std::max(0, r.P - tb.window + 1) >> 5 : 0, last = (T - 1) >> 5;
    CHECK((int)seen.size() == last - first + 1 && *seen.begin() == first && *seen.rbegin() == last);
    CHECK(may_see(tb, r.P, r.N, T - 1) && (first == 0 || !may_see(tb, r.P, r.N, 32 * first - 1)));
  }
}

}  // namespace

int main() {
  std::mt19937 rng(5);
  auto pick = [&](int n) { return (int)(rng() % (unsigned)n); };
  for (int tries = 0; tries < 600; ++tries) {
    Geometry g{};
    g.hkv = 1 << pick(4);
    g.group = 1 << pick(5);
    g.hq = g.hkv * g.group;
    g.cus = pick(5) ? 256 : 1 + pick(300);
    g.tb = pick(2) ? 64 : 32;
    TreeBatch tb{};
    tb.n = 1 + pick(tries % 8 ? 6 : kMaxBatch);
    tb.max_tokens = 1 + pick(kMaxNodes);
    tb.window = pick(2) ? 0 : 1 + pick(pick(2) ? 100 : 4000);
    std::vector<int> held(tb.n);
    for (int i = 0; i < tb.n; ++i) {
      held[i] = pick(8) ? 1 + pick(pick(3) ? 60 : 2000) : 0;
      const int64_t window = ((int64_t)tb.window + tb.max_tokens + 62) / 32;
      tb.units[i] = tb.window > 0 ? (int)std::min<int64_t>(held[i], window) : held[i];
    }
    const int64_t rows = tree_plan(g, tb);
    CHECK(tree_grid(tb) >= tb.part0[tb.n] && (tb.groups == 1 || tree_grid(tb) % 8 == 0));
    for (int turn = 0; turn < 3; ++turn) {  // (2: a replay past what the plan was made for)
      std::set<int64_t> used;
      for (int i = 0; i < tb.n; ++i) {
        const int most = 32 * (turn == 2 && pick(2) ? 4000 : held[i]);
        const int T = pick(3) ? most - pick(std::min(most, 70) + 1) : pick(most + 1);
        request(g, tb, rows, i, T, pick(7) ? 1 + pick(tb.max_tokens + 3) : 0, used);
      }
    }
  }
  std::puts("ok");
  return 0;
}

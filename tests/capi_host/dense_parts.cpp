// dense_parts.cpp -- the parts of dense decodes over random batches, as the
// workgroups of the launch see them: every unit of every sequence is read once
// for it, every partial has a row of its own inside the workspace, and the join
// finds exactly those that were written, also where a launch replays over
// sequences of other lengths.
#include <algorithm>
#include <random>
#include <set>

#include "stubs.h"

using namespace bsattn;

namespace {

struct Batch {
  Geometry g{};
  DenseBatch db{};
  std::vector<int> units;  // what each entry's pages hold
};

DenseJob& add(DenseBatch& db, int first, int count) {
  DenseJob& job = db.job[db.jobs++];
  job = DenseJob{};
  job.first = (int16_t)first;
  job.count = (int16_t)count;
  job.entry = db.order[first];
  job.seq = 1000 + job.entry;
  job.of = -1;
  return job;
}

Batch make(std::mt19937& rng, int n, int hkv, int group, int cus, int longest, bool share) {
  auto pick = [&](int k) { return (int)(rng() % (unsigned)k); };
  Batch b;
  b.g.hkv = hkv;
  b.g.group = group;
  b.g.hq = hkv * group;
  b.g.cus = cus;
  b.g.tb = pick(2) ? 64 : 32;
  b.g.kv_bits = pick(3) * 4;
  b.db.n = n;
  const int kind = pick(3);
  for (int i = 0; i < n; ++i)
    b.units.push_back(kind == 0 ? longest : kind == 1 ? pick(longest + 1) : pick(4) ? pick(std::min(longest, 40) + 1) : pick(longest + 1));
  std::vector<int> of(n, -1), rest(n);
  for (int i = 0; i < n; ++i) rest[i] = i;
  int placed = 0;
  if (share && group < 16) {
    std::shuffle(rest.begin(), rest.end(), rng);
    size_t at = 0;
    while (at + 1 < rest.size()) {
      const int count = std::min<int>(2 + pick(16 / group - 1), (int)(rest.size() - at));
      int least = INT32_MAX;
      for (int k = 0; k < count; ++k) least = std::min(least, b.units[rest[at + k]]);
      least -= least % 2;
      if (count >= 2 && least >= 32 && pick(4)) {
        for (int k = 0; k < count; ++k) {
          b.db.order[placed + k] = (int16_t)rest[at + k];
          of[rest[at + k]] = b.db.jobs;
        }
        add(b.db, placed, count).units = least - 2 * pick((least - 30) / 2);
        placed += count;
      }
      at += count;
    }
  }
  for (int i = 0; i < n; ++i) {
    b.db.order[placed] = (int16_t)i;
    DenseJob& job = add(b.db, placed++, 1);
    job.of = (int16_t)of[i];
    job.from = of[i] >= 0 ? b.db.job[of[i]].units : 0;
    job.units = b.units[i] - job.from;
  }
  return b;
}

// the launch over sequences that hold `units` now
void launch(const Batch& b, int parts, int64_t rows, const std::vector<int>& units) {
  const DenseBatch& db = b.db;
  const int64_t blocks = rows ? (rows - kJoinRows) / b.g.hq : 0;
  CHECK(rows == 0 || (rows > kJoinRows && (rows - kJoinRows) % b.g.hq == 0));
  CHECK(rows <= kPrefillRows);
  std::set<int64_t> used;                         // rows of partials, in blocks of hq
  std::vector<std::set<int64_t>> wrote(db.n);     // by entry
  std::vector<std::vector<int>> seen(db.n);       // units read for each entry
  std::vector<int> direct(db.n, 0), tables(db.n, 0);
  std::vector<DenseJoin> join(db.n);
  for (int e = 0; e < db.n; ++e) seen[e].assign(units[e], 0);
  for (int at = 0; at < parts; ++at) {
    int j = -1;
    for (int i = 0; i < db.jobs; ++i) j += db.job[i].part0 <= at;
    CHECK(j >= 0);
    const DenseJob& job = db.job[j];
    const int part = at - job.part0;
    const bool alone = job.count == 1;
    const int u0 = alone ? job.from : 0, held = alone ? std::max(0, units[job.entry] - job.from) : job.units;
    int cu = db.cu;
    if (alone && held > job.units) {
      const int most = std::max(1, (job.units + cu - 1) / cu);
      cu = std::max(cu, ((held + most - 1) / most + 3) & ~3);
    }
    const int own = (held + cu - 1) / cu;
    const bool whole = alone && own <= 1 && job.of < 0;
    if (alone && part == 0) {
      ++tables[job.entry];
      join[job.entry] = DenseJoin{job.shared0, job.step, job.shared, job.row0 - job.shared, job.shared + own};
    }
    const int ua = u0 + part * cu, ub = std::min(ua + cu, u0 + held);
    if (ub <= ua) {
      if (whole && part == 0) ++direct[job.entry];
      continue;
    }
    for (int k = 0; k < job.count; ++k) {
      const int e = db.order[job.first + k];
      for (int u = ua; u < ub; ++u) {
        CHECK(u < units[e]);
        ++seen[e][u];
      }
      if (whole) {
        ++direct[e];
        continue;
      }
      const int64_t row = (int64_t)job.row0 + (int64_t)part * job.count + k;
      CHECK(row >= 0 && row < blocks);
      CHECK(used.insert(row).second);
      wrote[e].insert(row);
    }
  }
  for (int e = 0; e < db.n; ++e) {
    for (int u = 0; u < units[e]; ++u) CHECK(seen[e][u] == 1);
    CHECK(tables[e] == 1);
    const DenseJoin& t = join[e];
    const bool joined = !(t.parts <= 1 && t.shared == 0);
    CHECK(direct[e] == (joined ? 0 : 1));
    std::set<int64_t> reads;
    if (joined)
      for (int p = 0; p < t.parts; ++p) CHECK(reads.insert(p < t.shared ? t.shared0 + (int64_t)p * t.step : t.own0 + p).second);
    CHECK(reads == wrote[e]);
    CHECK(rows > 0 || !joined);
  }
}

void check(std::mt19937& rng, Batch b) {
  auto pick = [&](int k) { return (int)(rng() % (unsigned)k); };
  int64_t rows = -1;
  const int parts = dense_plan(b.g, b.db, &rows);
  CHECK(parts >= b.db.n && b.db.cu >= 4 && b.db.cu % 4 == 0);
  launch(b, parts, rows, b.units);
  // (an entry may hold fewer tokens than its pages; a captured launch, which
  // has no shared jobs, may find any number)
  std::vector<int> other = b.units;
  bool shared = false;
  for (int j = 0; j < b.db.jobs; ++j) {
    const DenseJob& job = b.db.job[j];
    if (job.count > 1) shared = true;
    else other[job.entry] = job.from + pick(b.units[job.entry] - job.from + 1);
  }
  launch(b, parts, rows, other);
  // without a workspace: one part an entry, whatever it holds
  Batch whole = b;
  whole.db.cu = INT32_MAX / 32;
  whole.db.jobs = 0;
  for (int i = 0; i < b.db.n; ++i) {
    whole.db.order[i] = (int16_t)i;
    add(whole.db, i, 1).part0 = i;
  }
  launch(whole, b.db.n, 0, b.units);
  if (shared) return;
  for (int& u : other) u = pick(3) ? pick(24577) : 0;
  launch(b, parts, rows, other);
}

}  // namespace

int main() {
  std::mt19937 rng(7);
  auto pick = [&](int k) { return (int)(rng() % (unsigned)k); };
  const int heads[] = {1, 2, 4, 8, 16};
  const int lengths[] = {0, 1, 33, 64, 500, 3000, 24576};
  for (int i = 0; i < 1200; ++i)
    check(rng, make(rng, 1 + pick(kMaxBatch), heads[pick(5)], heads[pick(5)], pick(4) ? 256 : pick(300), lengths[pick(7)], pick(3) > 0));
  // the largest: 64 entries of 128 query heads that share, of 256 that do not
  for (int i = 0; i < 60; ++i) {
    check(rng, make(rng, kMaxBatch, 16, 8, 256, 24576, true));
    check(rng, make(rng, kMaxBatch, 16, 16, 256, 24576, false));
  }
  std::puts("ok");
  return 0;
}

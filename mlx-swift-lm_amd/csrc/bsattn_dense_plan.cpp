// bsattn_dense_plan.cpp -- how a dense decode's jobs are cut into the parts that
// its workgroups take (bsattn_dense.hip), and where their partials lie.
#include <algorithm>

#include "bsattn_internal.h"

namespace bsattn {

// Cuts the jobs into parts.
int dense_plan(const Geometry& g, DenseBatch& db, int64_t* rows) {
  int64_t all = 0;
  int most = 1;
  for (int j = 0; j < db.jobs; ++j) {
    all += db.job[j].units;
    most = std::max(most, db.job[j].units);
  }
  // Shared jobs first, for every head, then what the entries have of their own:
  // four prompts of 16001 int8 tokens, four branches each, 33.2 -> 29.8 us.
  // Where the entries are alike their parts stay together (8 x 32k bf16 161.6
  // us, head by head 163.4; 32 ragged windows 83.4 and 86.6)
  db.heads_first = db.job[0].count > 1;
  // One round of workgroups, two per CU: 8 x 32k bf16 tokens 162 us (three per
  // CU 167, four 165, six 169), 4 x 131k int4 99 (100, 110, 105), 4 x 262k int8
  // in 16-head groups 179 (185, 190, 199).  The parts are cut so that they all
  // fit into it: 9 x 13563 fp16 tokens, 16 kv heads, 153 us (576 workgroups 174),
  // 5 x 40k bf16 131 (152).
  const int64_t want = 2 * (int64_t)std::max(g.cus, 1);
  // (A branch's rest of a unit or two counts as a workgroup like any other: four
  // prompts of 16001 int8 tokens, four branches each, have 384 workgroups for
  // what is shared, of 44 units each, and 128 for the rests: 28.9 us.)
  auto fits = [&](int cu) {
    int64_t n = 0;
    for (int j = 0; j < db.jobs; ++j) n += std::max(1, (db.job[j].units + cu - 1) / cu);
    return n * g.hkv <= want;
  };
  auto cut = [&](int64_t workgroups) {
    const int64_t cu = std::max<int64_t>(4, (all * g.hkv + workgroups - 1) / workgroups);
    return ((int)std::min<int64_t>(cu, most) + 3) & ~3;
  };
  db.cu = cut(want);
  int lo = db.cu / 4, hi = (most + 3) / 4;  // in fours: the smallest that fits
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (fits(4 * mid)) hi = mid;
    else lo = mid + 1;
  }
  // Many sequences of different lengths, where the largest part of a round would
  // be far from the average: smaller parts, one after another (48 sequences of
  // 100 to 6000 bf16 tokens 104 us, in one round 111; affine caches, whose parts
  // cost more to begin, less small: 64 of 400 to 4000 int4 42 and 44).  More
  // sequences than a round takes: whole ones (33 x 300 tokens, 16 kv heads, 19
  // us, 24 in parts).
  const bool even = 4 * lo <= 32 || 2 * (int64_t)4 * lo * want <= 3 * all * g.hkv;
  if (!fits(4 * lo)) db.cu = cut(want);
  else db.cu = even ? 4 * lo : cut(g.kv_bits ? want : 3 * want);
  // (it ends: jobs of one part each, shared ones padded to 8, fit)
  static_assert((8 + 1) * kMaxBatch * 128 + kJoinRows <= kPrefillRows && kMaxBatch * 256 + kJoinRows <= kPrefillRows,
                "up to 128 query heads with shared jobs, 256 without");
  while (true) {
    int64_t parts = 0, blocks = 0;
    bool joined = false;
    for (int j = 0; j < db.jobs; ++j) {
      DenseJob& job = db.job[j];
      const bool direct = job.count == 1 && job.of < 0;
      int n = (job.units + db.cu - 1) / db.cu;
      if (job.count == 1) n = std::max(n, 1);  // (zeros for no tokens; the join's table)
      // (jobs of the same blocks: their n-th parts lie a multiple of 8
      // workgroups apart, whatever the grid's order, on the same XCD, whose L2
      // then holds them; two jobs of 4 x 8191 bf16 tokens 17.1 -> 14.6 us.
      // Where no two jobs read the same blocks the padding is empty workgroups
      // and nothing else.)
      if (job.count > 1) n = (n + 7) & ~7;
      job.part0 = (int32_t)parts;
      job.row0 = (int32_t)blocks;
      if (job.of >= 0) {  // (shared jobs come first)
        const DenseJob& with = db.job[job.of];
        job.shared = (int16_t)((with.units + db.cu - 1) / db.cu);
        job.step = with.count;
        job.shared0 = with.row0;
        while (db.order[with.first + job.shared0 - with.row0] != job.entry) ++job.shared0;
      }
      parts += n;
      blocks += (int64_t)n * job.count;
      joined = joined || n > 1 || !direct;
    }
    *rows = joined ? kJoinRows + blocks * g.hq : 0;
    if (*rows <= kPrefillRows) return (int)parts;
    db.cu *= 2;
  }
}

}  // namespace bsattn

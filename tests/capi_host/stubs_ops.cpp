// stubs_ops.cpp -- launchers of the operators around the cache for stubs.h:
// a fork writes the metadata and copies the page, the others do nothing.
#include "stubs.h"

using namespace bsattn;

namespace stub {
bsattn::DenseBatch last_dense;
}  // namespace stub

// every entry has a job of its own, and at most one with others, which hold
// the same units
static void check_jobs(const bsattn::DenseBatch& db) {
  stub::last_dense = db;
  CHECK(db.n >= 1 && db.n <= bsattn::kMaxBatch && db.jobs >= db.n && db.jobs <= bsattn::kMaxDenseJobs);
  std::vector<int> own(db.n, 0), with(db.n, 0), of(db.n, -1);
  for (int j = 0; j < db.jobs; ++j) {
    const bsattn::DenseJob& job = db.job[j];
    CHECK(job.count >= 1 && job.count <= 16 && job.first >= 0 && job.first + job.count <= 2 * bsattn::kMaxBatch);
    CHECK(job.units >= 0);
    CHECK(job.entry == db.order[job.first]);
    for (int k = 0; k < job.count; ++k) {
      const int e = db.order[job.first + k];
      CHECK(e >= 0 && e < db.n);
      if (job.count == 1) {
        ++own[e];
        CHECK(job.of == of[e] && job.from == (of[e] >= 0 ? db.job[of[e]].units : 0));
      } else {
        ++with[e];
        of[e] = j;
        CHECK(db.window == 0 && job.of < 0);
      }
    }
  }
  for (int e = 0; e < db.n; ++e) CHECK(own[e] == 1 && with[e] <= 1);
}

namespace bsattn {
using stub::run;
hipError_t launch_rotate(const Geometry& g, RotateBatch, int, hipStream_t, Timing*) { return run(g, nullptr); }
// (a job of n entries: `splits` parts)
int dense_plan(const Geometry& g, DenseBatch& db, int64_t* rows) {
  db.cu = 4;
  int parts = 0, blocks = 0;
  for (int j = 0; j < db.jobs; ++j) {
    db.job[j].part0 = parts;
    db.job[j].row0 = blocks;
    parts += stub::splits;
    blocks += stub::splits * db.job[j].count;
  }
  *rows = parts == db.n ? 0 : (int64_t)blocks * g.hq;
  return parts;
}
hipError_t launch_dense(const Geometry& g, const DenseBatch& db, int parts, const void*, void*, float* ws,
                        hipEvent_t done, hipStream_t s, Timing*) {
  CHECK((parts > db.n) == (ws != nullptr));
  check_jobs(db);
  {
    std::lock_guard<std::mutex> lock(stub::mu);
    stub::prefills.push_back({ws, (stub::Event*)done, parts});
  }
  const hipError_t e = run(g, nullptr);
  if (e == hipSuccess && done) (void)hipEventRecord(done, s);
  return e;
}
hipError_t launch_fork(const Geometry& g, const ForkBatch& fb, hipStream_t, Timing*) {
  const hipError_t e = run(g, nullptr);
  if (e != hipSuccess && !stub::applies) return e;
  const size_t bytes = (size_t)g.hkv * g.slab_bytes;
  for (int i = 0; i < fb.n; ++i) {
    const int full = fb.tokens[i] / g.tb;
    int32_t *from = g.meta + g.bt_off + (size_t)fb.src[i] * g.mbps, *to = g.meta + g.bt_off + (size_t)fb.dst[i] * g.mbps;
    std::memcpy(to, from, full * 4);
    CHECK((fb.tokens[i] % g.tb != 0) == (fb.tail_to[i] >= 0));
    if (fb.tail_to[i] >= 0) {
      to[full] = fb.tail_to[i];
      std::memcpy(g.pool + fb.tail_to[i] * bytes, g.pool + fb.tail_from[i] * bytes, bytes);
    }
    g.meta[fb.dst[i]] = fb.tokens[i];
    g.meta[g.cap_off + fb.dst[i]] = (full + (fb.tail_to[i] >= 0)) * g.tb;
  }
  return e;
}
}  // namespace bsattn

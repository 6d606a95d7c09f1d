// stubs_ops.cpp -- launchers of the operators around the cache for stubs.h:
// a fork writes the metadata and copies the page, the others do nothing.
#include "stubs.h"

using namespace bsattn;

namespace bsattn {
using stub::run;
hipError_t launch_rotate(const Geometry& g, RotateBatch, int, hipStream_t, Timing*) { return run(g, nullptr); }
int dense_plan(const Geometry&, const int32_t*, DenseBatch& db) {
  db.cu = 4;
  for (int i = 0; i < db.n; ++i) db.part0[i] = i * stub::splits;
  return db.n * stub::splits;
}
hipError_t launch_dense(const Geometry& g, const DenseBatch& db, int parts, const void*, void*, float* ws,
                        hipEvent_t done, hipStream_t s, Timing*) {
  CHECK((parts > db.n) == (ws != nullptr));
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

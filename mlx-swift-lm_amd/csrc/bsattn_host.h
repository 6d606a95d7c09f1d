// bsattn_host.h -- host side shared by the C ABI's sources (bsattn_capi.cpp,
// bsattn_ops.cpp): the cache handle, error reporting, device and capture
// guards, the split prefills' workspaces, sequence lists, metadata patches and
// the page bookkeeping.
//
// The host copy of lengths / block tables is authoritative; the device copy
// (`meta`) is brought up to date in stream order by small patch launches
// whose payload travels in the kernel arguments, so no host staging buffer
// can be overwritten while a copy is still pending.
#pragma once

#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <climits>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <memory>
#include <mutex>
#include <new>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/bsattn.h"
#include "bsattn_internal.h"

namespace bsattn {

// words of the device metadata to set: index and value
using Patches = std::vector<std::pair<int32_t, int32_t>>;

inline thread_local std::string g_err;  // message of the thread's last failed call

inline int fail(int code, const char* fmt, ...) noexcept {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  try {
    g_err = buf;
  } catch (...) {
    g_err.clear();  // no memory for the message: the status code still says what failed
  }
  return code;
}

// Handler of every entry point's function-try-block: no C++ exception
// crosses the ABI.  Host state is only changed after the allocations a call
// needs have succeeded, so a failed call leaves the cache as it was.
inline int on_exception() noexcept {
  try {
    throw;
  } catch (const std::bad_alloc&) {
    return fail(BSATTN_ERR_NOMEM, "host memory allocation failed");
  } catch (const std::length_error&) {
    return fail(BSATTN_ERR_NOMEM, "host container size limit exceeded");
  } catch (const std::exception& e) {
    return fail(BSATTN_ERR_INTERNAL, "internal error: %s", e.what());
  } catch (...) {
    return fail(BSATTN_ERR_INTERNAL, "internal error: unknown exception");
  }
}

inline int hip_fail(hipError_t e, const char* what) {
  return fail(BSATTN_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

#define HIP_TRY(call, what)              \
  do {                                   \
    hipError_t e_ = (call);              \
    if (e_ != hipSuccess) return hip_fail(e_, what); \
  } while (0)

}  // namespace bsattn

struct bsattn_cache {
  bsattn_desc d{};
  bsattn::Geometry geo{};
  int64_t num_pages = 0;
  size_t pool_bytes = 0, summ_bytes = 0, meta_words = 0;
  // per-launch workspaces, rows = batch entries of one launch
  float* scores = nullptr;    // [rows][hkv][sstride] + kScoreSlack
  int32_t* idx_ws = nullptr;  // [rows][hkv][nsel_max]
  float* partials = nullptr;  // [rows][hq][nsplit][D + 2]
  uint32_t* arrive = nullptr; // [kArriveWords] arrival counters of split merges, 0 between launches
  float* err_ws = nullptr;    // [rows][hkv][2][mfma_err_stride]: MFMA score bounds, chunk floors
  // split prefill partials of captured calls (a graph holds their addresses):
  // workspace and its rows, kept until the cache is destroyed
  std::vector<std::pair<float*, int64_t>> graph_ws;
  std::vector<int32_t> len;
  // set by bsattn_append_step: the device-side lengths may be ahead of `len`
  // until bsattn_sync
  bool stale = false;
  std::vector<std::vector<int32_t>> pages;
  std::vector<int32_t> free_pages;  // stack; back() is handed out next
  // holders of each page beyond the first: forks share the full blocks of
  // their prompt.  A page that a sequence may still write to (its last partial
  // block and those behind it) is never shared: a fork copies the partial
  // block, and so does a trim that ends inside a shared one.
  std::vector<int32_t> sharers;
  // metadata words that a failed launch may have left unset (or set ahead of
  // the host): sent before the next call's own (send_unsent)
  bsattn::Patches unsent;
  // the step that the cache was last mapped for (0: none, or the host has
  // changed one of its sequences since), its place among the step's caches, and
  // the step's sequences, also as a mark on each of the cache's
  uint64_t step = 0;
  int32_t step_layer = 0;
  std::vector<int32_t> step_seqs;
  std::vector<char> in_step;
  enum { kMapped, kAppended, kKept } step_state = kMapped;  // the last call with it
  // steps of which the map or this cache's append was captured: the host does not
  // see their replays
  struct CapturedStep {
    uint64_t stamp;     // of the step's last map
    int32_t layer;      // the cache's place in it
    bool map, append;   // which of them
    // requests of the captured map, its rows and the cache's place in it; whether
    // another captured one was for others, and whether the last map is, or was
    // captured itself
    std::shared_ptr<const std::vector<int32_t>> ids;
    int32_t rows, place;
    bool several, other, recorded;
    const bsattn_step* at;  // where the step lay then: another one there has taken its place
  };
  std::vector<CapturedStep> captured_steps;
  // opt-in per-kernel timing (bsattn_profile_*)
  bool profiling = false;
  std::vector<hipEvent_t> event_pool;
  std::vector<std::pair<hipEvent_t, hipEvent_t>> pending[bsattn::kProfKinds];
  double prof_ms[bsattn::kProfKinds] = {};
  int64_t prof_count[bsattn::kProfKinds] = {};
};

namespace bsattn {

struct DeviceGuard {
  int prev = -1;
  bool ok = false;
  explicit DeviceGuard(int dev) {
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    ok = hipSetDevice(dev) == hipSuccess;
  }
  ~DeviceGuard() {
    if (prev >= 0) (void)hipSetDevice(prev);
  }
};

// Lets this thread allocate, free and query events while any thread captures
// a graph, without invalidating the capture.
class RelaxedCapture {
 public:
  RelaxedCapture() { ok_ = hipThreadExchangeStreamCaptureMode(&mode_) == hipSuccess; }
  ~RelaxedCapture() {
    if (ok_) (void)hipThreadExchangeStreamCaptureMode(&mode_);
  }
  RelaxedCapture(const RelaxedCapture&) = delete;
  RelaxedCapture& operator=(const RelaxedCapture&) = delete;
  bool ok() const { return ok_; }

 private:
  hipStreamCaptureMode mode_ = hipStreamCaptureModeRelaxed;
  bool ok_ = false;
};

constexpr size_t kPrefillRowBytes = (kHeadDim + 2) * sizeof(float);

// ---------------------------------------------------------------------------
// Workspaces of the split prefills of one GPU (68 MB each), shared by its
// caches: a model has one cache per layer, and its layers' prefills follow
// each other on a stream.  A call takes the one that its stream used last, or
// one whose last user has finished; failing that another is allocated, up to
// kMost, and beyond that the call waits, on its stream, for another stream's.
// In each case the stream waits for the event of the last use (nothing to
// wait for on the same stream), so a handle that names another stream by now
// is no matter.  The lock is held from the choice until the event is
// recorded.  All are freed with the GPU's last cache.
// The event belongs to the merge's dispatch and has no system fence (only
// streams of the GPU wait for it): a call takes no longer with it than without
// (64 bf16 tokens behind 960, 19.9 and 19.7 us; recorded by itself, or with
// the fence, 20.9-22.6).
// ---------------------------------------------------------------------------
class PrefillSpaces {
 public:
  static PrefillSpaces* of(int device) {
    static PrefillSpaces all[kMaxDevices];
    return device >= 0 && device < kMaxDevices ? &all[device] : nullptr;
  }
  void add_cache() {
    std::lock_guard<std::mutex> lock(mu_);
    ++caches_;
  }
  void drop_cache() {  // (the device is current and idle)
    std::lock_guard<std::mutex> lock(mu_);
    if (--caches_ > 0) return;
    RelaxedCapture relaxed;
    for (int i = 0; i < count_; ++i) {
      (void)hipFree(spaces_[i].p);
      (void)hipEventDestroy(spaces_[i].done);
    }
    count_ = 0;
  }
  // launch(workspace, event that its last kernel must record), or launch(null,
  // null) when there is no workspace to be had
  template <typename F>
  hipError_t with(hipStream_t s, F launch) {
    std::unique_lock<std::mutex> lock(mu_);
    Space* sp = pick(s);
    if (sp && hipStreamWaitEvent(s, sp->done, 0) != hipSuccess) {
      (void)hipGetLastError();
      sp = nullptr;
    }
    if (!sp) {
      lock.unlock();
      return launch(nullptr, nullptr);
    }
    sp->stream = s;
    const hipError_t e = launch(sp->p, sp->done);
    // (part of the work may be under way without the event)
    if (e != hipSuccess && hipEventRecord(sp->done, s) != hipSuccess) (void)hipDeviceSynchronize();
    return e;
  }

 private:
  static constexpr int kMaxDevices = 64, kMost = 4;
  struct Space {
    float* p;
    hipEvent_t done;  // recorded by the last use
    hipStream_t stream;
  };
  Space* pick(hipStream_t s) {
    RelaxedCapture relaxed;
    if (!relaxed.ok()) return nullptr;
    for (int i = 0; i < count_; ++i)
      if (spaces_[i].stream == s) return &spaces_[i];
    for (int i = 0; i < count_; ++i) {
      if (hipEventQuery(spaces_[i].done) == hipSuccess) return &spaces_[i];
      (void)hipGetLastError();  // (not ready is no error of this call)
    }
    if (count_ < kMost) {
      Space n{nullptr, nullptr, s};
      if (hipMalloc((void**)&n.p, (size_t)kPrefillRows * kPrefillRowBytes) == hipSuccess) {
        if (hipEventCreateWithFlags(&n.done, hipEventDisableTiming | hipEventDisableSystemFence) == hipSuccess) {
          spaces_[count_] = n;
          return &spaces_[count_++];
        }
        (void)hipFree(n.p);
      }
      (void)hipGetLastError();
    }
    return count_ > 0 ? &spaces_[next_++ % count_] : nullptr;
  }
  std::mutex mu_;
  int caches_ = 0, count_ = 0;
  unsigned next_ = 0;
  Space spaces_[kMost] = {};
};

// the cache's own workspace of at least `rows` rows for a captured call, or
// null
inline float* graph_workspace(bsattn_cache* c, int64_t rows) {
  for (const auto& w : c->graph_ws)
    if (w.second >= rows) return w.first;
  RelaxedCapture relaxed;
  if (!relaxed.ok()) return nullptr;
  c->graph_ws.reserve(c->graph_ws.size() + 1);
  float* p = nullptr;
  if (hipMalloc((void**)&p, (size_t)rows * kPrefillRowBytes) != hipSuccess) {
    (void)hipGetLastError();
    return nullptr;
  }
  c->graph_ws.emplace_back(p, rows);
  return p;
}

// Seq list -> vector (validated, distinct)
inline int seq_list(const bsattn_cache* c, const int32_t* ids, int32_t n, std::vector<int32_t>& out) {
  if (n < 1) return fail(BSATTN_ERR_INVALID, "n_seqs must be >= 1 (got %d)", n);
  if (n > c->d.max_seqs) return fail(BSATTN_ERR_RANGE, "n_seqs %d exceeds max_seqs %d", n, c->d.max_seqs);
  out.resize(n);
  std::vector<char> seen(c->d.max_seqs, 0);
  for (int i = 0; i < n; ++i) {
    const int s = ids ? ids[i] : i;
    if (s < 0 || s >= c->d.max_seqs) return fail(BSATTN_ERR_RANGE, "sequence id %d out of range [0, %d)", s, c->d.max_seqs);
    if (seen[s]) return fail(BSATTN_ERR_INVALID, "sequence id %d listed twice", s);
    seen[s] = 1;
    out[i] = s;
  }
  return BSATTN_OK;
}

inline PatchBatch patch_batch(const std::pair<int32_t, int32_t>* p, size_t n) {
  PatchBatch pb{};
  pb.n = (int32_t)n;
  for (size_t i = 0; i < n; ++i) {
    pb.idx[i] = p[i].first;
    pb.val[i] = p[i].second;
  }
  return pb;
}

inline int send_patches(const bsattn_cache* c, const Patches& p, hipStream_t s) {
  for (size_t i = 0; i < p.size(); i += kMaxPatch) {
    const PatchBatch pb = patch_batch(p.data() + i, std::min<size_t>(kMaxPatch, p.size() - i));
    HIP_TRY(launch_patch(c->geo, pb, s), "patch launch");
  }
  return BSATTN_OK;
}

// whether work on s is recorded into a graph (also when that cannot be told)
inline bool capturing(hipStream_t s) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(s, &st) == hipSuccess) return st != hipStreamCaptureStatusNone;
  (void)hipGetLastError();
  return true;
}

// What an earlier call could not send; every call that changes the metadata,
// or launches work that reads it, starts here.  (The exports read block-table
// entries of tokens already held, which have been sent.)  Not into a graph,
// whose every replay would set the words back.
inline int send_unsent(bsattn_cache* c, hipStream_t s) {
  if (c->unsent.empty()) return BSATTN_OK;
  if (capturing(s))
    return fail(BSATTN_ERR_INVALID, "an earlier launch of this cache failed: make one call outside the capture first");
  if (int rc = send_patches(c, c->unsent, s)) return rc;
  c->unsent.clear();
  return BSATTN_OK;
}

// (after send_unsent)
inline int flush_patches(bsattn_cache* c, Patches& p, hipStream_t s) {
  const int rc = send_patches(c, p, s);
  if (rc) c->unsent.swap(p);
  return rc;
}

// device-side capacity of a sequence: tokens its pages hold
inline void cap_patch(const bsattn_cache* c, int seq, Patches& patches) {
  patches.emplace_back(c->geo.cap_off + seq, (int32_t)c->pages[seq].size() * c->d.block_size);
}

inline int release_pages(bsattn_cache* c, int seq, int keep_blocks,
                  Patches& patches) {
  auto& pg = c->pages[seq];
  int32_t* sharers = c->sharers.data();
  for (size_t i = pg.size(); i > (size_t)keep_blocks; --i) {
    const int32_t p = pg[i - 1];
    if (sharers[p] > 0) --sharers[p];
    else c->free_pages.push_back(p);
  }
  if (pg.size() > (size_t)keep_blocks) pg.resize(keep_blocks);
  cap_patch(c, seq, patches);
  return BSATTN_OK;
}

// bytes of a page's slabs
inline size_t page_slabs(const Geometry& g) { return (size_t)g.hkv * g.slab_bytes; }

// Profiling slots for one C-ABI call: null unless profiling is on and the
// stream is not being captured into a graph.
inline Timing* prof_slots(bsattn_cache* c, hipStream_t s, Timing* tm) {
  if (!c->profiling) return nullptr;
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(s, &st) != hipSuccess || st != hipStreamCaptureStatusNone) return nullptr;
  for (int k = 0; k < kProfKinds; ++k) {
    hipEvent_t ev[2];
    for (auto& e : ev) {
      if (!c->event_pool.empty()) {
        e = c->event_pool.back();
        c->event_pool.pop_back();
      } else if (hipEventCreate(&e) != hipSuccess) {
        e = nullptr;
      }
    }
    tm[k].start = ev[0];
    tm[k].stop = ev[1];
    tm[k].used = false;
  }
  return tm;
}

inline void prof_collect(bsattn_cache* c, Timing* tm) {
  if (!tm) return;
  for (int k = 0; k < kProfKinds; ++k) {
    if (tm[k].used && tm[k].start && tm[k].stop) {
      c->pending[k].emplace_back(tm[k].start, tm[k].stop);
    } else {
      if (tm[k].start) c->event_pool.push_back(tm[k].start);
      if (tm[k].stop) c->event_pool.push_back(tm[k].stop);
    }
  }
}

// workspace and event for the parts of a call: the cache's own where they fit
// (no event: a cache's calls follow each other), otherwise as for a split
// prefill
template <typename F>
hipError_t with_partials(bsattn_cache* c, int64_t rows, hipStream_t s, F launch) {
  if (rows <= (int64_t)std::min(kMaxBatch, c->d.max_seqs * kMaxQueries) * c->geo.hq * c->geo.nsplit)
    return launch(c->partials, nullptr);
  if (capturing(s)) return launch(graph_workspace(c, rows), nullptr);
  PrefillSpaces* spaces = PrefillSpaces::of(c->d.device);
  return spaces ? spaces->with(s, launch) : launch(nullptr, nullptr);
}

// The host has changed seqs: a step that is under way with one of them ends
inline void end_step(bsattn_cache* c, const std::vector<int32_t>& seqs) {
  if (c->step == 0) return;
  for (int s : seqs)
    if (c->in_step[s]) c->step = 0;
}

// Calls that need the exact token counts refuse while device-side appends
// (bsattn_append_step, bsattn_append_packed) may have moved them past the host's view.
inline int check_synced(const bsattn_cache* c) {
  if (c->stale)
    return fail(BSATTN_ERR_INVALID, "device-side lengths may be ahead of the host's view "
                                    "(bsattn_append_step): call bsattn_sync first");
  return BSATTN_OK;
}

}  // namespace bsattn

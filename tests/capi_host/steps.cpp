// steps.cpp -- verification steps on the host: what the calls refuse, when a
// step's map stops naming a cache's state, what reaches the launches (each
// cache's own slots and lengths, workspaces), and that a failed launch leaves
// the step where it was.
#include <algorithm>
#include <climits>
#include <string>

#include "stubs.h"

using namespace bsattn;

namespace stub {
std::vector<TreeBatch> trees;
std::vector<float*> tree_ws;
StepRows last_rows{};
}  // namespace stub

namespace bsattn {
using stub::run;
// the map by its definition
hipError_t launch_step_map(const StepMap& sm, hipStream_t, Timing*) {
  CHECK(sm.n >= 1 && sm.n <= kMaxBatch && sm.caches >= 1 && sm.caches <= kMaxStepCaches);
  if (stub::launches_left == 0) return hipErrorLaunchFailure;
  int64_t at = 0;
  std::vector<int> first(sm.n);
  for (int i = 0; i < sm.n; ++i) {
    const int64_t count = std::max(sm.counts[i], 0);
    bool fits = count <= sm.max_tokens && at + count <= sm.rows;
    for (int c = 0; c < sm.caches; ++c) {
      const StepCache& sc = sm.cache[c];
      fits = fits && sc.meta[sm.ids[i]] + count <= sc.meta[sc.cap_off + sm.ids[i]];
    }
    sm.starts[i] = (int32_t)std::min<int64_t>(at, sm.rows);
    sm.taken[i] = fits ? (int32_t)count : 0;
    for (int c = 0; c < sm.caches; ++c) {
      const StepCache& sc = sm.cache[c];
      const int len = sc.meta[sm.ids[i]];
      sm.ends[c * sm.n + i] = len + sm.taken[i];
      for (int t = 0; t < sm.taken[i]; ++t)
        sm.slots[(size_t)c * sm.rows + at + t] =
            sc.meta[sc.bt_off + (size_t)sm.ids[i] * sc.mbps + (len + t) / sc.tb] * sc.tb + (len + t) % sc.tb;
    }
    at += count;
  }
  return hipSuccess;
}
hipError_t launch_append_packed(const Geometry& g, const StepRows& sr, const void*, int64_t, int64_t, const void*, int64_t,
                                int64_t, hipStream_t, Timing*) {
  stub::last_rows = sr;
  const hipError_t e = run(g, nullptr);
  if (e != hipSuccess) return e;
  for (int i = 0; i < sr.n; ++i) {
    for (int t = 0; t < sr.taken[i]; ++t) CHECK(sr.slots[sr.starts[i] + t] >= 0 && sr.slots[sr.starts[i] + t] < sr.pages * g.tb);
    if (sr.taken[i]) g.meta[sr.ids[i]] = sr.ends[i];
  }
  return e;
}
hipError_t launch_keep(const Geometry& g, const StepRows& sr, const int32_t* kept, int width, const int32_t* n_kept,
                       hipStream_t, Timing*) {
  CHECK(kept && n_kept && width >= 1);
  stub::last_rows = sr;
  const hipError_t e = run(g, nullptr);
  if (e == hipSuccess)
    for (int i = 0; i < sr.n; ++i)
      if (sr.taken[i]) g.meta[sr.ids[i]] = sr.ends[i] - sr.taken[i] + std::min({n_kept[i], width, sr.taken[i]});
  return e;
}
hipError_t launch_tree(const Geometry& g, const TreeBatch& tb, const void*, void*, float* ws, hipEvent_t done, hipStream_t s,
                       Timing*) {
  bool parts = false;
  for (int i = 0; i < tb.n; ++i) parts = parts || tb.part0[i + 1] - tb.part0[i] > 1;
  CHECK(parts == (ws != nullptr));
  stub::trees.push_back(tb);
  stub::tree_ws.push_back(ws);
  const hipError_t e = run(g, nullptr);
  if (e == hipSuccess && done) (void)hipEventRecord(done, s);
  return e;
}
}  // namespace bsattn

alignas(16) static uint16_t x[8];

struct Arrays {
  std::vector<int32_t> starts, taken, requests, positions, slots, ends;
  std::vector<uint64_t> ancestors;
  bsattn_step st{};
  Arrays(int caches, int rows, int max_tokens) {
    starts.resize(65), taken.resize(64), requests.resize(rows), positions.resize(rows), slots.resize(rows * caches);
    ends.resize(64 * caches), ancestors.resize(rows);
    st.n_caches = caches, st.rows = rows, st.max_tokens = max_tokens;
    st.starts = starts.data(), st.taken = taken.data(), st.requests = requests.data(), st.positions = positions.data();
    st.ancestors = ancestors.data(), st.slots = slots.data(), st.ends = ends.data();
  }
};

static void refused(int rc, int code, const char* text) {
  if (rc != code || std::string(bsattn_last_error()).find(text) == std::string::npos) {
    std::printf("%d '%s', expected %d '%s'\n", rc, bsattn_last_error(), code, text);
    std::exit(1);
  }
}

static bsattn_cache* cache(int seqs, int blocks, int tokens, int hq = 8, int hkv = 2) {
  bsattn_desc d = small_desc(seqs, blocks);
  d.num_q_heads = hq;
  d.num_kv_heads = hkv;
  bsattn_cache* c = nullptr;
  CHECK(bsattn_cache_create(&d, &c) == BSATTN_OK);
  if (tokens) CHECK(bsattn_append(c, x, x, nullptr, seqs, tokens, nullptr) == BSATTN_OK);
  return c;
}

static void refusals() {
  bsattn_cache *a = cache(3, 8, 40), *b = cache(3, 8, 40), *other = cache(3, 8, 41);
  CHECK(bsattn_reserve(a, nullptr, 3, 16, nullptr) == BSATTN_OK && bsattn_reserve(b, nullptr, 3, 16, nullptr) == BSATTN_OK);
  Arrays s(2, 24, 8);
  bsattn_cache* both[] = {a, b};
  const int32_t counts[3] = {3, 0, 8}, parents[24] = {-1, 0, 0};
  auto map = [&]() { return bsattn_step_map(both, &s.st, counts, parents, nullptr, 3, nullptr); };
  auto append = [&](bsattn_cache* c) { return bsattn_append_packed(c, &s.st, x, nullptr, x, nullptr, nullptr); };
  auto attend = [&](bsattn_cache* c) { return bsattn_attend_tree(c, &s.st, x, nullptr, 0, nullptr, 1.f, x, nullptr); };
  const int32_t kept[3] = {0, 0, 0}, one[3] = {1, 1, 1};
  auto keep = [&](bsattn_cache* c) { return bsattn_keep(c, &s.st, kept, 1, one, nullptr); };
  // maps
  refused(bsattn_step_map(nullptr, &s.st, counts, nullptr, nullptr, 3, nullptr), BSATTN_ERR_INVALID, "null");
  refused(bsattn_step_map(both, nullptr, counts, nullptr, nullptr, 3, nullptr), BSATTN_ERR_INVALID, "null");
  refused(bsattn_step_map(both, &s.st, nullptr, nullptr, nullptr, 3, nullptr), BSATTN_ERR_INVALID, "null");
  refused(bsattn_step_map(both, &s.st, counts, nullptr, nullptr, 0, nullptr), BSATTN_ERR_INVALID, "n_seqs");
  refused(bsattn_step_map(both, &s.st, counts, nullptr, nullptr, 4, nullptr), BSATTN_ERR_RANGE, "n_seqs");
  refused(bsattn_step_map(both, &s.st, counts, nullptr, nullptr, 65, nullptr), BSATTN_ERR_RANGE, "64 requests");
  const int32_t twice[2] = {1, 1}, far[2] = {0, 3};
  refused(bsattn_step_map(both, &s.st, counts, nullptr, twice, 2, nullptr), BSATTN_ERR_INVALID, "twice");
  refused(bsattn_step_map(both, &s.st, counts, nullptr, far, 2, nullptr), BSATTN_ERR_RANGE, "out of range");
  for (int n : {0, -1, 129}) {
    s.st.n_caches = n;
    refused(map(), BSATTN_ERR_INVALID, "n_caches");
  }
  s.st.n_caches = 2;
  for (int n : {0, -5, (1 << 24) + 1, INT_MAX}) {
    s.st.rows = n;
    refused(map(), BSATTN_ERR_INVALID, "rows");
  }
  s.st.rows = 24;
  for (int n : {0, INT_MIN}) {
    s.st.max_tokens = n;
    refused(map(), BSATTN_ERR_INVALID, "max_tokens");
  }
  s.st.max_tokens = 65;
  refused(map(), BSATTN_ERR_INVALID, "at most 64 nodes");
  s.st.max_tokens = 8;
  for (void** p : {(void**)&s.st.starts, (void**)&s.st.taken, (void**)&s.st.requests, (void**)&s.st.positions,
                   (void**)&s.st.ancestors, (void**)&s.st.slots, (void**)&s.st.ends}) {
    void* was = *p;
    *p = nullptr;
    refused(map(), BSATTN_ERR_INVALID, "null array");
    *p = was;
  }
  bsattn_cache* same[] = {a, a};
  refused(bsattn_step_map(same, &s.st, counts, nullptr, nullptr, 3, nullptr), BSATTN_ERR_INVALID, "twice");
  bsattn_cache* longer[] = {a, other};
  refused(bsattn_step_map(longer, &s.st, counts, nullptr, nullptr, 3, nullptr), BSATTN_ERR_INVALID, "holds 40 tokens");
  bsattn_cache* small = cache(2, 8, 40);
  for (auto list : {std::vector<bsattn_cache*>{a, small}, {small, a}}) {  // (whichever comes first)
    refused(bsattn_step_map(list.data(), &s.st, counts, nullptr, nullptr, 3, nullptr), BSATTN_ERR_RANGE, "max_seqs 2");
    const int32_t ends[2] = {0, 2};
    refused(bsattn_step_map(list.data(), &s.st, counts, nullptr, ends, 2, nullptr), BSATTN_ERR_RANGE, "out of range");
    CHECK(bsattn_step_map(list.data(), &s.st, counts, nullptr, nullptr, 2, nullptr) == BSATTN_OK);
  }
  bsattn_cache_destroy(small);
  s.st.stamp = 0;
  bsattn_cache* none[] = {a, nullptr};
  refused(bsattn_step_map(none, &s.st, counts, nullptr, nullptr, 3, nullptr), BSATTN_ERR_INVALID, "null cache");
  // what comes before a map
  for (int rc : {append(a), attend(a), keep(a)}) refused(rc, BSATTN_ERR_INVALID, "bsattn_step_map");
  refused(bsattn_append_packed(nullptr, &s.st, x, nullptr, x, nullptr, nullptr), BSATTN_ERR_INVALID, "null");
  refused(bsattn_append_packed(a, nullptr, x, nullptr, x, nullptr, nullptr), BSATTN_ERR_INVALID, "null");
  // the order
  CHECK(map() == BSATTN_OK && s.st.n_seqs == 3 && s.st.stamp != 0);
  refused(attend(a), BSATTN_ERR_INVALID, "bsattn_append_packed");
  refused(keep(a), BSATTN_ERR_INVALID, "bsattn_append_packed");
  refused(append(other), BSATTN_ERR_INVALID, "not mapped");
  CHECK(append(a) == BSATTN_OK && stub::last_rows.slots == s.slots.data() && stub::last_rows.ends == s.ends.data());
  refused(attend(b), BSATTN_ERR_INVALID, "bsattn_append_packed");
  CHECK(append(b) == BSATTN_OK && stub::last_rows.slots == s.slots.data() + 24 && stub::last_rows.ends == s.ends.data() + 3);
  CHECK(attend(a) == BSATTN_OK && attend(b) == BSATTN_OK && attend(a) == BSATTN_OK);
  // tensors
  auto tree = [&](const void* q, const int64_t* qs, int window, const float* sinks, void* out) {
    return bsattn_attend_tree(a, &s.st, q, qs, window, sinks, 1.f, out, nullptr);
  };
  const int64_t odd[2] = {1024, 100}, back[2] = {-1024, 128}, wide[2] = {4096, 136};
  refused(tree(nullptr, nullptr, 0, nullptr, x), BSATTN_ERR_INVALID, "null");
  refused(tree(x, nullptr, 0, nullptr, nullptr), BSATTN_ERR_INVALID, "null");
  refused(tree(x + 1, nullptr, 0, nullptr, x), BSATTN_ERR_INVALID, "q must be 16-byte");
  refused(tree(x, nullptr, 0, nullptr, x + 4), BSATTN_ERR_INVALID, "out must be 16-byte");
  refused(tree(x, odd, 0, nullptr, x), BSATTN_ERR_INVALID, "strides");
  refused(tree(x, back, 0, nullptr, x), BSATTN_ERR_INVALID, "strides");
  refused(tree(x, nullptr, -1, nullptr, x), BSATTN_ERR_INVALID, "window");
  refused(tree(x, nullptr, 0, (const float*)((char*)x + 2), x), BSATTN_ERR_INVALID, "sinks");
  CHECK(tree(x, wide, 7, nullptr, x) == BSATTN_OK && stub::trees.back().qr == 4096 && stub::trees.back().qh == 136);
  refused(bsattn_append_packed(a, &s.st, x, odd, x, nullptr, nullptr), BSATTN_ERR_INVALID, "k strides");
  refused(bsattn_append_packed(a, &s.st, x, nullptr, x, back, nullptr), BSATTN_ERR_INVALID, "v strides");
  refused(bsattn_append_packed(a, &s.st, nullptr, nullptr, x, nullptr, nullptr), BSATTN_ERR_INVALID, "null");
  refused(bsattn_append_packed(a, &s.st, x, nullptr, x + 2, nullptr, nullptr), BSATTN_ERR_INVALID, "v must be");
  refused(bsattn_keep(a, &s.st, nullptr, 1, one, nullptr), BSATTN_ERR_INVALID, "null");
  refused(bsattn_keep(a, &s.st, kept, 1, nullptr, nullptr), BSATTN_ERR_INVALID, "null");
  refused(bsattn_keep(a, &s.st, kept, 0, one, nullptr), BSATTN_ERR_INVALID, "width");
  // kept: no attention after it, but another keep, or the append again
  CHECK(keep(a) == BSATTN_OK);
  refused(attend(a), BSATTN_ERR_INVALID, "moved");
  CHECK(attend(b) == BSATTN_OK && keep(a) == BSATTN_OK && append(a) == BSATTN_OK && attend(a) == BSATTN_OK);
  // what ends a step (device-side lengths ahead: host calls need a sync first)
  int32_t len = 0;
  CHECK(bsattn_seq_len(a, 0, &len) != BSATTN_OK || len == 40);
  refused(bsattn_append(a, x, x, nullptr, 3, 1, nullptr), BSATTN_ERR_INVALID, "bsattn_sync");
  CHECK(bsattn_sync(a, nullptr) == BSATTN_OK && bsattn_sync(b, nullptr) == BSATTN_OK);
  check_meta(a, 0, 43), check_meta(a, 1, 40), check_meta(a, 2, 48);
  CHECK(attend(a) == BSATTN_OK);  // (a sync moves nothing)
  CHECK(bsattn_append(a, x, x, nullptr, 3, 1, nullptr) == BSATTN_OK);
  for (int rc : {append(a), attend(a), keep(a)}) refused(rc, BSATTN_ERR_INVALID, "has changed since");
  CHECK(attend(b) == BSATTN_OK && bsattn_trim(b, nullptr, 3, 1, nullptr, nullptr) == BSATTN_OK);
  refused(attend(b), BSATTN_ERR_INVALID, "has changed since");
  refused(map(), BSATTN_ERR_INVALID, "tokens in the step's first cache");
  CHECK(bsattn_trim(a, nullptr, 3, 2, nullptr, nullptr) == BSATTN_OK && map() == BSATTN_OK && append(a) == BSATTN_OK);
  const uint64_t stamp = s.st.stamp;
  CHECK(map() == BSATTN_OK && s.st.stamp != stamp);
  Arrays t(1, 24, 8);
  CHECK(append(a) == BSATTN_OK && bsattn_step_map(both, &t.st, counts, nullptr, nullptr, 3, nullptr) == BSATTN_OK);
  refused(attend(a), BSATTN_ERR_INVALID, "not mapped");  // (mapped for another step)
  CHECK(append(b) == BSATTN_OK && bsattn_sync(a, nullptr) == BSATTN_OK && bsattn_sync(b, nullptr) == BSATTN_OK);
  CHECK(bsattn_reset(b, nullptr, 3, nullptr) == BSATTN_OK);
  refused(attend(b), BSATTN_ERR_INVALID, "has changed since");
  // a struct that is no longer what was mapped
  CHECK(bsattn_reset(a, nullptr, 3, nullptr) == BSATTN_OK && bsattn_append(a, x, x, nullptr, 3, 40, nullptr) == BSATTN_OK &&
        bsattn_reserve(a, nullptr, 3, 16, nullptr) == BSATTN_OK);
  CHECK(bsattn_step_map(both, &t.st, counts, nullptr, nullptr, 3, nullptr) == BSATTN_OK);
  for (int n : {0, 4, 65}) {
    t.st.n_seqs = n;
    refused(bsattn_append_packed(a, &t.st, x, nullptr, x, nullptr, nullptr), BSATTN_ERR_INVALID, "changed");
  }
  t.st.n_seqs = 3;
  t.st.ids[2] = 3;
  refused(bsattn_append_packed(a, &t.st, x, nullptr, x, nullptr, nullptr), BSATTN_ERR_INVALID, "changed");
  // chains of more tokens than a tree has: appended, not attended
  Arrays chunk(1, 24, 80);
  chunk.st.ancestors = nullptr;
  CHECK(bsattn_step_map(both, &chunk.st, counts, nullptr, nullptr, 3, nullptr) == BSATTN_OK);
  CHECK(bsattn_append_packed(a, &chunk.st, x, nullptr, x, nullptr, nullptr) == BSATTN_OK);
  refused(bsattn_attend_tree(a, &chunk.st, x, nullptr, 0, nullptr, 1.f, x, nullptr), BSATTN_ERR_INVALID, "at most 64");
  refused(bsattn_keep(a, &chunk.st, kept, 1, one, nullptr), BSATTN_ERR_INVALID, "at most 64");
  for (bsattn_cache* c : {a, b, other}) bsattn_cache_destroy(c);
}

// a launch that fails changes neither the step nor the caches
static void failures() {
  bsattn_cache* a = cache(2, 8, 40);
  CHECK(bsattn_reserve(a, nullptr, 2, 16, nullptr) == BSATTN_OK);
  Arrays s(1, 16, 8);
  const int32_t counts[2] = {3, 5}, kept[2] = {0, 0}, one[2] = {1, 1};
  auto failed = [&](auto call) {
    stub::launches_left = 0;
    CHECK(call() == BSATTN_ERR_HIP);
    stub::launches_left = -1;
  };
  auto map = [&]() { return bsattn_step_map(&a, &s.st, counts, nullptr, nullptr, 2, nullptr); };
  auto append = [&]() { return bsattn_append_packed(a, &s.st, x, nullptr, x, nullptr, nullptr); };
  auto attend = [&]() { return bsattn_attend_tree(a, &s.st, x, nullptr, 0, nullptr, 1.f, x, nullptr); };
  auto keep = [&]() { return bsattn_keep(a, &s.st, kept, 1, one, nullptr); };
  failed(map);
  refused(append(), BSATTN_ERR_INVALID, "not mapped");
  CHECK(map() == BSATTN_OK);
  failed(append);
  refused(attend(), BSATTN_ERR_INVALID, "bsattn_append_packed");
  CHECK(bsattn_append(a, x, x, nullptr, 2, 1, nullptr) == BSATTN_OK);  // (nothing is ahead of the host)
  CHECK(map() == BSATTN_OK && append() == BSATTN_OK);
  failed(attend);
  CHECK(attend() == BSATTN_OK);
  failed(keep);
  CHECK(attend() == BSATTN_OK && keep() == BSATTN_OK && bsattn_sync(a, nullptr) == BSATTN_OK);
  check_meta(a, 0, 42), check_meta(a, 1, 42);
  bsattn_cache_destroy(a);
}

// what was captured replays unseen: its step is taken at any time, others' rules stay
static void captures() {
  bsattn_cache *a = cache(2, 8, 40), *b = cache(2, 8, 40);
  CHECK(bsattn_reserve(a, nullptr, 2, 32, nullptr) == BSATTN_OK && bsattn_reserve(b, nullptr, 2, 32, nullptr) == BSATTN_OK);
  Arrays s(2, 16, 8), t(1, 16, 8), u(2, 16, 8);
  bsattn_cache *both[] = {a, b}, *swapped[] = {b, a};
  const int32_t counts[2] = {3, 5}, kept[2] = {0, 0}, one[2] = {1, 1};
  auto map = [&](bsattn_cache** l, Arrays& st) { return bsattn_step_map(l, &st.st, counts, nullptr, nullptr, 2, nullptr); };
  auto append = [&](bsattn_cache* c, Arrays& st) { return bsattn_append_packed(c, &st.st, x, nullptr, x, nullptr, nullptr); };
  auto attend = [&](bsattn_cache* c, Arrays& st) {
    return bsattn_attend_tree(c, &st.st, x, nullptr, 0, nullptr, 1.f, x, nullptr);
  };
  auto keep = [&](bsattn_cache* c, Arrays& st) { return bsattn_keep(c, &st.st, kept, 1, one, nullptr); };
  // a captured map: the host's appends do not end its step, nor do other steps' maps
  stub::capture = hipStreamCaptureStatusActive;
  CHECK(map(both, s) == BSATTN_OK && map(swapped, u) == BSATTN_OK);
  stub::capture = hipStreamCaptureStatusNone;
  CHECK(bsattn_append(a, x, x, nullptr, 2, 1, nullptr) == BSATTN_OK && bsattn_append(b, x, x, nullptr, 2, 1, nullptr) == BSATTN_OK);
  CHECK(keep(b, s) == BSATTN_OK && stub::last_rows.slots == s.slots.data() + 16 && attend(b, s) == BSATTN_OK);
  CHECK(append(b, u) == BSATTN_OK && stub::last_rows.slots == u.slots.data() && append(a, s) == BSATTN_OK);
  CHECK(stub::last_rows.slots == s.slots.data());
  CHECK(bsattn_sync(a, nullptr) == BSATTN_OK && bsattn_sync(b, nullptr) == BSATTN_OK);
  CHECK(bsattn_reset(a, nullptr, 2, nullptr) == BSATTN_OK && bsattn_append(a, x, x, nullptr, 2, 40, nullptr) == BSATTN_OK &&
        bsattn_reserve(a, nullptr, 2, 32, nullptr) == BSATTN_OK);
  // captured again: the earlier one's place, not one more
  CHECK(bsattn_reset(b, nullptr, 2, nullptr) == BSATTN_OK && bsattn_append(b, x, x, nullptr, 2, 40, nullptr) == BSATTN_OK &&
        bsattn_reserve(b, nullptr, 2, 32, nullptr) == BSATTN_OK);
  stub::capture = hipStreamCaptureStatusActive;
  const uint64_t before = s.st.stamp;
  CHECK(map(swapped, s) == BSATTN_OK && s.st.stamp != before && append(a, s) == BSATTN_OK);
  CHECK(stub::last_rows.slots == s.slots.data() + 16);
  stub::capture = hipStreamCaptureStatusNone;
  s.st.stamp = before;
  refused(append(a, s), BSATTN_ERR_INVALID, "not mapped");
  CHECK(bsattn_sync(a, nullptr) == BSATTN_OK);
  bsattn_cache_destroy(a);
  a = both[0] = cache(2, 8, 40);
  CHECK(bsattn_reserve(a, nullptr, 2, 32, nullptr) == BSATTN_OK);
  // a step mapped eagerly keeps its rules
  CHECK(map(both, t) == BSATTN_OK);
  refused(attend(a, t), BSATTN_ERR_INVALID, "bsattn_append_packed");
  refused(attend(b, t), BSATTN_ERR_INVALID, "not mapped");
  // until its append is captured
  stub::capture = hipStreamCaptureStatusActive;
  CHECK(append(a, t) == BSATTN_OK && attend(a, t) == BSATTN_OK);
  stub::capture = hipStreamCaptureStatusNone;
  CHECK(bsattn_sync(a, nullptr) == BSATTN_OK && map(both, t) == BSATTN_OK);
  CHECK(keep(a, t) == BSATTN_OK && attend(a, t) == BSATTN_OK && bsattn_sync(a, nullptr) == BSATTN_OK);
  CHECK(bsattn_append(a, x, x, nullptr, 2, 1, nullptr) == BSATTN_OK);
  refused(keep(a, t), BSATTN_ERR_INVALID, "has changed since");
  bsattn_cache_destroy(a);
  bsattn_cache_destroy(b);
}

// the workspace: none for short requests, the cache's own for few partials, the
// streams' for more (with the event that lets the next user in), one of the
// cache's for captures, and one part a request where there is none
static void workspaces() {
  const int L = 64 * 32;
  bsattn_cache* a = cache(4, 80, L, 16, 2);
  CHECK(bsattn_reserve(a, nullptr, 4, 64, nullptr) == BSATTN_OK);
  Arrays s(1, 256, 64);
  const int32_t counts[4] = {64, 64, 64, 64};
  auto attend = [&](int window, void* stream) {
    CHECK(bsattn_attend_tree(a, &s.st, x, nullptr, window, nullptr, 1.f, x, stream) == BSATTN_OK);
  };
  CHECK(bsattn_step_map(&a, &s.st, counts, nullptr, nullptr, 4, nullptr) == BSATTN_OK);
  CHECK(bsattn_append_packed(a, &s.st, x, nullptr, x, nullptr, nullptr) == BSATTN_OK);
  attend(1, nullptr);
  CHECK(stub::tree_ws.back() == nullptr && stub::trees.back().units[0] == (1 + 64 + 62) / 32);
  stub::waits.clear();
  attend(0, (void*)8);
  float* shared = stub::tree_ws.back();
  CHECK(shared && stub::trees.back().part0[4] > 4 && stub::trees.back().units[0] == 66);
  attend(0, (void*)16);  // (another stream waits for the first's use, or has its own)
  CHECK(stub::tree_ws.back() && (stub::tree_ws.back() != shared || !stub::waits.empty()));
  stub::capture = hipStreamCaptureStatusActive;
  attend(0, (void*)8);
  float* graph = stub::tree_ws.back();
  CHECK(graph && graph != shared);
  attend(0, (void*)16);
  CHECK(stub::tree_ws.back() == graph);
  stub::capture = hipStreamCaptureStatusNone;
  bsattn_cache* c = cache(4, 80, L, 16, 2);
  CHECK(bsattn_reserve(c, nullptr, 4, 64, nullptr) == BSATTN_OK);
  std::swap(a, c);
  CHECK(bsattn_step_map(&a, &s.st, counts, nullptr, nullptr, 4, nullptr) == BSATTN_OK);
  CHECK(bsattn_append_packed(a, &s.st, x, nullptr, x, nullptr, nullptr) == BSATTN_OK);
  stub::memory_limit = 0;
  stub::capture = hipStreamCaptureStatusActive;
  attend(0, (void*)8);
  stub::capture = hipStreamCaptureStatusNone;
  stub::memory_limit = SIZE_MAX;
  const TreeBatch& tb = stub::trees.back();
  CHECK(stub::tree_ws.back() == nullptr && tb.part0[4] == 4 && tb.cu >= 66);
  bsattn_cache_destroy(a);
  bsattn_cache_destroy(c);
}

int main() {
  refusals();
  failures();
  captures();
  workspaces();
  std::puts("ok");
  return 0;
}

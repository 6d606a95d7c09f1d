// bsattn_steps.cpp -- the C ABI's verification steps: maps, packed appends,
// tree attention, kept paths.  Argument checking and kernel sequencing.
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <vector>

#include "bsattn_host.h"

using namespace bsattn;

static_assert(BSATTN_STEP_SEQS == kMaxBatch && BSATTN_STEP_CACHES == kMaxStepCaches && BSATTN_TREE_NODES == kMaxNodes,
              "the header's limits are the kernels'");

namespace {

std::atomic<uint64_t> g_steps{0};  // names of the steps' maps
constexpr int kMostRows = 1 << 24;  // (row numbers and the launches' grids stay in 32 bits)

int check_sizes(const bsattn_step& st) {
  if (st.n_caches < 1 || st.n_caches > kMaxStepCaches)
    return fail(BSATTN_ERR_INVALID, "n_caches %d out of range [1, %d]", st.n_caches, kMaxStepCaches);
  if (st.rows < 1 || st.rows > kMostRows)
    return fail(BSATTN_ERR_INVALID, "rows %d out of range [1, %d]", st.rows, kMostRows);
  if (st.max_tokens < 1) return fail(BSATTN_ERR_INVALID, "max_tokens must be >= 1 (got %d)", st.max_tokens);
  if (!st.starts || !st.taken || !st.requests || !st.positions || !st.slots || !st.ends ||
      (!st.ancestors && st.max_tokens <= kMaxNodes))
    return fail(BSATTN_ERR_INVALID, "null array in the step");
  return BSATTN_OK;
}

using CapturedStep = bsattn_cache::CapturedStep;

// what was captured of a step (null: nothing)
CapturedStep* captured_step(bsattn_cache* c, uint64_t stamp) {
  for (CapturedStep& x : c->captured_steps)
    if (x.stamp == stamp) return &x;
  return nullptr;
}

// the stamp that a step's entry goes by before its map (0: it has none): its last
// one, or an earlier one where it was mapped for other caches since.  A step
// without a stamp is new, whatever lay there before.
uint64_t captured_before(const std::vector<CapturedStep>& steps, const bsattn_step* st, uint64_t before) {
  uint64_t own = 0;
  for (const CapturedStep& x : steps) {
    if (before != 0 && x.stamp == before) return before;
    if (before != 0 && x.at == st) own = x.stamp;
  }
  return own;
}

// the last call with the step that the cache is mapped for; one with another step
// (a captured one) changes its sequences under it.  A call that is only recorded
// moves nothing yet
void step_moves(bsattn_cache* c, const bsattn_step* st, bool captured, decltype(bsattn_cache::step_state) to) {
  if (captured || c->step == 0) return;
  if (c->step == st->stamp) {
    c->step_state = to;
    return;
  }
  for (int i = 0; i < st->n_seqs; ++i)
    if (c->in_step[st->ids[i]]) {
      c->step = 0;
      return;
    }
}

// the step's last map is the last that the cache was mapped for, and the
// cache's sequences are as they were then; or it was captured, and holds at its
// replays.  layer: the cache's place among the step's; ordered: whether the host
// knows the last call with it
int check_step(bsattn_cache* c, const bsattn_step* st, void* stream, int& layer, bool& ordered) {
  if (!c || !st) return fail(BSATTN_ERR_INVALID, "null argument");
  if (int rc = check_sizes(*st)) return rc;
  layer = st->stamp != 0 && c->step == st->stamp ? c->step_layer : -1;
  const CapturedStep* was = captured_step(c, st->stamp);
  if (was && was->map) layer = was->layer;
  ordered = !was;
  if (layer < 0)
    return fail(BSATTN_ERR_INVALID, "the cache was not mapped for this step, or has changed since: call bsattn_step_map");
  // (which map ran last, the host's or a replay's, it cannot tell: the arrays are
  // laid out for that one's requests)
  if (was && was->map && was->other && !(was->recorded && capturing((hipStream_t)stream)))
    return fail(BSATTN_ERR_INVALID, "the step's map was captured for other requests: use another step for these");
  if (st->n_seqs < 1 || st->n_seqs > std::min(kMaxBatch, c->d.max_seqs) || layer >= st->n_caches)
    return fail(BSATTN_ERR_INVALID, "the step has changed since its map");
  for (int i = 0; i < st->n_seqs; ++i)
    if (st->ids[i] < 0 || st->ids[i] >= c->d.max_seqs) return fail(BSATTN_ERR_INVALID, "the step has changed since its map");
  return BSATTN_OK;
}

int check_tree(const bsattn_step* st) {
  if (st->max_tokens > kMaxNodes)
    return fail(BSATTN_ERR_INVALID, "a step of up to %d tokens a request: trees have at most %d", st->max_tokens,
                kMaxNodes);
  return BSATTN_OK;
}

StepRows step_rows(const bsattn_cache* c, const bsattn_step& st, int layer) {
  StepRows sr{};
  sr.n = st.n_seqs;
  sr.rows = st.rows;
  sr.max_tokens = st.max_tokens;
  sr.pages = c->num_pages;
  sr.starts = st.starts;
  sr.taken = st.taken;
  sr.slots = st.slots + (size_t)layer * st.rows;
  sr.ends = st.ends + (size_t)layer * st.n_seqs;
  std::copy(st.ids, st.ids + st.n_seqs, sr.ids);
  return sr;
}

// rows [rows, heads, D] and the elements between their rows and heads
int packed_strides(const char* name, const void* x, const int64_t* strides, int heads, int64_t (&out)[2]) {
  if (!x) return fail(BSATTN_ERR_INVALID, "null argument");
  if ((uintptr_t)x % 16) return fail(BSATTN_ERR_INVALID, "%s must be 16-byte aligned", name);
  out[0] = strides ? strides[0] : (int64_t)heads * kHeadDim;
  out[1] = strides ? strides[1] : kHeadDim;
  for (int64_t st : out)
    if (st % 8 || st < 0)
      return fail(BSATTN_ERR_INVALID, "%s strides must be multiples of 8 elements and >= 0 (got %lld)", name,
                  (long long)st);
  return BSATTN_OK;
}

}  // namespace

extern "C" {

int bsattn_step_map(bsattn_cache* const* caches, bsattn_step* st, const int32_t* counts, const int32_t* parents,
                    const int32_t* seq_ids, int32_t n_seqs, void* stream) try {
  if (!caches || !st || !counts) return fail(BSATTN_ERR_INVALID, "null argument");
  if (int rc = check_sizes(*st)) return rc;
  if (n_seqs > kMaxBatch) return fail(BSATTN_ERR_RANGE, "n_seqs %d exceeds the %d requests of a step", n_seqs, kMaxBatch);
  if (parents && st->max_tokens > kMaxNodes)
    return fail(BSATTN_ERR_INVALID, "a tree has at most %d nodes (max_tokens is %d)", kMaxNodes, st->max_tokens);
  std::vector<int32_t> seqs;
  bool synced = true;
  int32_t least = 0;  // sequences of the smallest cache so far
  for (int l = 0; l < st->n_caches; ++l) {
    const bsattn_cache* c = caches[l];
    if (!c) return fail(BSATTN_ERR_INVALID, "null cache");
    if (c->d.device != caches[0]->d.device) return fail(BSATTN_ERR_INVALID, "the step's caches are on different GPUs");
    for (int k = 0; k < l; ++k)
      if (caches[k] == c) return fail(BSATTN_ERR_INVALID, "a cache is listed twice");
    // (what the smallest cache takes the others do)
    if (l == 0 || c->d.max_seqs < least)
      if (int rc = seq_list(c, seq_ids, n_seqs, seqs)) return rc;
    least = l == 0 ? c->d.max_seqs : std::min(least, c->d.max_seqs);
    if (c->num_pages * c->d.block_size > INT32_MAX)
      return fail(BSATTN_ERR_RANGE, "a pool of %lld tokens: slots are 32-bit", (long long)(c->num_pages * c->d.block_size));
    synced = synced && !c->stale;
  }
  if (synced)
    for (int l = 1; l < st->n_caches; ++l)
      for (int s : seqs)
        if (caches[l]->len[s] != caches[0]->len[s])
          return fail(BSATTN_ERR_INVALID, "sequence %d holds %d tokens in the step's first cache and %d in another", s,
                      caches[0]->len[s], caches[l]->len[s]);
  DeviceGuard dg(caches[0]->d.device);
  if (!dg.ok) return fail(BSATTN_ERR_HIP, "hipSetDevice(%d) failed", caches[0]->d.device);
  hipStream_t s = (hipStream_t)stream;
  StepMap sm{};
  sm.n = n_seqs;
  sm.rows = st->rows;
  sm.max_tokens = st->max_tokens;
  sm.caches = st->n_caches;
  sm.counts = counts;
  sm.parents = parents;
  sm.starts = st->starts;
  sm.taken = st->taken;
  sm.requests = st->requests;
  sm.positions = st->positions;
  sm.ancestors = st->ancestors;
  sm.slots = st->slots;
  sm.ends = st->ends;
  std::copy(seqs.begin(), seqs.end(), sm.ids);
  for (int l = 0; l < st->n_caches; ++l) {
    if (int rc = send_unsent(caches[l], s)) return rc;
    const Geometry& g = caches[l]->geo;
    sm.cache[l] = StepCache{g.meta, g.bt_off, g.cap_off, g.mbps, g.tb};
  }
  const bool captured = capturing(s);
  std::shared_ptr<const std::vector<int32_t>> ids;
  if (captured) {  // (nothing below throws)
    ids = std::make_shared<const std::vector<int32_t>>(seqs);
    for (int l = 0; l < st->n_caches; ++l) caches[l]->captured_steps.reserve(caches[l]->captured_steps.size() + 1);
  }
  Timing tm[kProfKinds];
  Timing* prof = prof_slots(caches[0], s, tm);
  const hipError_t e = launch_step_map(sm, s, prof);
  prof_collect(caches[0], prof);
  if (e != hipSuccess) return hip_fail(e, "step map launch");
  const uint64_t before = st->stamp;  // (what was captured under it goes by the new one)
  st->n_seqs = n_seqs;
  std::copy(seqs.begin(), seqs.end(), st->ids);
  st->stamp = ++g_steps;
  for (int l = 0; l < st->n_caches; ++l) {
    if (!captured) {  // (recorded: another step that is under way stays so)
      caches[l]->step = st->stamp;
      caches[l]->step_layer = l;
      caches[l]->step_state = bsattn_cache::kMapped;
      for (int sq : caches[l]->step_seqs) caches[l]->in_step[sq] = 0;
      caches[l]->step_seqs.assign(seqs.begin(), seqs.end());  // (within what create reserved)
      for (int sq : seqs) caches[l]->in_step[sq] = 1;
    }
    // (entries of steps whose memory this one has now have served)
    auto& steps = caches[l]->captured_steps;
    const uint64_t own = captured_before(steps, st, before);
    steps.erase(std::remove_if(steps.begin(), steps.end(),
                               [&](const CapturedStep& x) { return x.at == st && x.stamp != own; }),
                steps.end());
    // (a step that was captured stays so: its graph may replay after any map)
    CapturedStep* was = captured_step(caches[l], own);
    if (!was) {
      if (captured) steps.push_back({st->stamp, l, true, false, ids, st->rows, l, false, false, true, st});
      continue;
    }
    const bool other = was->map && (was->place != l || was->rows != st->rows || *was->ids != seqs);
    if (captured && !was->map) was->ids = ids, was->rows = st->rows, was->place = l;
    was->stamp = st->stamp;
    was->layer = l;
    was->map |= captured;
    was->several |= captured && other;
    was->other = other || was->several;
    was->recorded = captured;
    was->at = st;
  }
  return BSATTN_OK;
} catch (...) {
  return on_exception();
}

int bsattn_append_packed(bsattn_cache* c, const bsattn_step* st, const void* k, const int64_t* k_strides,
                         const void* v, const int64_t* v_strides, void* stream) try {
  int layer;
  bool ordered;
  if (int rc = check_step(c, st, stream, layer, ordered)) return rc;
  int64_t ks[2], vs[2];
  if (int rc = packed_strides("k", k, k_strides, c->geo.hkv, ks)) return rc;
  if (int rc = packed_strides("v", v, v_strides, c->geo.hkv, vs)) return rc;
  DeviceGuard dg(c->d.device);
  if (!dg.ok) return fail(BSATTN_ERR_HIP, "hipSetDevice(%d) failed", c->d.device);
  hipStream_t s = (hipStream_t)stream;
  if (int rc = send_unsent(c, s)) return rc;
  const bool captured = capturing(s);
  if (captured) c->captured_steps.reserve(c->captured_steps.size() + 1);  // (nothing below throws)
  Timing tm[kProfKinds];
  Timing* prof = prof_slots(c, s, tm);
  const hipError_t e = launch_append_packed(c->geo, step_rows(c, *st, layer), k, ks[0], ks[1], v, vs[0], vs[1], s, prof);
  prof_collect(c, prof);
  if (e != hipSuccess) return hip_fail(e, "packed append launch");
  c->stale = true;
  step_moves(c, st, captured, bsattn_cache::kAppended);
  if (captured) {
    if (CapturedStep* was = captured_step(c, st->stamp)) was->append = true;
    else c->captured_steps.push_back({st->stamp, layer, false, true, nullptr, 0, 0, false, false, false, st});
  }
  return BSATTN_OK;
} catch (...) {
  return on_exception();
}

int bsattn_attend_tree(bsattn_cache* c, const bsattn_step* st, const void* q, const int64_t* q_strides, int32_t window,
                       const float* sinks, float scale, void* out, void* stream) try {
  int layer;
  bool ordered;
  if (int rc = check_step(c, st, stream, layer, ordered)) return rc;
  if (int rc = check_tree(st)) return rc;
  if (ordered && c->step_state != bsattn_cache::kAppended)
    return fail(BSATTN_ERR_INVALID, c->step_state == bsattn_cache::kKept
                                        ? "the step's tokens have moved (bsattn_keep)"
                                        : "the step's tokens are not in the cache: call bsattn_append_packed");
  if (!out) return fail(BSATTN_ERR_INVALID, "null argument");
  if ((uintptr_t)out % 16) return fail(BSATTN_ERR_INVALID, "out must be 16-byte aligned");
  if (window < 0) return fail(BSATTN_ERR_INVALID, "window must be >= 0 (got %d)", window);
  if ((uintptr_t)sinks % 4) return fail(BSATTN_ERR_INVALID, "sinks must be 4-byte aligned");
  const Geometry& g = c->geo;
  int64_t qs[2];
  if (int rc = packed_strides("q", q, q_strides, g.hq, qs)) return rc;
  DeviceGuard dg(c->d.device);
  if (!dg.ok) return fail(BSATTN_ERR_HIP, "hipSetDevice(%d) failed", c->d.device);
  hipStream_t s = (hipStream_t)stream;
  if (int rc = send_unsent(c, s)) return rc;
  TreeBatch tb{};
  tb.n = st->n_seqs;
  tb.max_tokens = std::min(st->max_tokens, st->rows);
  tb.window = window;
  tb.sl2 = scale * 1.4426950408889634f;
  tb.sinks = sinks;
  tb.starts = st->starts;
  tb.taken = st->taken;
  tb.ancestors = st->ancestors;
  tb.qr = qs[0];
  tb.qh = qs[1];
  for (int i = 0; i < tb.n; ++i) {
    tb.ids[i] = st->ids[i];
    // (the device-side length is at most what the pages hold; a window can
    // begin and end inside a unit, and the tree's positions follow it)
    int64_t units = (int64_t)c->pages[tb.ids[i]].size() * (g.tb / 32);
    if (window > 0) units = std::min<int64_t>(units, ((int64_t)window + tb.max_tokens + 62) / 32);
    tb.units[i] = (int32_t)units;
  }
  const int64_t rows = tree_plan(g, tb);
  Timing tm[kProfKinds];
  Timing* prof = prof_slots(c, s, tm);
  auto run = [&](float* ws, hipEvent_t done) {
    if (ws) return launch_tree(g, tb, q, out, ws, done, s, prof);
    TreeBatch whole = tb;  // (without a workspace: one part a request)
    whole.cu = INT32_MAX / 32;
    for (int i = 0; i <= whole.n; ++i) whole.part0[i] = i;
    return launch_tree(g, whole, q, out, nullptr, nullptr, s, prof);
  };
  const hipError_t e = rows == 0 ? launch_tree(g, tb, q, out, nullptr, nullptr, s, prof) : with_partials(c, rows, s, run);
  prof_collect(c, prof);
  if (e != hipSuccess) return hip_fail(e, "tree attention launch");
  return BSATTN_OK;
} catch (...) {
  return on_exception();
}

int bsattn_keep(bsattn_cache* c, const bsattn_step* st, const int32_t* kept, int32_t width, const int32_t* n_kept,
                void* stream) try {
  int layer;
  bool ordered;
  if (int rc = check_step(c, st, stream, layer, ordered)) return rc;
  if (int rc = check_tree(st)) return rc;
  if (ordered && c->step_state == bsattn_cache::kMapped)
    return fail(BSATTN_ERR_INVALID, "the step's tokens are not in the cache: call bsattn_append_packed");
  if (!kept || !n_kept) return fail(BSATTN_ERR_INVALID, "null argument");
  if (width < 1) return fail(BSATTN_ERR_INVALID, "width must be >= 1 (got %d)", width);
  DeviceGuard dg(c->d.device);
  if (!dg.ok) return fail(BSATTN_ERR_HIP, "hipSetDevice(%d) failed", c->d.device);
  hipStream_t s = (hipStream_t)stream;
  if (int rc = send_unsent(c, s)) return rc;
  Timing tm[kProfKinds];
  Timing* prof = prof_slots(c, s, tm);
  const hipError_t e = launch_keep(c->geo, step_rows(c, *st, layer), kept, width, n_kept, s, prof);
  prof_collect(c, prof);
  if (e != hipSuccess) return hip_fail(e, "keep launch");
  c->stale = true;
  step_moves(c, st, capturing(s), bsattn_cache::kKept);
  return BSATTN_OK;
} catch (...) {
  return on_exception();
}

}  // extern "C"

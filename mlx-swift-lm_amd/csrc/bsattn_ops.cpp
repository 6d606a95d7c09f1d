// bsattn_ops.cpp -- the C ABI's operators around the cache: dense decode,
// forks, rotary positions and the norms before them.  Argument checking and kernel
// sequencing.
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <vector>

#include "bsattn_host.h"

using namespace bsattn;

namespace {

int check_rope(const bsattn_rope& r) {
  if (!r.theta) return fail(BSATTN_ERR_INVALID, "null rope angles");
  if (r.dims < 2 || r.dims > kHeadDim || r.dims % 2)
    return fail(BSATTN_ERR_INVALID, "rope dims %d unsupported (even, 2 to %d)", r.dims, kHeadDim);
  if (r.interleaved != 0 && r.interleaved != 1)
    return fail(BSATTN_ERR_INVALID, "rope interleaved must be 0 or 1 (got %d)", r.interleaved);
  if (!std::isfinite(r.factor)) return fail(BSATTN_ERR_INVALID, "rope factor must be finite");
  if (r.reserved != 0) return fail(BSATTN_ERR_INVALID, "rope reserved field must be 0");
  if ((uintptr_t)r.theta % 8) return fail(BSATTN_ERR_INVALID, "rope angles must be 8-byte aligned");
  return BSATTN_OK;
}

// tensor i of the batch: x [n, heads, L, D] with its strides, into out
int set_tensor(RotateBatch& rb, int i, const char* name, const void* x, const int64_t* strides, int heads, int L,
               void* out) {
  if (((uintptr_t)x | (uintptr_t)out) % 16)
    return fail(BSATTN_ERR_INVALID, "%s and its output must be 16-byte aligned", name);
  const int64_t dense[3] = {(int64_t)heads * L * kHeadDim, (int64_t)L * kHeadDim, kHeadDim};
  const int64_t* st = strides ? strides : dense;
  for (int j = 0; j < 3; ++j) {
    if (st[j] % 8 || st[j] < 0)
      return fail(BSATTN_ERR_INVALID, "%s strides must be multiples of 8 elements and >= 0 (got %lld)", name,
                  (long long)st[j]);
    if (x == out && st[j] != dense[j])
      return fail(BSATTN_ERR_INVALID, "%s can be rotated in place only when it is dense", name);
  }
  rb.x[i] = (const uint16_t*)x;
  rb.out[i] = (uint16_t*)out;
  rb.heads[i] = heads;
  rb.sb[i] = st[0];
  rb.sh[i] = st[1];
  rb.sl[i] = st[2];
  return BSATTN_OK;
}

int rotate_impl(bsattn_cache* c, const bsattn_rope& rope, RotateBatch& rb, const int32_t* seq_ids, int32_t n_seqs,
                int32_t n_tokens, const int32_t* positions, hipStream_t s) {
  std::vector<int32_t> seqs;
  int rc = seq_list(c, seq_ids, n_seqs, seqs);
  if (rc) return rc;
  DeviceGuard dg(c->d.device);
  if (!dg.ok) return fail(BSATTN_ERR_HIP, "hipSetDevice(%d) failed", c->d.device);
  if (!positions && (rc = send_unsent(c, s))) return rc;
  rb.theta = rope.theta;
  rb.dims = rope.dims;
  rb.interleaved = rope.interleaved;
  rb.m = rope.factor;
  rb.pos = positions;
  rb.L = n_tokens;
  for (int i0 = 0; i0 < n_seqs; i0 += kMaxBatch) {
    const int n = std::min(kMaxBatch, n_seqs - i0);
    rb.b0 = i0;
    for (int i = 0; i < n; ++i) rb.ids[i] = seqs[i0 + i];
    Timing tm[kProfKinds];
    Timing* prof = prof_slots(c, s, tm);
    const hipError_t e = launch_rotate(c->geo, rb, n, s, prof);
    prof_collect(c, prof);
    if (e != hipSuccess) return hip_fail(e, "rotate launch");
  }
  return BSATTN_OK;
}

// a job of the `count` entries order[first] ..
DenseJob& add_job(DenseBatch& db, const int32_t* ids, int first, int count) {
  DenseJob& job = db.job[db.jobs++];
  job = DenseJob{};
  job.first = (int16_t)first;
  job.count = (int16_t)count;
  job.entry = db.order[first];
  job.seq = ids[job.entry];
  job.of = -1;
  return job;
}

// Units of 32 tokens that a shared prefix must have to be read apart from its
// sequences' rest.  32 heads in groups of 4, one cache again and again (and
// caches in turn, past what the Infinity Cache holds), together against apart:
//   bf16  2 branches of 2048 tokens  9.8 and 10.1 us (9.9 and 11.2), of 4096
//         10.1, 13.2 (11.6, 16.1), of 8191 11.6, 12.5 (15.7, 14.6), of 16384
//         18.2, 26.0 (19.8, 28.6); 8 of 1100 10.1, 14.0 (10.1, 17.4)
//   int8  2 of 8191 11.7, 11.3 (12.4, 11.7), of 16384 15.1, 17.2 (16.2, 19.0)
//   int4  2 of 8191 11.5, 11.0 (11.6, 11.2), of 65536 25.4, 31.2 (25.5, 30.8)
// Two branches in groups of 8 lose most: 8191 bf16 tokens 11.1 and 9.6 us
// (11.5, 10.5).  Below this 32 branches of 600 tokens take 16.9 together, 14.1
// apart.
constexpr int kSharedUnits = 32;

// Jobs of a launch of the sequences ids[0, n): the full blocks that entries
// share, read once for as many as fill the columns, and each entry's rest.  A
// block is shared only with all those before it (forks share from the beginning, trims take
// from the end), so the longest common prefix is found by bisection.  Not with
// a window, and not in a capture: its replays may find other sequences.
//
// Shared jobs fill all 16 columns, and then every job of the launch does: for
// affine caches a unit takes about 5 / 4 of the time of one with half of them
// (2 branches of 2000 tokens beside 4 sequences of 60k int4 tokens 74 us with
// the branches together and 60 apart; int8, 40k, 69 and 58; bf16, 16k, 47 both).
void dense_jobs(const bsattn_cache* c, const int32_t* ids, DenseBatch& db, hipStream_t s, bool share = true) {
  const Geometry& g = c->geo;
  const int per_block = g.tb / 32, most = 16 / g.group;
  int16_t of[kMaxBatch];  // an entry's shared job, or -1
  std::fill(of, of + kMaxBatch, (int16_t)-1);
  db.jobs = 0;
  db.again = 0;
  int placed = 0;
  int64_t saved = 0, left = 0;  // units read fewer times, and read
  auto sharing = [&](int i) {
    const auto& pg = c->pages[ids[i]];
    return !pg.empty() && c->sharers[pg[0]] > 0;
  };
  bool any = false;
  for (int i = 0; i < db.n && !any; ++i) any = sharing(i);
  if (share && any && db.window == 0 && most > 1 && !capturing(s)) {
    for (int i = 0; i < db.n; ++i) {
      if (of[i] >= 0 || !sharing(i)) continue;
      const auto& pi = c->pages[ids[i]];
      std::pair<int32_t, int32_t> found[kMaxBatch];  // blocks in common, entry
      int n = 0;
      for (int j = i + 1; j < db.n; ++j) {
        const auto& pj = c->pages[ids[j]];
        if (of[j] >= 0 || pj.empty() || pj[0] != pi[0]) continue;
        int lo = 1, hi = (int)std::min(pi.size(), pj.size());  // the first lo are common, none from hi on
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (pi[mid] == pj[mid]) lo = mid + 1;
          else hi = mid;
        }
        found[n++] = {lo, j};
      }
      std::sort(found, found + n, [](auto a, auto b) { return a.first != b.first ? a.first > b.first : a.second < b.second; });
      // the k that save most: k readings of what the k-th has in common
      int best = 0;
      for (int k = 1; k <= std::min(n, most - 1); ++k)
        if (found[k - 1].first * per_block >= kSharedUnits &&
            (int64_t)k * found[k - 1].first > (best ? (int64_t)best * found[best - 1].first : 0))
          best = k;
      if (!best) continue;
      const int units = found[best - 1].first * per_block;
      db.order[placed] = (int16_t)i;
      for (int k = 0; k < best; ++k) db.order[placed + 1 + k] = (int16_t)found[k].second;
      for (int k = 0; k <= best; ++k) of[db.order[placed + k]] = (int16_t)db.jobs;
      for (int j = 0; j < db.jobs; ++j) db.again |= c->pages[db.job[j].seq][0] == pi[0];
      add_job(db, ids, placed, best + 1).units = units;
      left += units;
      saved += (int64_t)best * units;
      placed += best + 1;
    }
  }
  for (int i = 0; i < db.n; ++i) {
    db.order[placed] = (int16_t)i;
    DenseJob& job = add_job(db, ids, placed++, 1);
    job.of = of[i];
    job.from = of[i] >= 0 ? db.job[of[i]].units : 0;
    // (the pages may hold fewer tokens than fit them; a window can begin and
    // end inside a unit)
    int64_t units = (int64_t)c->pages[ids[i]].size() * per_block - job.from;
    if (db.window > 0) units = std::min<int64_t>(units, ((int64_t)db.window + 62) / 32);
    job.units = (int)units;
    left += units;
  }
  if (saved > 0 && g.kv_bits != 0 && 4 * saved < left) dense_jobs(c, ids, db, s, false);
}

}  // namespace

extern "C" {

int bsattn_decode_dense(bsattn_cache* c, const void* q, const int32_t* seq_ids, int32_t n_seqs, int32_t window,
                        const float* sinks, float scale, void* out, void* stream) try {
  if (!c || !q || !out) return fail(BSATTN_ERR_INVALID, "null argument");
  if (window < 0) return fail(BSATTN_ERR_INVALID, "window must be >= 0 (got %d)", window);
  if (((uintptr_t)q | (uintptr_t)out) % 16) return fail(BSATTN_ERR_INVALID, "q and out must be 16-byte aligned");
  if ((uintptr_t)sinks % 4) return fail(BSATTN_ERR_INVALID, "sinks must be 4-byte aligned");
  std::vector<int32_t> seqs;
  int rc = seq_list(c, seq_ids, n_seqs, seqs);
  if (rc) return rc;
  DeviceGuard dg(c->d.device);
  if (!dg.ok) return fail(BSATTN_ERR_HIP, "hipSetDevice(%d) failed", c->d.device);
  hipStream_t s = (hipStream_t)stream;
  rc = send_unsent(c, s);
  if (rc) return rc;
  const Geometry& g = c->geo;
  for (int i0 = 0; i0 < n_seqs; i0 += kMaxBatch) {
    DenseBatch db{};
    db.n = std::min(kMaxBatch, n_seqs - i0);
    db.window = window;
    db.sl2 = scale * 1.4426950408889634f;
    db.sinks = sinks;
    const int32_t* ids = seqs.data() + i0;
    dense_jobs(c, ids, db, s);
    int64_t rows = 0;
    const int parts = dense_plan(g, db, &rows);
    const uint16_t* qq = (const uint16_t*)q + (size_t)i0 * g.hq * kHeadDim;
    uint16_t* oo = (uint16_t*)out + (size_t)i0 * g.hq * kHeadDim;
    Timing tm[kProfKinds];
    Timing* prof = prof_slots(c, s, tm);
    auto run = [&](float* ws, hipEvent_t done) {
      if (ws) return launch_dense(g, db, parts, qq, oo, ws, done, s, prof);
      DenseBatch whole = db;  // (without a workspace: one part an entry)
      whole.cu = INT32_MAX / 32;
      whole.jobs = 0;
      whole.again = whole.heads_first = 0;
      for (int i = 0; i < db.n; ++i) {
        whole.order[i] = (int16_t)i;
        add_job(whole, ids, i, 1).part0 = i;
      }
      return launch_dense(g, whole, db.n, qq, oo, nullptr, nullptr, s, prof);
    };
    const hipError_t e = rows == 0 ? launch_dense(g, db, parts, qq, oo, nullptr, nullptr, s, prof)
                                   : with_partials(c, rows, s, run);
    prof_collect(c, prof);
    if (e != hipSuccess) return hip_fail(e, "dense decode launch");
  }
  return BSATTN_OK;
} catch (...) {
  return on_exception();
}

int bsattn_fork(bsattn_cache* c, const int32_t* src_ids, const int32_t* dst_ids, int32_t n, const int32_t* n_tokens,
                void* stream) try {
  if (!c || !src_ids || !dst_ids) return fail(BSATTN_ERR_INVALID, "null argument");
  int rc = check_synced(c);
  if (rc) return rc;
  std::vector<int32_t> dst;
  rc = seq_list(c, dst_ids, n, dst);
  if (rc) return rc;
  const int tb = c->d.block_size;
  std::vector<char> is_dst(c->d.max_seqs, 0);
  for (int sq : dst) {
    is_dst[sq] = 1;
    if (c->len[sq] != 0 || !c->pages[sq].empty())
      return fail(BSATTN_ERR_INVALID, "sequence %d is not empty: a fork needs an empty one (bsattn_reset)", sq);
  }
  std::vector<int32_t> tokens(n), tails;  // tails: the pairs with a partial block
  for (int i = 0; i < n; ++i) {
    const int sq = src_ids[i];
    if (sq < 0 || sq >= c->d.max_seqs)
      return fail(BSATTN_ERR_RANGE, "sequence id %d out of range [0, %d)", sq, c->d.max_seqs);
    if (is_dst[sq]) return fail(BSATTN_ERR_INVALID, "sequence %d is forked from and to", sq);
    tokens[i] = n_tokens ? n_tokens[i] : c->len[sq];
    if (tokens[i] < 0 || tokens[i] > c->len[sq])
      return fail(BSATTN_ERR_RANGE, "a fork of %d tokens from sequence %d, which holds %d", tokens[i], sq, c->len[sq]);
    if (tokens[i] % tb) tails.push_back(i);
  }
  if (tails.size() > c->free_pages.size())
    return fail(BSATTN_ERR_NO_PAGES, "page pool exhausted: need %zu pages, %zu free", tails.size(),
                c->free_pages.size());
  DeviceGuard dg(c->d.device);
  if (!dg.ok) return fail(BSATTN_ERR_HIP, "hipSetDevice(%d) failed", c->d.device);
  hipStream_t s = (hipStream_t)stream;
  if (capturing(s)) return fail(BSATTN_ERR_INVALID, "a fork cannot be captured");
  rc = send_unsent(c, s);
  if (rc) return rc;
  // every allocation first: the new rows, and what takes a failed launch back
  std::vector<std::vector<int32_t>> rows(n);
  Patches undo;
  for (int i = 0; i < n; ++i) {
    const auto& pg = c->pages[src_ids[i]];
    rows[i].reserve((tokens[i] + tb - 1) / tb);
    rows[i].assign(pg.begin(), pg.begin() + tokens[i] / tb);
    undo.emplace_back(dst[i], 0);
    undo.emplace_back(c->geo.cap_off + dst[i], 0);
  }
  for (size_t t = 0; t < tails.size(); ++t) rows[tails[t]].push_back(c->free_pages[c->free_pages.size() - 1 - t]);
  for (int i0 = 0; i0 < n; i0 += kMaxBatch) {
    ForkBatch fb{};
    fb.n = std::min(kMaxBatch, n - i0);
    for (int i = 0; i < fb.n; ++i) {
      const bool partial = tokens[i0 + i] % tb != 0;
      fb.src[i] = src_ids[i0 + i];
      fb.dst[i] = dst[i0 + i];
      fb.tokens[i] = tokens[i0 + i];
      fb.tail_from[i] = partial ? c->pages[src_ids[i0 + i]][tokens[i0 + i] / tb] : -1;
      fb.tail_to[i] = partial ? rows[i0 + i].back() : -1;
    }
    Timing tm[kProfKinds];
    Timing* prof = prof_slots(c, s, tm);
    const hipError_t e = launch_fork(c->geo, fb, s, prof);
    prof_collect(c, prof);
    if (e != hipSuccess) {
      c->unsent.swap(undo);
      return hip_fail(e, "fork launch");
    }
  }
  c->free_pages.resize(c->free_pages.size() - tails.size());
  for (int i = 0; i < n; ++i) {
    int32_t* sharers = c->sharers.data();
    for (const int32_t *p = rows[i].data(), *end = p + tokens[i] / tb; p != end; ++p) ++sharers[*p];
    c->pages[dst[i]].swap(rows[i]);
    c->len[dst[i]] = tokens[i];
  }
  // (a step's own tokens may lie in pages that its sequence shares now)
  end_step(c, dst);
  for (int i = 0; i < n; ++i)
    if (c->in_step[src_ids[i]]) c->step = 0;
  return BSATTN_OK;
} catch (...) {
  return on_exception();
}

int bsattn_rotate(bsattn_cache* c, const bsattn_rope* rope, const void* x, const int64_t* strides, int32_t heads,
                  const int32_t* seq_ids, int32_t n_seqs, int32_t n_tokens, const int32_t* positions, void* out,
                  void* stream) try {
  if (!c || !rope || !x || !out) return fail(BSATTN_ERR_INVALID, "null argument");
  if (int rc = check_rope(*rope)) return rc;
  if (n_tokens < 1) return fail(BSATTN_ERR_INVALID, "n_tokens must be >= 1 (got %d)", n_tokens);
  if (heads < 1 || heads > 65535) return fail(BSATTN_ERR_INVALID, "heads %d out of range [1, 65535]", heads);
  RotateBatch rb{};
  if (int rc = set_tensor(rb, 0, "x", x, strides, heads, n_tokens, out)) return rc;
  return rotate_impl(c, *rope, rb, seq_ids, n_seqs, n_tokens, positions, (hipStream_t)stream);
} catch (...) {
  return on_exception();
}

int bsattn_norm_rotate(bsattn_cache* c, const bsattn_rope* rope, const void* q, const int64_t* q_strides,
                       const void* k, const int64_t* k_strides, const void* q_weight, const void* k_weight, float eps,
                       float weight_offset, const int32_t* seq_ids, int32_t n_seqs, int32_t n_tokens,
                       const int32_t* positions, void* q_out, void* k_out, void* stream) try {
  if (!c || !rope || !q || !k || !q_out || !k_out) return fail(BSATTN_ERR_INVALID, "null argument");
  if (!q_weight != !k_weight) return fail(BSATTN_ERR_INVALID, "one norm weight without the other");
  if (int rc = check_rope(*rope)) return rc;
  if (n_tokens < 1) return fail(BSATTN_ERR_INVALID, "n_tokens must be >= 1 (got %d)", n_tokens);
  if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail(BSATTN_ERR_INVALID, "eps must be finite and >= 0");
  if (!std::isfinite(weight_offset)) return fail(BSATTN_ERR_INVALID, "weight_offset must be finite");
  if (((uintptr_t)q_weight | (uintptr_t)k_weight) % 16)
    return fail(BSATTN_ERR_INVALID, "the norm weights must be 16-byte aligned");
  if (q_out == k_out || q_out == k || k_out == q)
    return fail(BSATTN_ERR_INVALID, "queries and keys need outputs of their own");
  RotateBatch rb{};
  if (int rc = set_tensor(rb, 0, "queries", q, q_strides, c->geo.hq, n_tokens, q_out)) return rc;
  if (int rc = set_tensor(rb, 1, "keys", k, k_strides, c->geo.hkv, n_tokens, k_out)) return rc;
  rb.w[0] = (const uint16_t*)q_weight;
  rb.w[1] = (const uint16_t*)k_weight;
  rb.eps = eps;
  rb.woff = weight_offset;
  return rotate_impl(c, *rope, rb, seq_ids, n_seqs, n_tokens, positions, (hipStream_t)stream);
} catch (...) {
  return on_exception();
}

}  // extern "C"

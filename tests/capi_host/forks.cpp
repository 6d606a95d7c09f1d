// forks.cpp -- the page bookkeeping of forks: sequences that append, fork, trim
// and reset in any order hold the tokens they should, whatever they share; no
// page is lost or handed out twice; a call that fails changes nothing.
#include <algorithm>
#include <random>
#include <set>

#include "stubs.h"

namespace stub {
extern bsattn::DenseBatch last_dense;
}

alignas(16) static uint16_t kv[8];
static const int kSeqs = 6, kBlocks = 8, kTb = 32;

// tokens of each sequence as the caller knows them, written into the pages
// beside the library (the stub appends do not)
static std::vector<std::vector<int>> model(kSeqs);
static int next_token = 1;

static std::vector<int32_t> pages_of(bsattn_cache* c, int seq) {
  int32_t n = 0;
  std::vector<int32_t> p(kBlocks);
  CHECK(bsattn_seq_pages(c, seq, p.data(), kBlocks, &n) == BSATTN_OK);
  p.resize(n);
  return p;
}
static int32_t* slot(int page, int at) {
  const bsattn::Geometry& g = stub::last;
  return (int32_t*)(g.pool + (size_t)page * g.hkv * g.slab_bytes) + at;
}

static void check_all(bsattn_cache* c, int pages_in_all) {
  std::set<int32_t> used;
  for (int s = 0; s < kSeqs; ++s) {
    check_meta(c, s, (int)model[s].size());
    const auto p = pages_of(c, s);
    CHECK(p.size() >= (model[s].size() + kTb - 1) / kTb);
    for (size_t t = 0; t < model[s].size(); ++t) CHECK(*slot(p[t / kTb], t % kTb) == model[s][t]);
    used.insert(p.begin(), p.end());
    // what the sequence may write to is its own
    for (size_t b = model[s].size() / kTb; b < p.size(); ++b)
      for (int o = 0; o < kSeqs; ++o)
        if (o != s) {
          const auto q = pages_of(c, o);
          CHECK(std::find(q.begin(), q.end(), p[b]) == q.end());
        }
  }
  bsattn_info info;
  CHECK(bsattn_cache_info(c, &info) == BSATTN_OK);
  CHECK((int64_t)used.size() + info.free_pages == pages_in_all);
}

static void runs(unsigned seed, int num_pages) {
  std::mt19937 rng(seed);
  auto pick = [&](int n) { return (int)(rng() % (unsigned)n); };
  bsattn_desc d = small_desc(kSeqs, kBlocks);
  d.num_pages = num_pages;
  bsattn_cache* c = nullptr;
  CHECK(bsattn_cache_create(&d, &c) == BSATTN_OK);
  for (auto& m : model) m.clear();
  const int32_t all[kSeqs] = {0, 1, 2, 3, 4, 5};
  CHECK(bsattn_reset(c, all, kSeqs, nullptr) == BSATTN_OK);  // (the stub's geometry is this cache's)
  for (int step = 0; step < 400; ++step) {
    // every now and then a launch fails, having written the metadata or not
    const bool fails = pick(10) == 0;
    stub::applies = pick(2);
    const int s = pick(kSeqs), n = 1 + pick(70);
    std::vector<int32_t> ids(all, all + kSeqs);
    std::shuffle(ids.begin(), ids.end(), rng);
    ids.resize(1 + pick(kSeqs));
    stub::launches_left = fails ? pick(2) : -1;
    int rc = 0;
    switch (pick(5)) {
      case 0:
      case 1:
        rc = bsattn_append(c, kv, kv, &s, 1, n, nullptr);
        if (rc == BSATTN_OK) {
          const auto p = pages_of(c, s);
          for (int i = 0; i < n; ++i) {
            const int t = (int)model[s].size();
            model[s].push_back(next_token);
            *slot(p[t / kTb], t % kTb) = next_token++;
          }
        }
        break;
      case 2: {
        std::vector<int32_t> src, dst, len;
        for (int x : ids)
          if (model[x].empty() && x != s) {
            src.push_back(s);
            dst.push_back(x);
            len.push_back(pick(3) == 0 ? pick((int)model[s].size() + 1) : (int)model[s].size());
          }
        if (dst.empty()) break;
        rc = bsattn_fork(c, src.data(), dst.data(), (int)dst.size(), len.data(), nullptr);
        if (rc == BSATTN_OK)
          for (size_t i = 0; i < dst.size(); ++i) model[dst[i]].assign(model[s].begin(), model[s].begin() + len[i]);
        if (rc == BSATTN_ERR_INVALID)  // (an empty sequence may hold pages that an append of it reserved)
          CHECK(std::any_of(dst.begin(), dst.end(), [&](int x) { return !pages_of(c, x).empty(); }));
        break;
      }
      case 3:
        rc = bsattn_trim(c, ids.data(), (int)ids.size(), n, nullptr, nullptr);
        // (a trim whose patches fail has trimmed: they are sent later)
        if (rc == BSATTN_OK || (rc == BSATTN_ERR_HIP && fails)) {
          int32_t len = 0;
          CHECK(bsattn_seq_len(c, ids[0], &len) == BSATTN_OK);
          const bool done = rc == BSATTN_OK || len != (int)model[ids[0]].size() || model[ids[0]].empty();
          if (done)
            for (int x : ids) model[x].resize(model[x].size() - std::min<size_t>(model[x].size(), n));
        }
        break;
      case 4:
        if (pick(3)) break;
        rc = bsattn_reset(c, ids.data(), 1, nullptr);
        int32_t len = 0;
        CHECK(bsattn_seq_len(c, ids[0], &len) == BSATTN_OK);
        if (len == 0) model[ids[0]].clear();
        break;
    }
    CHECK(rc == BSATTN_OK || rc == BSATTN_ERR_HIP || rc == BSATTN_ERR_NO_PAGES || rc == BSATTN_ERR_RANGE ||
          rc == BSATTN_ERR_INVALID);
    CHECK(rc != BSATTN_ERR_HIP || fails);
    stub::launches_left = -1;
    // (what could not be sent goes with the next call)
    CHECK(bsattn_decode(c, kv, all, kSeqs, 1.f, kv, nullptr, nullptr) == BSATTN_OK);
    check_all(c, num_pages);
  }
  bsattn_cache* copy = nullptr;
  CHECK(bsattn_copy(c, &copy, nullptr) == BSATTN_OK);
  CHECK(bsattn_reset(c, all, kSeqs, nullptr) == BSATTN_OK);
  bsattn_info info;
  CHECK(bsattn_cache_info(c, &info) == BSATTN_OK && info.free_pages == num_pages);
  CHECK(bsattn_decode(copy, kv, all, kSeqs, 1.f, kv, nullptr, nullptr) == BSATTN_OK);
  check_all(copy, num_pages);
  CHECK(bsattn_reset(copy, all, kSeqs, nullptr) == BSATTN_OK);
  CHECK(bsattn_cache_info(copy, &info) == BSATTN_OK && info.free_pages == num_pages);
  bsattn_cache_destroy(c);
  bsattn_cache_destroy(copy);
}

// the jobs of a dense decode over forks of forks: what is read for several
// sequences at once is in the same pages for each of them, and worth it
static void shared_jobs(unsigned seed, int hq, int hkv) {
  std::mt19937 rng(seed);
  auto pick = [&](int n) { return (int)(rng() % (unsigned)n); };
  const int seqs = 80, blocks = 64;
  bsattn_desc d = small_desc(seqs, blocks);
  d.num_q_heads = hq;
  d.num_kv_heads = hkv;
  d.block_size = seed % 2 ? 32 : 64;
  bsattn_cache* c = nullptr;
  CHECK(bsattn_cache_create(&d, &c) == BSATTN_OK);
  std::vector<int32_t> len(seqs, 0), ids;
  for (int s = 0; s < seqs; ++s) {
    const int from = s ? pick(s) : 0;
    if (s > 3 && len[from] && pick(5)) {
      len[s] = 1 + pick(len[from]);
      if (pick(2)) len[s] = len[from];
      CHECK(bsattn_fork(c, &from, &s, 1, &len[s], nullptr) == BSATTN_OK);
    }
    const int more = pick(3) ? pick(300) : pick(2) * 1500;
    if (more && len[s] + more <= blocks * d.block_size) {
      CHECK(bsattn_append(c, kv, kv, &s, 1, more, nullptr) == BSATTN_OK);
      len[s] += more;
    }
    ids.push_back(s);
  }
  for (int tries = 0; tries < 20; ++tries) {
    std::shuffle(ids.begin(), ids.end(), rng);
    const int n = 1 + pick(64), window = pick(4) ? 0 : 100;
    stub::splits = 3;
    CHECK(bsattn_decode_dense(c, kv, ids.data(), n, window, nullptr, 1.f, kv, nullptr) == BSATTN_OK);
    const bsattn::DenseBatch& db = stub::last_dense;
    const int per_block = d.block_size / 32, cols = hq / hkv;
    CHECK(db.n == n);
    for (int j = 0; j < db.jobs; ++j) {
      const bsattn::DenseJob& job = db.job[j];
      CHECK(job.count * cols <= 16);
      if (job.count == 1) continue;
      CHECK(window == 0 && job.units >= 16 && job.units % per_block == 0);
      std::vector<int32_t> lead;
      for (int k = 0; k < job.count; ++k) {
        const int seq = ids[db.order[job.first + k]];
        CHECK(len[seq] >= 32 * job.units);
        std::vector<int32_t> p(blocks);
        int32_t held = 0;
        CHECK(bsattn_seq_pages(c, seq, p.data(), blocks, &held) == BSATTN_OK && held * per_block >= job.units);
        p.resize(job.units / per_block);
        if (k == 0) lead = p;
        CHECK(p == lead);
      }
    }
    // (two of the same prompt are found)
    stub::capture = hipStreamCaptureStatusActive;
    CHECK(bsattn_decode_dense(c, kv, ids.data(), n, 0, nullptr, 1.f, kv, nullptr) == BSATTN_OK);
    CHECK(stub::last_dense.jobs == n);
    stub::capture = hipStreamCaptureStatusNone;
  }
  // eight branches of one prompt of 40 blocks
  std::vector<int32_t> all(seqs), src(8, 0), dst;
  for (int s = 0; s < seqs; ++s) all[s] = s;
  CHECK(bsattn_reset(c, all.data(), seqs, nullptr) == BSATTN_OK);
  CHECK(bsattn_append(c, kv, kv, all.data(), 1, 40 * d.block_size + 3, nullptr) == BSATTN_OK);
  for (int i = 0; i < 8; ++i) dst.push_back(10 + i);
  CHECK(bsattn_fork(c, src.data(), dst.data(), 8, nullptr, nullptr) == BSATTN_OK);
  CHECK(bsattn_decode_dense(c, kv, dst.data(), 8, 0, nullptr, 1.f, kv, nullptr) == BSATTN_OK);
  const int per_job = std::min(8, 16 / (hq / hkv));
  CHECK(stub::last_dense.jobs == 8 + (per_job > 1 ? 8 / per_job : 0));
  if (per_job > 1) CHECK(stub::last_dense.job[0].count == per_job && stub::last_dense.job[0].units == 40 * d.block_size / 32);
  // beside a sequence that is many times as long: not worth the other columns
  // of affine caches
  for (int bits : {0, 4}) {
    bsattn_desc b = small_desc(8, 512);
    b.num_q_heads = hq;
    b.num_kv_heads = hkv;
    b.kv_bits = bits;
    b.group_size = 64;
    b.num_pages = 500;
    b.block_size = 64;
    bsattn_cache* q = nullptr;
    CHECK(bsattn_cache_create(&b, &q) == BSATTN_OK);
    const int32_t two[2] = {0, 1}, from[3] = {1, 1, 1}, to[3] = {2, 3, 4}, with[4] = {0, 2, 3, 4};
    CHECK(bsattn_append(q, kv, kv, &two[0], 1, 400 * 64, nullptr) == BSATTN_OK);
    CHECK(bsattn_append(q, kv, kv, &two[1], 1, 20 * 64 + 1, nullptr) == BSATTN_OK);
    CHECK(bsattn_fork(q, from, to, 3, nullptr, nullptr) == BSATTN_OK);
    CHECK(bsattn_decode_dense(q, kv, to, 3, 0, nullptr, 1.f, kv, nullptr) == BSATTN_OK);
    CHECK(stub::last_dense.jobs == (per_job > 1 ? 4 : 3));
    CHECK(bsattn_decode_dense(q, kv, with, 4, 0, nullptr, 1.f, kv, nullptr) == BSATTN_OK);
    CHECK(stub::last_dense.jobs == (per_job > 1 && bits == 0 ? 5 : 4) && stub::last_dense.again == 0);
    bsattn_cache_destroy(q);
  }
  stub::splits = 1;
  bsattn_cache_destroy(c);
}

int main() {
  for (unsigned seed = 0; seed < 6; ++seed) {
    shared_jobs(seed, 8, 2);
    shared_jobs(seed, 4, 4);
    shared_jobs(seed, 16, 2);
    shared_jobs(seed, 16, 1);
  }
  for (unsigned seed = 0; seed < 40; ++seed) runs(seed, 8 + (int)(seed % 4) * 12);
  // captured: a fork, and a trim that would copy a page, are refused
  const bsattn_desc d = small_desc(4, 8);
  bsattn_cache* c = nullptr;
  CHECK(bsattn_cache_create(&d, &c) == BSATTN_OK);
  const int32_t zero = 0, one = 1, two = 2, ids[2] = {0, 1};
  CHECK(bsattn_append(c, kv, kv, &zero, 1, 100, nullptr) == BSATTN_OK);
  CHECK(bsattn_fork(c, &zero, &one, 1, nullptr, nullptr) == BSATTN_OK);
  stub::capture = hipStreamCaptureStatusActive;
  CHECK(bsattn_fork(c, &zero, &two, 1, nullptr, nullptr) == BSATTN_ERR_INVALID);
  CHECK(bsattn_trim(c, &one, 1, 20, nullptr, nullptr) == BSATTN_ERR_INVALID);  // (ends inside block 2)
  CHECK(bsattn_trim(c, &one, 1, 4, nullptr, nullptr) == BSATTN_OK);            // (at its end)
  stub::capture = hipStreamCaptureStatusNone;
  int32_t len = 0;
  CHECK(bsattn_seq_len(c, 1, &len) == BSATTN_OK && len == 96);
  // null and bad arguments
  CHECK(bsattn_fork(nullptr, &zero, &two, 1, nullptr, nullptr) == BSATTN_ERR_INVALID);
  CHECK(bsattn_fork(c, nullptr, &two, 1, nullptr, nullptr) == BSATTN_ERR_INVALID);
  CHECK(bsattn_fork(c, &zero, nullptr, 1, nullptr, nullptr) == BSATTN_ERR_INVALID);
  CHECK(bsattn_fork(c, &zero, &two, 0, nullptr, nullptr) == BSATTN_ERR_INVALID);
  CHECK(bsattn_fork(c, &zero, &one, 1, nullptr, nullptr) == BSATTN_ERR_INVALID);
  CHECK(bsattn_fork(c, &two, &two, 1, nullptr, nullptr) == BSATTN_ERR_INVALID);
  const int32_t far = 101, neg = -1, id9 = 9;
  CHECK(bsattn_fork(c, &zero, &two, 1, &far, nullptr) == BSATTN_ERR_RANGE);
  CHECK(bsattn_fork(c, &zero, &two, 1, &neg, nullptr) == BSATTN_ERR_RANGE);
  CHECK(bsattn_fork(c, &id9, &two, 1, nullptr, nullptr) == BSATTN_ERR_RANGE);
  CHECK(bsattn_fork(c, &zero, &id9, 1, nullptr, nullptr) == BSATTN_ERR_RANGE);
  alignas(16) static uint16_t buf[64];
  alignas(8) static double theta[64];
  uint16_t* odd = buf + 1;
  CHECK(bsattn_decode_dense(nullptr, buf, ids, 2, 0, nullptr, 1.f, buf, nullptr) == BSATTN_ERR_INVALID);
  CHECK(bsattn_decode_dense(c, nullptr, ids, 2, 0, nullptr, 1.f, buf, nullptr) == BSATTN_ERR_INVALID);
  CHECK(bsattn_decode_dense(c, buf, ids, 2, -1, nullptr, 1.f, buf, nullptr) == BSATTN_ERR_INVALID);
  CHECK(bsattn_decode_dense(c, odd, ids, 2, 0, nullptr, 1.f, buf, nullptr) == BSATTN_ERR_INVALID);
  CHECK(bsattn_decode_dense(c, buf, ids, 2, 0, (const float*)((char*)buf + 2), 1.f, buf, nullptr) == BSATTN_ERR_INVALID);
  CHECK(bsattn_decode_dense(c, buf, ids, 0, 0, nullptr, 1.f, buf, nullptr) == BSATTN_ERR_INVALID);
  CHECK(bsattn_decode_dense(c, buf, &id9, 1, 0, nullptr, 1.f, buf, nullptr) == BSATTN_ERR_RANGE);
  bsattn_rope rope{theta, 64, 0, 1.f, 0};
  auto rotate = [&](const bsattn_rope& r, const void* x, const int64_t* st, int heads, int L, void* out) {
    return bsattn_rotate(c, &r, x, st, heads, ids, 2, L, nullptr, out, nullptr);
  };
  CHECK(rotate(rope, buf, nullptr, 1, 1, buf + 32) == BSATTN_OK);
  CHECK(rotate(rope, buf, nullptr, 1, 1, buf) == BSATTN_OK);  // in place
  const int64_t view[3] = {512, 128, 256}, bad[3] = {512, 128, 4}, back[3] = {512, 128, -128};
  CHECK(rotate(rope, buf, view, 1, 1, buf + 32) == BSATTN_OK);
  CHECK(rotate(rope, buf, view, 1, 1, buf) == BSATTN_ERR_INVALID);
  CHECK(rotate(rope, buf, bad, 1, 1, buf + 32) == BSATTN_ERR_INVALID);
  CHECK(rotate(rope, buf, back, 1, 1, buf + 32) == BSATTN_ERR_INVALID);
  CHECK(rotate(rope, odd, nullptr, 1, 1, buf + 32) == BSATTN_ERR_INVALID);
  CHECK(rotate(rope, buf, nullptr, 0, 1, buf + 32) == BSATTN_ERR_INVALID);
  CHECK(rotate(rope, buf, nullptr, 1, 0, buf + 32) == BSATTN_ERR_INVALID);
  for (bsattn_rope r : {bsattn_rope{nullptr, 64, 0, 1.f, 0}, bsattn_rope{theta, 63, 0, 1.f, 0}, bsattn_rope{theta, 0, 0, 1.f, 0},
                        bsattn_rope{theta, 130, 0, 1.f, 0}, bsattn_rope{theta, 64, 2, 1.f, 0},
                        bsattn_rope{theta, 64, 0, 1.f / 0.f, 0}, bsattn_rope{theta, 64, 0, 1.f, 1}})
    CHECK(rotate(r, buf, nullptr, 1, 1, buf + 32) == BSATTN_ERR_INVALID);
  auto norm = [&](const void* qw, const void* kw, float eps, float off, void* q_out, void* k_out) {
    return bsattn_norm_rotate(c, &rope, buf, nullptr, buf + 8, nullptr, qw, kw, eps, off, ids, 2, 1, nullptr, q_out, k_out,
                              nullptr);
  };
  CHECK(norm(buf, buf, 0.f, 0.f, buf + 32, buf + 40) == BSATTN_OK);
  CHECK(norm(nullptr, nullptr, 0.f, 0.f, buf + 32, buf + 40) == BSATTN_OK);
  CHECK(norm(buf, nullptr, 0.f, 0.f, buf + 32, buf + 40) == BSATTN_ERR_INVALID);
  CHECK(norm(odd, buf, 0.f, 0.f, buf + 32, buf + 40) == BSATTN_ERR_INVALID);
  CHECK(norm(buf, buf, -1.f, 0.f, buf + 32, buf + 40) == BSATTN_ERR_INVALID);
  CHECK(norm(buf, buf, 0.f, 1.f / 0.f, buf + 32, buf + 40) == BSATTN_ERR_INVALID);
  CHECK(norm(buf, buf, 0.f, 0.f, buf + 32, buf + 32) == BSATTN_ERR_INVALID);
  CHECK(norm(buf, buf, 0.f, 0.f, buf + 8, buf + 32) == BSATTN_ERR_INVALID);
  // the dense decode's parts go through the cache's own workspace where they
  // fit (64 rows of 8 heads and 2 splits), else through the split prefills':
  // one for a stream, the cache's own in a capture, none when there is no memory
  auto dense = [&](hipStream_t s) { return bsattn_decode_dense(c, buf, ids, 2, 0, nullptr, 1.f, buf, s); };
  stub::prefills.clear();
  CHECK(dense(nullptr) == BSATTN_OK && stub::prefills.back().ws == nullptr);
  stub::splits = 5;
  CHECK(dense(nullptr) == BSATTN_OK);
  const stub::Prefill own = stub::prefills.back();
  CHECK(own.ws && !own.done && own.nsplit == 10 &&
        stub::memory.at(own.ws) == 64u * 8 * 2 * (bsattn::kHeadDim + 2) * sizeof(float));
  stub::splits = 64;
  CHECK(dense(nullptr) == BSATTN_OK && stub::prefills.back().ws == own.ws);
  stub::splits = 65;
  CHECK(dense(nullptr) == BSATTN_OK);
  const stub::Prefill first = stub::prefills.back();
  CHECK(first.ws && first.ws != own.ws && first.done && first.nsplit == 130);
  CHECK(dense(nullptr) == BSATTN_OK && stub::prefills.back().ws == first.ws);
  CHECK(dense((hipStream_t)16) == BSATTN_OK && stub::prefills.back().ws != first.ws);
  stub::capture = hipStreamCaptureStatusActive;
  CHECK(dense(nullptr) == BSATTN_OK);
  const stub::Prefill graph = stub::prefills.back();
  CHECK(graph.ws && !graph.done && stub::memory.at(graph.ws) == 130u * 8 * (bsattn::kHeadDim + 2) * sizeof(float));
  stub::capture = hipStreamCaptureStatusNone;
  CHECK(dense(nullptr) == BSATTN_OK && stub::prefills.back().ws == first.ws);
  stub::launches_left = 0;
  CHECK(dense(nullptr) == BSATTN_ERR_HIP);
  stub::launches_left = -1;
  bsattn_cache_destroy(c);
  CHECK(stub::memory.empty());
  CHECK(bsattn_cache_create(&d, &c) == BSATTN_OK);
  stub::memory_limit = 1000;
  CHECK(dense(nullptr) == BSATTN_OK && stub::prefills.back().ws == nullptr && stub::prefills.back().nsplit == 2);
  stub::memory_limit = SIZE_MAX;
  bsattn_cache_destroy(c);
  std::puts("ok");
  return 0;
}

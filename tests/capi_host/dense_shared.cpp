// dense_shared.cpp -- which blocks a dense decode reads for several sequences
// at once: some whenever two of the call's have 32 units and more in common
// (no window, no capture, room in the columns for two), and then only as many
// as each of the members has in common with the others.
#include <algorithm>
#include <random>

#include "stubs.h"

namespace stub {
extern bsattn::DenseBatch last_dense;
}

alignas(16) static uint16_t kv[8];

static void run(unsigned seed, int hq, int hkv, int tb) {
  std::mt19937 rng(seed);
  auto pick = [&](int n) { return (int)(rng() % (unsigned)n); };
  const int seqs = 40, blocks = 96, per_block = tb / 32, group = hq / hkv;
  bsattn_desc d = small_desc(seqs, blocks);
  d.num_q_heads = hq;
  d.num_kv_heads = hkv;
  d.block_size = tb;
  bsattn_cache* c = nullptr;
  CHECK(bsattn_cache_create(&d, &c) == BSATTN_OK);
  std::vector<std::vector<int32_t>> pages(seqs);
  std::vector<int32_t> len(seqs, 0), ids;
  for (int s = 0; s < seqs; ++s) {
    const int from = s ? pick(s) : 0;
    if (s > 2 && len[from] && pick(4)) {
      // (often near the least that is read together)
      len[s] = std::min(len[from], pick(2) ? 1 + pick(len[from]) : 32 * 30 + pick(160));
      CHECK(bsattn_fork(c, &from, &s, 1, &len[s], nullptr) == BSATTN_OK);
    }
    const int more = pick(3) ? pick(400) : 1100 + pick(900);
    if (more && len[s] + more <= blocks * tb) {
      CHECK(bsattn_append(c, kv, kv, &s, 1, more, nullptr) == BSATTN_OK);
      len[s] += more;
    }
    int32_t held = 0;
    pages[s].resize(blocks);
    CHECK(bsattn_seq_pages(c, s, pages[s].data(), blocks, &held) == BSATTN_OK);
    pages[s].resize(held);
    ids.push_back(s);
  }
  auto common = [&](int a, int b) {  // units
    size_t n = 0;
    while (n < pages[a].size() && n < pages[b].size() && pages[a][n] == pages[b][n]) ++n;
    return (int)n * per_block;
  };
  int found = 0, none = 0;
  for (int tries = 0; tries < 60; ++tries) {
    std::shuffle(ids.begin(), ids.end(), rng);
    const int n = 1 + pick(tries % 2 ? 4 : seqs), window = pick(5) ? 0 : 5000;
    const bool captured = pick(6) == 0;
    stub::capture = captured ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    CHECK(bsattn_decode_dense(c, kv, ids.data(), n, window, nullptr, 1.f, kv, nullptr) == BSATTN_OK);
    stub::capture = hipStreamCaptureStatusNone;
    int most = 0;
    for (int i = 0; i < n; ++i)
      for (int j = 0; j < i; ++j) most = std::max(most, common(ids[i], ids[j]));
    const bool should = most >= 32 && window == 0 && !captured && group < 16;
    const bsattn::DenseBatch& db = stub::last_dense;
    int shared = 0;
    for (int j = 0; j < db.jobs; ++j) {
      const bsattn::DenseJob& job = db.job[j];
      if (job.count == 1) continue;
      ++shared;
      CHECK(job.units >= 32 && job.count * group <= 16);
      for (int a = 0; a < job.count; ++a)
        for (int b = 0; b < a; ++b)
          CHECK(common(ids[db.order[job.first + a]], ids[db.order[job.first + b]]) >= job.units);
    }
    CHECK((shared > 0) == should);
    (should ? found : none) += 1;
  }
  CHECK(none > 5 && (group == 16 || found > 5));
  bsattn_cache_destroy(c);
}

int main() {
  for (unsigned seed = 0; seed < 4; ++seed)
    for (int tb : {32, 64}) {
      run(seed, 8, 2, tb);
      run(seed, 4, 4, tb);
      run(seed, 16, 2, tb);
      run(seed, 16, 1, tb);
    }
  std::puts("ok");
  return 0;
}

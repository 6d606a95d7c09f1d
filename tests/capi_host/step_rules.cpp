// step_rules.cpp -- which calls with a step are taken and which are refused,
// around captures and around host calls for other sequences.  The launches'
// stand-ins and the helpers are steps.cpp's.
#include "../../mlx-swift-lm_amd/csrc/bsattn_host.h"

#define main steps_main
#include "steps.cpp"
#undef main

struct Rig {
  bsattn_cache *a, *b;
  bsattn_cache* both[2];
  const int32_t counts[3] = {3, 5, 2}, kept[3] = {0, 0, 0}, one[3] = {1, 1, 1};
  explicit Rig(int seqs = 2) : a(cache(seqs, 16, 40)), b(cache(seqs, 16, 40)), both{a, b} { reserve(); }
  ~Rig() {
    bsattn_cache_destroy(a);
    bsattn_cache_destroy(b);
  }
  void sync() {
    for (bsattn_cache* c : both) CHECK(bsattn_sync(c, nullptr) == BSATTN_OK);
  }
  void reserve() {
    for (bsattn_cache* c : both) CHECK(bsattn_reserve(c, nullptr, c->d.max_seqs, 32, nullptr) == BSATTN_OK);
  }
  // a host call for every sequence
  void more() {
    sync();
    for (bsattn_cache* c : both) CHECK(bsattn_append(c, x, x, nullptr, c->d.max_seqs, 1, nullptr) == BSATTN_OK);
    reserve();
  }
  int map(Arrays& s, int n = 2, const int32_t* ids = nullptr, bool swap = false) {
    bsattn_cache* swapped[2] = {b, a};
    return bsattn_step_map(swap ? swapped : both, &s.st, counts, nullptr, ids, n, nullptr);
  }
  int append(bsattn_cache* c, Arrays& s) { return bsattn_append_packed(c, &s.st, x, nullptr, x, nullptr, nullptr); }
  int attend(bsattn_cache* c, Arrays& s) {
    return bsattn_attend_tree(c, &s.st, x, nullptr, 0, nullptr, 1.f, x, nullptr);
  }
  int keep(bsattn_cache* c, Arrays& s) { return bsattn_keep(c, &s.st, kept, 1, one, nullptr); }
  template <typename F>
  void captured(F calls) {
    stub::capture = hipStreamCaptureStatusActive;
    calls();
    stub::capture = hipStreamCaptureStatusNone;
  }
};

// an eager map of a step whose map was captured: the graph may still replay
static void eager_map_of_a_captured_step() {
  Rig r;
  Arrays s(2, 16, 8);
  r.captured([&] { CHECK(r.map(s) == BSATTN_OK); });
  CHECK(r.map(s) == BSATTN_OK);
  r.more();
  // (here the graph replays)
  for (bsattn_cache* c : r.both) CHECK(r.append(c, s) == BSATTN_OK && r.attend(c, s) == BSATTN_OK && r.keep(c, s) == BSATTN_OK);
  for (int turn = 0; turn < 5; ++turn) {
    r.captured([&] { CHECK(r.map(s) == BSATTN_OK); });
    CHECK(r.map(s) == BSATTN_OK);
    r.more();
    CHECK(r.keep(r.b, s) == BSATTN_OK && stub::last_rows.slots == s.slots.data() + 16);
  }
}

// a captured append takes the order checks from its own step only
static void captured_append_of_another_step() {
  Rig r;
  Arrays s(2, 16, 8), t(2, 16, 8);
  CHECK(r.map(s) == BSATTN_OK);
  r.captured([&] { CHECK(r.append(r.a, s) == BSATTN_OK); });
  CHECK(r.keep(r.a, s) == BSATTN_OK && r.append(r.b, s) == BSATTN_OK && r.keep(r.b, s) == BSATTN_OK);
  for (int turn = 0; turn < 2; ++turn) {
    CHECK(r.map(t) == BSATTN_OK);
    for (bsattn_cache* c : r.both) {
      refused(r.attend(c, t), BSATTN_ERR_INVALID, "bsattn_append_packed");
      refused(r.keep(c, t), BSATTN_ERR_INVALID, "bsattn_append_packed");
      CHECK(r.append(c, t) == BSATTN_OK && r.attend(c, t) == BSATTN_OK && r.keep(c, t) == BSATTN_OK);
      refused(r.attend(c, t), BSATTN_ERR_INVALID, "moved");
    }
    // its own: taken as it comes after a map, in that cache
    CHECK(r.map(s) == BSATTN_OK && r.attend(r.a, s) == BSATTN_OK && r.keep(r.a, s) == BSATTN_OK && r.attend(r.a, s) == BSATTN_OK);
    refused(r.attend(r.b, s), BSATTN_ERR_INVALID, "bsattn_append_packed");
    CHECK(r.append(r.b, s) == BSATTN_OK && r.keep(r.b, s) == BSATTN_OK);
    r.more();
    refused(r.keep(r.a, s), BSATTN_ERR_INVALID, "has changed since");
  }
}

// what is recorded moves nothing: a step that is under way stays where it is
static void captures_beside_a_step() {
  Rig r;
  Arrays s(2, 16, 8), t(2, 16, 8);
  CHECK(r.map(t) == BSATTN_OK && r.append(r.a, t) == BSATTN_OK);
  r.captured([&] {
    CHECK(r.map(s) == BSATTN_OK && r.append(r.a, s) == BSATTN_OK && r.attend(r.a, s) == BSATTN_OK && r.keep(r.a, s) == BSATTN_OK);
  });
  CHECK(r.attend(r.a, t) == BSATTN_OK);
  // a captured keep
  r.captured([&] { CHECK(r.keep(r.a, t) == BSATTN_OK); });
  CHECK(r.attend(r.a, t) == BSATTN_OK && r.keep(r.a, t) == BSATTN_OK);
  refused(r.attend(r.a, t), BSATTN_ERR_INVALID, "moved");
}

// a captured map and eager ones for other requests: the arrays may be either's
static void other_requests() {
  Rig r(3);
  const char* text = "captured for other requests";
  const int32_t back[2] = {1, 0}, far[2] = {0, 2};
  Arrays s(2, 16, 8);
  r.captured([&] { CHECK(r.map(s) == BSATTN_OK); });
  CHECK(r.append(r.a, s) == BSATTN_OK && r.append(r.b, s) == BSATTN_OK && r.keep(r.a, s) == BSATTN_OK);
  for (int how = 0; how < 5; ++how) {
    if (how == 0) CHECK(r.map(s, 1) == BSATTN_OK);
    if (how == 1) CHECK(r.map(s, 3) == BSATTN_OK);
    if (how == 2) CHECK(r.map(s, 2, back) == BSATTN_OK);
    if (how == 3) CHECK(r.map(s, 2, far) == BSATTN_OK);
    if (how == 4) CHECK(r.map(s, 2, nullptr, true) == BSATTN_OK);
    // (here the graph may have replayed)
    for (bsattn_cache* c : r.both)
      for (int rc : {r.append(c, s), r.attend(c, s), r.keep(c, s)}) refused(rc, BSATTN_ERR_INVALID, text);
    // nor into a graph of its own, where the map is not
    r.captured([&] { refused(r.append(r.a, s), BSATTN_ERR_INVALID, text); });
    // mapped as it was captured
    CHECK(r.map(s) == BSATTN_OK && r.append(r.b, s) == BSATTN_OK && r.keep(r.a, s) == BSATTN_OK);
  }
  // captured for two lists: within each capture they are known
  r.captured([&] {
    CHECK(r.map(s, 2, far) == BSATTN_OK && r.append(r.a, s) == BSATTN_OK && r.attend(r.a, s) == BSATTN_OK && r.keep(r.a, s) == BSATTN_OK);
  });
  for (const int32_t* ids : {(const int32_t*)nullptr, far}) {
    refused(r.keep(r.a, s), BSATTN_ERR_INVALID, text);
    CHECK(r.map(s, 2, ids) == BSATTN_OK);
  }
  refused(r.keep(r.a, s), BSATTN_ERR_INVALID, text);
  // another step for these
  Arrays t(2, 16, 8);
  CHECK(r.map(t, 2, far) == BSATTN_OK && r.append(r.a, t) == BSATTN_OK && r.attend(r.a, t) == BSATTN_OK && r.keep(r.a, t) == BSATTN_OK);
}

// host calls for other sequences leave a step under way; those for one of its own end it
static void other_sequences() {
  Rig r(6);
  bsattn_cache* c = r.a;
  const int32_t ids[2] = {4, 1}, free_one = 2, other = 0, own = 4, second = 1;
  CHECK(bsattn_reset(c, &free_one, 1, nullptr) == BSATTN_OK);
  Arrays s(1, 16, 8);
  auto begin = [&] {
    CHECK(bsattn_sync(c, nullptr) == BSATTN_OK && r.map(s, 2, ids) == BSATTN_OK && r.append(c, s) == BSATTN_OK &&
          r.attend(c, s) == BSATTN_OK && bsattn_sync(c, nullptr) == BSATTN_OK);
  };
  int32_t got = 0;
  auto calls = [&](int how, const int32_t* id) {
    switch (how) {
      case 0: return bsattn_append(c, x, x, id, 1, 3, nullptr);
      case 1: return bsattn_append_decode(c, x, x, x, id, 1, 1.f, x, nullptr, nullptr);
      case 2: return bsattn_append_step(c, x, x, id, 1, nullptr);
      case 3: return bsattn_trim(c, id, 1, 1, &got, nullptr);
      default: return bsattn_reset(c, id, 1, nullptr);
    }
  };
  for (int how = 0; how < 5; ++how) {
    begin();
    CHECK(calls(how, &other) == BSATTN_OK);
    CHECK(r.attend(c, s) == BSATTN_OK && r.keep(c, s) == BSATTN_OK);
    for (const int32_t* id : {&own, &second}) {
      begin();
      CHECK(calls(how, id) == BSATTN_OK);
      for (int rc : {r.append(c, s), r.attend(c, s), r.keep(c, s)}) refused(rc, BSATTN_ERR_INVALID, "has changed since");
      CHECK(bsattn_sync(c, nullptr) == BSATTN_OK);
      if (how == 4)
        CHECK(bsattn_append(c, x, x, id, 1, 40, nullptr) == BSATTN_OK && bsattn_reserve(c, id, 1, 32, nullptr) == BSATTN_OK);
    }
    CHECK(bsattn_reset(c, &other, 1, nullptr) == BSATTN_OK && bsattn_append(c, x, x, &other, 1, 40, nullptr) == BSATTN_OK);
    CHECK(bsattn_reserve(c, nullptr, 6, 32, nullptr) == BSATTN_OK && bsattn_reset(c, &free_one, 1, nullptr) == BSATTN_OK);
  }
  // a fork between others, from the step's, to the step's
  begin();
  CHECK(bsattn_fork(c, &other, &free_one, 1, nullptr, nullptr) == BSATTN_OK && r.keep(c, s) == BSATTN_OK);
  begin();
  CHECK(bsattn_reset(c, &free_one, 1, nullptr) == BSATTN_OK && r.attend(c, s) == BSATTN_OK);
  CHECK(bsattn_fork(c, &own, &free_one, 1, nullptr, nullptr) == BSATTN_OK);
  refused(r.keep(c, s), BSATTN_ERR_INVALID, "has changed since");
  CHECK(bsattn_reset(c, &own, 1, nullptr) == BSATTN_OK);
  begin();
  CHECK(s.taken[0] == 0);  // (it holds no pages)
  CHECK(bsattn_fork(c, &other, &own, 1, nullptr, nullptr) == BSATTN_OK);
  refused(r.keep(c, s), BSATTN_ERR_INVALID, "has changed since");
  // the marks are the last map's
  const int32_t two[2] = {0, 3};
  CHECK(r.map(s, 2, two) == BSATTN_OK && r.append(c, s) == BSATTN_OK && bsattn_sync(c, nullptr) == BSATTN_OK);
  CHECK(bsattn_trim(c, ids, 2, 1, nullptr, nullptr) == BSATTN_OK && r.keep(c, s) == BSATTN_OK && bsattn_sync(c, nullptr) == BSATTN_OK);
  CHECK(bsattn_trim(c, two + 1, 1, 1, nullptr, nullptr) == BSATTN_OK);
  refused(r.keep(c, s), BSATTN_ERR_INVALID, "has changed since");
}

// steps that come and go, each captured: what is kept of them does not grow with their number
static void many_captured_steps() {
  Rig r;
  Arrays s(2, 16, 8), t(2, 16, 8);
  r.captured([&] { CHECK(r.map(t) == BSATTN_OK && r.append(r.a, t) == BSATTN_OK); });
  const bsattn_step fresh = Arrays(2, 16, 8).st;
  for (int turn = 0; turn < 100; ++turn) {
    const bsattn_step was = s.st;
    s.st = fresh;  // (a new struct in the old one's memory, with the old arrays)
    s.st.starts = was.starts, s.st.taken = was.taken, s.st.requests = was.requests, s.st.positions = was.positions;
    s.st.ancestors = was.ancestors, s.st.slots = was.slots, s.st.ends = was.ends;
    if (turn % 3 == 0) CHECK(r.map(s) == BSATTN_OK);
    r.captured([&] { CHECK((turn % 3 == 0 || r.map(s) == BSATTN_OK) && r.append(r.a, s) == BSATTN_OK); });
    CHECK(r.a->captured_steps.size() <= 2 && r.b->captured_steps.size() <= 2);
  }
  // the others are as they were
  CHECK(r.attend(r.a, t) == BSATTN_OK && r.append(r.b, t) == BSATTN_OK && r.keep(r.a, s) == BSATTN_OK);
  // one that was mapped for other caches in between has not changed
  Arrays u(2, 16, 8);
  r.captured([&] { CHECK(r.map(u) == BSATTN_OK); });
  bsattn_cache* alone = cache(2, 16, 40);
  u.st.n_caches = 1;
  CHECK(bsattn_step_map(&alone, &u.st, r.counts, nullptr, nullptr, 2, nullptr) == BSATTN_OK);
  refused(r.keep(r.a, u), BSATTN_ERR_INVALID, "not mapped");
  u.st.n_caches = 2;
  CHECK(r.map(u) == BSATTN_OK && r.keep(r.a, u) == BSATTN_OK && r.map(u, 1) == BSATTN_OK);
  refused(r.keep(r.a, u), BSATTN_ERR_INVALID, "captured for other requests");
  bsattn_cache_destroy(alone);
}

// what runs of a captured step changes its sequences: another step of theirs ends, one of others does not
static void captured_step_beside_a_step() {
  const int32_t mine[2] = {0, 1}, theirs[2] = {2, 1}, apart[2] = {2, 3};
  for (bool keeps : {false, true})
    for (const int32_t* ids : {theirs, apart}) {
      Rig r(4);
      Arrays s(2, 16, 8), t(2, 16, 8);
      CHECK(r.map(s, 2, ids) == BSATTN_OK);  // (so that its arrays hold something)
      r.captured([&] { CHECK(r.map(s, 2, ids) == BSATTN_OK); });
      CHECK(r.map(t, 2, mine) == BSATTN_OK);
      for (bsattn_cache* c : r.both) {
        CHECK(r.append(c, t) == BSATTN_OK && r.attend(c, t) == BSATTN_OK && r.attend(c, s) == BSATTN_OK);
        CHECK(r.attend(c, t) == BSATTN_OK);  // (attention changes nothing)
        CHECK((keeps ? r.keep(c, s) : r.append(c, s)) == BSATTN_OK);
        if (ids == apart) CHECK(r.attend(c, t) == BSATTN_OK && r.keep(c, t) == BSATTN_OK);
        else
          for (int rc : {r.append(c, t), r.attend(c, t), r.keep(c, t)}) refused(rc, BSATTN_ERR_INVALID, "has changed since");
      }
    }
}

int main() {
  eager_map_of_a_captured_step();
  captured_append_of_another_step();
  captures_beside_a_step();
  other_requests();
  other_sequences();
  many_captured_steps();
  captured_step_beside_a_step();
  std::puts("ok");
  return 0;
}

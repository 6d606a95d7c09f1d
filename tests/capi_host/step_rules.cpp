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
  // nor do calls with another step that was captured
  CHECK(r.append(r.b, s) == BSATTN_OK);
  refused(r.attend(r.b, t), BSATTN_ERR_INVALID, "bsattn_append_packed");
  CHECK(r.append(r.b, t) == BSATTN_OK && r.attend(r.b, t) == BSATTN_OK);
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

int main() {
  eager_map_of_a_captured_step();
  captured_append_of_another_step();
  captures_beside_a_step();
  other_requests();
  std::puts("ok");
  return 0;
}

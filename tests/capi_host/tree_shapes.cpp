// tree_shapes.cpp -- how tree attentions are launched: reads calls from stdin
// (query and kv heads, tokens per block, the longest request's new tokens, the
// window or 0, the requests' number, then the tokens that each holds, in pages that take
// 64 more), makes them over the stand-ins of steps.cpp and prints each launch's
// column tiles and whether its waves hold one.
#define main steps_main
#include "steps.cpp"
#undef main

int main() {
  int hq, hkv, tb, most, window, n;
  while (std::scanf("%d %d %d %d %d %d", &hq, &hkv, &tb, &most, &window, &n) == 6) {
    bsattn_desc d = small_desc(n, 1024);
    d.num_q_heads = hq;
    d.num_kv_heads = hkv;
    d.block_size = tb;
    bsattn_cache* c = nullptr;
    CHECK(bsattn_cache_create(&d, &c) == BSATTN_OK);
    for (int32_t i = 0; i < n; ++i) {
      int tokens = 0;
      CHECK(std::scanf("%d", &tokens) == 1 && bsattn_append(c, x, x, &i, 1, tokens, nullptr) == BSATTN_OK);
      CHECK(bsattn_reserve(c, &i, 1, 64, nullptr) == BSATTN_OK);
    }
    Arrays s(1, 64 * n, most);
    const std::vector<int32_t> counts(n, most);
    CHECK(bsattn_step_map(&c, &s.st, counts.data(), nullptr, nullptr, n, nullptr) == BSATTN_OK);
    CHECK(bsattn_append_packed(c, &s.st, x, nullptr, x, nullptr, nullptr) == BSATTN_OK);
    CHECK(bsattn_attend_tree(c, &s.st, x, nullptr, window, nullptr, 1.f, x, nullptr) == BSATTN_OK);
    std::printf("%d %d\n", stub::trees.back().tiles, (int)stub::trees.back().narrow);
    bsattn_cache_destroy(c);
  }
  return 0;
}

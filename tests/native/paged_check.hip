// Host-side check of the rules that deal a batch's cached tokens to workgroups (plz_paged.h), built
// with asserts on and run on the CPU by tests/test_paged.py: the walk of the attention kernel and of
// the kernel that joins its parts, restated, over many batches.
#undef NDEBUG
#include <cassert>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <vector>

#include "plz_paged.h"

using namespace plz::paged;
static long checks = 0;

struct Part {
  int b;
  bool ends;
};

static void check_batch(const std::vector<int>& lens, int cap, int parts, int waves) {
  int total = 0;
  for (int n : lens) total += tiles_of(n, cap);
  if (total == 0) return;
  const Deal d = deal(total, parts * waves);
  assert(d.runs >= 1 && d.runs <= parts * waves);
  assert(run_begin(d, 0) == 0 && run_begin(d, d.runs) == total);
  std::vector<int> seen(total, 0), tiles_done(lens.size(), 0);
  std::map<std::pair<int, int>, int> part;  // (workgroup, place) -> request
  std::vector<std::pair<int, int>> open(parts, {-1, 0});
  for (int w = 0; w < parts; ++w) {
    std::vector<std::map<int, Part>> left(waves);  // a wave's parts by place
    for (int wave = 0; wave < waves; ++wave) {
      const int i = w * waves + wave;
      if (i >= d.runs) continue;
      const int r0 = run_begin(d, i), r1 = run_begin(d, i + 1);
      assert(r0 < r1);
      for (int p = r0; p < r1; ++p) assert(run_of(d, p) == i);
      int b = 0, first = 0;  // the request that holds tile r0
      while (first + tiles_of(lens[b], cap) <= r0) first += tiles_of(lens[b++], cap);
      for (;; ++b) {
        assert(b < (int)lens.size());
        const int n = tiles_of(lens[b], cap);
        if (n == 0) continue;
        const int t0 = r0 - first > 0 ? r0 - first : 0, t1 = r1 - first < n ? r1 - first : n;
        assert(t0 < t1);
        for (int t = t0; t < t1; ++t) {
          assert(t * TILE < lens[b]);  // a tile's first token exists
          ++seen[first + t];
        }
        if (t0 > 0 || t1 < n)
          assert(left[wave].emplace(place_of(t0 > 0), Part{b, t1 == n}).second);
        else
          tiles_done[b] += n;
        first += n;
        if (first >= r1) break;
      }
    }
    // the workgroup's join, as the kernel does it
    for (int start = -1; start < waves; ++start) {
      if (!left[start < 0 ? 0 : start].count(start < 0 ? 0 : 1)) continue;
      const int b = left[start < 0 ? 0 : start][start < 0 ? 0 : 1].b;
      bool ended = start < 0 && left[0][0].ends;
      for (int m = (start < 0 ? 0 : start) + 1; !ended && m < waves && left[m].count(0); ++m) {
        assert(left[m][0].b == b);
        ended = left[m][0].ends;
      }
      if (start >= 0 && ended) {
        tiles_done[b] += tiles_of(lens[b], cap);
        continue;
      }
      assert(part.emplace(std::make_pair(w, start < 0 ? 0 : 1), b).second);
      if (start >= 0) {
        int before = 0;
        for (int k = 0; k < b; ++k) before += tiles_of(lens[k], cap);
        assert(open[w].first == -1);
        open[w] = {b, run_of(d, before + tiles_of(lens[b], cap) - 1) / waves};
      }
    }
  }
  for (int s : seen) assert(s == 1);
  size_t joined = 0;
  for (int w = 0; w < parts; ++w) {
    if (open[w].first < 0) continue;
    assert(open[w].second > w);
    for (int i = w; i <= open[w].second; ++i, ++joined)
      assert(part.at({i, i == w ? 1 : 0}) == open[w].first);
    tiles_done[open[w].first] += tiles_of(lens[open[w].first], cap);
  }
  assert(joined == part.size());
  for (size_t b = 0; b < lens.size(); ++b) assert(tiles_done[b] == tiles_of(lens[b], cap));
  ++checks;
}

int main() {
  srand(7);
  for (int cap : {16, 64, 4096, 1 << 20})
    for (int parts : {1, 2, 12, 96, 768})
      for (int waves : {1, 4, 8})
        for (int it = 0; it < 60; ++it) {
          std::vector<int> lens(1 + rand() % (it % 3 ? 9 : 400));
          for (int& n : lens) {
            const int k = rand() % 6;
            n = k == 0 ? 0 : k == 1 ? -rand() % 9 : k == 2 ? cap + rand() % 3 : k == 3 ? rand() % 40
                : rand() % (cap < 9000 ? cap + 1 : 9000);
          }
          check_batch(lens, cap, parts, waves);
        }
  check_batch({1 << 24}, 1 << 24, 768, 4);  // one long request
  for (int p : {0, 1, (1 << 30) - 1}) {     // as many tiles as the entry point takes
    const Deal d = deal(1 << 30, 4096);
    const int w = run_of(d, p);
    assert(run_begin(d, w) <= p && p < run_begin(d, w + 1));
    ++checks;
  }
  printf("paged runs: %ld checks passed\n", checks);
  return 0;
}

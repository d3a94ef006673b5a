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

static void check_batch(const std::vector<int>& lens, int cap, int parts, int waves) {
  int total = 0;
  for (int n : lens) total += tiles_of(n, cap);
  if (total == 0) return;
  const int runs = run_count(total, parts, waves);
  assert(runs >= 1 && runs <= parts && (runs == 1 || total / runs >= 1));
  assert(run_begin(total, runs, 0) == 0 && run_begin(total, runs, runs) == total);
  std::vector<int> seen(total, 0);
  std::map<std::pair<int, int>, int> slot;  // (run, slot) -> request
  for (int w = 0; w < runs; ++w) {
    const int r0 = run_begin(total, runs, w), r1 = run_begin(total, runs, w + 1);
    assert(r0 < r1);
    for (int p = r0; p < r1; ++p) assert(run_of(total, runs, p) == w);
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
      if (!(t0 == 0 && t1 == n)) assert(slot.emplace(std::make_pair(w, (int)(t0 == 0)), b).second);
      first += n;
      if (first >= r1) break;
    }
  }
  for (int s : seen) assert(s == 1);
  int first = 0;
  size_t joined = 0;
  for (size_t b = 0; b < lens.size(); ++b) {
    const int n = tiles_of(lens[b], cap);
    if (n == 0) continue;
    const int w0 = run_of(total, runs, first), w1 = run_of(total, runs, first + n - 1);
    if (w0 != w1)
      for (int w = w0; w <= w1; ++w) {
        assert(slot.at({w, (int)(w == w0)}) == (int)b);
        ++joined;
      }
    first += n;
  }
  assert(joined == slot.size());
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
    const int w = run_of(1 << 30, 768, p);
    assert(run_begin(1 << 30, 768, w) <= p && p < run_begin(1 << 30, 768, w + 1));
    ++checks;
  }
  printf("paged runs: %ld checks passed\n", checks);
  return 0;
}

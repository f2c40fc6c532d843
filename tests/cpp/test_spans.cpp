// Random spans of up to four lists: the answer is that of all pairs.
#include <cstdio>
#include <random>
#include <vector>

#include "spans.hpp"

int main() {
  std::mt19937 rng(1);
  int meets = 0, wrong = 0;
  for (int trial = 0; trial < 20000; ++trial) {
    const int lists = 1 + rng() % 4, room = 20 << rng() % 8;
    std::vector<std::vector<b200cp::Span>> spans(lists);
    std::vector<b200cp::SpanList> args;
    struct One {
      b200cp::Span s;
      bool written;
    };
    std::vector<One> all;
    for (int k = 0; k < lists; ++k) {
      const bool written = rng() % 3 != 0;
      const int n = rng() % 5;
      for (int i = 0; i < n; ++i) {
        const uintptr_t b = 1 + rng() % room;
        spans[k].push_back({b, b + rng() % 8});
        all.push_back({spans[k].back(), written});
      }
      args.push_back({spans[k].data(), spans[k].size(), written});
    }
    bool want = false;
    for (size_t i = 0; i < all.size(); ++i)
      for (size_t j = 0; j < i; ++j)
        want |= (all[i].written || all[j].written) && all[i].s.begin < all[i].s.end && all[j].s.begin < all[j].s.end &&
                all[i].s.begin < all[j].s.end && all[j].s.begin < all[i].s.end;
    const bool got = b200cp::spans_meet(args.data(), args.size());
    meets += want;
    wrong += got != want;
  }
  std::printf("%d of 20000 meet, %d wrong\n", meets, wrong);
  return wrong == 0 && meets > 2000 && meets < 18000 ? 0 : 1;
}

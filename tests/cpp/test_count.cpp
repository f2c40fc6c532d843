// A count is asked for once, also where it is zero; an error is not remembered.
#include <atomic>
#include <cstdio>
#include <initializer_list>

#include "raise_limit.hpp"

int main() {
  int asked = 0, wrong = 0;
  for (const int value : {0, 1, 7}) {
    std::atomic<int> slot{0};
    int n = -1;
    asked = 0;
    wrong += b200cp::remembered_count(slot, &n, [&](int*) { ++asked; return 5; }) != 5;
    for (int k = 0; k < 3; ++k) {
      n = -1;
      wrong += b200cp::remembered_count(slot, &n, [&](int* out) { ++asked; *out = value; return 0; }) != 0 || n != value;
    }
    wrong += asked != 2;
  }
  std::printf("%d wrong\n", wrong);
  return wrong ? 1 : 0;
}

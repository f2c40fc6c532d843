// Whether memory that a call writes meets other memory of the call.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace b200cp {

struct Span {   // begin == end: nothing
  uintptr_t begin, end;
};
struct SpanList {   // sorted by the check where it is not
  Span* at;
  size_t count;
  bool written;
};

// True where two spans meet of which at least one is written (of the same list or of two).  The lists of a step are those of its parameters, its
// gradients and so on, mostly in the order of their addresses each: they are passed once, the least span of all lists next, beside how far
// the spans before it reach.
inline bool spans_meet(SpanList* lists, size_t n) {
  const auto before = [](const Span& a, const Span& b) { return a.begin < b.begin; };
  for (size_t k = 0; k < n; ++k)
    if (!std::is_sorted(lists[k].at, lists[k].at + lists[k].count, before)) std::sort(lists[k].at, lists[k].at + lists[k].count, before);
  uintptr_t end = 0, written_end = 0;
  for (;;) {
    SpanList* next = nullptr;
    uintptr_t until = UINTPTR_MAX;   // where the first of the other lists begins
    for (size_t k = 0; k < n; ++k) {
      if (!lists[k].count) continue;
      if (!next || lists[k].at->begin < next->at->begin) {
        if (next) until = next->at->begin;
        next = lists + k;
      } else {
        until = std::min(until, lists[k].at->begin);
      }
    }
    if (!next) return false;
    for (; next->count && next->at->begin <= until; ++next->at, --next->count) {
      const Span s = *next->at;
      if (s.begin == s.end) continue;
      if (s.begin < (next->written ? end : written_end)) return true;
      end = std::max(end, s.end);
      if (next->written) written_end = std::max(written_end, s.end);
    }
  }
}

}  // namespace b200cp

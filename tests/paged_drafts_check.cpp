// Checks how calls of drafted tokens are cut into items, compiled for the host: over random batches,
// requests that do not fit among them, the items of a call are no more than its launch is made for, those
// of cut requests no more than its workspace holds, and each request's items cover its attended subtiles.
// Prints "ok" or the batch that failed.
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "paged_index.h"

using namespace ssa;

#define CHECK(x)                                                                              \
  do {                                                                                        \
    if (!(x)) {                                                                               \
      std::printf("%s: batch %d, B=%d cap=%lld window=%d items=%d M=%d G=%d\n", #x, batch, B, \
                  (long long)cap, window, items, M, G);                                       \
      return 1;                                                                               \
    }                                                                                         \
  } while (0)

int main() {
  std::mt19937 rng(1);
  auto upto = [&](long long n) { return (long long)(rng() % (unsigned long long)(n + 1)); };
  for (int batch = 0; batch < 4000; ++batch) {
    const int B = 1 + (int)upto(batch % 3 ? 8 : 300), page = 16 * (1 + (int)upto(20));
    const int64_t cap = page * (1 + upto(batch % 2 ? 12 : 3000));
    const int windows[] = {0, 0, 1, 2, 15, 16, 17, 100, 1000, 0x7fffffff};
    const int window = windows[upto(9)], Ms[] = {16, 32, 64, 128}, M = Ms[upto(3)];
    const int G = 1 + (int)upto(20), items = 1 + (int)upto(batch % 5 ? 40 : 1536);
    const int words = upto(1) ? 0 : 1 + (int)upto(31);
    std::vector<int> lens(B), cu(B + 1);
    for (int b = 0; b < B; ++b) cu[b + 1] = cu[b] + (int)(upto(2) ? upto(upto(1) ? 40 : 1100) : 0);
    const int64_t N = cu[B] + upto(5);
    for (int b = 0; b < B; ++b) {
      const int n = cu[b + 1] - cu[b];
      const int edge[] = {n, n - 1, n + 1, (int)cap, (int)cap + 1, -1, -0x7fffffff - 1, 0x7fffffff};
      lens[b] = upto(2) ? n + (int)upto(cap) : edge[upto(7)];
    }
    float work = 0;
    int64_t all_tiles = 0;
    std::vector<DraftSpan> spans(B);
    for (int b = 0; b < B; ++b) {
      const DraftSpan s = spans[b] = draft_span(lens[b], cu[b], cu[b + 1], N, window, words, cap);
      const int n = cu[b + 1] - cu[b];
      CHECK(s.n == n);
      CHECK(s.span.ok == (n > 0 && lens[b] >= n && lens[b] <= cap && (!words || n <= 32 * words)));
      const int tiles = draft_tiles(s, G, M);
      CHECK((int64_t)tiles * M >= (int64_t)n * G && (int64_t)(tiles - 1) * M < (int64_t)std::max(n, 1) * G);
      CHECK(draft_units(s) >= (n > 0) && (n > 0 || draft_units(s) == 0));
      all_tiles += tiles;
      work += (float)tiles * (float)draft_units(s);
    }
    CHECK(N == 0 || all_tiles <= draft_most_tiles(B, N, G, M));
    const int chunk = draft_chunk(work, (float)items);
    const int64_t keys = window > 0 ? std::min<int64_t>(cap, (int64_t)window + N + 15) : cap;
    const int64_t most = paged_most_units(keys, 0);
    int64_t made = 0, parts = 0;
    for (int b = 0; b < B; ++b) {
      const DraftSpan& s = spans[b];
      const int units = draft_units(s), splits = paged_items(units, chunk);
      const int64_t of = (int64_t)draft_tiles(s, G, M) * splits;
      made += of;
      parts += splits > 1 ? of : 0;
      CHECK(units <= most);
      if (!s.span.ok) {
        CHECK(splits <= 1);
        continue;
      }
      CHECK(s.ctx == lens[b] - s.n && s.span.len == lens[b]);
      CHECK(s.span.first <= s.ctx && (window == 0 ? s.span.first == 0
                                                  : s.span.first == std::max(0, s.ctx - window + 1)));
      int at = s.span.first / 16;
      for (int j = 0; j < splits; ++j) {
        const PagedRange r = paged_item_range(s.span, units, j, splits);
        CHECK(r.begin == at && r.end > r.begin && r.end - r.begin <= (int64_t)chunk * kPagedUnit);
        at = r.end;
      }
      CHECK(at == (lens[b] - 1) / 16 + 1);
      CHECK((at * 16 - 1) / page < cap / page);
    }
    CHECK(made <= all_tiles + items && made <= all_tiles * most);
    CHECK(parts <= 2 * items);
  }
  // offsets that do not ascend or pass the call's rows make a request none
  const int bad[][2] = {{-1, 3}, {5, 4}, {0, 11}, {-2147483647 - 1, 2147483647}, {11, 12}};
  for (const auto& c : bad)
    if (draft_span(100, c[0], c[1], 10, 0, 0, 1000).n != 0) return 1;
  std::puts("ok");
  return 0;
}

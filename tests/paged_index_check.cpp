// Checks the paged attention's cutting of requests into items, compiled for the host: over random
// batches every attended subtile lies in exactly one item, no more items than the workspace holds,
// and no index leaves the table. Prints "ok" or the batch that failed.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "paged_index.h"

using namespace ssa;

#define CHECK(x)                                                                            \
  do {                                                                                      \
    if (!(x)) {                                                                             \
      std::printf("%s: batch %d, B=%d cap=%lld window=%d items=%d\n", #x, batch, B,       \
                  (long long)cap, window, items);                                           \
      return 1;                                                                             \
    }                                                                                       \
  } while (0)

int main() {
  std::mt19937 rng(1);
  auto upto = [&](long long n) { return (long long)(rng() % (unsigned long long)(n + 1)); };
  for (int batch = 0; batch < 4000; ++batch) {
    const int B = 1 + (int)upto(batch % 3 ? 8 : 300), page = 16 * (1 + (int)upto(20));
    const int64_t cap = page * (1 + upto(batch % 2 ? 12 : 3000));
    const int windows[] = {0, 0, 1, 2, 15, 16, 17, 100, 1000, 0x7fffffff};
    const int window = windows[upto(9)];
    const int items = 1 + (int)upto(batch % 5 ? 40 : 1024);
    std::vector<int> lens(B);
    for (int& n : lens) {
      const int edge[] = {0, 1, 15, 16, 17, (int)cap, (int)cap - 1, -1, (int)cap + 1, -0x7fffffff};
      n = upto(1) ? (int)upto(cap) : edge[upto(9)];
    }
    int units = 0;
    for (int n : lens) units += paged_units(paged_span(n, window, cap));
    const int chunk = paged_chunk(units, items);
    CHECK(chunk >= 1);
    int64_t made = 0;
    const int64_t most = paged_most_units(cap, window);
    for (int n : lens) {
      const PagedSpan s = paged_span(n, window, cap);
      CHECK(s.ok == (n >= 0 && n <= cap));
      const int u = paged_units(s), k = paged_items(u, chunk);
      CHECK(u <= most);
      made += k;
      if (!s.ok || n == 0) {
        CHECK(u == 0 && k == 0);
        const PagedRange r = paged_item_range(s, 0, 0, 1);
        CHECK(r.begin == 0 && r.end <= 1);
        continue;
      }
      CHECK(s.len == n && s.first >= 0 && s.first < n);
      CHECK(window == 0 ? s.first == 0 : n - s.first == (n < window ? n : window));
      int at = s.first / 16;
      for (int j = 0; j < k; ++j) {
        const PagedRange r = paged_item_range(s, u, j, k);
        CHECK(r.begin == at && r.end > r.begin);
        CHECK(r.end - r.begin <= chunk * kPagedUnit);
        at = r.end;
      }
      CHECK(at == (n + 15) / 16);
      CHECK((at * 16 - 1) / page < cap / page);
    }
    CHECK(made <= paged_most_items(B, items, most));
  }
  for (int d = 1; d <= 4096; ++d) {
    const PageDiv div = page_div(d);
    for (int k = 0; k < 200; ++k) {
      const int64_t q = k < 3 ? k : upto((1 << 28) / d);
      for (int64_t x = q * d - 1; x <= q * d + 1; ++x)
        if (x >= 0 && x < 1 << 28 && page_of((int)x, div) != x / d) {
          std::printf("%lld / %d\n", (long long)x, d);
          return 1;
        }
      const int64_t page = 16 * d, len = k < 4 ? 0x7fffffff - k : upto(k % 2 ? 5 * page : 0x7fffffff);
      if (paged_pages((int)len, (int)page, div) != (len + page - 1) / page) {
        std::printf("pages of %lld tokens at %d\n", (long long)len, (int)page);
        return 1;
      }
    }
  }
  std::puts("ok");
  return 0;
}

// Checks how many items a call aims at, compiled for the host: the work of up to 65,535 requests is added
// up in fp32 as the kernel's 64 lanes do, a run of requests each and then pairwise, and the units per item
// that follow must cover the work of all, exactly. Units at and below powers of two, where sums of small
// terms lose most. Prints "ok" or the batch that failed.
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "paged_index.h"

using namespace ssa;

int main() {
  std::mt19937 rng(2);
  auto upto = [&](long long n) { return (long long)(rng() % (unsigned long long)(n + 1)); };
  for (int batch = 0; batch < 3000; ++batch) {
    const int counts[] = {65535, 65536 - 64, 30000, 1000, 65, 64, 3}, B = counts[upto(batch % 50 ? 6 : 0)];
    const int kind = batch % 6, power = 1 << upto(24);
    std::vector<int> units(B), tiles(B);
    const int run = (B + 63) / 64;
    for (int b = 0; b < B; ++b) {
      const bool first = b % run == 0;
      units[b] = kind == 0 ? (first ? 1 << 24 : 1)               // what is added vanishes
                 : kind == 1 ? (first ? power : 1)
                 : kind == 2 ? std::max(1, power - 1)
                 : kind == 3 ? 32767
                             : 1 + (int)upto(power);
      tiles[b] = kind < 3 ? 1 : 1 + (int)upto(kind == 5 ? 3000 : 3);
    }
    float lane[64], next[64];
    double work = 0;  // below 2^53: exact
    for (int l = 0; l < 64; ++l) {
      lane[l] = 0;
      for (int b = std::min(l * run, B); b < std::min(l * run + run, B); ++b) {
        volatile float x = (float)tiles[b] * (float)units[b], sum = lane[l] + x;
        lane[l] = sum;
        work += (double)tiles[b] * units[b];
      }
    }
    for (int off = 1; off < 64; off *= 2) {
      for (int l = 0; l < 64; ++l) next[l] = lane[l] + lane[l ^ off];
      std::copy(next, next + 64, lane);
    }
    for (int items : {1, 7, 96, 128, 256, 512, 768, 1024, 1536}) {
      const int chunk = draft_chunk(lane[0], (float)items);
      if (chunk < 1000000000 && (double)chunk * items < work) {
        std::printf("batch %d: B=%d kind %d power %d items %d: chunk %d covers %.0f of %.0f (sum %.0f)\n", batch,
                    B, kind, power, items, chunk, (double)chunk * items, work, (double)lane[0]);
        return 1;
      }
      // nor much more than needed
      if ((double)chunk * items > work * 1.0002 + 2.0 * items) return 2;
    }
  }
  std::puts("ok");
  return 0;
}

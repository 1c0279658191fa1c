// Index arithmetic of the paged key-value cache, shared by its kernels and compiled for the host by
// its tests: which keys a request attends and how a call's keys are cut into items. No memory is
// touched here; a length or page id that does not fit its table is answered, never followed.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define SSA_HD __host__ __device__ inline
#else
#define SSA_HD inline
#endif

namespace ssa {

// Keys [first, len) of a request: the last `window` of its `len` keys (window 0: all of them).
// ok: 0 <= len <= cap, cap = table width x page size.
struct PagedSpan {
  int first, len;
  bool ok;
};

SSA_HD PagedSpan paged_span(int len, int window, int64_t cap) {
  PagedSpan s{0, 0, len >= 0 && (int64_t)len <= cap};
  if (!s.ok) return s;
  s.len = len;
  s.first = window > 0 && len > window ? len - window : 0;
  return s;
}

// A request's keys are cut at multiples of 16 (a subtile, never across pages: pages hold a multiple
// of 16 tokens) and dealt out in units of kPagedUnit subtiles.
constexpr int kPagedUnit = 8;

SSA_HD int paged_units(const PagedSpan& s) {
  if (s.len == 0) return 0;
  const int subtiles = (s.len - 1) / 16 + 1 - s.first / 16;
  return (subtiles + kPagedUnit - 1) / kPagedUnit;
}

// The most units a request can have: its table row's keys, or its window's from any offset.
SSA_HD int64_t paged_most_units(int64_t cap, int window) {
  const int64_t keys = window > 0 && (int64_t)window + 15 < cap ? (int64_t)window + 15 : cap;
  return (keys + 16 * kPagedUnit - 1) / (16 * kPagedUnit);
}

// The most items that B requests make when a call aims at `items`.
SSA_HD int64_t paged_most_items(int64_t B, int64_t items, int64_t most_units) {
  const int64_t cut = items + B, all = B * most_units;
  return cut < all ? cut : all;
}

// Units per item so that a call's `units` make at most `items` items besides one more per request.
// (The units of a call are held below 2^31.)
SSA_HD int paged_chunk(int units, int items) {
  return units <= items ? 1 : (int)(((unsigned)units + (unsigned)items - 1) / (unsigned)items);
}

SSA_HD int paged_items(int units, int chunk) {
  return (int)(((unsigned)units + (unsigned)chunk - 1) / (unsigned)chunk);
}

// Subtiles [begin, end) of item j of n: the request's units spread evenly over its items.
struct PagedRange {
  int begin, end;
};

SSA_HD PagedRange paged_item_range(const PagedSpan& s, int units, int j, int n) {
  const int a = s.first / 16, last = (s.len - 1) / 16 + 1;
  const int each = (int)((unsigned)units / (unsigned)n), more = units - each * n;
  PagedRange r;
  r.begin = a + (j * each + (j < more ? j : more)) * kPagedUnit;
  r.end = r.begin + (each + (j < more ? 1 : 0)) * kPagedUnit;
  if (r.end > last) r.end = last;
  return r;
}

// Division of a subtile's number (below 2^28: lengths are below 2^31) by the subtiles of a page, D up
// to 4096, as a multiplication: mul = ceil(2^(31 + shift) / D), 2^shift <= D < 2^(shift + 1), is off
// by less than 1 in 2^(31 + shift) / D > 2^30, more than any quotient's distance from the next.
struct PageDiv {
  unsigned mul;
  int shift;
};

SSA_HD PageDiv page_div(int subtiles) {
  PageDiv d{0, 0};
  while ((2 << d.shift) <= subtiles) ++d.shift;
  d.mul = (unsigned)((((uint64_t)1 << (31 + d.shift)) + (unsigned)subtiles - 1) /
                     (unsigned)subtiles);
  return d;
}

SSA_HD int page_of(int subtile, const PageDiv& d) {
  return (int)(((uint64_t)((unsigned)subtile * 2u) * d.mul >> 32) >> d.shift);
}

// Pages that hold len tokens.
SSA_HD int paged_pages(int len, int page, const PageDiv& d) {
  return page_of((int)(((unsigned)len + 15u) / 16u) + page / 16 - 1, d);
}

}  // namespace ssa

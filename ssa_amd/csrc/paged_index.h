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

// Drafted tokens: request b's are rows [cu[b], cu[b + 1]) of the call's N, its last n tokens of the
// cache. ctx: the tokens before them, the first at position ctx. Keys [span.first, span.len) are
// attended by some of its rows: a row's position is ctx or later, its window ends there.
// n is 0 where the offsets do not fit N; span.ok: the tokens fit the cache and the masks (of `words`
// 32-bit words a row; 0: every token attends those before it).
struct DraftSpan {
  int ctx, n;
  PagedSpan span;
};

SSA_HD DraftSpan draft_span(int len, int c0, int c1, int64_t N, int window, int words,
                            int64_t cap) {
  DraftSpan s{0, c0 >= 0 && c1 >= c0 && (int64_t)c1 <= N ? c1 - c0 : 0, {0, 0, false}};
  if (s.n == 0) return s;
  s.span.ok = len >= s.n && (int64_t)len <= cap && (words == 0 || (int64_t)s.n <= 32ll * words);
  if (!s.span.ok) return s;
  s.ctx = len - s.n;
  s.span.len = len;
  s.span.first = window > 0 && s.ctx >= window ? s.ctx - window + 1 : 0;
  return s;
}

// Units of keys; one where rows are only answered (a length that does not fit).
SSA_HD int draft_units(const DraftSpan& s) {
  return s.n == 0 ? 0 : s.span.ok ? paged_units(s.span) : 1;
}

// Tiles of M rows, a row a drafted token and one of the G query heads of a key head (a call's rows are
// held below 2^31).
SSA_HD int draft_tiles(const DraftSpan& s, int G, int M) {
  return (int)(((unsigned)s.n * (unsigned)G + (unsigned)M - 1u) / (unsigned)M);
}

// Units per item so that `work` units (of every row tile) make at most `items` items besides one more per
// row tile. work is a sum in fp32 of up to 65,535 requests' by 64 lanes: 1,024 additions one after the
// other, 6 across the lanes, 3 roundings of a term, 2 here, 2^-24 each, make it at most 6.2 10^-5 too small.
SSA_HD int draft_chunk(float work, float items) {
  const float c = work / items * 1.0001f;
  return c >= 1e9f ? 1000000000 : (int)c + 1;
}

// The most row tiles that N tokens of B requests make, and the most items of requests that are cut
// in more than one (each of their parts is kept for the join): fewer than two per item aimed at.
SSA_HD int64_t draft_most_tiles(int64_t B, int64_t N, int64_t G, int M) {
  return N * G / M + (B < N ? B : N);
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

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

SSA_HD int paged_pages(int len, int page) { return (int)(((int64_t)len + page - 1) / page); }

}  // namespace ssa

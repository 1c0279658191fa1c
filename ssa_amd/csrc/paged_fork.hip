// Requests of the paged key-value cache that share pages: forked, cut short and ended, with the pages that
// no request lists any more given back; and the pages that have to be copied for it.
#include <algorithm>

#include "paged_parts.h"

namespace ssa {
namespace {

// ---- rows of the table from other rows ---------------------------------------------------------

struct ForkRow;

// What the call's rows say of a page: the first row that listed it and changes with the first entry there
// (a row may list a page twice), the first row that will hold it as its last, partly filled page, whether a
// row will hold it whole.
struct PageUse {
  unsigned long long holder;
  int first_part, whole;
};

constexpr unsigned long long kNoHolder = ~0ull;

__device__ inline unsigned long long holder_of(int b, int e) {
  return (unsigned long long)b << 32 | (unsigned)e;
}

struct ForkParams {
  const int32_t* src;  // NULL: every row itself
  const int32_t* new_lens;
  int32_t* lens;
  int32_t* table;
  int64_t table_stride, W, cap;
  int B, page;
  int32_t* free_pages;
  int64_t P;
  int32_t* nfree;
  int32_t* source;
  int32_t* target;
  int32_t* tokens;
  int32_t* status;
  PageDiv div;
  // workspace
  PageUse* use;       // (P)
  int32_t* old;       // (B, W): the held entries of the table before
  ForkRow* rows;      // (B)
  int32_t* given;     // (units): pages given back, then the sum of those before
  int32_t* bad;       // (units)
  int32_t* taken;     // (B): whether a page is taken, then the pages taken before it (-1: none)
  int32_t* top;       // (B): the stack's top before, the first page on top
  int32_t* nfree0;    // (1): free pages before
  int32_t* left;      // (1): free pages after, -1: nothing changes
  int64_t units;      // of at most kForkEntries entries of a row
  int chunks;         // of a row
};

constexpr int kForkEntries = 1024, kForkLoads = kForkEntries / 64;

// A row's change.
struct ForkRow {
  int from, len, want, have, whole, need;  // pages held before, to hold whole and to hold
  int ok, same;
};

__device__ inline ForkRow fork_row(const ForkParams& p, int b) {
  ForkRow r;
  r.len = p.lens[b];
  r.want = p.new_lens[b];
  r.from = p.src ? p.src[b] : b;
  r.ok = r.len >= 0 && r.len <= p.cap && r.want >= 0;
  if (r.want > 0) {
    r.ok = r.ok && r.from >= 0 && r.from < p.B;
    const int of = r.ok ? p.lens[r.from] : 0;
    r.ok = r.ok && of <= p.cap && r.want <= of;
  }
  if (!r.ok || r.want == 0) r.from = b;  // no page is taken from there
  r.have = r.ok ? paged_pages(r.len, p.page, p.div) : 0;
  r.need = r.ok ? paged_pages(r.want, p.page, p.div) : 0;
  r.whole = r.need - (r.need > 0 && r.want < r.need * p.page ? 1 : 0);
  r.same = r.ok && r.want == r.len && (r.want == 0 || r.from == b);
  return r;
}

// f(k, entry) for this lane's entries of a chunk below `end`; k counts to kForkLoads.
template <class F>
__device__ inline void each_entry(int chunk, int end, F f) {
  const int first = chunk * kForkEntries, lane = threadIdx.x & 63;
#pragma unroll
  for (int k = 0; k < kForkLoads; ++k) {
    if (first + k * 64 >= end) return;
    const int e = first + k * 64 + lane;
    if (e < end) f(k, e);
  }
}

// A page is given back where no row lists it any more, and copied where two rows would write it; both are
// known once every row has said what it will hold, so the call is steps between which all units (chunks of
// a row's entries, a wave each) are done. Counts that are kept from call to call instead would have to be
// right at every resize too.
// 1: the table's held entries are kept, the uses of their pages cleared.
__device__ inline void fork_clear(const ForkParams& p, int unit) {
  const int b = unit / p.chunks, chunk = unit - b * p.chunks;
  const ForkRow r = fork_row(p, b);
  bool bad = !r.ok;
  const int32_t* const row = p.table + b * p.table_stride;
  int id[kForkLoads];
  each_entry(chunk, r.have, [&](int k, int e) { id[k] = row[e]; });
  each_entry(chunk, r.have, [&](int k, int e) {
    p.old[b * p.W + e] = id[k];
    if (id[k] < 0 || id[k] >= p.P) bad = true;
    else p.use[id[k]] = PageUse{kNoHolder, 0x7fffffff, 0};
  });
  const bool any = __any(bad);
  if ((threadIdx.x & 63) == 0) {
    p.bad[unit] = any;
    if (chunk == 0) {
      p.rows[b] = r;
      const int nfree = *p.nfree, at = nfree - 1 - b;
      p.top[b] = at >= 0 && at < p.P ? p.free_pages[at] : -1;
      if (b == 0) *p.nfree0 = nfree;
    }
  }
}

// 2: the uses of the pages.
__device__ inline void fork_mark(const ForkParams& p, int unit) {
  const int b = unit / p.chunks, chunk = unit - b * p.chunks;
  const ForkRow r = p.rows[b];
  const int32_t* const mine = p.old + b * p.W;
  const int32_t* const theirs = p.old + r.from * p.W;
  int id[kForkLoads];
  each_entry(chunk, r.need, [&](int k, int e) { id[k] = theirs[e]; });
  each_entry(chunk, r.need, [&](int k, int e) {
    if (id[k] < 0 || id[k] >= p.P) return;
    if (e < r.whole) p.use[id[k]].whole = 1;
    else atomicMin(&p.use[id[k]].first_part, b);
  });
  if (r.same) return;
  each_entry(chunk, r.have, [&](int k, int e) { id[k] = mine[e]; });
  each_entry(chunk, r.have, [&](int k, int e) {
    if (id[k] >= 0 && id[k] < p.P) atomicMin(&p.use[id[k]].holder, holder_of(b, e));
  });
}

// Whether row b gives back a page of this use at entry e.
__device__ inline bool gives(const PageUse& u, int b, int e) {
  return !u.whole && u.first_part == 0x7fffffff && u.holder == holder_of(b, e);
}

// Whether row b needs a copy of its last page: another row holds it whole or was first.
__device__ inline bool copies(const PageUse& u, int b) { return u.whole || u.first_part != b; }

// 3: pages given back by the unit, and whether its row takes one.
__device__ inline void fork_count(const ForkParams& p, int unit) {
  const int b = unit / p.chunks, chunk = unit - b * p.chunks, lane = threadIdx.x & 63;
  const ForkRow r = p.rows[b];
  if (chunk == 0 && lane == 0) {
    bool take = false;
    if (r.whole < r.need) {
      const int id = p.old[r.from * p.W + r.whole];
      take = id >= 0 && id < p.P && copies(p.use[id], b);
    }
    p.taken[b] = take;
  }
  int n = 0;
  if (!r.same) {
    int id[kForkLoads];
    each_entry(chunk, r.have, [&](int k, int e) { id[k] = p.old[b * p.W + e]; });
    each_entry(chunk, r.have, [&](int k, int e) {
      if (id[k] >= 0 && id[k] < p.P) n += gives(p.use[id[k]], b, e);
    });
  }
  n = lane_sums(n).all;
  if (lane == 0) p.given[unit] = n;
}

constexpr int kForkThreads = 1024, kForkWaves = kForkThreads / 64;

// All or nothing: -1 or the pages lacking, 0 where the call fits.
__device__ inline int fork_status(const ForkParams& p, bool bad, int64_t taken, int64_t given) {
  const int nfree = *p.nfree0;
  const int64_t lack = taken - nfree;
  if (bad || nfree < 0 || nfree > p.P || nfree - taken + given > p.P) return -1;
  return lack > 0 ? (int)lack : 0;
}

// 4, by one workgroup: sums of the units and rows before each, and the free pages after.
__device__ inline void fork_sum(const ForkParams& p) {
  __shared__ int64_t s_wave[kForkWaves];
  __shared__ int64_t s_all;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  bool bad = false;
  for (int64_t u = tid; u < p.units; u += kForkThreads) bad |= p.bad[u] != 0;
  bad = __syncthreads_or(bad);
  // x becomes the sum before it; a row that takes no page keeps -1
  auto scan = [&](int32_t* x, int64_t n, bool mark) {
    int64_t sum = 0;
    for (int64_t i0 = 0; i0 < n; i0 += kForkThreads) {
      const int64_t i = i0 + tid;
      const int64_t v = i < n ? x[i] : 0;
      const LaneSums<int64_t> s = lane_sums(v);
      __syncthreads();
      if (lane == 63) s_wave[wv] = s.upto;
      __syncthreads();
      if (wv == 0) {
        const int64_t w = lane < kForkWaves ? s_wave[lane] : 0;
        const LaneSums<int64_t> t = lane_sums(w);
        if (lane < kForkWaves) s_wave[lane] = t.upto - w;
        if (lane == 0) s_all = t.all;
      }
      __syncthreads();
      if (i < n)
        x[i] = mark && v == 0 ? -1 : (int)min(sum + s_wave[wv] + s.upto - v, (int64_t)0x7fffffff);
      sum += s_all;
    }
    return sum;
  };
  const int64_t taken = scan(p.taken, p.B, true), given = scan(p.given, p.units, false);
  if (tid == 0) {
    const int status = fork_status(p, bad, taken, given);
    *p.status = status;
    *p.left = status == 0 ? (int)(*p.nfree0 - taken + given) : -1;
  }
}

// What a unit of step 5 goes by: the free pages after (-1: nothing changes), its row's place among the
// pages taken, the pages given back before it.
struct ForkPlace {
  int left, taken, given;
};

// 5: the pages taken, those given back onto the stack, the new rows and lengths.
__device__ inline void fork_write(const ForkParams& p, int unit, const ForkPlace& at_) {
  const int b = unit / p.chunks, chunk = unit - b * p.chunks, lane = threadIdx.x & 63;
  const ForkRow r = p.rows[b];
  const int fresh = at_.left >= 0 && at_.taken >= 0 ? p.top[at_.taken] : -1;
  const bool takes = at_.left >= 0 && at_.taken >= 0;
  if (chunk == 0 && lane == 0) {
    p.source[b] = takes ? p.old[r.from * p.W + r.whole] : -1;
    p.target[b] = fresh;
    p.tokens[b] = takes ? r.want - r.whole * p.page : 0;
    if (b == 0 && at_.left >= 0) *p.nfree = at_.left;
  }
  if (at_.left < 0) return;
  int32_t* const row = p.table + b * p.table_stride;
  if (!r.same) {
    int id[kForkLoads];
    unsigned int give = 0;
    each_entry(chunk, r.have, [&](int k, int e) { id[k] = p.old[b * p.W + e]; });
    each_entry(chunk, r.have, [&](int k, int e) {
      give |= gives(p.use[id[k]], b, e) ? 1u << k : 0u;
    });
    int at = at_.left - 1 - at_.given;
#pragma unroll
    for (int k = 0; k < kForkLoads; ++k) {
      if (chunk * kForkEntries + k * 64 >= r.have) break;
      const unsigned long long all = __ballot(give >> k & 1);
      if (give >> k & 1) p.free_pages[at - __popcll(all & ((1ull << lane) - 1))] = id[k];
      at -= __popcll(all);
    }
    const int32_t* const theirs = p.old + r.from * p.W;
    each_entry(chunk, max(r.have, r.need), [&](int, int e) {
      row[e] = e >= r.need ? -1 : e == r.whole && takes ? fresh : theirs[e];
    });
    if (chunk == 0 && lane == 0) p.lens[b] = r.want;
  } else if (takes && chunk == r.whole / kForkEntries && lane == 0) {
    row[r.whole] = fresh;
  }
}

__device__ inline ForkPlace fork_place(const ForkParams& p, int unit) {  // after step 4
  return ForkPlace{*p.left, p.taken[unit / p.chunks], p.given[unit]};
}

// 4 and 5 at once, each wave adding up the units and rows by itself: a launch fewer where these are few.
__device__ inline void fork_sum_write(const ForkParams& p, int unit) {
  const int lane = threadIdx.x & 63, b = unit / p.chunks;
  int64_t given = 0, given_all = 0, taken = 0, taken_all = 0;
  bool bad = false;
  for (int u = lane; u < p.units; u += 64) {
    const int n = p.given[u];
    given_all += n;
    given += u < unit ? n : 0;
    bad |= p.bad[u] != 0;
  }
  for (int y = lane; y < p.B; y += 64) {
    const int n = p.taken[y];
    taken_all += n;
    taken += y < b ? n : 0;
  }
  given = lane_sums(given).all;
  given_all = lane_sums(given_all).all;
  taken = lane_sums(taken).all;
  taken_all = lane_sums(taken_all).all;
  const int status = fork_status(p, __any(bad), taken_all, given_all);
  if (unit == 0 && lane == 0) *p.status = status;
  fork_write(p, unit, ForkPlace{status == 0 ? (int)(*p.nfree0 - taken_all + given_all) : -1,
                                p.taken[b] ? (int)taken : -1, (int)given});
}

// The steps as launches of their own, four units a workgroup. Bound by their launches and the chains of
// memory latencies in each (row, page id, the page's use): 64 rows of up to 500 pages 15 us, forked or
// ended.
__global__ __launch_bounds__(256) void paged_fork_clear_kernel(ForkParams p) {
  const int64_t u = (int64_t)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  if (u < p.units) fork_clear(p, (int)u);
}
__global__ __launch_bounds__(256) void paged_fork_mark_kernel(ForkParams p) {
  const int64_t u = (int64_t)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  if (u < p.units) fork_mark(p, (int)u);
}
__global__ __launch_bounds__(256) void paged_fork_count_kernel(ForkParams p) {
  const int64_t u = (int64_t)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  if (u < p.units) fork_count(p, (int)u);
}
__global__ __launch_bounds__(kForkThreads) void paged_fork_sum_kernel(ForkParams p) { fork_sum(p); }
template <bool SUM>
__global__ __launch_bounds__(256) void paged_fork_write_kernel(ForkParams p) {
  const int64_t u = (int64_t)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  if (u >= p.units) return;
  if constexpr (SUM) fork_sum_write(p, (int)u);
  else fork_write(p, (int)u, fork_place(p, (int)u));
}

// Up to so many units each wave adds them up by itself: 64 requests of 1,000 tokens 11.3 us a fork for
// 13.7 with the sums in a launch of their own, 512 of 500 15.4 for 14.2, 4,096 of 300 47.5 for 25.6. (All
// steps in one launch of one workgroup: 2 requests 33 us for 8.2, 64 56 for 11.3.)
constexpr int64_t kForkSums = 256;

struct ForkLayout {
  int64_t chunks, units;
  size_t old, rows, given, bad, taken, top, nfree0, left, bytes;
};

ForkLayout fork_layout(int64_t B, int64_t W, int64_t pages) {
  ForkLayout y{};
  y.chunks = (W + kForkEntries - 1) / kForkEntries;
  y.units = B * y.chunks;
  y.rows = (size_t)pages * sizeof(PageUse);
  y.old = y.rows + (size_t)B * sizeof(ForkRow);
  y.given = y.old + (size_t)B * W * 4;
  y.bad = y.given + (size_t)y.units * 4;
  y.taken = y.bad + (size_t)y.units * 4;
  y.top = y.taken + (size_t)B * 4;
  y.nfree0 = y.top + (size_t)B * 4;
  y.left = y.nfree0 + 4;
  y.bytes = (y.left + 4 + 15) / 16 * 16;
  return y;
}

// ---- pages copied ------------------------------------------------------------------------------

struct CopyParams {
  char* kpool;
  char* vpool;
  const int32_t* source;
  const int32_t* target;
  const int32_t* tokens;  // NULL: whole pages
  int64_t pages;
  int page, Hkv, vecs, layers;                     // vecs: 16-byte pieces of a row
  int64_t kpl, kpp, kph, kps, vpl, vpp, vph, vps;  // bytes
};

// Division by a number of the call: an estimate that is one or two short, and its correction.
struct Quotient {
  unsigned d, mul;
  __device__ explicit Quotient(unsigned by) : d(by), mul(0xffffffffu / by) {}
  __device__ unsigned operator()(unsigned x, unsigned& rest) const {
    unsigned q = __umulhi(x, mul);
    rest = x - q * d;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool more = rest >= d;
      q += more;
      rest -= more ? d : 0;
    }
    return q;
  }
};

constexpr int kCopyBatch = 8;

// A thread moves 16-byte pieces of the copied tokens' keys and values, kCopyBatch of them on their way
// at a time; a workgroup row (y) a page, x over a page's pieces of all layers. Bound by memory: 96 pages
// of up to 128 tokens, 8 heads of 128 in 4 layers (16-bit, 200 MB in all), 45 us, 4.4 TB/s.
__global__ __launch_bounds__(256) void paged_copy_kernel(CopyParams p) {
  const int i = blockIdx.y;
  const int64_t from = p.source[i], to = p.target[i];
  const int n = p.tokens ? min(p.tokens[i], p.page) : p.page;
  if (from < 0 || from >= p.pages || to < 0 || to >= p.pages || from == to || n <= 0) return;
  const unsigned per = n * p.vecs;  // pieces of a layer's keys or values of a head
  const unsigned all = 2u * p.layers * p.Hkv * per, step = gridDim.x * 256;
  const Quotient block(per), slot_of(p.vecs), head(p.Hkv);
  for (unsigned x0 = blockIdx.x * 256 + threadIdx.x; x0 < all; x0 += step * kCopyBatch) {
    u32x4 v[kCopyBatch];
    char* at[kCopyBatch];
#pragma unroll
    for (int u = 0; u < kCopyBatch; ++u) {
      const unsigned x = x0 + u * step;
      if (x >= all) break;
      unsigned r, c, h;
      const unsigned of = block(x, r), slot = slot_of(r, c), lv = head(of, h);
      const bool val = lv & 1;
      char* const base = (val ? p.vpool : p.kpool) + (lv >> 1) * (val ? p.vpl : p.kpl) +
                         h * (val ? p.vph : p.kph) + slot * (val ? p.vps : p.kps) + c * 16;
      const int64_t pp = val ? p.vpp : p.kpp;
      v[u] = *(const u32x4*)(base + from * pp);
      at[u] = base + to * pp;
    }
#pragma unroll
    for (int u = 0; u < kCopyBatch; ++u) {
      if (x0 + u * step >= all) break;
      *(u32x4*)at[u] = v[u];
    }
  }
}

}  // namespace
}  // namespace ssa

using namespace ssa;

extern "C" size_t ssa_paged_fork_workspace_size(int64_t B, int64_t W, int64_t pages) {
  if (B <= 0 || W <= 0 || pages <= 0 || !fits_int(B) || !fits_int(W) || !fits_int(pages)) return 0;
  return fork_layout(B, W, pages).bytes;
}

extern "C" int ssa_paged_fork(const int32_t* src, const int32_t* new_lens, int32_t* lens,
                              int32_t* table, int64_t table_stride, int64_t B, int64_t W,
                              int64_t page, int32_t* free_pages, int64_t pages, int32_t* nfree,
                              int32_t* source, int32_t* target, int32_t* tokens, int32_t* status,
                              void* workspace, size_t workspace_bytes, ssa_stream_t stream) {
  const char* const who = "ssa_paged_fork";
  SSA_REQUIRE(new_lens && lens && table && free_pages && nfree && source && target &&
                  tokens && status, SSA_ERR_INVALID, "%s: NULL argument", who);
  SSA_REQUIRE(B > 0 && fits_int(B) && W > 0 && table_stride >= W && pages > 0 && fits_int(pages),
              SSA_ERR_INVALID, "%s: bad shape (B=%lld, W=%lld, pages=%lld)", who, (long long)B,
              (long long)W, (long long)pages);
  SSA_REQUIRE(page > 0 && page % 16 == 0 && page <= 65536, SSA_ERR_UNSUPPORTED,
              "%s: page of %lld tokens (a multiple of 16 up to 65536)", who, (long long)page);
  SSA_REQUIRE(W <= 0x7fffffff / page, SSA_ERR_UNSUPPORTED,
              "%s: a table row of %lld pages holds more than 2^31 - 1 tokens", who, (long long)W);
  const ForkLayout y = fork_layout(B, W, pages);
  SSA_REQUIRE(fits_int(y.units) && fits_launch((y.units + 3) / 4, 256), SSA_ERR_UNSUPPORTED,
              "%s: %lld table rows of %lld pages", who, (long long)B, (long long)W);
  SSA_REQUIRE(workspace_bytes >= y.bytes && workspace && aligned16(workspace), SSA_ERR_WORKSPACE,
              "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, y.bytes,
              workspace_bytes);
  char* const ws = (char*)workspace;
  ForkParams p{src, new_lens, lens, table, table_stride, W, W * page, (int)B, (int)page,
               free_pages, pages, nfree, source, target, tokens, status,
               page_div((int)page / 16), (PageUse*)ws, (int32_t*)(ws + y.old),
               (ForkRow*)(ws + y.rows), (int32_t*)(ws + y.given), (int32_t*)(ws + y.bad),
               (int32_t*)(ws + y.taken), (int32_t*)(ws + y.top), (int32_t*)(ws + y.nfree0),
               (int32_t*)(ws + y.left), y.units, (int)y.chunks};
  hipStream_t st = (hipStream_t)stream;
  const unsigned grid = (unsigned)((y.units + 3) / 4);
  paged_fork_clear_kernel<<<grid, 256, 0, st>>>(p);
  SSA_TRY(launch_status("paged_fork_clear_kernel"));
  paged_fork_mark_kernel<<<grid, 256, 0, st>>>(p);
  SSA_TRY(launch_status("paged_fork_mark_kernel"));
  paged_fork_count_kernel<<<grid, 256, 0, st>>>(p);
  SSA_TRY(launch_status("paged_fork_count_kernel"));
  if (y.units <= kForkSums) {
    paged_fork_write_kernel<true><<<grid, 256, 0, st>>>(p);
    return launch_status("paged_fork_write_kernel");
  }
  paged_fork_sum_kernel<<<1, kForkThreads, 0, st>>>(p);
  SSA_TRY(launch_status("paged_fork_sum_kernel"));
  paged_fork_write_kernel<false><<<grid, 256, 0, st>>>(p);
  return launch_status("paged_fork_write_kernel");
}

extern "C" int ssa_paged_copy(void* kpool, void* vpool, int dtype, int64_t layers, int64_t Hkv,
                              int64_t d, int64_t pages, int64_t page, const int64_t* strides,
                              const int32_t* source, const int32_t* target, const int32_t* tokens,
                              int64_t n, ssa_stream_t stream) {
  const char* const who = "ssa_paged_copy";
  SSA_REQUIRE(kpool && vpool && strides && source && target, SSA_ERR_INVALID, "%s: NULL argument",
              who);
  SSA_TRY(check_pool(who, dtype, Hkv, d, pages, page));
  SSA_REQUIRE(n >= 0 && n <= 65535 && layers > 0 && fits_int(layers), SSA_ERR_INVALID,
              "%s: %lld pages of %lld layers (at most 65535 pages)", who, (long long)n,
              (long long)layers);
  const int es = dtype_size(dtype);
  // strides: kpool(layer,page,head,slot), vpool(layer,page,head,slot)
  SSA_REQUIRE(rows16(kpool, strides, 4, es) && rows16(vpool, strides + 4, 4, es), SSA_ERR_INVALID,
              "%s: rows must start at multiples of 16 bytes", who);
  const int64_t vecs = d * es / 16;
  // counted in 32 bits, up to a step of all workgroups past the end
  SSA_REQUIRE(layers <= (1 << 30) / (Hkv * page * vecs), SSA_ERR_UNSUPPORTED,
              "%s: %lld layers (a page of at most 32 GiB over all of them)", who, (long long)layers);
  if (n == 0) return SSA_OK;
  const int64_t pieces = 2 * layers * Hkv * page * vecs;
  // at most eight workgroups a CU for all pages, each with kCopyBatch pieces a thread or more
  const int64_t blocks = std::max<int64_t>(
      1, std::min((pieces + 256 * kCopyBatch - 1) / (256 * kCopyBatch), (2048 + n - 1) / n));
  CopyParams p{(char*)kpool, (char*)vpool, source, target, tokens, pages, (int)page, (int)Hkv,
               (int)vecs, (int)layers,
               strides[0] * es, strides[1] * es, strides[2] * es, strides[3] * es,
               strides[4] * es, strides[5] * es, strides[6] * es, strides[7] * es};
  paged_copy_kernel<<<dim3((unsigned)blocks, (unsigned)n), 256, 0, (hipStream_t)stream>>>(p);
  return launch_status("paged_copy_kernel");
}

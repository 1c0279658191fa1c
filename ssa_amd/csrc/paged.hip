// The paged key-value cache: pages taken and given back from the requests' lengths, new tokens'
// keys and values stored through their slots, and one new token's attention over its pages.
//
// A pool holds `pages` pages of `page` tokens: (pages, Hkv, page, d) by strides (page, head, slot).
// Request b's token j lies in page table[b][j / page] at slot j % page.
#include <algorithm>

#include "paged_parts.h"

namespace ssa {
namespace {

// ---- lengths -> pages, slots, positions --------------------------------------------------------

struct ResizeParams {
  int32_t* lens;
  const int32_t* new_lens;
  int32_t* table;
  int64_t table_stride, B, W;
  int page;
  int32_t* free_pages;
  int64_t P;
  int32_t* nfree;
  int64_t* slots;
  int32_t* pos;
  int64_t T;
  int32_t* cu;
  int32_t* status;
  PageDiv div;
};

constexpr int kResizeThreads = 1024, kResizeWaves = kResizeThreads / 64;

// A request's change: pages taken, pages given back, new tokens.
template <class I>
struct Change {
  I x[3];
};

template <class I>
struct ScanRoom {
  I of[3][kResizeWaves], all[3];
};

// Exclusive prefix of the threads' changes (c becomes it) and their sum; threads past n hold none.
template <class I>
__device__ inline Change<I> block_scan(Change<I>& c, int64_t n, ScanRoom<I>& room) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  if (wv * 64 < n) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const LaneSums<I> s = lane_sums(c.x[i]);
      c.x[i] = s.upto - c.x[i];
      if (lane == 63) room.of[i][wv] = s.upto;
    }
  } else if (lane < 3) {
    room.of[lane][wv] = 0;
  }
  __syncthreads();
  if (wv < 3) {
    const I x = lane < kResizeWaves ? room.of[wv][lane] : 0;
    const LaneSums<I> s = lane_sums(x);
    if (lane < kResizeWaves) room.of[wv][lane] = s.upto - x;
    if (lane == 0) room.all[wv] = s.all;
  }
  __syncthreads();
  Change<I> all;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    c.x[i] += room.of[i][wv];
    all.x[i] = room.all[i];
  }
  __syncthreads();
  return all;
}

__device__ inline Change<int> change_of(int len, int new_len, const ResizeParams& p) {
  const int have = paged_pages(len, p.page, p.div), need = paged_pages(new_len, p.page, p.div);
  return Change<int>{{max(need - have, 0), max(have - need, 0), max(new_len - len, 0)}};
}

// Slots of more tokens are a launch of their own: 3,840 tokens of 64 requests 10.7 us in this launch
// and 11.5 in two, 15,000 of 1,000 requests 23.8 and 13.8 (each with the giving back).
constexpr int kSlotsInside = 4 * kResizeThreads;

// Calls f(request, its nth page, t) for the pages t < count of a tile of n requests whose prefix sums
// are `at`.
template <class F>
__device__ inline void each_page(const int* at, int n, int count, F f) {
  for (int t = threadIdx.x; t < count; t += kResizeThreads) {
    const int i = last_at_most(at, n, t);
    f(i, t - at[i], t);
  }
}

// One workgroup: totals first (all or nothing), then tiles of one request per thread whose pages and
// tokens are shared out over the threads by a search in the tile's prefix sums. The free pages are a
// stack; a page given back lands where a take of the same order would find it, so growing and
// shrinking back restores the stack. Takes are read before gives are written (they overlap).
// Bound by its chain of memory latencies and, past some thousand pages, by one CU's instructions: 256
// requests grown by a token 3 us, 13,000 pages taken for 64 prompts 8 to 10.
__global__ __launch_bounds__(kResizeThreads) void paged_resize_kernel(ResizeParams p) {
  __shared__ ScanRoom<int> room;
  __shared__ ScanRoom<int64_t> room64;
  __shared__ int s_flags[kResizeWaves];
  __shared__ int s_at[kResizeThreads], s_new[kResizeThreads], s_have[kResizeThreads],
      s_len[kResizeThreads];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t cap = p.W * p.page;
  const int nfree = *p.nfree;
  const bool one = p.B <= kResizeThreads;  // one tile: its scan gives the totals
  // bad: a length or count that does not fit; large: sums may pass 31 bits; many: more than a page or
  // a token of one request
  bool bad = nfree < 0 || nfree > p.P, large = !one, many = !one;
  Change<int> before{{0, 0, 0}};
  Change<int64_t> total{{0, 0, 0}};
  int len = 0, want = 0;  // the tile's request of this thread
  for (int64_t b = tid; b < p.B; b += kResizeThreads) {
    len = p.lens[b];
    want = p.new_lens[b];
    const PagedSpan o = paged_span(len, 0, cap), n = paged_span(want, 0, cap);
    bad |= !o.ok || !n.ok;
    before = change_of(o.len, n.len, p);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      total.x[i] += before.x[i];
      large |= before.x[i] >= 1 << 20;
      many |= before.x[i] > 1;
    }
  }
  const int flags = (__any(bad) ? 1 : 0) | (__any(large) ? 2 : 0) | (__any(many) ? 4 : 0);
  if (lane == 0) s_flags[tid >> 6] = flags;
  const Change<int> own = before;
  Change<int> all = block_scan(before, p.B, room);
  const int f = s_flags[lane & (kResizeWaves - 1)];
  bad = __any(f & 1);
  large = __any(f & 2);
  many = __any(f & 4);
  if (large) {
    total = block_scan(total, kResizeThreads, room64);
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i) total.x[i] = all.x[i];
  }
  const int64_t lack = total.x[0] - nfree;
  const int status = bad || nfree - total.x[0] + total.x[1] > p.P ? -1
                     : total.x[2] > p.T ? -2
                     : lack > 0 ? (int)min(lack, (int64_t)0x7fffffff) : 0;
  if (tid == 0) *p.status = status;
  const bool inside = p.T <= kSlotsInside;
  const int live = status == 0 ? (int)total.x[2] : 0;  // slots that are written below
  if (inside) {
    for (int t = live + tid; t < p.T; t += kResizeThreads) {
      p.slots[t] = -1;
      if (p.pos) p.pos[t] = 0;
    }
  }
  if (status != 0) {
    for (int64_t b = tid; b <= p.B; b += kResizeThreads) p.cu[b] = 0;
    return;
  }
  const int top = nfree - (int)total.x[0], left = top + (int)total.x[1];
  if (!many && inside) {  // a step of single tokens: every thread serves its own request
    // the table entry of the page taken, given back or written to
    const int e = own.x[1] ? paged_pages(want, p.page, p.div) : page_of(len / 16, p.div);
    int32_t* const entry = p.table + tid * p.table_stride + e;
    int pg = 0;
    if (own.x[0]) pg = p.free_pages[nfree - 1 - before.x[0]];
    else if (own.x[1] || own.x[2]) pg = *entry;
    __syncthreads();  // takes are read before gives are written
    if (own.x[0]) *entry = pg;
    if (own.x[1]) {
      *entry = -1;
      p.free_pages[left - 1 - before.x[1]] = pg;
    }
    if (own.x[2]) {
      p.slots[before.x[2]] = (int64_t)pg * p.page + (len - e * p.page);
      if (p.pos) p.pos[before.x[2]] = len;
    }
    if (tid < p.B) {
      p.cu[tid] = before.x[2];
      p.lens[tid] = want;
    }
    if (tid == 0) {
      p.cu[p.B] = all.x[2];
      *p.nfree = left;
    }
    return;
  }
  int taken = 0, added = 0;
  for (int64_t b0 = 0; b0 < p.B; b0 += kResizeThreads) {
    const int64_t b = b0 + tid;
    const int n = (int)min(p.B - b0, (int64_t)kResizeThreads);
    if (large) {
      len = tid < n ? p.lens[b] : 0;
      want = tid < n ? p.new_lens[b] : 0;
      before = change_of(len, want, p);
      all = block_scan(before, n, room);
    }
    s_have[tid] = paged_pages(len, p.page, p.div);
    s_at[tid] = before.x[0];
    s_new[tid] = before.x[2];
    s_len[tid] = len;
    if (tid < n) p.cu[b] = added + before.x[2];
    __syncthreads();
    each_page(s_at, n, all.x[0], [&](int i, int nth, int t) {
      p.table[(b0 + i) * p.table_stride + s_have[i] + nth] = p.free_pages[nfree - 1 - (taken + t)];
    });
    if (inside) {
      for (int t = tid; t < all.x[2]; t += kResizeThreads) {
        const int i = last_at_most(s_new, n, t), pos = s_len[i] + t - s_new[i];
        const int e = page_of(pos / 16, p.div), fresh = e - s_have[i];
        // a page of this call from the stack it came from, an earlier one from the table
        const int64_t pg = fresh >= 0 ? p.free_pages[nfree - 1 - (taken + s_at[i] + fresh)]
                                      : p.table[(b0 + i) * p.table_stride + e];
        p.slots[added + t] = pg * p.page + (pos - e * p.page);
        if (p.pos) p.pos[added + t] = pos;
      }
    }
    taken += all.x[0];
    added += all.x[2];
    __syncthreads();
  }
  if (tid == 0) p.cu[p.B] = added;
  int given = 0;
  for (int64_t b0 = 0; total.x[1] > 0 && b0 < p.B; b0 += kResizeThreads) {
    const int64_t b = b0 + tid;
    const int n = (int)min(p.B - b0, (int64_t)kResizeThreads);
    if (large) {
      len = tid < n ? p.lens[b] : 0;
      want = tid < n ? p.new_lens[b] : 0;
      before = change_of(len, want, p);
      all = block_scan(before, n, room);
    }
    s_have[tid] = paged_pages(want, p.page, p.div);  // what is kept
    s_at[tid] = before.x[1];
    __syncthreads();
    each_page(s_at, n, all.x[1], [&](int i, int nth, int t) {
      int32_t* e = p.table + (b0 + i) * p.table_stride + s_have[i] + nth;
      p.free_pages[left - 1 - (given + t)] = *e;
      *e = -1;
    });
    given += all.x[1];
    __syncthreads();
  }
  if (one) {
    if (tid < p.B) p.lens[tid] = want;
  } else {
    for (int64_t b = tid; b < p.B; b += kResizeThreads) p.lens[b] = p.new_lens[b];
  }
  if (tid == 0) *p.nfree = left;
}

// Slots and positions of the new tokens, a thread each (after the pages are in the table).
__global__ __launch_bounds__(256) void paged_slots_kernel(ResizeParams p) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= p.T) return;
  int64_t slot = -1;
  int pos = 0;
  if (t < p.cu[p.B]) {
    const int b = last_at_most(p.cu, (int)p.B, (int)t);
    pos = p.lens[b] - p.cu[b + 1] + (int)t;
    const int e = page_of(pos / 16, p.div);
    slot = (int64_t)p.table[b * p.table_stride + e] * p.page + (pos - e * p.page);
  }
  p.slots[t] = slot;
  if (p.pos) p.pos[t] = pos;
}

// ---- keys and values into their slots ----------------------------------------------------------

struct AppendParams {
  const char* k;
  const char* v;
  char* kpool;
  char* vpool;
  const int64_t* slots;
  int64_t T, pages;
  int page, Hkv, vecs;                                 // vecs: 16-byte pieces of a row
  int64_t kst, ksh, vst, vsh;                          // bytes
  int64_t kpp, kph, kps, vpp, vph, vps;                // bytes
};

// A thread moves one 16-byte piece of a key row and of its value row. Bound by memory: 65,436 tokens of
// 2 heads of 64 (bf16, 67 MB in all) 11.8 us, 5.7 TB/s.
__global__ __launch_bounds__(256) void paged_append_kernel(AppendParams p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = p.Hkv * p.vecs;
  if (i >= p.T * per) return;
  const int64_t t = i / per;
  const int r = (int)(i - t * per), h = r / p.vecs, c = (r - h * p.vecs) * 16;
  const int64_t slot = p.slots[t];
  if (slot < 0 || slot >= p.pages * p.page) return;
  const int64_t pg = slot / p.page, off = slot - pg * p.page;
  const u32x4 a = *(const u32x4*)(p.k + t * p.kst + h * p.ksh + c);
  const u32x4 b = *(const u32x4*)(p.v + t * p.vst + h * p.vsh + c);
  *(u32x4*)(p.kpool + pg * p.kpp + h * p.kph + off * p.kps + c) = a;
  *(u32x4*)(p.vpool + pg * p.vpp + h * p.vph + off * p.vps + c) = b;
}

// ---- attention of one new token ----------------------------------------------------------------

struct AttendParams {
  const char* q;
  char* kpool;
  char* vpool;
  char* out;
  float* lse;
  const char* k_new;
  const char* v_new;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* status;  // of the resize before, or NULL
  int64_t table_stride, cap, pages;
  int B, Hq, Hkv, G, d, page, window;
  float scale_log2;
  int64_t qb, qh, ob, oh;                 // elements
  int64_t kpp, kph, kps, vpp, vph, vps;   // elements
  int64_t knb, knh, vnb, vnh;             // elements
  PageDiv div;           // by the subtiles of a page
  int64_t stream_units;  // units of a key head from which a call streams
  int RT, items, units;  // row tiles of 16 heads; items aimed at (0: one per request); grid units
  float* part;           // (item, query head, DP): parts of rows that several items share
  float* part_ml;        // (item, query head, 2): their m and l
  int32_t* info;         // per request: its first item and their number
};

// One item of a call: the subtiles [begin, end) of request b, item j of n; `first_item` is the index
// of the request's item 0 among all.
struct Item {
  int b, j, n, begin, end, first_item;
  bool stream;  // the call reads more than stays in the caches
  PagedSpan span;
};

// The tokens of a table row; none fits after a refused resize (every row is then answered as bad).
__device__ inline int64_t row_cap(const AttendParams& p) {
  return p.status && *p.status != 0 ? -1 : p.cap;
}

// Finds item `index` from the lengths alone, each wave for itself: every lane sums a run of
// requests, the wave adds the runs up. False past the last item. Up to 64 requests the lengths are one
// load; past that the time grows with the square of the batch, as every workgroup reads all lengths: 256
// requests of 20 to 200 keys in a table 4,096 tokens wide 16 us, 1,024 65, 4,096 600, 16,384 7.8 ms (in a
// table of 208, an item per request: 7, 17, 61, 233 us); 1,024 of 500 to 1,500 keys 135 us and 97, 4,096
// of these 880 and 350.
__device__ inline bool find_item(const AttendParams& p, int index, Item& it) {
  const int lane = threadIdx.x & 63;
  const int64_t cap = row_cap(p);
  if (p.items == 0) {  // an item per request
    it.b = index;
    it.span = paged_span(p.lens[index], p.window, cap);
    it.j = 0;
    it.n = 1;
    it.first_item = index;
    it.stream = p.stream_units == 0;
    const int units = paged_units(it.span);
    const PagedRange r = paged_item_range(it.span, units, 0, 1);
    it.begin = r.begin;
    it.end = units ? r.end : r.begin;
    return true;
  }
  // the requests in runs, a run per lane; up to 64 requests one each, whose numbers stay in registers
  const int run = (p.B + 63) / 64, b0 = min(lane * run, p.B), b1 = min(b0 + run, p.B);
  int len = 0, own = 0, units = 0, n = 0;
  for (int b = b0; b < b1; ++b) {
    len = p.lens[b];
    own = paged_units(paged_span(len, p.window, cap));
    units += own;
  }
  const int all = lane_sums(units).all, chunk = paged_chunk(all, p.items);
  it.stream = all >= p.stream_units;
  if (run == 1) {
    n = paged_items(own, chunk);
  } else {
    for (int b = b0; b < b1; ++b)
      n += paged_items(paged_units(paged_span(p.lens[b], p.window, cap)), chunk);
  }
  const int upto = lane_sums(n).upto;
  const unsigned long long past = __ballot(upto > index);
  if (past == 0) return false;
  const int owner = __builtin_ctzll(past);
  it.first_item = __builtin_amdgcn_readlane(upto - n, owner);
  it.b = owner * run;
  if (run == 1) {
    len = __builtin_amdgcn_readlane(len, owner);
    own = __builtin_amdgcn_readlane(own, owner);
    it.n = __builtin_amdgcn_readlane(n, owner);
  } else {
    for (;; ++it.b) {
      len = p.lens[it.b];
      own = paged_units(paged_span(len, p.window, cap));
      it.n = paged_items(own, chunk);
      if (index < it.first_item + it.n) break;
      it.first_item += it.n;
    }
  }
  it.span = paged_span(len, p.window, cap);
  it.j = index - it.first_item;
  const PagedRange r = paged_item_range(it.span, own, it.j, it.n);
  it.begin = r.begin;
  it.end = r.end;
  return true;
}

__device__ inline Item uniform(const Item& x) {
  return Item{uniform(x.b),     uniform(x.j),   uniform(x.n),
              uniform(x.begin), uniform(x.end), uniform(x.first_item),
              uniform((int)x.stream) != 0,
              PagedSpan{uniform(x.span.first), uniform(x.span.len), uniform((int)x.span.ok) != 0}};
}

// The wave of a request's last keys stores the new token's key and value into the slot of position j
// at its start: its own later loads see them, and the row tiles of a key head each store the same
// bytes rather than wait for one another. (Kept in LDS until the last tile instead, a short request
// takes 0.2 us longer.)
template <int ES>
__device__ inline void store_new(const AttendParams& p, int b, int g, int j) {
  const int e = page_of(j / 16, p.div), per = p.d * ES / 16;
  const int64_t pg = p.table[b * p.table_stride + e], off = j - e * p.page;
  if (pg >= 0 && pg < p.pages) {
    const char* k = p.k_new + (b * p.knb + g * p.knh) * ES;
    const char* v = p.v_new + (b * p.vnb + g * p.vnh) * ES;
    char* kto = p.kpool + (pg * p.kpp + g * p.kph + off * p.kps) * ES;
    char* vto = p.vpool + (pg * p.vpp + g * p.vph + off * p.vps) * ES;
    for (int i = threadIdx.x & 63; i < 2 * per; i += 64) {
      const int c = (i < per ? i : i - per) * 16;
      *(u32x4*)((i < per ? kto : vto) + c) = *(const u32x4*)((i < per ? k : v) + c);
    }
  }
  wave_lds_sync();
}

// Attention over one item by a workgroup, its tiles in four runs, one a wave. Scores are K Q^T: a
// product's result then has a head per lane column and the keys in the very order that the second
// product, V^T P^T, takes its weights in, so weights never move between lanes and a head's statistics
// belong to its lanes. A lane's values are loaded a row at a time and turned into operands by
// byte permutes: no LDS, no transposed copy. Bound by the reading of K and V: a wave's next keys are in
// flight while it weighs the current values and the other way round; 16 lanes of 16 heads serve
// any group of query heads, as the matrix units wait for memory anyway. 1,048,577 tokens (bf16, 14 / 2
// heads of 64) 92 us with the join, 5.8 TB/s; a kernel that only reads as much takes 96 without the
// non-temporal hint and 88 with it. Equal shares that run on over several requests cost every short call 1 us or more
// for 2 % of a mixed batch. MT: tiles of 16 query heads served by one reading. ACROSS: the waves take
// a key head each, over all of the item's tiles.
template <int DT, int DP, int MT, bool ACROSS, int WPE>
__global__ __launch_bounds__(kAttendWaves * 64, WPE) void paged_attend_kernel(AttendParams p) {
  using T = Tile<DT, DP>;
  constexpr int NT = T::NT, NC = T::NC, VB = T::VB, LC = T::LC, LW = T::LW, NA = T::NA;
  constexpr int NW = kAttendWaves, HEADS = ACROSS ? NW : 1, NR = ACROSS ? 1 : NW / 2;
  __shared__ f32x4 red[NR][MT][ACROSS ? 1 : NA][64];
  __shared__ float red_m[NR][MT][64], red_l[NR][MT][64];
  const int wv = uniform(threadIdx.x >> 6);
  // row tiles of one (item, key head) are 8 workgroups apart: on one XCD, whose L2 they share
  const int id = blockIdx.x, rt = (id >> 3) % p.RT, unit = (id >> 3) / p.RT * 8 + (id & 7);
  const int groups = p.Hkv / HEADS, item = unit / groups;
  const int g = unit % groups * HEADS + (ACROSS ? wv : 0);
  Item found;
  if (unit >= p.units || !find_item(p, item, found)) return;
  const Item it = uniform(found);
  const int first = it.span.first, len = it.span.len;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int head0 = rt * MT * 16 + col;  // of MT tiles of 16 heads
  const int tiles = (it.end - it.begin + NT - 1) / NT;
  const int i0 = ACROSS ? 0 : uniform((int)((int64_t)tiles * wv / NW));
  const int i1 = ACROSS ? tiles : uniform((int)((int64_t)tiles * (wv + 1) / NW));

  __shared__ u32x4 q_lds[T::kQInLds ? MT : 1][T::kQInLds ? NC : 1][64];
  u32x4 q[MT][T::kQInLds ? 1 : NC];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (T::kQInLds && c % NW != wv) continue;
      const int at = c * 64 + grp * 16, head = head0 + mt * 16;
      u32x4 x = {0, 0, 0, 0};
      if (head < p.G && at < p.d * T::ES)
        x = *(const u32x4*)(p.q + (it.b * p.qb + (int64_t)(g * p.G + head) * p.qh) * T::ES + at);
      if constexpr (T::kQInLds) q_lds[mt][c][lane] = x;
      else q[mt][c] = x;
    }
  if constexpr (T::kQInLds) __syncthreads();

  const char* const kbase = p.kpool + g * p.kph * T::ES;
  const char* const vbase = p.vpool + g * p.vph * T::ES;
  const int64_t kpp = p.kpp * T::ES, vpp = p.vpp * T::ES;
  const int kps = (int)p.kps * T::ES, vps = (int)p.vps * T::ES, row_bytes = p.d * T::ES;

  const int koff = col * kps + grp * 16;
  int vcol[VB];
#pragma unroll
  for (int vb = 0; vb < VB; ++vb) {
    const int c = vb * T::CB * T::ES + col * LW * 4;
    vcol[vb] = c < row_bytes ? c : 0;  // columns past d are computed and not written
  }
  const int32_t* const row = p.table + it.b * p.table_stride;
  // page and offset of 64 subtiles at a time, one per lane; the next 64 are on their way
  int pid = 0, poff = 0, pid_next = 0, batch = it.begin + i0 * NT;
  unsigned long long bad = 0;
  const int sub_end = min(it.begin + i1 * NT, it.end);
  auto pages_at = [&](int s) {
    s += lane;
    return s < sub_end ? row[page_of(s, p.div)] : 0;
  };
  auto take_pages = [&](int x) {
    bad |= __ballot(x < 0 || x >= p.pages);
    pid = x < 0 || x >= p.pages ? 0 : x;
    poff = (batch + lane) * 16 - page_of(batch + lane, p.div) * p.page;
  };
  if (i0 < i1) {
    const int x = pages_at(batch);
    pid_next = pages_at(batch + 64);
    if (p.k_new && sub_end * 16 >= len) store_new<T::ES>(p, it.b, g, len - 1);
    take_pages(x);
  }

  Rows<DT, DP> rows;
  Softmax<NA> st[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    st[mt].m = -INFINITY;
    st[mt].l = 0.0f;
#pragma unroll
    for (int i = 0; i < NA; ++i) st[mt].acc[i] = f32x4{0, 0, 0, 0};
  }

  // pages of tile i's subtiles (the last one again past the wave's end)
  int64_t pg[NT];
  int off[NT];
  auto locate = [&](int i) {
    const int s = it.begin + i * NT;
    if (s >= batch + 64) {
      batch += 64;
      take_pages(pid_next);
      pid_next = pages_at(batch + 64);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int x = min(s + t, sub_end - 1) - batch;
      pg[t] = __builtin_amdgcn_readlane(pid, x);
      off[t] = __builtin_amdgcn_readlane(poff, x);
    }
  };
  auto load_k_as = [&](auto aux, int piece) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const Buffer src = buffer_at(kbase + (pg[t] * kpp + (int64_t)off[t] * kps));
#pragma unroll
      for (int c = 0; c < NC / T::KP; ++c) {
        const int at = (piece * (NC / T::KP) + c) * 64;
        rows.k[t][c] = __builtin_bit_cast(
            u32x4, load_words<4, aux.value>(src, at + grp * 16 < row_bytes ? koff + at : kOutside));
      }
    }
  };
  auto load_v_as = [&](auto aux, int i) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const Buffer src = buffer_at(vbase + (pg[t] * vpp + (int64_t)off[t] * vps));
      // rows that do not count may hold anything: read as zero
      const int lo = max(first - (it.begin + i * NT + t) * 16, 0);
      const int count = min(len - (it.begin + i * NT + t) * 16, 16) - lo;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = grp * 4 + r, at = (unsigned)(n - lo) < (unsigned)max(count, 0) ? n * vps
                                                                                    : kOutside;
#pragma unroll
        for (int vb = 0; vb < VB; ++vb)
          rows.v[t][r][vb] = load_words<LW, aux.value>(src, at + vcol[vb]);
      }
    }
  };
  constexpr bool kMayStream = DP < 512;  // there its second set of loads costs the registers
  using Plain = std::integral_constant<int, 0>;
  using Stream = std::integral_constant<int, kStream>;
  auto load_k = [&](int piece) {
    if (kMayStream && it.stream) load_k_as(Stream{}, piece);
    else load_k_as(Plain{}, piece);
  };
  auto load_v = [&](int i) {
    if (kMayStream && it.stream) load_v_as(Stream{}, i);
    else load_v_as(Plain{}, i);
  };

  if (i0 < i1) {
    locate(i0);
    load_k(0);
    load_v(i0);
  }
  for (int i = i0; i < i1; ++i) {
    const int j0 = (it.begin + i * NT) * 16;
    const bool edge = j0 < first || len - j0 < NT * 16;
    if constexpr (T::kQInLds) asm volatile("" ::: "memory");  // read the queries here, every time
    // scores: lane column a head, rows the keys 4 grp + r of each subtile
    // fp32 adds its products in kChains chains: against 64 bits one over the whole head left up to
    // 3.1 times the error of the same in plain operations, four 1.3 times at most, for 1.5% more
    // time or less (eight requests of up to 16K keys, 106.4 -> 107.9 us, on another box 110.3 -> 110.6). At 64 columns two are as
    // short, and four spilled.
    constexpr int kChains = DT != SSA_F32 ? 1 : DP == 64 ? 2 : 4;
    f32x4 s[MT][NT], chain[MT][NT][kChains];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < kChains; ++e) chain[mt][t][e] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      constexpr int per = NC / T::KP;
      if (c > 0 && c % per == 0) load_k(c / per);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        u32x4 qc;
        if constexpr (T::kQInLds) qc = q_lds[mt][c][lane];
        else qc = q[mt][c];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (DT == SSA_F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              f32x4& x = chain[mt][t][e % kChains];
              const unsigned int a = rows.k[t][c % per][e], b = qc[e];
              x = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a), __uint_as_float(b), x,
                                                       0, 0, 0);
            }
          } else {
            chain[mt][t][0] = mfma16(rows.k[t][c % per], qc, chain[mt][t][0], DT == SSA_BF16);
          }
        }
      }
    }
    const bool more = i + 1 < i1;
    if (more) {
      locate(i + 1);
      load_k(0);
    }
    constexpr int PARTS = kParts<DT>;
    u32x4 w[MT][PARTS];  // the weights in 16-bit parts
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      Softmax<NA>& o = st[mt];
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const auto& of = chain[mt][t];
          float x = of[0][r];
          if constexpr (kChains == 2) x += of[1][r];
          if constexpr (kChains == 4) x = (x + of[1][r]) + (of[2][r] + of[3][r]);
          x *= p.scale_log2;
          if (edge) {
            const int j = j0 + t * 16 + grp * 4 + r;
            if (j < first || j >= len) x = -INFINITY;
          }
          s[mt][t][r] = x;
          mx = fmaxf(mx, x);
        }
      mx = fmaxf(mx, lane_xor(mx, 16));
      mx = fmaxf(mx, lane_xor(mx, 32));
      if (__any(mx > o.m)) {  // a head without a finite score so far stays at -inf, its sums at 0
        const float m = fmaxf(o.m, mx);
        const float a = __builtin_amdgcn_exp2f(o.m - (m == -INFINITY ? 0.0f : m));
        o.m = m;
        o.l *= a;
#pragma unroll
        for (int n = 0; n < NA; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) o.acc[n][r] *= a;
      }
      const float base = (o.m == -INFINITY ? 0.0f : o.m) - T::kShift;
      float sum = 0.0f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[mt][t][r] = __builtin_amdgcn_exp2f(s[mt][t][r] - base);
          sum += s[mt][t][r];
        }
      o.l += sum;
      if constexpr (DT != SSA_F32) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            unsigned int x[PARTS];
            split<DT>(s[mt][t][2 * h], s[mt][t][2 * h + 1], x);
#pragma unroll
            for (int i = 0; i < PARTS; ++i) w[mt][i][2 * t + h] = x[i];
          }
      }
    }
#pragma unroll
    for (int vb = 0; vb < VB; ++vb)
#pragma unroll
      for (int e = 0; e < LC; ++e) {
        if constexpr (DT == SSA_F32) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                f32x4& acc = st[mt].acc[vb * LC + e];
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(
                    __uint_as_float(rows.v[t][r][vb].w[e]), s[mt][t][r], acc, 0, 0, 0);
              }
        } else {
          // column e of the lane's values, key after key
          u32x4 vt;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              vt[2 * t + h] = __builtin_amdgcn_perm(
                  rows.v[t][2 * h + 1][vb].w[e / 2], rows.v[t][2 * h][vb].w[e / 2],
                  e % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            f32x4& acc = st[mt].acc[vb * LC + e];
#pragma unroll
            for (int i = 0; i < PARTS; ++i) acc = mfma16(vt, w[mt][i], acc, DT == SSA_BF16);
          }
        }
      }
    if (more) load_v(i + 1);
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    st[mt].l += lane_xor(st[mt].l, 16);
    st[mt].l += lane_xor(st[mt].l, 32);
    if (bad != 0 || !it.span.ok) st[mt].l = NAN;
  }

  if constexpr (!ACROSS) {
    // the waves' results, half of them into the other half at a time
#pragma unroll
    for (int half = NW / 2; half >= 1; half >>= 1) {
      if (wv >= half && wv < 2 * half) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          red_m[wv - half][mt][lane] = st[mt].m;
          red_l[wv - half][mt][lane] = st[mt].l;
#pragma unroll
          for (int n = 0; n < NA; ++n) red[wv - half][mt][n][lane] = st[mt].acc[n];
        }
      }
      __syncthreads();
      if (wv < half) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          join(st[mt], red_m[wv][mt][lane], red_l[wv][mt][lane], &red[wv][mt][0][lane], 64);
      }
      __syncthreads();
    }
    if (wv != 0) return;
  }

  if (p.items != 0 && it.j == 0 && g == 0 && rt == 0 && lane == 0) {
    p.info[2 * it.b] = it.first_item;
    p.info[2 * it.b + 1] = it.n;
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const Softmax<NA>& o = st[mt];
    const int h = g * p.G + head0 + mt * 16;
    if (head0 + mt * 16 >= p.G) break;
    const float inv = len == 0 && it.span.ok ? 0.0f : 1.0f / o.l;
    const int64_t part = (int64_t)item * p.Hq + h, to = it.b * p.ob + h * p.oh;
#pragma unroll
    for (int vb = 0; vb < VB; ++vb)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < LC; e += 4) {
          const int c = vb * T::CB + LC * (grp * 4 + r) + e;
          if (c >= p.d) continue;
          f32x4 x;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = o.acc[vb * LC + e + i][r];
          if (it.n > 1) {
            *(f32x4*)(p.part + part * DP + c) = x;
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] *= inv;
            store_row4<DT>(p.out, to + c, x);
          }
        }
    if (grp != 0) continue;
    if (it.n > 1) {
      p.part_ml[part * 2] = o.m;
      p.part_ml[part * 2 + 1] = o.l;
    } else if (p.lse) {
      p.lse[(int64_t)it.b * p.Hq + h] = len == 0 && it.span.ok ? -INFINITY
          : (o.m - T::kShift + __builtin_amdgcn_logf(o.l)) * kLn2;
    }
  }
}

constexpr int kJoinBatch = 8;

// Joins a row's parts: a workgroup per (request, query head), DP / 4 threads across a part's row and
// the parts shared out over the workgroup's splits, kJoinBatch of them on their way at a time. Rows
// without keys, and of lengths that do not fit, are answered here. Bound by its chain of three memory
// latencies: 3.5 us for 14 rows of 33 parts, 6 for 2,048 rows of 1 to 12.
template <int DT, int DP, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_join_kernel(AttendParams p) {
  constexpr int PER = DP / 4, NS = THREADS / PER, WAVES = THREADS / 64;
  __shared__ f32x4 red[WAVES][PER < 64 ? PER : 64];
  __shared__ float red_m[WAVES], red_l[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6);
  const int h = blockIdx.x, b = blockIdx.y, c = tid % PER * 4, split = tid / PER;
  const int len = p.lens[b], first = p.info[2 * b], parts = p.info[2 * b + 1];
  const PagedSpan s = paged_span(len, p.window, row_cap(p));
  Softmax<1> st;
  st.m = -INFINITY;
  st.l = s.ok ? 0.0f : NAN;
  st.acc[0] = f32x4{0, 0, 0, 0};
  if (s.len > 0) {
    if (parts <= 1) return;  // written by its one item
    for (int i = split; i < parts; i += NS * kJoinBatch) {
      float m[kJoinBatch], l[kJoinBatch], mx = st.m;
      f32x4 a[kJoinBatch];
#pragma unroll
      for (int u = 0; u < kJoinBatch; ++u) {
        const int at = i + u * NS;
        const int64_t row = (int64_t)(first + at) * p.Hq + h;
        const bool in = at < parts;
        m[u] = in ? p.part_ml[row * 2] : -INFINITY;
        l[u] = in ? p.part_ml[row * 2 + 1] : 0.0f;
        a[u] = in ? *(const f32x4*)(p.part + row * DP + c) : f32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int u = 0; u < kJoinBatch; ++u) mx = fmaxf(mx, m[u]);
      const float base = mx == -INFINITY ? 0.0f : mx, x = __builtin_amdgcn_exp2f(st.m - base);
      st.m = mx;
      st.l *= x;
#pragma unroll
      for (int r = 0; r < 4; ++r) st.acc[0][r] *= x;
#pragma unroll
      for (int u = 0; u < kJoinBatch; ++u) {
        const float y = __builtin_amdgcn_exp2f(m[u] - base);
        st.l += l[u] * y;
#pragma unroll
        for (int r = 0; r < 4; ++r) st.acc[0][r] += a[u][r] * y;
      }
    }
    // splits within a wave, then the waves' (past 256 columns a split is two waves)
#pragma unroll
    for (int off = 32; off >= PER; off >>= 1) {
      f32x4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = lane_xor(st.acc[0][r], off);
      const float m = lane_xor(st.m, off), l = lane_xor(st.l, off);
      join(st, m, l, &o, 0);
    }
    constexpr int STEP = PER > 64 ? PER / 64 : 1;
    if (lane < PER) red[wv][lane] = st.acc[0];
    if (lane == 0) {
      red_m[wv] = st.m;
      red_l[wv] = st.l;
    }
    __syncthreads();
    if (tid >= PER) return;
#pragma unroll
    for (int w = STEP; w < WAVES; w += STEP)
      join(st, red_m[wv + w], red_l[wv + w], &red[wv + w][lane], 0);
  }
  if (tid >= PER) return;
  const float inv = s.len == 0 && s.ok ? 0.0f : 1.0f / st.l;
#pragma unroll
  for (int r = 0; r < 4; ++r) st.acc[0][r] *= inv;
  if (c < p.d) store_row4<DT>(p.out, b * p.ob + h * p.oh + c, st.acc[0]);
  if (p.lse && tid == 0)
    p.lse[(int64_t)b * p.Hq + h] = s.len == 0 && s.ok ? -INFINITY
        : (st.m - (DT == SSA_F16 ? kF16Shift : 0.0f) + __builtin_amdgcn_logf(st.l)) * kLn2;
}

// Whether a call is one launch, a request an item: no request passes 512 keys (8 us a call; parts and
// their join 11), or 2048 in 512 or more (request, key head, row tile) triples (256 x 1,000 keys, 4 key
// heads: 48 us; cut 60). With few triples and more keys the cut wins: 2,000 keys of 8 heads 12 and 24.
// What a request may reach counts, the table's width, as the lengths are the device's: 64 requests of 100
// to 500 keys (8 key heads of 128) 18.8 us in a table of 496, 24.6 in one of 32,768; of 2 heads of 64 7.7
// and 10.1.
bool one_launch(int64_t triples, int64_t units) {
  return units <= 4 || (units <= 16 && triples >= 512);
}

// Whether a wave serves two tiles of 16 query heads from one reading of the keys and values (past head
// dim 128 their registers do not fit). It makes fewer, longer workgroups: 16-bit calls that may read
// more than the caches hold win (128 requests of 2,000 to 9,000 keys, 20 heads of 128 on one: 77 us
// for 84; 64 of 2,000 to 20,000, 48 on two: 124 for 137), smaller ones lose (64 of 500 to 4,000, 32 on
// one: 23 for 19); in fp32 the matrix products count too (8 of 2,000 to 9,000, 40 on two: 26 for 31).
//
// A workgroup's waves take a key head each instead of a run of keys each where a token's heads lie side
// by side (token-major pools): four rows of 128 or 256 bytes are then read at about the same time, one at
// a time leaves memory at 5.4 TB/s of 6.1: 64 requests of 64 to 32,768 keys (8 heads of 128, 16-bit)
// 235 us for 250, 16 of 8,192 100 for 114 (of head dim 64 55 for 67). Longer rows gain nothing (fp32 63 for
// 61), heads that lie apart lose (235 for 219), and so do calls of little to read, whose waves then have
// four tiles each to begin with (one of 4,096 keys 15 for 13; one of 32,768 33 for 30).
constexpr int64_t kAcrossBytes = (int64_t)32 << 20;

enum Serve { kOneTile, kTwoTiles, kAcross };

bool may_serve_two(int64_t G, int64_t d) { return G > 16 && d <= 128; }
bool may_serve_across(int64_t G, int64_t Hkv, int64_t d) {
  return G <= 16 && Hkv % kAttendWaves == 0 && d <= 128;
}

// strides: kpool's and vpool's (page, head, slot)
Serve serve(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t d, int64_t W, int64_t page,
            int64_t window, const int64_t* strides) {
  const int64_t units = paged_most_units(W * page, (int)window);
  // whether the call may read so much
  auto reads = [&](int64_t bytes) { return B * units >= bytes / unit_bytes(dtype, d, Hkv); };
  if (may_serve_two(Hq / Hkv, d) && (dtype == SSA_F32 || reads(kStreamBytes))) return kTwoTiles;
  if (may_serve_across(Hq / Hkv, Hkv, d) && dtype != SSA_F32 && strides[1] < strides[2] &&
      strides[4] < strides[5] && B > 1 && reads(kAcrossBytes) && !one_launch(B * Hkv, units))
    return kAcross;
  return kOneTile;
}

// How a call of these sizes is cut: known on the host without the lengths.
// Unless it is one launch, items for about `target` workgroups, what the CUs hold at once (four a CU at
// head dim 64, two at 256, one at 512; three at 128, and there twice as many even out uneven lengths
// better: 64 mixed requests 267 us for 1536, 286 for 768). A single request is even by itself and has the
// most parts to join: 512 (1M tokens 102 us, 106 for 1024).
struct Layout {
  int64_t RT, items, max_items;  // items: 0 when every request is one item
  int dp;
  size_t part_ml, info, bytes;  // offsets into the workspace, which starts with the parts
};

Layout layout(int64_t B, int64_t Hq, int64_t Hkv, int64_t d, int64_t W, int64_t page,
              int64_t window, Serve how) {
  Layout y{};
  const bool two = how == kTwoTiles;
  const int64_t heads = how == kAcross ? Hkv / kAttendWaves : Hkv;  // of a workgroup each
  y.RT = (Hq / Hkv + (two ? 31 : 15)) / (two ? 32 : 16);
  y.dp = d <= 64 ? 64 : d <= 128 ? 128 : d <= 256 ? 256 : 512;
  const int64_t units = paged_most_units(W * page, (int)window);
  y.max_items = B;
  if (one_launch(B * Hkv * y.RT, units)) return y;
  const int64_t target = y.dp == 512             ? 256
                         : y.dp == 256 || B == 1 ? 512
                         : y.dp == 128           ? (two ? 1024 : 1536)
                                                 : 1024;
  y.items = std::max<int64_t>(1, target / (heads * y.RT));
  y.max_items = paged_most_items(B, y.items, units);
  const size_t parts = (size_t)y.max_items * Hq;
  y.part_ml = parts * y.dp * 4;
  y.info = y.part_ml + parts * 2 * 4;
  y.bytes = (y.info + (size_t)B * 8 + 15) / 16 * 16;
  return y;
}

template <int DT, int DP, int MT, bool ACROSS, int WPE>
int run_attend(const AttendParams& p, int64_t blocks, hipStream_t st) {
  paged_attend_kernel<DT, DP, MT, ACROSS, WPE><<<(unsigned)blocks, kAttendWaves * 64, 0, st>>>(p);
  SSA_TRY(launch_status("paged_attend_kernel"));
  if (p.items == 0) return SSA_OK;
  // 16 to 4 splits of a row's parts; 1024 threads take 10 us more for 4,096 rows of a few parts, and
  // 256 at head dim 512 (2 splits) 1.6 us more for 128 rows
  constexpr int JOIN = DP <= 128 ? 256 : 512;
  paged_join_kernel<DT, DP, JOIN><<<dim3(p.Hq, p.B), JOIN, 0, st>>>(p);
  return launch_status("paged_join_kernel");
}

template <int DT>
int run_attend_dim(const AttendParams& p, int dp, Serve how, int64_t blocks, hipStream_t st) {
  const bool two = how == kTwoTiles;
  if constexpr (DT != SSA_F32) {
    if (how == kAcross)
      return dp == 64 ? run_attend<DT, 64, 1, true, 4>(p, blocks, st)
                      : run_attend<DT, 128, 1, true, 3>(p, blocks, st);
  }
  switch (dp) {
    case 64:
      if (two) return run_attend<DT, 64, 2, false, DT == SSA_F32 ? 2 : 3>(p, blocks, st);
      return run_attend<DT, 64, 1, false, DT == SSA_F32 ? 3 : 4>(p, blocks, st);
    case 128:
      if (two) return run_attend<DT, 128, 2, false, 2>(p, blocks, st);
      return run_attend<DT, 128, 1, false, 3>(p, blocks, st);
    case 256: return run_attend<DT, 256, 1, false, 2>(p, blocks, st);
    default: return run_attend<DT, 512, 1, false, 1>(p, blocks, st);
  }
}

}  // namespace
}  // namespace ssa

using namespace ssa;

extern "C" int ssa_paged_resize(int32_t* lens, const int32_t* new_lens, int32_t* table,
                                int64_t table_stride, int64_t B, int64_t W, int64_t page,
                                int32_t* free_pages, int64_t pages, int32_t* nfree,
                                int64_t* slots, int32_t* pos, int64_t T, int32_t* cu,
                                int32_t* status, ssa_stream_t stream) {
  SSA_REQUIRE(lens && new_lens && table && free_pages && nfree && cu && status, SSA_ERR_INVALID,
              "ssa_paged_resize: NULL argument");
  SSA_REQUIRE(B > 0 && fits_int(B) && W > 0 && table_stride >= W && pages > 0 && fits_int(pages),
              SSA_ERR_INVALID, "ssa_paged_resize: bad shape (B=%lld, W=%lld, pages=%lld)",
              (long long)B, (long long)W, (long long)pages);
  SSA_REQUIRE(page > 0 && page % 16 == 0 && page <= 65536, SSA_ERR_UNSUPPORTED,
              "ssa_paged_resize: page of %lld tokens (a multiple of 16 up to 65536)",
              (long long)page);
  SSA_REQUIRE(W <= 0x7fffffff / page, SSA_ERR_UNSUPPORTED,
              "ssa_paged_resize: a table row of %lld pages holds more than 2^31 - 1 tokens",
              (long long)W);
  SSA_REQUIRE(fits_int(T) && (T == 0 || slots), SSA_ERR_INVALID,
              "ssa_paged_resize: T=%lld slots", (long long)T);
  ResizeParams p{lens,  new_lens, table, table_stride, B, W,  (int)page, free_pages,
                 pages, nfree,    slots, pos,          T, cu, status,    page_div((int)page / 16)};
  hipStream_t st = (hipStream_t)stream;
  paged_resize_kernel<<<1, kResizeThreads, 0, st>>>(p);
  SSA_TRY(launch_status("paged_resize_kernel"));
  if (T > kSlotsInside) {
    paged_slots_kernel<<<(unsigned)((T + 255) / 256), 256, 0, st>>>(p);
    SSA_TRY(launch_status("paged_slots_kernel"));
  }
  return SSA_OK;
}

extern "C" int ssa_paged_append(const void* k, const void* v, void* kpool, void* vpool, int dtype,
                                int64_t T, int64_t Hkv, int64_t d, int64_t pages, int64_t page,
                                const int64_t* strides, const int64_t* slots,
                                ssa_stream_t stream) {
  SSA_REQUIRE(k && v && kpool && vpool && strides && slots, SSA_ERR_INVALID,
              "ssa_paged_append: NULL argument");
  SSA_TRY(check_pool("ssa_paged_append", dtype, Hkv, d, pages, page));
  SSA_REQUIRE(fits_int(T), SSA_ERR_INVALID, "ssa_paged_append: T=%lld tokens", (long long)T);
  const int es = dtype_size(dtype);
  SSA_REQUIRE(rows16(k, strides, 2, es) && rows16(v, strides + 2, 2, es) &&
                  rows16(kpool, strides + 4, 3, es) && rows16(vpool, strides + 7, 3, es),
              SSA_ERR_INVALID, "ssa_paged_append: rows must start at multiples of 16 bytes");
  if (T == 0) return SSA_OK;
  AppendParams p{(const char*)k, (const char*)v, (char*)kpool, (char*)vpool, slots, T, pages,
                 (int)page, (int)Hkv, (int)(d * es / 16),
                 strides[0] * es, strides[1] * es, strides[2] * es, strides[3] * es,
                 strides[4] * es, strides[5] * es, strides[6] * es, strides[7] * es,
                 strides[8] * es, strides[9] * es};
  const int64_t blocks = (T * p.Hkv * p.vecs + 255) / 256;
  SSA_REQUIRE(fits_launch(blocks, 256), SSA_ERR_UNSUPPORTED, "ssa_paged_append: %lld tokens in one call",
              (long long)T);
  paged_append_kernel<<<(unsigned)blocks, 256, 0, (hipStream_t)stream>>>(p);
  return launch_status("paged_append_kernel");
}

extern "C" size_t ssa_paged_attend_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t d,
                                                  int64_t W, int64_t page, int64_t window) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || d <= 0 || d > 512 || W <= 0 || page <= 0 ||
      !fits_int(window) || W > 0x7fffffff / page)
    return 0;
  const size_t one = layout(B, Hq, Hkv, d, W, page, window, kOneTile).bytes;
  if (may_serve_two(Hq / Hkv, d))
    return std::max(one, layout(B, Hq, Hkv, d, W, page, window, kTwoTiles).bytes);
  if (may_serve_across(Hq / Hkv, Hkv, d))
    return std::max(one, layout(B, Hq, Hkv, d, W, page, window, kAcross).bytes);
  return one;
}

extern "C" int ssa_paged_attend(const void* q, void* kpool, void* vpool, void* out, float* lse,
                                int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t d,
                                int64_t pages, int64_t page, const int32_t* table,
                                int64_t table_stride, int64_t W, const int32_t* lens,
                                const void* k_new, const void* v_new, const int64_t* strides,
                                float scale, int64_t window, const int32_t* status,
                                void* workspace, size_t workspace_bytes,
                                ssa_stream_t stream) {
  SSA_REQUIRE(q && kpool && vpool && out && table && lens && strides, SSA_ERR_INVALID,
              "ssa_paged_attend: NULL argument");
  SSA_REQUIRE((k_new == nullptr) == (v_new == nullptr), SSA_ERR_INVALID,
              "ssa_paged_attend: k_new and v_new come together");
  SSA_TRY(check_pool("ssa_paged_attend", dtype, Hkv, d, pages, page));
  SSA_REQUIRE(B > 0 && B <= 65535 && Hq > 0 && Hq <= 65535 && Hq % Hkv == 0, SSA_ERR_INVALID,
              "ssa_paged_attend: B=%lld, Hq=%lld, Hkv=%lld (at most 65535 rows; Hq a multiple of "
              "Hkv)", (long long)B, (long long)Hq, (long long)Hkv);
  SSA_REQUIRE(W > 0 && table_stride >= W && W <= 0x7fffffff / page, SSA_ERR_INVALID,
              "ssa_paged_attend: table of %lld pages a row, stride %lld (at most 2^31 - 1 tokens)",
              (long long)W, (long long)table_stride);
  SSA_REQUIRE(fits_int(window), SSA_ERR_INVALID, "ssa_paged_attend: window %lld",
              (long long)window);
  const int es = dtype_size(dtype);
  // strides: q(b,h), kpool(page,head,slot), vpool(page,head,slot), out(b,h), k_new(b,h), v_new(b,h)
  SSA_REQUIRE(rows16(q, strides, 2, es) && rows16(kpool, strides + 2, 3, es) &&
                  rows16(vpool, strides + 5, 3, es) && rows16(out, strides + 8, 2, es) &&
                  (!k_new || (rows16(k_new, strides + 10, 2, es) &&
                              rows16(v_new, strides + 12, 2, es))),
              SSA_ERR_INVALID, "ssa_paged_attend: rows must start at multiples of 16 bytes");
  SSA_REQUIRE(strides[4] < (1 << 24) && strides[7] < (1 << 24), SSA_ERR_UNSUPPORTED,
              "ssa_paged_attend: slots 2^24 elements apart or more");
  SSA_REQUIRE(B * paged_most_units(W * page, (int)window) <= 0x7fffffff, SSA_ERR_UNSUPPORTED,
              "ssa_paged_attend: %lld table rows of %lld tokens (2^38 in all at most)",
              (long long)B, (long long)(W * page));
  const Serve how = serve(dtype, B, Hq, Hkv, d, W, page, window, strides + 2);
  const Layout y = layout(B, Hq, Hkv, d, W, page, window, how);
  SSA_REQUIRE(workspace_bytes >= y.bytes && (y.bytes == 0 || (workspace && aligned16(workspace))),
              SSA_ERR_WORKSPACE, "ssa_paged_attend: needs a 16-byte aligned workspace of %zu bytes, "
              "got %zu", y.bytes, workspace_bytes);
  AttendParams p{};
  p.q = (const char*)q;
  p.kpool = (char*)kpool;
  p.vpool = (char*)vpool;
  p.out = (char*)out;
  p.lse = lse;
  p.k_new = (const char*)k_new;
  p.v_new = (const char*)v_new;
  p.table = table;
  p.lens = lens;
  p.status = status;
  p.table_stride = table_stride;
  p.cap = W * page;
  p.pages = pages;
  p.B = (int)B;
  p.Hq = (int)Hq;
  p.Hkv = (int)Hkv;
  p.G = (int)(Hq / Hkv);
  p.d = (int)d;
  p.page = (int)page;
  p.window = (int)window;
  p.scale_log2 = scale * kLog2e;
  int64_t* const st[14] = {&p.qb, &p.qh, &p.kpp, &p.kph, &p.kps, &p.vpp, &p.vph,
                           &p.vps, &p.ob, &p.oh, &p.knb, &p.knh, &p.vnb, &p.vnh};
  for (int i = 0; i < (k_new ? 14 : 10); ++i) *st[i] = strides[i];
  p.div = page_div((int)page / 16);
  p.RT = (int)y.RT;
  p.items = (int)y.items;
  // What does not fit the 256 MB last-level cache is read past it: 537 MB 94 us with the hint, 102
  // without; 105 MB that the cache holds 30 and 27. Row tiles read it twice, the second time from L2:
  // 300 MB with two of them 110 us with the hint, 83 without.
  p.stream_units = y.RT > 1 ? INT64_MAX : kStreamBytes / unit_bytes(dtype, d, Hkv);
  if (y.items == 0 && B * paged_most_units(W * page, (int)window) >= p.stream_units)
    p.stream_units = 0;
  p.part = (float*)workspace;
  p.part_ml = (float*)((char*)workspace + y.part_ml);
  p.info = (int32_t*)((char*)workspace + y.info);
  const int64_t units = y.max_items * (how == kAcross ? Hkv / kAttendWaves : Hkv);
  const int64_t blocks = (units + 7) / 8 * 8 * y.RT;
  SSA_REQUIRE(fits_launch(blocks, kAttendWaves * 64), SSA_ERR_UNSUPPORTED,
              "ssa_paged_attend: too many rows in one call");
  p.units = (int)units;
  hipStream_t hs = (hipStream_t)stream;
  if (dtype == SSA_F32) return run_attend_dim<SSA_F32>(p, y.dp, how, blocks, hs);
  if (dtype == SSA_F16) return run_attend_dim<SSA_F16>(p, y.dp, how, blocks, hs);
  return run_attend_dim<SSA_BF16>(p, y.dp, how, blocks, hs);
}

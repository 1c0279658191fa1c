// Drafted tokens over the paged key-value cache: their masks and positions from their parents, their
// attention over the cache (every one over the context and its own ancestors), and the accepted ones
// moved together.
//
// Request b's drafted tokens are rows [cu[b], cu[b + 1]) of a call's N and the last n = cu[b + 1] -
// cu[b] of its lens[b] tokens of the cache.
#include <float.h>

#include <algorithm>

#include "paged_parts.h"

namespace ssa {
namespace {

constexpr int kMaxWords = 32;  // of a mask: 1024 drafted tokens a request

// ---- parents -> masks, positions ---------------------------------------------------------------

struct MaskParams {
  const int32_t* parents;
  const int32_t* cu;
  const int32_t* lens;
  int32_t* masks;
  int32_t* pos;
  int64_t N;
  int B, words;
  int first;  // the launch's first request
  bool all;   // whether each of its workgroups looks at all offsets
};

// A token's way up so far: the next ancestor's place plus 1 (0: none), the tokens on the way, and
// whether one of them has a parent that does not fit.
__device__ inline unsigned int way(int anc, int steps, bool bad) {
  return (unsigned)(anc + 1) | (unsigned)steps << 16 | (bad ? 1u << 31 : 0);
}

// A workgroup for a request and four words of its masks, a thread a token. Every round joins a token's
// way with that of the ancestor where it ends, so its length doubles: a chain of 1024 takes ten rounds.
// The last workgroups answer the rows that no request's offsets hold, and all rows where the offsets
// descend (they may be two requests' then). Bound by launch and barrier latency: 64 trees of up to 64 tokens
// 3.7 us, 8 of 1,024 11.4.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void paged_draft_masks_kernel(MaskParams p) {
  __shared__ unsigned int ways[THREADS];
  __shared__ u32x4 seen[THREADS];
  const int b = p.first + blockIdx.x, t = threadIdx.x, w0 = blockIdx.y * 4;
  const int count = min(4, p.words - w0);
  auto store = [&](int64_t row, const u32x4& m, int pos) {
    for (int i = 0; i < count; ++i) p.masks[row * p.words + w0 + i] = m[i];
    if (w0 == 0) p.pos[row] = pos;
  };
  bool falls = false;
  if (p.all)
    for (int i = t; i < p.B; i += THREADS) falls |= p.cu[i + 1] < p.cu[i];
  if (b == p.B) {
    falls = __syncthreads_or(falls);
    const int end = p.cu[p.B];
    const int64_t first = falls || end < 0 ? p.N : min((int64_t)max(p.cu[0], 0), p.N);
    for (int64_t row = t; row < first; row += THREADS) store(row, u32x4{}, -1);
    for (int64_t row = max((int64_t)end, first) + t; row < p.N; row += THREADS) store(row, u32x4{}, 0);
    return;
  }
  const int c0 = p.cu[b], c1 = p.cu[b + 1];
  const DraftSpan s = draft_span(p.lens[b], c0, c1, p.N, 0, p.words, 0x7fffffff);
  const bool mine = s.span.ok && t < s.n;
  const int parent = mine ? p.parents[(int64_t)c0 + t] : -1;
  if (__syncthreads_or(falls)) return;
  if (!s.span.ok) {  // of offsets that pass the rows, those that are there
    const int64_t to = min((int64_t)c1, p.N);
    for (int64_t row = max(c0, 0) + t; row < to; row += THREADS) store(row, u32x4{}, -1);
    return;
  }
  const bool bad = parent < -1 || parent >= t;
  unsigned int own = way(bad ? -1 : parent, 1, mine && bad);
  u32x4 m{};
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = t >> 5 == w0 + i ? 1u << (t & 31) : 0;
  ways[t] = own;
  seen[t] = m;
  while (__syncthreads_or((own & 0xffff) != 0)) {
    const int at = (int)(own & 0xffff) - 1;
    if (at >= 0) {
      const unsigned int up = ways[at];
      m |= seen[at];
      own = (up & 0xffff) | (own & 0x7fff0000u) + (up & 0x7fff0000u) | ((own | up) & 1u << 31);
    }
    __syncthreads();
    ways[t] = own;
    seen[t] = m;
  }
  if (!mine) return;
  const bool fits = own >> 31 == 0;
  store((int64_t)c0 + t, fits ? m : u32x4{}, fits ? s.ctx + (int)(own >> 16 & 0x7fff) - 1 : -1);
}

// Up to so many requests every workgroup looks at all offsets; past them the last ones do, in a launch of
// their own that finds all rows written.
constexpr int64_t kMaskScan = 1024;

// ---- attention of drafted tokens ---------------------------------------------------------------

struct DraftParams {
  const char* q;
  const char* kpool;
  const char* vpool;
  char* out;
  float* lse;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;
  const int32_t* masks;   // NULL: a chain
  const int32_t* pos;
  const int32_t* status;  // of the resize before, or NULL
  int64_t table_stride, cap, pages, N;
  int B, Hq, Hkv, G, d, page, window, words;
  bool clear;  // rows behind the last token become zeros
  float scale_log2;
  int64_t qt, qh, ot, oh;                // elements
  int64_t kpp, kph, kps, vpp, vph, vps;  // elements
  PageDiv div;           // by the subtiles of a page
  int64_t stream_units;  // units of a key head from which a call streams
  int64_t items;         // items aimed at, 0: no row tile is cut
  int64_t blocks;        // workgroups for row tiles; kRestBlocks more follow
  int64_t max_parts;     // row tiles of parts that the workspace holds
  float* part;           // (part, row of the tile, DP)
  float* part_ml;        // (part, row of the tile, 2): their m and l
  int32_t* info;         // per request: its first part and the splits of its row tiles
};

constexpr int kRestBlocks = 8;

// What one workgroup does: split j of n of a row tile of request b and key head g.
struct DraftItem {
  int b, g, tile, tiles, j, n, begin, end, past, first_part, c0;  // past: the end of its share of the pages
  bool stream;
  DraftSpan s;
};

__device__ inline DraftSpan draft_of(const DraftParams& p, int b) {
  return draft_span(p.lens[b], p.cu[b], p.cu[b + 1], p.N, p.window, p.words, p.cap);
}

// Finds workgroup `id`'s item from the lengths alone, each wave for itself: every lane sums a run of
// requests, the wave adds the runs up. Of the call's row tiles an XCD takes a run, the tiles of the
// same keys next to each other: its L2 serves them together. False past the last one, and for all where
// the offsets descend (rest_rows answers). (Equal shares of all units instead, a workgroup going on from one
// row tile to the next, cost a short call 8 us, and a mixed batch 550 us for 313: a unit takes as long with
// few rows as with many.)
template <int M>
__device__ inline bool find_draft(const DraftParams& p, int id, DraftItem& it) {
  const int lane = threadIdx.x & 63;
  const int run = (p.B + 63) / 64, b0 = min(lane * run, p.B), b1 = min(b0 + run, p.B);
  DraftSpan own{};
  int units = 0, tiles = 0;
  float work = 0.0f;
  bool falls = false;
  for (int b = b0; b < b1; ++b) {
    own = draft_of(p, b);
    falls |= p.cu[b + 1] < p.cu[b];
    units = draft_units(own);
    tiles = draft_tiles(own, p.G, M);
    work += (float)tiles * (float)units;
  }
  if (__any(falls)) return false;
  int chunk = 0x7fffffff;
  it.stream = p.stream_units == 0;
  if (p.items != 0) {
    const float all = lane_sums(work).all;
    chunk = draft_chunk(all, (float)p.items);
    it.stream = all >= (float)p.stream_units;
  }
  int n = 0, parts = 0;
  auto count = [&](int of, int u) {
    const int splits = paged_items(u, chunk);
    n += of * splits;
    parts += splits > 1 ? of * splits : 0;
  };
  if (run == 1) {
    count(tiles, units);
  } else {
    for (int b = b0; b < b1; ++b) {
      const DraftSpan s = draft_of(p, b);
      count(draft_tiles(s, p.G, M), draft_units(s));
    }
  }
  const LaneSums<int> sums = lane_sums(n);
  const int all = sums.all * p.Hkv, per = (int)(((unsigned)all + 7u) / 8u);
  const int index = (id & 7) * per + (id >> 3);
  if ((id >> 3) >= per || index >= all) return false;
  const unsigned long long past = __ballot(sums.upto * p.Hkv > index);
  if (past == 0) return false;
  const int owner = __builtin_ctzll(past);
  const LaneSums<int> part_sums = lane_sums(parts);
  int first = __builtin_amdgcn_readlane(sums.upto - n, owner);
  int part = __builtin_amdgcn_readlane(part_sums.upto - parts, owner);
  it.b = owner * run;
  for (;; ++it.b) {
    it.s = draft_of(p, it.b);
    units = draft_units(it.s);
    tiles = draft_tiles(it.s, p.G, M);
    it.n = paged_items(units, chunk);
    if (run == 1 || it.b + 1 >= min((owner + 1) * run, p.B) ||
        index < (first + tiles * it.n) * p.Hkv) break;
    first += tiles * it.n;
    part += it.n > 1 ? tiles * it.n : 0;
  }
  const unsigned int at = (unsigned)(index - first * p.Hkv);
  if (tiles <= 0 || at / (unsigned)tiles >= (uint64_t)it.n * p.Hkv) return false;
  it.c0 = p.cu[it.b];
  it.tiles = tiles;
  const unsigned int row = at / (unsigned)tiles;
  it.tile = (int)(at - row * tiles);
  it.j = (int)(row / (unsigned)p.Hkv);
  it.g = (int)(row - (unsigned)it.j * p.Hkv);
  it.stream = it.stream && it.tiles == 1;
  // a bound on what is written: offsets that ascend make no more parts than the workspace holds
  const int64_t part0 = (int64_t)part * p.Hkv, part_end = part0 + (int64_t)tiles * it.n * p.Hkv;
  it.first_part = it.n > 1 && (part < 0 || part_end > p.max_parts) ? -1 : (int)part0;
  it.begin = it.end = it.past = 0;
  if (it.s.span.ok) {
    const PagedRange r = paged_item_range(it.s.span, units, it.j, it.n);
    it.begin = r.begin;
    it.end = it.past = r.end;
    if (!p.masks) {  // a chain: none of the tile's tokens attends keys past its last one
      const unsigned int last = ((unsigned)it.tile * M + M - 1) / (unsigned)p.G;
      const int seen = (it.s.ctx + (int)min(last, (unsigned)it.s.n - 1)) / 16 + 1;
      it.end = min(it.end, max(seen, it.begin));
    }
  }
  return true;
}

__device__ inline DraftItem uniform(const DraftItem& x) {
  return DraftItem{uniform(x.b),     uniform(x.g),   uniform(x.tile), uniform(x.tiles),
                   uniform(x.j),     uniform(x.n),   uniform(x.begin), uniform(x.end),
                   uniform(x.past),  uniform(x.first_part), uniform(x.c0), uniform((int)x.stream) != 0,
                   DraftSpan{uniform(x.s.ctx), uniform(x.s.n),
                             PagedSpan{uniform(x.s.span.first), uniform(x.s.span.len),
                                       uniform((int)x.s.span.ok) != 0}}};
}

// Which of the 64 keys from j0 on a row attends: bit j - j0. tok, pos: the row's place among its request's n
// drafted tokens and its position.
__device__ inline uint64_t attended_keys(const DraftParams& p, const DraftItem& it, int tok, int pos, int j0) {
  const int ctx = it.s.ctx, i0 = j0 - ctx;  // the first key's place among the drafted ones
  const int64_t start = p.window > 0 ? (int64_t)pos - p.window + 1 : 0;  // below 0: keys' positions may be too
  auto below = [](int64_t x) { return x <= 0 ? 0ull : x >= 64 ? ~0ull : (1ull << x) - 1; };
  const uint64_t context = below(-(int64_t)i0) & ~below(start - j0);
  if (i0 + 64 <= 0) return context;
  uint64_t bits;
  if (!p.masks) {
    bits = below((int64_t)tok - i0 + 1) & ~below(start - j0);
  } else {
    const int32_t* const words = p.masks + ((int64_t)it.c0 + tok) * p.words;
    auto word = [&](int w) { return w >= 0 && w < p.words ? (uint64_t)(unsigned)words[w] : 0ull; };
    const int w = i0 >> 5, r = i0 & 31;
    const uint64_t lo = word(w) | word(w + 1) << 32;
    bits = r ? lo >> r | word(w + 2) << (64 - r) : lo;
    bits &= below((int64_t)it.s.n - i0);
    if (p.window > 0) {
      for (uint64_t left = bits; left; left &= left - 1) {
        const int x = __builtin_ctzll(left);
        if (p.pos[(int64_t)it.c0 + i0 + x] < start) bits &= ~(1ull << x);
      }
    }
  }
  return context | (bits & ~below(-(int64_t)i0) & below((int64_t)it.s.n - i0));
}

// Whether pages that an item's tile does not read, of tokens past all of its own, are in the table's row but
// not in the pool: they make the request one that does not fit all the same.
__device__ inline bool bad_past(const DraftParams& p, const DraftItem& it, const int32_t* row) {
  bool bad = false;
  for (int s = it.end + (int)(threadIdx.x & 63); s < it.past; s += 64) {
    const int x = row[page_of(s, p.div)];
    bad |= x < 0 || x >= p.pages;
  }
  return __any(bad);
}

// Rows that no request's items answer, by block `id` of kRestBlocks: those behind the last request's become
// zeros where the call wants them cleared; NaN are those before the first, those of requests whose offsets
// pass the rows, and all of them where the offsets descend or the resize was refused.
template <int DT>
__device__ inline void rest_rows(const DraftParams& p, int id) {
  constexpr int ES = DT == SSA_F32 ? 4 : 2;
  __shared__ int s_lo, s_hi;  // the first and last offset among the rows
  const int tid = threadIdx.x;
  if (tid == 0) {
    s_lo = 0x7fffffff;
    s_hi = -1;
  }
  __syncthreads();
  int lo = 0x7fffffff, hi = -1;
  bool falls = false;
  for (int b = tid; b <= p.B; b += 256) {
    const int c = p.cu[b];
    if (c >= 0) lo = min(lo, c);
    if (c <= p.N) hi = max(hi, c);
    falls |= b > 0 && c < p.cu[b - 1];
  }
  if (lo != 0x7fffffff) atomicMin(&s_lo, lo);
  if (hi >= 0) atomicMax(&s_hi, hi);
  falls = __syncthreads_or(falls);
  if (falls && p.items != 0)  // nothing to join
    for (int b = id * 256 + tid; b < p.B; b += kRestBlocks * 256) p.info[2 * b + 1] = 1;
  const int end = p.cu[p.B];
  const bool fits = end >= 0 && end <= p.N;
  const int64_t first = falls || (p.status && *p.status != 0) ? p.N : min((int64_t)s_lo, p.N);
  const int64_t last = fits && !p.clear ? p.N : max((int64_t)s_hi, first);
  const int per = p.d * ES / 16;
  const int64_t rows = (first + p.N - last) * p.Hq;
  for (int64_t i = id * 256 + tid; i < rows * per; i += kRestBlocks * 256) {
    const int64_t row = i / per, n = row / p.Hq, h = row - n * p.Hq, t = n < first ? n : last + n - first;
    const bool bad = n < first || !fits;
    const int64_t to = t * p.ot + h * p.oh + (i - row * per) * (16 / ES);
    const float x = bad ? NAN : 0.0f;
    const f32x4 v = {x, x, x, x};
    store_row4<DT>(p.out, to, v);
    if constexpr (ES == 2) store_row4<DT>(p.out, to + 4, v);
    if (p.lse && i == row * per) p.lse[t * p.Hq + h] = bad ? NAN : -INFINITY;
  }
}

// The value a row's sums give: m -INFINITY: no key is attended; l NaN: the row is answered as bad.
__device__ inline float row_scale(float m, float l) {
  return l != l ? NAN : m == -INFINITY ? 0.0f : 1.0f / l;
}

__device__ inline float row_lse(float m, float l, float shift) {
  return l != l ? NAN : m == -INFINITY ? -INFINITY
                                       : (m - shift + __builtin_amdgcn_logf(l)) * kLn2;
}

// Whether a 16-bit (two a word) or 32-bit value is infinite or NaN.
template <int DT>
__device__ inline bool not_finite(unsigned int w) {
  if constexpr (DT == SSA_F32) return (w & 0x7f800000u) == 0x7f800000u;
  constexpr unsigned int e = DT == SSA_BF16 ? 0x7f80u : 0x7c00u;
  return (w & e) == e || (w & e << 16) == e << 16;
}

// The value with what is infinite or NaN made zero.
template <int DT>
__device__ inline unsigned int finite_part(unsigned int w) {
  if constexpr (DT == SSA_F32) return (w & 0x7f800000u) == 0x7f800000u ? 0u : w;
  constexpr unsigned int e = DT == SSA_BF16 ? 0x7f80u : 0x7c00u;
  if ((w & e) == e) w &= 0xffff0000u;
  if ((w & e << 16) == e << 16) w &= 0xffffu;
  return w;
}

// What is not finite in the value as a number of the type: 1 for +inf, 2^8 for -inf, 2^15 for NaN, 0.
template <int DT>
__device__ inline unsigned int kind_of(unsigned int w) {
  if constexpr (DT == SSA_F32) {
    const unsigned int x = w & 0x7fffffffu;
    return x < 0x7f800000u ? 0u : x > 0x7f800000u ? 0x47000000u : w >> 31 ? 0x43800000u : 0x3f800000u;
  } else {
    constexpr unsigned int e = DT == SSA_BF16 ? 0x7f80u : 0x7c00u;
    constexpr unsigned int pos = DT == SSA_BF16 ? 0x3f80u : 0x3c00u;
    constexpr unsigned int neg = DT == SSA_BF16 ? 0x4380u : 0x5c00u;
    constexpr unsigned int nan = DT == SSA_BF16 ? 0x4700u : 0x7800u;
    auto half = [&](unsigned int h) {
      const unsigned int x = h & 0x7fffu;
      return x < e ? 0u : x > e ? nan : h >> 15 ? neg : pos;
    };
    return half(w & 0xffffu) | half(w >> 16) << 16;
  }
}

// Two 16-bit numbers, 0 or 1.
template <int DT>
__device__ inline unsigned int pack16(bool a, bool b) {
  constexpr unsigned int one = DT == SSA_BF16 ? 0x3f80u : 0x3c00u;
  return (a ? one : 0u) | (b ? one << 16 : 0u);
}

// What sums of kinds say: with[r] over keys of a weight, without over those of weight zero.
__device__ inline float not_finite_sum(float with, float without) {
  const int kinds = (int)with;
  float v = kinds >= 1 << 15 || without > 0.0f ? NAN : 0.0f;
  if (kinds & 0xff) v += INFINITY;
  if (kinds & 0x7f00) v -= INFINITY;
  return v;
}

// Attention of a row tile (MT times 16 rows, a row a drafted token's query head of the key head) over
// an item's keys, its tiles of keys in four runs, one a wave; the layout of products and loads is
// paged_attend_kernel's, a row where that has a head. Tiles of keys that some row does not attend (the
// drafted ones, the last, a window's first) take their masks from the rows' words; their lowest score
// -FLT_MAX stands for attended keys, so that -INFINITY means a row without any. A value that is infinite
// or NaN there reaches the rows that do not attend it as 0 x infinity: where a result is NaN, the wave
// does its keys again with care, such values taken out of the product and added to the rows that attend
// them. Bound by the reading of keys and values: 32 requests of 8,000 keys, 4 tokens of 4 heads a key head
// (8 heads of 128, bf16) 184 us, 5.7 TB/s; one token a request 184, for which paged_attend_kernel takes 170.
template <int DT, int DP, int MT, int WPE>
__global__ __launch_bounds__(kAttendWaves * 64, WPE) void paged_drafts_kernel(DraftParams p) {
  using T = Tile<DT, DP>;
  constexpr int NT = T::NT, NC = T::NC, VB = T::VB, LC = T::LC, LW = T::LW, NA = T::NA;
  constexpr int NW = kAttendWaves, NR = NW / 2, M = MT * 16;
  __shared__ f32x4 red[NR][MT][NA][64];
  __shared__ float red_m[NR][MT][64], red_l[NR][MT][64];
  const int wv = uniform(threadIdx.x >> 6);
  if (blockIdx.x >= p.blocks) {
    rest_rows<DT>(p, (int)(blockIdx.x - p.blocks));
    return;
  }
  if (p.status && *p.status != 0) return;
  DraftItem found;
  if (!find_draft<M>(p, blockIdx.x, found)) return;
  const DraftItem it = uniform(found);
  const int ctx = it.s.ctx, n = it.s.n, first = it.s.span.first, len = it.s.span.len;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int tiles = (it.end - it.begin + NT - 1) / NT;
  const int i0 = uniform((int)((int64_t)tiles * wv / NW));
  const int i1 = uniform((int)((int64_t)tiles * (wv + 1) / NW));

  // this lane's rows: drafted token, head and position; past the last row the last again
  int tok[MT], head[MT], rpos[MT];
  bool real[MT];
  int late = 0;  // the latest first key of the tile's rows
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const unsigned int x = it.tile * M + mt * 16 + col;
    const int t = (int)(x / (unsigned)p.G);
    real[mt] = t < n;
    tok[mt] = min(t, n - 1);
    head[mt] = it.g * p.G + (int)(x - (unsigned)t * p.G);
    rpos[mt] = !p.masks ? ctx + tok[mt] : p.pos[(int64_t)it.c0 + tok[mt]];
    if (p.window > 0 && rpos[mt] >= p.window) late = max(late, rpos[mt] - p.window + 1);
  }
  if (p.window > 0) {
    late = max(late, lane_xor(late, 1));
    late = max(late, lane_xor(late, 2));
    late = max(late, lane_xor(late, 4));
    late = max(late, lane_xor(late, 8));
  }
  late = uniform(late);

  __shared__ u32x4 q_lds[T::kQInLds ? MT : 1][T::kQInLds ? NC : 1][64];
  u32x4 q[MT][T::kQInLds ? 1 : NC];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (T::kQInLds && c % NW != wv) continue;
      const int at = c * 64 + grp * 16;
      u32x4 x = {0, 0, 0, 0};
      if (real[mt] && at < p.d * T::ES)
        x = *(const u32x4*)(p.q + (((int64_t)it.c0 + tok[mt]) * p.qt + head[mt] * p.qh) * T::ES + at);
      if constexpr (T::kQInLds) q_lds[mt][c][lane] = x;
      else q[mt][c] = x;
    }
  if constexpr (T::kQInLds) __syncthreads();

  const char* const kbase = p.kpool + it.g * p.kph * T::ES;
  const char* const vbase = p.vpool + it.g * p.vph * T::ES;
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
  int pid = 0, poff = 0, pid_next = 0, batch = 0;
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
  Rows<DT, DP> rows;
  Softmax<NA> st[MT];

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
        const int x = grp * 4 + r, at = (unsigned)(x - lo) < (unsigned)max(count, 0) ? x * vps
                                                                                    : kOutside;
#pragma unroll
        for (int vb = 0; vb < VB; ++vb)
          rows.v[t][r][vb] = load_words<LW, aux.value>(src, at + vcol[vb]);
      }
    }
  };
  constexpr bool kMayStream = DP < 512 && MT == 1;
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
  // which of this lane's keys of the tile from j0 on its row attends: bit 4 t + r
  auto attended = [&](int mt, int j0) {
    const uint64_t keys = attended_keys(p, it, tok[mt], rpos[mt], j0) >> grp * 4;
    unsigned int bits = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) bits |= (unsigned)(keys >> t * 16 & 15) << t * 4;
    return bits;
  };
  auto each_value = [&](auto f) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int vb = 0; vb < VB; ++vb)
#pragma unroll
          for (int x = 0; x < LW; ++x) f(rows.v[t][r][vb].w[x]);
  };
  // Adds the tile's infinite and NaN values to the rows that attend them: products of their kinds, as
  // numbers (1, 2^8 and 2^15 add up without carries), with ones at the keys of a weight, and with ones
  // at the keys whose weight is zero, where 0 x infinity is NaN.
  auto add_not_finite = [&](const f32x4 (&s)[MT][NT], const unsigned int (&allow)[MT]) {
    f32x4 some[MT][NT], none[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool yes = allow[mt] >> (t * 4 + r) & 1;
          some[mt][t][r] = yes && !(s[mt][t][r] == 0.0f) ? 1.0f : 0.0f;
          none[mt][t][r] = yes && s[mt][t][r] == 0.0f ? 1.0f : 0.0f;
        }
#pragma unroll
    for (int vb = 0; vb < VB; ++vb)
#pragma unroll
      for (int e = 0; e < LC; ++e)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          f32x4 x{}, y{};
          if constexpr (DT == SSA_F32) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float kind = __uint_as_float(kind_of<DT>(rows.v[t][r][vb].w[e]));
                x = __builtin_amdgcn_mfma_f32_16x16x4f32(kind, some[mt][t][r], x, 0, 0, 0);
                y = __builtin_amdgcn_mfma_f32_16x16x4f32(kind, none[mt][t][r], y, 0, 0, 0);
              }
          } else {
            u32x4 kinds, a, b;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                kinds[2 * t + h] = kind_of<DT>(__builtin_amdgcn_perm(
                    rows.v[t][2 * h + 1][vb].w[e / 2], rows.v[t][2 * h][vb].w[e / 2],
                    e % 2 ? 0x07060302u : 0x05040100u));
                a[2 * t + h] = pack16<DT>(some[mt][t][2 * h] != 0.0f, some[mt][t][2 * h + 1] != 0.0f);
                b[2 * t + h] = pack16<DT>(none[mt][t][2 * h] != 0.0f, none[mt][t][2 * h + 1] != 0.0f);
              }
            x = mfma16(kinds, a, x, DT == SSA_BF16);
            y = mfma16(kinds, b, y, DT == SSA_BF16);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) st[mt].acc[vb * LC + e][r] += not_finite_sum(x[r], y[r]);
        }
  };

  auto walk = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      st[mt].m = -INFINITY;
      st[mt].l = 0.0f;
#pragma unroll
      for (int i = 0; i < NA; ++i) st[mt].acc[i] = f32x4{0, 0, 0, 0};
    }
    batch = it.begin + i0 * NT;
    if (i0 < i1) {
      const int x = pages_at(batch);
      pid_next = pages_at(batch + 64);
      take_pages(x);
      locate(i0);
      load_k(0);
      load_v(i0);
    }
    for (int i = i0; i < i1; ++i) {
      const int j0 = (it.begin + i * NT) * 16;
      const bool edge = j0 < late || ctx - j0 < NT * 16;
      if constexpr (T::kQInLds) asm volatile("" ::: "memory");  // read the queries here, every time
      // scores: lane column a row, rows the keys 4 grp + r of each subtile; fp32 in kChains chains, as
      // paged_attend_kernel
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
      unsigned int allow[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        Softmax<NA>& o = st[mt];
        allow[mt] = edge ? attended(mt, j0) : 0xffu;
        float mx = allow[mt] ? -FLT_MAX : -INFINITY;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const auto& of = chain[mt][t];
            float x = of[0][r];
            if constexpr (kChains == 2) x += of[1][r];
            if constexpr (kChains == 4) x = (x + of[1][r]) + (of[2][r] + of[3][r]);
            x *= p.scale_log2;
            if (edge && !(allow[mt] >> (t * 4 + r) & 1)) x = -INFINITY;
            s[mt][t][r] = x;
            mx = fmaxf(mx, x);
          }
        mx = fmaxf(mx, lane_xor(mx, 16));
        mx = fmaxf(mx, lane_xor(mx, 32));
        if (__any(mx > o.m)) {  // a row without a key so far stays at -inf, its sums at 0
          const float m = fmaxf(o.m, mx);
          const float a = __builtin_amdgcn_exp2f(o.m - (m == -INFINITY ? 0.0f : m));
          o.m = m;
          o.l *= a;
#pragma unroll
          for (int x = 0; x < NA; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) o.acc[x][r] *= a;
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
              for (int y = 0; y < PARTS; ++y) w[mt][y][2 * t + h] = x[y];
            }
        }
      }
      if (careful.value && edge) {
        bool odd = false;
        each_value([&](unsigned int& v) { odd |= not_finite<DT>(v); });
        if (__any(odd)) {
          add_not_finite(s, allow);
          each_value([&](unsigned int& v) { v = finite_part<DT>(v); });
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
              for (int y = 0; y < PARTS; ++y) acc = mfma16(vt, w[mt][y], acc, DT == SSA_BF16);
            }
          }
        }
      if (more) load_v(i + 1);
    }
  };
  walk(std::false_type{});
  bool nan = false;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) nan |= st[mt].acc[i][r] != st[mt].acc[i][r];
  if (__any(nan)) walk(std::true_type{});
  const bool misfit = bad != 0 || !it.s.span.ok || (wv == 0 && bad_past(p, it, row));
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    st[mt].l += lane_xor(st[mt].l, 16);
    st[mt].l += lane_xor(st[mt].l, 32);
    if (misfit || rpos[mt] < ctx) st[mt].l = NAN;
  }

  // the waves' results, half of them into the other half at a time
#pragma unroll
  for (int half = NW / 2; half >= 1; half >>= 1) {
    if (wv >= half && wv < 2 * half) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        red_m[wv - half][mt][lane] = st[mt].m;
        red_l[wv - half][mt][lane] = st[mt].l;
#pragma unroll
        for (int x = 0; x < NA; ++x) red[wv - half][mt][x][lane] = st[mt].acc[x];
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

  if (p.items != 0 && it.j == 0 && it.g == 0 && it.tile == 0 && lane == 0) {
    p.info[2 * it.b] = it.first_part;
    p.info[2 * it.b + 1] = it.n;
  }
  if (it.n > 1 && it.first_part < 0) return;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const Softmax<NA>& o = st[mt];
    if (!real[mt]) continue;
    const float inv = row_scale(o.m, o.l);
    const int64_t token = (int64_t)it.c0 + tok[mt], to = token * p.ot + head[mt] * p.oh;
    const int64_t part =
        ((int64_t)it.first_part + ((int64_t)it.j * p.Hkv + it.g) * it.tiles + it.tile) * M +
        mt * 16 + col;
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
          for (int y = 0; y < 4; ++y) x[y] = o.acc[vb * LC + e + y][r];
          if (it.n > 1) {
            *(f32x4*)(p.part + part * DP + c) = x;
          } else {
#pragma unroll
            for (int y = 0; y < 4; ++y) x[y] *= inv;
            store_row4<DT>(p.out, to + c, x);
          }
        }
    if (grp != 0) continue;
    if (it.n > 1) {
      p.part_ml[part * 2] = o.m;
      p.part_ml[part * 2 + 1] = o.l;
    } else if (p.lse) {
      p.lse[token * p.Hq + head[mt]] = row_lse(o.m, o.l, T::kShift);
    }
  }
}

// ---- many rows -----------------------------------------------------------------------------------

// A tile of keys or values in LDS is rows of DP 16-bit numbers; 16-byte chunk c of row r lies at chunk
// c ^ tile_swz(r), so that the 16 lanes of a ds_read_b128 phase (rows r..r + 15) and the 32 of a
// transposing read (four rows and four chunks, or eight and two) meet every bank once.
template <int DP>
__device__ inline int tile_swz(int r) {
  if constexpr (DP == 64)  // two rows fill the banks
    return (r >> 1 & 1) << 2 | (r >> 2 & 1) << 1 | (r >> 3 & 1);
  return (r & 3) << 2 | (r >> 2 & 1) << 1 | (r >> 3 & 1);
}

// 16 bytes of each lane from memory to LDS, the wave's one after the other from `to` on.
template <int AUX>
__device__ inline void load_lds(const char* from, unsigned char* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)to, 16, 0, AUX);
}

// Weights of two keys as 16-bit parts: bf16's three, each rounded to 8 bits of what the ones before leave,
// hold them exactly (two left up to 2^-17 of a weight; the third costs 16 tokens over 1M 149 -> 189 us, 16
// trees of 64 182 -> 222); fp16's two, cut to 11 bits each, leave 2^-20, and the output keeps 11 bits. A part
// may be negative or zero: the walk that meets infinite values takes them out of the products first.
template <int DT>
__device__ inline void parts_of(float p0, float p1, unsigned int (&w)[kParts<DT>]) {
  if constexpr (DT == SSA_BF16) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      w[i] = __builtin_bit_cast(unsigned int, bf16x2{(__bf16)p0, (__bf16)p1});
      asm("" : "+v"(w[i]));  // the halves are taken from it, not rounded once more
      p0 -= __uint_as_float(w[i] << 16);
      p1 -= __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    const auto h = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(p0, p1));
    w[0] = __builtin_bit_cast(unsigned int, h);
    w[1] = __builtin_bit_cast(unsigned int, __builtin_amdgcn_cvt_pkrtz(p0 - (float)h[0],
                                                                       p1 - (float)h[1]));
  }
}

// Products of RW x RW numbers over 1024 / RW columns (32 bytes of 16 lanes each, or 16 of 32).
template <int DT>
__device__ inline f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
  return mfma16(a, b, c, DT == SSA_BF16);
}
template <int DT>
__device__ inline f32x16 mfma(const u32x4& a, const u32x4& b, const f32x16& c) {
  if constexpr (DT == SSA_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Attention of a tile of rows over an item's keys, a wave's RW rows (16 or 32) against all of them:
// tiles of KT keys go from memory to LDS, one ahead of the products, and serve the four waves.
// Scores are K Q^T: lane column a row, so its statistics and its weights stay in its lanes and are the
// second product's operand as they are; values are transposed by the LDS reads. A lane's scores come in
// quads: r of quad q is key 4 GR q + 4 grp + r, GR = 64 / RW lanes of a row. bf16 weights, whose
// exponents suffice, go by the maximum of a row's first keys (fp16's maximum rises with the scores), and
// nothing looks for infinite or NaN values: where a sum or a result is too large or not finite, the item is
// done again with care (the maximum raised tile by tile, values that are not finite taken out of the
// products as in paged_drafts_kernel).
// 16 tokens of 7 heads (of 64) over 1,048,561 keys, 537 MB: 178 us and 14 for the join after it; its products
// and weights alone take 160, its loads alone 95. 16 trees of 64 tokens over 2,000 to 9,000 keys (32 / 8 heads
// of 128): 198 us and 20, alone 174 and 110; matrix units busy 35 % of the time in both.
// Rings of three and four tiles, with fewer workgroups a CU, took as long or longer.
template <int DT, int DP, int RW, int KT, int WPE>
__global__ __launch_bounds__(256, WPE) void paged_drafts_tile_kernel(DraftParams p) {
  typedef typename std::conditional<RW == 16, f32x4, f32x16>::type Acc;
  constexpr int NW = 4, M = NW * RW, GR = 64 / RW, ROW = DP * 2, TILE = KT * ROW;
  constexpr int KD = ROW / (16 * GR), DB = DP / RW, AR = RW * RW / 64;  // steps, blocks, results a lane
  constexpr int NS = KT / RW, NQ = KT / (4 * GR), SUB = KT / 16;  // products, quads, subtiles of a tile
  constexpr int CH = ROW / 16, RPI = 64 / CH, LPW = KT / RPI / NW;  // chunks, rows, loads of a wave
  constexpr int PARTS = kParts<DT>;  // of a weight
  constexpr float kShift = DT == SSA_F16 ? kF16Shift : 0.0f;
  constexpr float kGrow = DT == SSA_F16 ? 1.0f : 8.0f;  // fp16 weights end at 2^16
  // a stage is the keys' tile and the values'; objects of their own, so that the compiler's waits for
  // one are not for the other
  __shared__ __attribute__((aligned(1024))) unsigned char st0[2 * TILE];
  __shared__ __attribute__((aligned(1024))) unsigned char st1[2 * TILE];
  if (blockIdx.x >= p.blocks) {
    rest_rows<DT>(p, (int)(blockIdx.x - p.blocks));
    return;
  }
  if (p.status && *p.status != 0) return;
  DraftItem found;
  if (!find_draft<M>(p, blockIdx.x, found)) return;
  const DraftItem it = uniform(found);
  const int wv = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane % RW, grp = lane / RW;
  const int ctx = it.s.ctx, n = it.s.n, first = it.s.span.first, len = it.s.span.len;
  const int tiles = (it.end - it.begin + SUB - 1) / SUB;

  const unsigned int x = it.tile * M + wv * RW + col;
  const int t0 = (int)(x / (unsigned)p.G), tok = min(t0, n - 1);
  const int head = it.g * p.G + (int)(x - (unsigned)t0 * p.G);
  const bool real = t0 < n, any = __any(real);  // a wave without rows loads and waits with the others
  const int rpos = !p.masks ? ctx + tok : p.pos[(int64_t)it.c0 + tok];
  // the latest first key of the wave's rows
  int late = p.window > 0 && rpos >= p.window ? rpos - p.window + 1 : 0;
  if (p.window > 0) {
#pragma unroll
    for (int i = 1; i < RW; i <<= 1) late = max(late, lane_xor(late, i));
  }
  late = uniform(late);

  // the queries take the scale's sign, so that larger products are larger scores; one of 0 is next to it
  const unsigned int sign = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
  const float scale = fmaxf(fabsf(p.scale_log2), FLT_MIN);
  u32x4 q[KD];
#pragma unroll
  for (int c = 0; c < KD; ++c) {
    const int at = (c * GR + grp) * 16;
    q[c] = u32x4{};
    if (real && at < p.d * 2)
      q[c] = *(const u32x4*)(p.q + (((int64_t)it.c0 + tok) * p.qt + head * p.qh) * 2 + at) ^ sign;
  }

  const char* const kbase = p.kpool + it.g * p.kph * 2;
  const char* const vbase = p.vpool + it.g * p.vph * 2;
  const int64_t kpp = p.kpp * 2, vpp = p.vpp * 2;
  const int kps = (int)p.kps * 2, vps = (int)p.vps * 2, row_bytes = p.d * 2;
  const int32_t* const row = p.table + it.b * p.table_stride;

  // page and offset of 64 subtiles at a time, one per lane; the next 64 are on their way
  int pid = 0, poff = 0, pid_next = 0, batch = 0;
  unsigned long long bad = 0;
  auto pages_at = [&](int s) {
    s += lane;
    return s < it.end ? row[page_of(s, p.div)] : 0;
  };
  auto take_pages = [&](int v) {
    bad |= __ballot(v < 0 || v >= p.pages);
    pid = v < 0 || v >= p.pages ? 0 : v;
    poff = (batch + lane) * 16 - page_of(batch + lane, p.div) * p.page;
  };

  // load j of this wave: rows (j NW + wv) RPI.. of the tile, a lane a chunk. With up to 16 chunks a row
  // a row's place in its subtile of 16, and so its swizzle, is the same for every j; with 32 it is for
  // every other j, and the swizzle's other bit moves along.
  const int lchunk = lane % CH;
  auto load_row = [&](int j) { return ((j * NW + wv) * RPI + lane / CH) & 15; };
  auto issue = [&](unsigned char* to, int i) __attribute__((always_inline)) {
    const int s0 = it.begin + i * SUB;
    if (s0 >= batch + 64) {
      batch += 64;
      take_pages(pid_next);
      pid_next = pages_at(batch + 64);
    }
    const bool full = DP == p.d && s0 * 16 >= first && len - s0 * 16 >= KT && s0 + SUB <= it.end;
    auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < LPW; ++j) {
        const int u = j * NW + wv, s = s0 + u * RPI / 16, at = min(s, it.end - 1) - batch;
        const int r = load_row(j), c = lchunk ^ tile_swz<DP>(r);
        const int64_t pg = __builtin_amdgcn_readlane(pid, at);
        const int64_t off = __builtin_amdgcn_readlane(poff, at);
        f(kbase + (pg * kpp + off * kps) + (unsigned)(r * kps + c * 16),
          vbase + (pg * vpp + off * vps) + (unsigned)(r * vps + c * 16), to + u * 1024,
          (int)(s * 16u + r), c * 16 < row_bytes, s < it.end);
      }
    };
    if (full && it.stream) {
      each([&](const char* k, const char* v, unsigned char* at, int, bool, bool) {
        load_lds<kStream>(k, at);
        load_lds<kStream>(v, at + TILE);
      });
    } else if (full) {
      each([&](const char* k, const char* v, unsigned char* at, int, bool, bool) {
        load_lds<0>(k, at);
        load_lds<0>(v, at + TILE);
      });
    } else {  // columns past d and rows that do not count are read as zero
      each([&](const char* k, const char* v, unsigned char* at, int key, bool in, bool own) {
        const char* const zero = (const char*)kZeroRow + lchunk * 16;
        const bool counts = in & own & (key >= first) & (key < len);
        load_lds<0>(in ? k : zero, at);
        load_lds<0>(counts ? v : zero, at + TILE);
      });
    }
  };

  // LDS reads: keys row RW t + col, chunk GR c + grp; values (transposing) rows 4 GR q + 4 grp + (0..3)
  // of quads q = 2 st and 2 st + 1, 16 columns of the block (RW 32: the upper lanes the other 16)
  const int kswz = (tile_swz<DP>(col & 15) ^ grp) * 16, krow = col * ROW;
  const int vrow = 4 * grp + (lane & 15) / 4;
  const int vchunk = (RW == 32 ? 2 * (lane >> 4 & 1) : 0) + (lane >> 1 & 1);
  const int vat0 = vrow * ROW + (lane & 1) * 8, vswz0 = (tile_swz<DP>(vrow & 15) ^ vchunk) * 16;
  const int vat1 = vat0 + 4 * GR * ROW;
  const int vswz1 = (tile_swz<DP>((vrow + 4 * GR) & 15) ^ vchunk) * 16;

  float m, l;
  Acc acc[DB];
  auto compute = [&](const unsigned char* ks, int i, auto careful) __attribute__((always_inline)) {
    const unsigned char* const vs = ks + TILE;
    const int s0 = it.begin + i * SUB, j0 = s0 * 16;
    // up to the tile of the latest first key: past it every row has a maximum or no key of the context
    const bool edge = j0 <= late || ctx - j0 < KT || s0 + SUB > it.end;
    Acc sum_of[NS];
#pragma unroll
    for (int t = 0; t < NS; ++t) {
      sum_of[t] = Acc{};
#pragma unroll
      for (int c = 0; c < KD; ++c) {
        const u32x4 a = *(const u32x4*)(ks + t * RW * ROW + krow + (kswz ^ c * GR * 16));
        sum_of[t] = mfma<DT>(a, q[c], sum_of[t]);
      }
    }
    float s[NQ][4];
#pragma unroll
    for (int t = 0; t < NS; ++t)
#pragma unroll
      for (int r = 0; r < AR; ++r) s[(t * AR + r) / 4][r % 4] = sum_of[t][r];
    // bit 4 q + r: whether the row attends r of quad q
    unsigned int allow = NQ == 8 ? ~0u : (1u << 4 * NQ % 32) - 1;
    float mx = -FLT_MAX;
    if (edge) {
      uint64_t keys = attended_keys(p, it, tok, rpos, j0);
      const int own = min(it.end - s0, SUB) * 16;  // past the item's end the next item's keys lie
      if (own < 64) keys &= (1ull << own) - 1;
      keys >>= 4 * grp;
      allow = 0;
#pragma unroll
      for (int y = 0; y < NQ; ++y) allow |= (unsigned)(keys >> 4 * GR * y & 15) << 4 * y;
      if (allow == 0) mx = -INFINITY;
#pragma unroll
      for (int y = 0; y < NQ; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[y][r] = allow & 1u << (4 * y + r) ? s[y][r] : -INFINITY;
    }
    if (DT != SSA_BF16 || edge || i == 0 || careful.value) {
      float top = s[0][0];
#pragma unroll
      for (int y = 0; y < NQ; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, s[y][r]);
      mx = fmaxf(mx, top * scale);
      if constexpr (RW == 16) mx = fmaxf(mx, lane_xor(mx, 16));
      mx = fmaxf(mx, lane_xor(mx, 32));
      if (__any(mx > m + kGrow)) {
        const float up = fmaxf(m, mx);
        const float a = __builtin_amdgcn_exp2f(m - (up == -INFINITY ? 0.0f : up));
        m = up;
        l *= a;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r = 0; r < AR; ++r) acc[db][r] *= a;
      }
    }
    const float base = (m == -INFINITY ? 0.0f : m) - kShift;
    float sum = 0.0f;
#pragma unroll
    for (int y = 0; y < NQ; ++y)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[y][r] = __builtin_amdgcn_exp2f(fmaf(s[y][r], scale, -base));
        sum += s[y][r];
      }
    l += sum;
#pragma unroll
    for (int st = 0; st < NQ / 2; ++st) {
      u32x4 w[PARTS];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float* const of = &s[2 * st + y / 2][y % 2 * 2];
        unsigned int parts[PARTS];
        parts_of<DT>(of[0], of[1], parts);
#pragma unroll
        for (int k = 0; k < PARTS; ++k) w[k][y] = parts[k];
      }
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const unsigned char* const at = vs + st * 8 * GR * ROW;
        const uint2 lo = lds_read_tr(at + vat0 + (vswz0 ^ db * RW * 2));
        const uint2 up = lds_read_tr(at + vat1 + (vswz1 ^ db * RW * 2));
        u32x4 v = {lo.x, lo.y, up.x, up.y};
        if constexpr (careful.value) {
          u32x4 kinds, some, none;
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            kinds[y] = kind_of<DT>(v[y]);
            v[y] = finite_part<DT>(v[y]);
            const float* const of = &s[2 * st + y / 2][y % 2 * 2];
            const unsigned int yes = allow >> (4 * (2 * st + y / 2) + y % 2 * 2);
            some[y] = pack16<DT>(yes & 1 && !(of[0] == 0.0f), yes & 2 && !(of[1] == 0.0f));
            none[y] = pack16<DT>(yes & 1 && of[0] == 0.0f, yes & 2 && of[1] == 0.0f);
          }
          if (__any((kinds[0] | kinds[1] | kinds[2] | kinds[3]) != 0)) {
            const Acc with = mfma<DT>(kinds, some, Acc{}), without = mfma<DT>(kinds, none, Acc{});
#pragma unroll
            for (int r = 0; r < AR; ++r) acc[db][r] += not_finite_sum(with[r], without[r]);
          }
        }
#pragma unroll
        for (int k = 0; k < PARTS; ++k) acc[db] = mfma<DT>(v, w[k], acc[db]);
      }
    }
  };
  auto begin = [&] {
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = Acc{};
    batch = it.begin;
    const int v = pages_at(batch);
    pid_next = pages_at(batch + 64);
    take_pages(v);
  };
  begin();
  if (tiles > 0) issue(st0, 0);
  for (int i = 0; i < tiles; i += 2) {
    dma_barrier();  // tile i is there for all waves; tile i - 1 is read no more
    if (i + 1 < tiles) issue(st1, i + 1);
    if (any) compute(st0, i, std::false_type{});
    if (i + 1 >= tiles) break;
    dma_barrier();
    if (i + 2 < tiles) issue(st0, i + 2);
    if (any) compute(st1, i + 1, std::false_type{});
  }
  bool off = !(l < 0x1p100f);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < AR; ++r) off |= !(fabsf(acc[db][r]) < INFINITY);
  if (__syncthreads_or(off && real)) {
    begin();
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
      __syncthreads();
      issue(st0, i);
      dma_barrier();
      if (any) compute(st0, i, std::true_type{});
    }
  }
  if constexpr (RW == 16) l += lane_xor(l, 16);
  l += lane_xor(l, 32);
  const bool misfit = bad != 0 || !it.s.span.ok || bad_past(p, it, row);
  if (misfit || rpos < ctx) l = NAN;

  if (p.items != 0 && it.j == 0 && it.g == 0 && it.tile == 0 && threadIdx.x == 0) {
    p.info[2 * it.b] = it.first_part;
    p.info[2 * it.b + 1] = it.n;
  }
  if (!real || (it.n > 1 && it.first_part < 0)) return;
  const float inv = row_scale(m, l);
  const int64_t token = (int64_t)it.c0 + tok, to = token * p.ot + head * p.oh;
  const int64_t part = ((int64_t)it.first_part + ((int64_t)it.j * p.Hkv + it.g) * it.tiles + it.tile) * M +
                       wv * RW + col;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g = 0; g < AR / 4; ++g) {
      const int c = RW * db + 4 * GR * g + 4 * grp;
      if (c >= p.d) continue;
      f32x4 y;
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = acc[db][4 * g + r];
      if (it.n > 1) {
        *(f32x4*)(p.part + part * DP + c) = y;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] *= inv;
        store_row4<DT>(p.out, to + c, y);
      }
    }
  if (grp != 0) return;
  if (it.n > 1) {
    p.part_ml[part * 2] = m;
    p.part_ml[part * 2 + 1] = l;
  } else if (p.lse) {
    p.lse[token * p.Hq + head] = row_lse(m, l, kShift);
  }
}

// Joins the parts of rows whose tiles were cut: a wave per row (a token's query head), its lanes over
// the columns, four waves a workgroup. Bound by memory: 32,768 rows of 3 to 11 parts of 128 columns (98 MB)
// 20 us; by latency where rows are few, 4 us, or 14 where each has many parts (224 rows over 1M keys). BATCH:
// parts of a row (and split of the wave) on their way at a time: 16 where rows are few and long, 4 where the
// rows fill the card (kFewJoins has both sides).
template <int DT, int DP, int M, int BATCH>
__global__ __launch_bounds__(256) void paged_drafts_join_kernel(DraftParams p) {
  constexpr int PER = DP / 4, NS = PER < 64 ? 64 / PER : 1, NV = PER > 64 ? PER / 64 : 1;
  const int lane = threadIdx.x & 63;
  const unsigned int id = blockIdx.x * 4 + uniform(threadIdx.x >> 6), token = id / (unsigned)p.Hq;
  const int64_t row = token;
  if (row >= p.N || (p.status && *p.status != 0)) return;
  const int h = (int)(id - token * p.Hq), g = h / p.G;
  const int b = last_at_most(p.cu, p.B, (int)row), c0 = p.cu[b], c1 = p.cu[b + 1];
  const DraftSpan s = draft_of(p, b);
  if (row < c0 || row >= c1 || s.n == 0) return;  // rest_rows answers
  const int first = p.info[2 * b], parts = p.info[2 * b + 1];
  if (parts <= 1) return;  // written by its one item
  const unsigned int x = (unsigned)(row - c0) * p.G + (h - g * p.G), tile = x / M;
  const int64_t tiles = draft_tiles(s, p.G, M), step = tiles * p.Hkv;
  const bool held = first >= 0 && first + step * parts <= p.max_parts;
  const int64_t at = ((held ? first : 0) + g * tiles + tile) * M + x % M;
  const int split = lane / PER % NS, c = lane % PER * 4;
  Softmax<NV> st;
  st.m = -INFINITY;
  st.l = held ? 0.0f : NAN;
#pragma unroll
  for (int v = 0; v < NV; ++v) st.acc[v] = f32x4{0, 0, 0, 0};
  for (int i = split; held && i < parts; i += NS * BATCH) {
    float m[BATCH], l[BATCH], mx = st.m;
    f32x4 a[BATCH][NV];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const bool in = i + u * NS < parts;
      const int64_t from = at + (in ? i + u * NS : 0) * step * M;
      m[u] = in ? p.part_ml[from * 2] : -INFINITY;
      l[u] = in ? p.part_ml[from * 2 + 1] : 0.0f;
#pragma unroll
      for (int v = 0; v < NV; ++v)
        a[u][v] = in ? *(const f32x4*)(p.part + from * DP + v * 256 + c) : f32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) mx = fmaxf(mx, m[u]);
    const float base = mx == -INFINITY ? 0.0f : mx, y = __builtin_amdgcn_exp2f(st.m - base);
    st.m = mx;
    st.l *= y;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int r = 0; r < 4; ++r) st.acc[v][r] *= y;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const float z = __builtin_amdgcn_exp2f(m[u] - base);
      st.l += l[u] * z;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int r = 0; r < 4; ++r) st.acc[v][r] += a[u][v][r] * z;
    }
  }
#pragma unroll
  for (int off = 32; off >= PER; off >>= 1) {
    f32x4 o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = lane_xor(st.acc[0][r], off);
    const float m = lane_xor(st.m, off), l = lane_xor(st.l, off);
    Softmax<1> one{st.m, st.l, {st.acc[0]}};
    join(one, m, l, &o, 0);
    st.m = one.m;
    st.l = one.l;
    st.acc[0] = one.acc[0];
  }
  const float inv = row_scale(st.m, st.l);
  const int64_t to = row * p.ot + h * p.oh;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
#pragma unroll
    for (int r = 0; r < 4; ++r) st.acc[v][r] *= inv;
    if (lane < PER && v * 256 + c < p.d) store_row4<DT>(p.out, to + v * 256 + c, st.acc[v]);
  }
  if (p.lse && lane == 0)
    p.lse[row * p.Hq + h] = row_lse(st.m, st.l, DT == SSA_F16 ? kF16Shift : 0.0f);
}

// How a call of these sizes is cut: known on the host without the lengths.
struct DraftLayout {
  int64_t items, blocks, max_parts;  // items: 0 when no row tile is cut
  int dp, M;
  size_t part_ml, info, bytes;  // offsets into the workspace, which starts with the parts
};

// Two tiles of 16 rows a wave where requests have more rows on average (past head dim 128 their
// registers do not fit).
DraftLayout draft_layout(int dtype, int64_t B, int64_t N, int64_t Hq, int64_t Hkv, int64_t d, int64_t W,
                         int64_t page, int64_t window) {
  DraftLayout y{};
  const int64_t G = Hq / Hkv;
  y.dp = d <= 64 ? 64 : d <= 128 ? 128 : d <= 256 ? 256 : 512;
  // Rows of a key head; of a request rows / B on average. Tiles of 16 rows, whose waves take a run of keys
  // each, win up to there; past them tiles that the waves share (bf16, 32 requests of 8,000 keys, 8 heads
  // of 128): 16 rows a request 176 us for 207, 20 rows 212 for 216, 64 231 for 353. Past 64 rows tiles of
  // 128: 128 rows 330 us for 347 (two of 64), 96 299 for 313, 64 275 for 230. fp32, 32 rows: 121 for 125 (two
  // of 16).
  const int64_t rows = N * G;
  if (dtype == SSA_F32) y.M = y.dp <= 128 && rows > 16 * B ? 32 : 16;
  else y.M = y.dp == 512 || rows <= 16 * B ? 16 : y.dp == 256 || rows <= 64 * B ? 64 : 128;
  const int64_t tiles = draft_most_tiles(B, N, G, y.M) * Hkv;
  const int64_t cap = W * page;
  const int64_t units = paged_most_units(window > 0 ? std::min(cap, window + N + 15) : cap, 0);
  const auto rounded = [](int64_t x) { return (x + 7) / 8 * 8; };  // an XCD's run each
  y.blocks = rounded(tiles);
  if (units <= 4 || (units <= 16 && tiles >= 512)) return y;
  // Workgroups aimed at: what the CUs hold at once (one a CU at head dim 512, two at 256, three or four
  // below), or twice that below 256 where it evens out uneven requests. Three a CU and twice as many: 64 mixed
  // requests 280 us and 266, 16 trees of 64 tokens 229 and 218; one request is even by itself: 16 tokens over
  // 1M 181 and 192, 8 over 1M 120 and 133, over 100K of 8 key heads 16 tokens 92 and 116, 4 tokens 84 and 92
  // (so are two alike, which the host cannot know: 50,000 each 90 and 115). Head dim 256, two a CU and one and
  // a half: 8 requests of 8,000 keys 71 and 79, one of 60,000 68 and 74, 64 of 2,000 68 and 78, windows of
  // 2,048 of 48 requests 79 and 95, of 1,024 of 32 requests 48 and 43, 20 of 500 to 9,000 100 and 82.
  const int64_t target = y.dp == 512 ? 256 : y.dp == 256 ? 512 : B == 1 ? 768 : y.M >= 64 ? 1536 : 1024;
  y.items = std::max<int64_t>(1, target / Hkv);
  y.blocks = rounded(std::min(tiles + y.items * Hkv, tiles * units));
  y.max_parts = std::min(2 * y.items * Hkv, y.blocks);
  const size_t held = (size_t)y.max_parts * y.M;
  y.part_ml = held * y.dp * 4;
  y.info = y.part_ml + held * 2 * 4;
  y.bytes = (y.info + (size_t)B * 8 + 15) / 16 * 16;
  return y;
}

// Rows up to which a join takes 16 parts at a time (the whole call with 4 and with 16: 32 rows of 100,000 keys
// 31.7 and 28.8 us, 256 45.7 and 42.5, 1,024 in 8 requests of 8,000 23.8 and 23.5, 1,536 103.9 and 102.1,
// 2,048 in one request 156.7 and 158.2, in 16 29.1 and 29.1, 4,096 in 32 28.9 and 29.6).
constexpr int64_t kFewJoins = 1024;

template <int DT, int DP, int M, int KT, int WPE>
int run_drafts(const DraftParams& p, hipStream_t st) {
  const unsigned blocks = (unsigned)(p.blocks + kRestBlocks);
  if constexpr (KT != 0)
    paged_drafts_tile_kernel<DT, DP, M / 4, KT, WPE><<<blocks, 256, 0, st>>>(p);
  else
    paged_drafts_kernel<DT, DP, M / 16, WPE><<<blocks, kAttendWaves * 64, 0, st>>>(p);
  SSA_TRY(launch_status("paged_drafts_kernel"));
  if (p.items == 0) return SSA_OK;
  const int64_t rows = p.N * p.Hq, joins = (rows + 3) / 4;
  if (rows <= kFewJoins) paged_drafts_join_kernel<DT, DP, M, 16><<<(unsigned)joins, 256, 0, st>>>(p);
  else paged_drafts_join_kernel<DT, DP, M, 4><<<(unsigned)joins, 256, 0, st>>>(p);
  return launch_status("paged_drafts_join_kernel");
}

template <int DT>
int run_drafts_dim(const DraftParams& p, const DraftLayout& y, hipStream_t st) {
  constexpr bool f32 = DT == SSA_F32;
  if constexpr (!f32) {
    if (y.M == 64 && y.dp == 64) return run_drafts<DT, 64, 64, 64, 4>(p, st);
    if (y.M == 64 && y.dp == 128) return run_drafts<DT, 128, 64, 32, 4>(p, st);
    if (y.M == 64 && y.dp == 256) return run_drafts<DT, 256, 64, 32, 2>(p, st);
    if (y.M == 128 && y.dp == 64) return run_drafts<DT, 64, 128, 64, 3>(p, st);
    if (y.M == 128 && y.dp == 128) return run_drafts<DT, 128, 128, 64, 2>(p, st);
  } else {
    if (y.M == 32 && y.dp == 64) return run_drafts<DT, 64, 32, 0, 2>(p, st);
    if (y.M == 32 && y.dp == 128) return run_drafts<DT, 128, 32, 0, 2>(p, st);
  }
  switch (y.dp) {
    case 64: return run_drafts<DT, 64, 16, 0, f32 ? 3 : 4>(p, st);
    case 128: return run_drafts<DT, 128, 16, 0, 2>(p, st);
    case 256: return run_drafts<DT, 256, 16, 0, 2>(p, st);
    default: return run_drafts<DT, 512, 16, 0, 1>(p, st);
  }
}

// ---- accepted tokens moved together ------------------------------------------------------------

struct KeepParams {
  char* kpool;
  char* vpool;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;
  const int32_t* path;
  const int32_t* counts;
  int32_t* new_lens;
  int64_t table_stride, path_stride, cap, pages;
  int width;                                           // of a path
  int page, Hkv, vecs, columns;                        // vecs: 16-byte pieces of a row
  int64_t kpl, kpp, kph, kps, vpl, vpp, vph, vps;      // bytes
  PageDiv div;
};

constexpr int kKeepThreads = 64, kKeepBatch = 32;

// Whether a request's tokens move by its own check, or (all or none) by those of a launch before it.
enum Keep { kKeepEach, kKeepCheck, kKeepAll };

// A workgroup for a request and 64 columns (a column: 16 bytes of a layer's keys or values of a head,
// over all tokens), a thread a column. An accepted token never moves up and they move in order, so a
// column's tokens are read kKeepBatch at a time before any of these is written, and none that is
// written is read again. All or nothing: every workgroup of a request checks its whole path first, and
// with kKeepAll looks at what the launch before it (kKeepCheck) found of every request. Bound
// by the longest path's column: 24 requests with 200 of 600 tokens moved in 8 layers (5 heads of 80, fp32,
// 93 MB in all) 38 us; 64 with 2 in 24 layers 4.1.
template <Keep KEEP>
__global__ __launch_bounds__(kKeepThreads) void paged_keep_kernel(KeepParams p) {
  __shared__ int64_t s_from[2][kKeepThreads], s_to[2][kKeepThreads];  // of keys and values
  __shared__ int s_first;
  const int b = blockIdx.y, tid = threadIdx.x;
  const int len = p.lens[b], c0 = p.cu[b], c1 = p.cu[b + 1], count = p.counts[b];
  const int n = c1 - c0, ctx = len - n;
  bool bad = c0 < 0 || c1 < c0 || len < 0 || len > p.cap || n > len || count < 0 || count > n ||
             count > p.width;
  const int32_t* const path = p.path + b * p.path_stride;
  const int32_t* const row = p.table + b * p.table_stride;
  auto place = [&](int at, int& page, int& slot) {  // of drafted token `at`
    const int j = ctx + at, e = page_of(j / 16, p.div);
    page = row[e];
    slot = j - e * p.page;
    return page >= 0 && page < p.pages;
  };
  if (tid == 0) s_first = 0x7fffffff;
  __syncthreads();
  if (!bad) {
    bool wrong = false;
    int moved = 0x7fffffff;
    for (int i = tid; i < count; i += kKeepThreads) {
      const int at = path[i], before = i > 0 ? path[i - 1] : -1;
      int page, slot;
      if (before >= at || at < 0 || at >= n || !place(at, page, slot) || !place(i, page, slot))
        wrong = true;
      else if (at != i) moved = min(moved, i);
    }
    if (moved != 0x7fffffff) atomicMin(&s_first, moved);
    bad = __syncthreads_or(wrong);
  }
  if (KEEP != kKeepAll && blockIdx.x == 0 && tid == 0) p.new_lens[b] = bad ? -1 : ctx + count;
  if (KEEP == kKeepCheck || bad || s_first >= count) return;
  if constexpr (KEEP == kKeepAll) {
    bool none = false;
    for (int i = tid; i < (int)gridDim.y; i += kKeepThreads) none |= p.new_lens[i] < 0;
    if (__any(none)) return;
  }
  const int first = s_first, column = blockIdx.x * kKeepThreads + tid;
  const int c = column % p.vecs, of = column / p.vecs, h = of % p.Hkv, lv = of / p.Hkv;
  const bool mine = column < p.columns, v = lv & 1;
  char* const base = (v ? p.vpool : p.kpool) + (lv >> 1) * (v ? p.vpl : p.kpl) +
                     h * (v ? p.vph : p.kph) + c * 16;
  for (int i0 = first; i0 < count; i0 += kKeepThreads) {
    const int m = min(count - i0, kKeepThreads);
    __syncthreads();
    if (tid < m) {
      int page, slot;
      place(path[i0 + tid], page, slot);
      s_from[0][tid] = page * p.kpp + slot * p.kps;
      s_from[1][tid] = page * p.vpp + slot * p.vps;
      place(i0 + tid, page, slot);
      s_to[0][tid] = page * p.kpp + slot * p.kps;
      s_to[1][tid] = page * p.vpp + slot * p.vps;
    }
    __syncthreads();
    if (!mine) continue;
    for (int i = 0; i < m; i += kKeepBatch) {
      u32x4 x[kKeepBatch];
#pragma unroll
      for (int g = 0; g < kKeepBatch; g += 8) {
        if (i + g >= m) break;
#pragma unroll
        for (int u = g; u < g + 8; ++u) {
          x[u] = *(const u32x4*)(base + s_from[v][min(i + u, m - 1)]);
        }
      }
#pragma unroll
      for (int g = 0; g < kKeepBatch; g += 8) {
        if (i + g >= m) break;
#pragma unroll
        for (int u = g; u < g + 8; ++u)
          if (i + u < m) *(u32x4*)(base + s_to[v][i + u]) = x[u];
      }
    }
  }
}

// Whether the n ints from a on and the m from b on share any.
bool overlap(const int32_t* a, int64_t n, const int32_t* b, int64_t m) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return a && b && n > 0 && m > 0 && x < y + (uintptr_t)m * 4 && y < x + (uintptr_t)n * 4;
}

int check_table(const char* who, int64_t W, int64_t table_stride, int64_t page) {
  SSA_REQUIRE(W > 0 && table_stride >= W && W <= 0x7fffffff / page, SSA_ERR_INVALID,
              "%s: table of %lld pages a row, stride %lld (at most 2^31 - 1 tokens)", who,
              (long long)W, (long long)table_stride);
  return SSA_OK;
}

}  // namespace
}  // namespace ssa

using namespace ssa;

extern "C" int ssa_paged_draft_masks(const int32_t* parents, const int32_t* cu,
                                     const int32_t* lens, int64_t B, int64_t N, int64_t words,
                                     int32_t* masks, int32_t* pos, ssa_stream_t stream) {
  SSA_REQUIRE(cu && lens && (N == 0 || (parents && masks && pos)), SSA_ERR_INVALID,
              "ssa_paged_draft_masks: NULL argument");
  SSA_REQUIRE(B > 0 && B < 0x7fffffff && fits_int(N), SSA_ERR_INVALID,
              "ssa_paged_draft_masks: bad shape (B=%lld, N=%lld)", (long long)B, (long long)N);
  SSA_REQUIRE(words > 0 && words <= kMaxWords, SSA_ERR_UNSUPPORTED,
              "ssa_paged_draft_masks: masks of %lld words (1 to %d)", (long long)words, kMaxWords);
  const int threads = words <= 2 ? 64 : words <= 8 ? 256 : 1024;
  SSA_REQUIRE(fits_launch((B + 1) * ((words + 3) / 4), threads), SSA_ERR_UNSUPPORTED,
              "ssa_paged_draft_masks: %lld requests in one call", (long long)B);
  if (N == 0) return SSA_OK;
  for (const int32_t* in : {parents, cu, lens}) {  // read by workgroups that others may be ahead of
    const int64_t n = in == parents ? N : in == cu ? B + 1 : B;
    SSA_REQUIRE(!overlap(masks, N * words, in, n) && !overlap(pos, N, in, n), SSA_ERR_INVALID,
                "ssa_paged_draft_masks: an output lies over an input");
  }
  hipStream_t st = (hipStream_t)stream;
  auto run = [&](int64_t first, int64_t blocks, bool all) {
    MaskParams p{parents, cu, lens, masks, pos, N, (int)B, (int)words, (int)first, all};
    const dim3 grid((unsigned)blocks, (unsigned)((words + 3) / 4));
    if (threads == 64) paged_draft_masks_kernel<64><<<grid, 64, 0, st>>>(p);
    else if (threads == 256) paged_draft_masks_kernel<256><<<grid, 256, 0, st>>>(p);
    else paged_draft_masks_kernel<1024><<<grid, 1024, 0, st>>>(p);
    return launch_status("paged_draft_masks_kernel");
  };
  if (B <= kMaskScan) return run(0, B + 1, true);
  SSA_TRY(run(0, B, false));
  return run(B, 1, true);
}

extern "C" size_t ssa_paged_attend_drafts_workspace_size(int dtype, int64_t B, int64_t N, int64_t Hq,
                                                         int64_t Hkv, int64_t d, int64_t W,
                                                         int64_t page, int64_t window) {
  if (dtype_size(dtype) == 0 || B <= 0 || N <= 0 || !fits_int(N) || Hq <= 0 || Hkv <= 0 || Hq % Hkv || d <= 0 || d > 512 ||
      W <= 0 || page <= 0 || !fits_int(window) || W > 0x7fffffff / page)
    return 0;
  return draft_layout(dtype, B, N, Hq, Hkv, d, W, page, window).bytes;
}

extern "C" int ssa_paged_attend_drafts(const void* q, const void* kpool, const void* vpool,
                                       void* out, float* lse, int dtype, int64_t B, int64_t N,
                                       int64_t Hq, int64_t Hkv, int64_t d, int64_t pages,
                                       int64_t page, const int32_t* table, int64_t table_stride,
                                       int64_t W, const int32_t* lens, const int32_t* cu,
                                       const int32_t* masks, const int32_t* pos, int64_t words,
                                       const int64_t* strides, float scale, int64_t window,
                                       const int32_t* status, int clear_rest, void* workspace,
                                       size_t workspace_bytes, ssa_stream_t stream) {
  const char* const who = "ssa_paged_attend_drafts";
  SSA_REQUIRE(q && kpool && vpool && out && table && lens && cu && strides, SSA_ERR_INVALID,
              "%s: NULL argument", who);
  SSA_REQUIRE((masks == nullptr) == (pos == nullptr) && (masks == nullptr) == (words == 0),
              SSA_ERR_INVALID, "%s: masks, pos and words come together", who);
  SSA_REQUIRE(words >= 0 && words <= kMaxWords, SSA_ERR_UNSUPPORTED,
              "%s: masks of %lld words (1 to %d)", who, (long long)words, kMaxWords);
  SSA_TRY(check_pool(who, dtype, Hkv, d, pages, page));
  SSA_REQUIRE(B > 0 && B <= 65535 && N > 0 && fits_int(N) && Hq > 0 && Hq <= 65535 &&
                  Hq % Hkv == 0, SSA_ERR_INVALID,
              "%s: B=%lld, N=%lld, Hq=%lld, Hkv=%lld (at most 65535 requests; Hq a multiple of "
              "Hkv)", who, (long long)B, (long long)N, (long long)Hq, (long long)Hkv);
  SSA_TRY(check_table(who, W, table_stride, page));
  SSA_REQUIRE(fits_int(window), SSA_ERR_INVALID, "%s: window %lld", who, (long long)window);
  const int es = dtype_size(dtype);
  // strides: q(t,h), kpool(page,head,slot), vpool(page,head,slot), out(t,h)
  SSA_REQUIRE(rows16(q, strides, 2, es) && rows16(kpool, strides + 2, 3, es) &&
                  rows16(vpool, strides + 5, 3, es) && rows16(out, strides + 8, 2, es),
              SSA_ERR_INVALID, "%s: rows must start at multiples of 16 bytes", who);
  SSA_REQUIRE(strides[4] < (1 << 24) && strides[7] < (1 << 24), SSA_ERR_UNSUPPORTED,
              "%s: slots 2^24 elements apart or more", who);
  const DraftLayout y = draft_layout(dtype, B, N, Hq, Hkv, d, W, page, window);
  SSA_REQUIRE(workspace_bytes >= y.bytes && (y.bytes == 0 || (workspace && aligned16(workspace))),
              SSA_ERR_WORKSPACE, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who,
              y.bytes, workspace_bytes);
  SSA_REQUIRE(fits_launch(y.blocks + kRestBlocks, kAttendWaves * 64) && fits_int(N * Hq) &&
                  fits_launch((N * Hq + 3) / 4, 256), SSA_ERR_UNSUPPORTED,
              "%s: too many rows in one call", who);
  DraftParams p{};
  p.q = (const char*)q;
  p.kpool = (const char*)kpool;
  p.vpool = (const char*)vpool;
  p.out = (char*)out;
  p.lse = lse;
  p.table = table;
  p.lens = lens;
  p.cu = cu;
  p.masks = masks;
  p.pos = pos;
  p.status = status;
  p.table_stride = table_stride;
  p.cap = W * page;
  p.pages = pages;
  p.N = N;
  p.B = (int)B;
  p.Hq = (int)Hq;
  p.Hkv = (int)Hkv;
  p.G = (int)(Hq / Hkv);
  p.d = (int)d;
  p.page = (int)page;
  p.window = (int)window;
  p.words = (int)words;
  p.clear = clear_rest != 0;
  p.scale_log2 = scale * kLog2e;
  int64_t* const st[10] = {&p.qt,  &p.qh,  &p.kpp, &p.kph, &p.kps,
                           &p.vpp, &p.vph, &p.vps, &p.ot,  &p.oh};
  for (int i = 0; i < 10; ++i) *st[i] = strides[i];
  p.div = page_div((int)page / 16);
  p.stream_units = kStreamBytes / unit_bytes(dtype, d, Hkv);
  p.items = y.items;
  p.blocks = y.blocks;
  p.max_parts = y.max_parts;
  p.part = (float*)workspace;
  p.part_ml = (float*)((char*)workspace + y.part_ml);
  p.info = (int32_t*)((char*)workspace + y.info);
  hipStream_t hs = (hipStream_t)stream;
  if (dtype == SSA_F32) return run_drafts_dim<SSA_F32>(p, y, hs);
  if (dtype == SSA_F16) return run_drafts_dim<SSA_F16>(p, y, hs);
  return run_drafts_dim<SSA_BF16>(p, y, hs);
}

namespace {

int keep(const char* who, bool all, void* kpool, void* vpool, int dtype, int64_t layers, int64_t Hkv,
         int64_t d, int64_t pages, int64_t page, const int64_t* strides, const int32_t* table,
         int64_t table_stride, int64_t W, const int32_t* lens, const int32_t* cu, int64_t B,
         const int32_t* path, int64_t path_stride, int64_t width, const int32_t* counts,
         int32_t* new_lens, ssa_stream_t stream) {
  SSA_REQUIRE(kpool && vpool && strides && table && lens && cu && counts && new_lens &&
                  (path || width == 0), SSA_ERR_INVALID, "%s: NULL argument", who);
  SSA_TRY(check_pool(who, dtype, Hkv, d, pages, page));
  SSA_REQUIRE(B > 0 && B <= 65535 && layers > 0 && fits_int(layers) && fits_int(width) &&
                  path_stride >= 0, SSA_ERR_INVALID,
              "%s: B=%lld, layers=%lld, paths of %lld (at most 65535 requests)", who, (long long)B,
              (long long)layers, (long long)width);
  SSA_REQUIRE(kpool != vpool, SSA_ERR_INVALID, "%s: keys and values in the same memory", who);
  SSA_TRY(check_table(who, W, table_stride, page));
  const int es = dtype_size(dtype);
  // strides: kpool(layer,page,head,slot), vpool(layer,page,head,slot)
  SSA_REQUIRE(rows16(kpool, strides, 4, es) && rows16(vpool, strides + 4, 4, es), SSA_ERR_INVALID,
              "%s: rows must start at multiples of 16 bytes", who);
  const int64_t vecs = d * es / 16, columns = 2 * layers * Hkv * vecs;
  const int64_t blocks = (columns + kKeepThreads - 1) / kKeepThreads;
  SSA_REQUIRE(fits_int(columns) && fits_launch(blocks * B, kKeepThreads), SSA_ERR_UNSUPPORTED,
              "%s: %lld layers of %lld requests in one call", who, (long long)layers, (long long)B);
  // a request's workgroups read its length while the first of them writes the new one
  SSA_REQUIRE(!overlap(new_lens, B, lens, B) && !overlap(new_lens, B, counts, B) &&
                  !overlap(new_lens, B, cu, B + 1) &&
                  !overlap(new_lens, B, path, (B - 1) * path_stride + width) &&
                  !overlap(new_lens, B, table, (B - 1) * table_stride + W),
              SSA_ERR_INVALID, "%s: new_lens lies over an input", who);
  KeepParams p{(char*)kpool, (char*)vpool, table, lens, cu, path, counts, new_lens,
               table_stride, path_stride, W * page, pages, (int)width,
               (int)page, (int)Hkv, (int)vecs, (int)columns,
               strides[0] * es, strides[1] * es, strides[2] * es, strides[3] * es,
               strides[4] * es, strides[5] * es, strides[6] * es, strides[7] * es,
               page_div((int)page / 16)};
  const dim3 grid((unsigned)blocks, (unsigned)B);
  hipStream_t st = (hipStream_t)stream;
  if (!all) {
    paged_keep_kernel<kKeepEach><<<grid, kKeepThreads, 0, st>>>(p);
  } else {
    paged_keep_kernel<kKeepCheck><<<dim3(1, (unsigned)B), kKeepThreads, 0, st>>>(p);
    SSA_TRY(launch_status("paged_keep_kernel"));
    paged_keep_kernel<kKeepAll><<<grid, kKeepThreads, 0, st>>>(p);
  }
  return launch_status("paged_keep_kernel");
}

}  // namespace

extern "C" int ssa_paged_keep(void* kpool, void* vpool, int dtype, int64_t layers, int64_t Hkv,
                              int64_t d, int64_t pages, int64_t page, const int64_t* strides,
                              const int32_t* table, int64_t table_stride, int64_t W,
                              const int32_t* lens, const int32_t* cu, int64_t B,
                              const int32_t* path, int64_t path_stride, int64_t width,
                              const int32_t* counts, int32_t* new_lens, ssa_stream_t stream) {
  return keep("ssa_paged_keep", false, kpool, vpool, dtype, layers, Hkv, d, pages, page, strides, table,
              table_stride, W, lens, cu, B, path, path_stride, width, counts, new_lens, stream);
}

extern "C" int ssa_paged_keep_all(void* kpool, void* vpool, int dtype, int64_t layers, int64_t Hkv,
                                  int64_t d, int64_t pages, int64_t page, const int64_t* strides,
                                  const int32_t* table, int64_t table_stride, int64_t W,
                                  const int32_t* lens, const int32_t* cu, int64_t B,
                                  const int32_t* path, int64_t path_stride, int64_t width,
                                  const int32_t* counts, int32_t* new_lens, ssa_stream_t stream) {
  return keep("ssa_paged_keep_all", true, kpool, vpool, dtype, layers, Hkv, d, pages, page, strides,
              table, table_stride, W, lens, cu, B, path, path_stride, width, counts, new_lens, stream);
}

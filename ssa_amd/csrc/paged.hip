// The paged key-value cache: pages taken and given back from the requests' lengths, new tokens'
// keys and values stored through their slots, and one new token's attention over its pages.
//
// A pool holds `pages` pages of `page` tokens: (pages, Hkv, page, d) by strides (page, head, slot).
// Request b's token j lies in page table[b][j / page] at slot j % page.
#include <math.h>

#include "common.h"
#include "paged_index.h"

namespace ssa {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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
};

constexpr int kResizeThreads = 1024;

// Sum over the workgroup of three counts (every thread receives them).
__device__ inline void block_sum3(int64_t (&x)[3], int64_t (*red)[3]) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
  for (int c = 0; c < 3; ++c) {
    for (int off = 32; off >= 1; off >>= 1) x[c] += __shfl_xor(x[c], off);
    if (lane == 0) red[wv][c] = x[c];
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < 3; ++c) {
    x[c] = 0;
    for (int w = 0; w < kResizeThreads / 64; ++w) x[c] += red[w][c];
  }
  __syncthreads();
}

// Exclusive prefix over the workgroup's threads; total: the sum over all of them.
__device__ inline int block_scan(int x, int* red, int* total) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int s = x;
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(s, off);
    if (lane >= off) s += y;
  }
  if (lane == 63) red[wv] = s;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kResizeThreads / 64; ++w) {
    if (w < wv) before += red[w];
    all += red[w];
  }
  __syncthreads();
  *total = all;
  return before + s - x;
}

// The last i < n with at[i] <= x (at ascending, at[0] <= x): the request a page or token is of.
template <class It>
__device__ inline int last_at_most(It at, int n, int x) {
  int lo = 0, hi = n;  // at[lo] <= x < at[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One workgroup: totals first (all or nothing), then tiles of one request per thread whose pages
// are shared out over the threads by a search in the tile's prefix sums. The free pages are a
// stack; a page given back lands where a take of the same order would find it, so growing and
// shrinking back restores the stack. Takes are read before gives are written (they overlap).
__global__ __launch_bounds__(kResizeThreads) void paged_resize_kernel(ResizeParams p) {
  __shared__ int64_t red3[kResizeThreads / 64][3];
  __shared__ int red[kResizeThreads / 64];
  __shared__ int s_at[kResizeThreads], s_have[kResizeThreads], s_need[kResizeThreads];
  __shared__ int s_bad;
  const int tid = threadIdx.x;
  const int64_t cap = p.W * p.page;
  const int nfree = *p.nfree;
  if (tid == 0) s_bad = nfree < 0 || nfree > p.P;
  __syncthreads();
  int64_t sum[3] = {0, 0, 0};  // taken, given, new tokens
  for (int64_t b = tid; b < p.B; b += kResizeThreads) {
    const PagedSpan o = paged_span(p.lens[b], 0, cap), n = paged_span(p.new_lens[b], 0, cap);
    if (!o.ok || !n.ok) {
      s_bad = 1;
      continue;
    }
    const int have = paged_pages(o.len, p.page), need = paged_pages(n.len, p.page);
    sum[0] += max(need - have, 0);
    sum[1] += max(have - need, 0);
    sum[2] += max(n.len - o.len, 0);
  }
  block_sum3(sum, red3);
  const int64_t lack = sum[0] - nfree;
  const int status = s_bad || nfree - sum[0] + sum[1] > p.P ? -1
                     : sum[2] > p.T ? -2
                     : lack > 0 ? (int)min(lack, (int64_t)0x7fffffff) : 0;
  if (tid == 0) *p.status = status;
  if (status != 0) {
    for (int64_t b = tid; b <= p.B; b += kResizeThreads) p.cu[b] = 0;
    return;
  }
  const int top = nfree - (int)sum[0], left = top + (int)sum[1];
  int taken = 0, added = 0, given = 0;
  for (int64_t b0 = 0; b0 < p.B; b0 += kResizeThreads) {
    const int64_t b = b0 + tid;
    const int n = (int)min(p.B - b0, (int64_t)kResizeThreads);
    const int o = tid < n ? p.lens[b] : 0, w = tid < n ? p.new_lens[b] : 0;
    const int have = paged_pages(o, p.page), need = paged_pages(w, p.page);
    int all;
    const int at_new = block_scan(max(w - o, 0), red, &all);
    if (tid < n) p.cu[b] = added + at_new;
    added += all;
    s_have[tid] = have;
    s_at[tid] = block_scan(max(need - have, 0), red, &all);
    __syncthreads();
    for (int t = tid; t < all; t += kResizeThreads) {
      const int i = last_at_most(s_at, n, t);
      p.table[(b0 + i) * p.table_stride + s_have[i] + t - s_at[i]] =
          p.free_pages[nfree - 1 - (taken + t)];
    }
    taken += all;
    __syncthreads();
  }
  if (tid == 0) p.cu[p.B] = added;
  if (sum[1] > 0) {
    for (int64_t b0 = 0; b0 < p.B; b0 += kResizeThreads) {
      const int64_t b = b0 + tid;
      const int n = (int)min(p.B - b0, (int64_t)kResizeThreads);
      const int have = paged_pages(tid < n ? p.lens[b] : 0, p.page);
      const int need = paged_pages(tid < n ? p.new_lens[b] : 0, p.page);
      int all;
      s_need[tid] = need;
      s_at[tid] = block_scan(max(have - need, 0), red, &all);
      __syncthreads();
      for (int t = tid; t < all; t += kResizeThreads) {
        const int i = last_at_most(s_at, n, t);
        int32_t* e = p.table + (b0 + i) * p.table_stride + s_need[i] + t - s_at[i];
        p.free_pages[left - 1 - (given + t)] = *e;
        *e = -1;
      }
      given += all;
      __syncthreads();
    }
  }
  for (int64_t b = tid; b < p.B; b += kResizeThreads) p.lens[b] = p.new_lens[b];
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
    const int e = pos / p.page;
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

// A thread moves one 16-byte piece of a key row and of its value row.
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
  int64_t table_stride, cap, pages;
  int B, Hq, Hkv, G, d, page, window;
  float scale_log2;
  int64_t qb, qh, ob, oh;                 // elements
  int64_t kpp, kph, kps, vpp, vph, vps;   // elements
  int64_t knb, knh, vnb, vnh;             // elements
};

template <int DT>
__device__ inline float load_elem(const char* base, int64_t i) {
  if constexpr (DT == SSA_F32) return ((const float*)base)[i];
  else if constexpr (DT == SSA_F16) return (float)((const _Float16*)base)[i];
  else return (float)((const __bf16*)base)[i];
}

template <int DT>
__device__ inline void store_elem(char* base, int64_t i, float x) {
  if constexpr (DT == SSA_F32) ((float*)base)[i] = x;
  else if constexpr (DT == SSA_F16) ((_Float16*)base)[i] = (_Float16)x;
  else ((__bf16*)base)[i] = (__bf16)x;
}

// The new token's key and value into the slot of position len - 1, an element per thread.
template <int DT>
__global__ __launch_bounds__(256) void paged_store_new_kernel(AttendParams p) {
  const int b = blockIdx.y, h = blockIdx.x;
  const PagedSpan s = paged_span(p.lens[b], p.window, p.cap);
  if (s.len == 0) return;
  const int e = (s.len - 1) / p.page, off = (s.len - 1) - e * p.page;
  const int64_t pg = p.table[b * p.table_stride + e];
  if (pg < 0 || pg >= p.pages) return;
  for (int c = threadIdx.x; c < p.d; c += 256) {
    store_elem<DT>(p.kpool, pg * p.kpp + h * p.kph + off * p.kps + c,
                   load_elem<DT>(p.k_new, b * p.knb + h * p.knh + c));
    store_elem<DT>(p.vpool, pg * p.vpp + h * p.vph + off * p.vps + c,
                   load_elem<DT>(p.v_new, b * p.vnb + h * p.vnh + c));
  }
}

// One wave per (request, query head): 64 keys at a time, a key's score per lane, the running maximum
// and sum in fp32, the values added up with a lane's columns in registers.
template <int DT>
__global__ __launch_bounds__(64) void paged_attend_rows_kernel(AttendParams p) {
  __shared__ float qs[512], ps[64];
  __shared__ int64_t vs[64];
  const int lane = threadIdx.x, b = blockIdx.y, h = blockIdx.x, g = h / p.G;
  const PagedSpan s = paged_span(p.lens[b], p.window, p.cap);
  for (int c = lane; c < p.d; c += 64) qs[c] = load_elem<DT>(p.q, b * p.qb + h * p.qh + c);
  __syncthreads();
  float m = -INFINITY, l = 0.0f, acc[8] = {};
  bool bad = !s.ok;
  for (int j0 = s.first; j0 < s.len; j0 += 64) {
    const int j = j0 + lane, n = min(64, s.len - j0);
    float x = -INFINITY;
    int64_t vrow = 0;
    if (j < s.len) {
      const int e = j / p.page, off = j - e * p.page;
      int64_t pg = p.table[b * p.table_stride + e];
      if (pg < 0 || pg >= p.pages) {
        bad = true;
        pg = 0;
      }
      const int64_t krow = pg * p.kpp + g * p.kph + off * p.kps;
      vrow = pg * p.vpp + g * p.vph + off * p.vps;
      x = 0.0f;
      for (int c = 0; c < p.d; ++c) x += qs[c] * load_elem<DT>(p.kpool, krow + c);
      x *= p.scale_log2;
    }
    float mx = x;
    for (int off = 32; off >= 1; off >>= 1) mx = fmaxf(mx, lane_xor(mx, off));
    const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.0f : mn;
    const float w = exp2f(x - base), a = exp2f(m - base);
    float sum = w;
    for (int off = 32; off >= 1; off >>= 1) sum += lane_xor(sum, off);
    l = l * a + sum;
    m = mn;
    ps[lane] = w;
    vs[lane] = vrow;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = lane + 64 * i;
      if (c >= p.d) break;
      float y = acc[i] * a;
      for (int t = 0; t < n; ++t) y += ps[t] * load_elem<DT>(p.vpool, vs[t] + c);
      acc[i] = y;
    }
    __syncthreads();
  }
  bad = __any(bad);
  const float inv = s.len == 0 ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = lane + 64 * i;
    if (c < p.d) store_elem<DT>(p.out, b * p.ob + h * p.oh + c, bad ? NAN : acc[i] * inv);
  }
  if (p.lse && lane == 0)
    p.lse[(int64_t)b * p.Hq + h] = bad ? NAN : s.len == 0 ? -INFINITY : (m + log2f(l)) * kLn2;
}

bool fits_int(int64_t x) { return x >= 0 && x <= 0x7fffffff; }

// Rows of 16-byte pieces: the base and every stride (elements) a multiple of 16 bytes.
bool rows16(const void* base, const int64_t* strides, int n, int es) {
  if (!aligned16(base)) return false;
  for (int i = 0; i < n; ++i)
    if (strides[i] * es % 16 != 0) return false;
  return true;
}

// Checks shared by the entry points that touch a pool.
int check_pool(const char* who, int dtype, int64_t Hkv, int64_t d, int64_t pages, int64_t page) {
  SSA_REQUIRE(dtype_size(dtype) != 0, SSA_ERR_UNSUPPORTED, "%s: unknown dtype %d", who, dtype);
  SSA_REQUIRE(Hkv > 0 && Hkv <= 65535 && pages > 0 && fits_int(pages), SSA_ERR_INVALID,
              "%s: bad pool (Hkv=%lld, pages=%lld)", who, (long long)Hkv, (long long)pages);
  SSA_REQUIRE(d > 0 && d % 8 == 0 && d <= 512, SSA_ERR_UNSUPPORTED,
              "%s: head dim %lld (a multiple of 8 up to 512)", who, (long long)d);
  SSA_REQUIRE(page > 0 && page % 16 == 0 && page <= 65536, SSA_ERR_UNSUPPORTED,
              "%s: page of %lld tokens (a multiple of 16 up to 65536)", who, (long long)page);
  return SSA_OK;
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
  ResizeParams p{lens,  new_lens, table, table_stride, B,   W,     (int)page, free_pages,
                 pages, nfree,    slots, pos,          T,   cu,    status};
  hipStream_t st = (hipStream_t)stream;
  paged_resize_kernel<<<1, kResizeThreads, 0, st>>>(p);
  SSA_TRY(launch_status("paged_resize_kernel"));
  if (T > 0) {
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
  SSA_REQUIRE(fits_int(blocks), SSA_ERR_UNSUPPORTED, "ssa_paged_append: %lld tokens in one call",
              (long long)T);
  paged_append_kernel<<<(unsigned)blocks, 256, 0, (hipStream_t)stream>>>(p);
  return launch_status("paged_append_kernel");
}

extern "C" size_t ssa_paged_attend_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t d,
                                                  int64_t W, int64_t page, int64_t window) {
  return 0;
}

extern "C" int ssa_paged_attend(const void* q, void* kpool, void* vpool, void* out, float* lse,
                                int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t d,
                                int64_t pages, int64_t page, const int32_t* table,
                                int64_t table_stride, int64_t W, const int32_t* lens,
                                const void* k_new, const void* v_new, const int64_t* strides,
                                float scale, int64_t window, void* workspace,
                                size_t workspace_bytes, ssa_stream_t stream) {
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
  AttendParams p{(const char*)q, (char*)kpool, (char*)vpool, (char*)out, lse, (const char*)k_new,
                 (const char*)v_new, table, lens, table_stride, W * page, pages, (int)B, (int)Hq,
                 (int)Hkv, (int)(Hq / Hkv), (int)d, (int)page, (int)window, scale * kLog2e,
                 strides[0], strides[1], strides[8], strides[9], strides[2], strides[3],
                 strides[4], strides[5], strides[6], strides[7],
                 k_new ? strides[10] : 0, k_new ? strides[11] : 0, k_new ? strides[12] : 0,
                 k_new ? strides[13] : 0};
  hipStream_t st = (hipStream_t)stream;
  const dim3 new_grid((unsigned)Hkv, (unsigned)B), grid((unsigned)Hq, (unsigned)B);
#define SSA_PAGED_RUN(DT)                                             \
  do {                                                                \
    if (k_new) {                                                      \
      paged_store_new_kernel<DT><<<new_grid, 256, 0, st>>>(p);        \
      SSA_TRY(launch_status("paged_store_new_kernel"));               \
    }                                                                 \
    paged_attend_rows_kernel<DT><<<grid, 64, 0, st>>>(p);             \
  } while (0)
  if (dtype == SSA_F32) SSA_PAGED_RUN(SSA_F32);
  else if (dtype == SSA_F16) SSA_PAGED_RUN(SSA_F16);
  else SSA_PAGED_RUN(SSA_BF16);
#undef SSA_PAGED_RUN
  return launch_status("paged_attend_rows_kernel");
}

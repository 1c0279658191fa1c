// Device and host parts that the paged cache's kernels share: sums over a wave, the layout of the
// attention's tiles and products, its running softmax, checks of the entry points' pools.
#pragma once

#include <math.h>

#include <type_traits>

#include "common.h"
#include "paged_index.h"

namespace ssa {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ inline int other_lane(int x, int j) { return lane_xor(x, j); }
__device__ inline float other_lane(float x, int j) { return lane_xor(x, j); }
__device__ inline int64_t other_lane(int64_t x, int j) {
  const unsigned int lo = lane_xor((unsigned int)x, j), hi = lane_xor((unsigned int)(x >> 32), j);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// Sums over the wave and up to (and with) each lane: a block of lanes takes the sum of the block
// beside it, and its upper lanes add it to their prefix.
template <class I>
struct LaneSums {
  I all, upto;
};

template <class I>
__device__ inline LaneSums<I> lane_sums(I x) {
  const int lane = threadIdx.x & 63;
  LaneSums<I> s{x, x};
  auto step = [&](I y, int off) {
    s.upto += lane & off ? y : 0;
    s.all += y;
  };
  step(other_lane(s.all, 1), 1);
  step(other_lane(s.all, 2), 2);
  step(other_lane(s.all, 4), 4);
  step(other_lane(s.all, 8), 8);
  step(other_lane(s.all, 16), 16);
  step(other_lane(s.all, 32), 32);
  return s;
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

// Four values at element i (a multiple of 4) of a row, rounded to the type.
template <int DT>
__device__ inline void store_row4(char* base, int64_t i, const f32x4& x) {
  if constexpr (DT == SSA_F32) {
    *(f32x4*)(base + i * 4) = x;
  } else {
    unsigned int w[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float y = x[r];
      if constexpr (DT == SSA_BF16) w[r] = __builtin_bit_cast(unsigned short, (__bf16)y);
      else w[r] = __builtin_bit_cast(unsigned short, (_Float16)y);
    }
    *(uint2*)(base + i * 2) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
  }
}

constexpr float kF16Shift = 14.0f;
constexpr int64_t kStreamBytes = (int64_t)192 << 20;

// How a call is laid out, by type and padded head dim DP. The 16-bit products take 32 keys at once
// (two subtiles), the fp32 ones 4, so their tile is one subtile where registers are short.
template <int DT, int DP>
struct Tile {
  static constexpr int ES = DT == SSA_F32 ? 4 : 2;
  static constexpr int NT = DT == SSA_F32 && DP > 64 ? 1 : 2;  // subtiles of 16 keys
  static constexpr int NC = DP * ES / 64;                      // 64-byte chunks of a key row
  static constexpr int CB = DT == SSA_F32 ? 64 : DP < 128 ? DP : 128;  // columns of a value block
  static constexpr int LC = CB / 16;                           // of them a lane's
  static constexpr int LW = LC * ES / 4;                       // in words
  static constexpr int VB = DP / CB;
  static constexpr int NA = DP / 16;  // accumulators of 16 columns x 16 heads
  static constexpr bool kQInLds = NC >= 8;         // queries: registers are short
  static constexpr int KP = NC >= 32 ? 4 : NC >= 16 ? 2 : 1;  // pieces that a tile's keys are taken in
  // fp16 weights are taken up to 2^14 so that the small ones keep their bits
  static constexpr float kShift = DT == SSA_F16 ? kF16Shift : 0.0f;
};

__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A wave's running softmax over its keys for 16 query heads: lane l holds head l % 16, accumulator
// (vb, e) the columns vb CB + LC (4 (l / 16) + r) + e, r = 0..3. m: the largest score (log2 units),
// l: sum of 2^(score - m + kShift) over the lane's own keys until they are added up.
template <int NA>
struct Softmax {
  float m, l;
  f32x4 acc[NA];
};

// Scales (m, l, acc) of two disjoint key sets to their common maximum and adds them.
template <int NA>
__device__ inline void join(Softmax<NA>& a, float m, float l, const f32x4* acc, int stride) {
  const float mx = fmaxf(a.m, m), base = mx == -INFINITY ? 0.0f : mx;
  const float x = __builtin_amdgcn_exp2f(a.m - base), y = __builtin_amdgcn_exp2f(m - base);
  a.m = mx;
  a.l = a.l * x + l * y;
#pragma unroll
  for (int i = 0; i < NA; ++i) {
    const f32x4 o = acc[i * stride];
#pragma unroll
    for (int r = 0; r < 4; ++r) a.acc[i][r] = a.acc[i][r] * x + o[r] * y;
  }
}

__device__ inline f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c, bool bf16) {
  if (bf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// A weight's 16-bit parts: bf16 holds 8 of its 24 bits, fp16 11 (of 22: the output rounds to 11).
template <int DT>
constexpr int kParts = DT == SSA_BF16 ? 3 : 2;

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Two weights as sums of 16-bit parts, each the leading bits of what the ones before leave. bf16: three
// hold the weight exactly; with two 0.4 % of the outputs fell on the other side of their rounding, with
// three 0.05 %, as many as in plain fp32 operations. The third's product costs up to 2.5 % (one request of
// 1M tokens 90.2 -> 92.4 us, 128 of 2,000 to 9,000 with 20 heads on one 75.7 -> 77.1, 64 mixed ones 0.2 %).
// A part of another sign than the first, or zero where that is not, would turn an infinite value into NaN:
// none is negative, and instead of zero they are the smallest subnormal (fp16: 2^-38 of the largest
// weight; below that the first part is zero too and such a value gives NaN).
template <int DT>
__device__ inline void split(float p0, float p1, unsigned int (&w)[kParts<DT>]) {
  if constexpr (DT == SSA_BF16) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned int a = __float_as_uint(p0) & 0xffff0000u;
      const unsigned int b = __float_as_uint(p1) & 0xffff0000u;
      w[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      p0 -= __uint_as_float(a);
      p1 -= __uint_as_float(b);
    }
    w[2] = __builtin_bit_cast(unsigned int, bf16x2{(__bf16)p0, (__bf16)p1});
  } else {
    const auto h = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(p0, p1));
    w[0] = __builtin_bit_cast(unsigned int, h);
    w[1] = __builtin_bit_cast(unsigned int, f16x2{(_Float16)(p0 - (float)h[0]),
                                                  (_Float16)(p1 - (float)h[1])});
  }
  const u16x2 one = {1, 1};
  const u16x2 least = __builtin_elementwise_min(__builtin_bit_cast(u16x2, w[0]), one);
#pragma unroll
  for (int i = 1; i < kParts<DT>; ++i)
    w[i] = __builtin_bit_cast(
        unsigned int, __builtin_elementwise_max(__builtin_bit_cast(u16x2, w[i]), least));
}

template <int W>
struct Words {
  unsigned int w[W];
};

// Loads through a buffer descriptor: a uniform base, a lane's 32-bit offset; an offset past the
// descriptor's size reads as zero and touches no memory.
typedef __amdgpu_buffer_rsrc_t Buffer;
constexpr int kSpan = 0x7fffffff, kOutside = -0x7fffffff - 1;

__device__ inline Buffer buffer_at(const char* p) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, kSpan, 0x00027000);
}

// AUX: 0, or kStream for the non-temporal hint.
constexpr int kStream = 2;

template <int W, int AUX>
__device__ inline Words<W> load_words(Buffer b, int off) {
  if constexpr (W == 4)
    return __builtin_bit_cast(Words<W>, __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, AUX));
  else
    return __builtin_bit_cast(Words<W>, __builtin_amdgcn_raw_buffer_load_b64(b, off, 0, AUX));
}

// The rows of a lane's keys and values as they come from the cache, in the layouts of the products'
// operands: keys lane l: row l % 16 of the subtile, 16 bytes at 64 c + 16 (l / 16) (the columns'
// order within a product does not matter: queries lie alike); values: rows 4 (l / 16) + r, the
// columns of Softmax.
template <int DT, int DP>
struct Rows {
  using T = Tile<DT, DP>;
  u32x4 k[T::NT][T::NC / T::KP];
  Words<T::LW> v[T::NT][4][T::VB];
};

// With eight a unit's waves have a subtile each, half a tile: 128 requests of 2,000 to 9,000 keys, 20
// heads on one, 97 us for 86.
constexpr int kAttendWaves = 4;

bool fits_int(int64_t x) { return x >= 0 && x <= 0x7fffffff; }

// Whether a launch's threads can be counted: in 32 bits.
bool fits_launch(int64_t blocks, int threads) { return blocks <= 0xffffffffll / threads; }

// Rows of 16-byte pieces: the base and every stride (elements, none negative) a multiple of 16 bytes.
bool rows16(const void* base, const int64_t* strides, int n, int es) {
  if (!aligned16(base)) return false;
  for (int i = 0; i < n; ++i)
    if (strides[i] < 0 || strides[i] * es % 16 != 0) return false;
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

// Bytes of the keys and values of one unit of every key head.
int64_t unit_bytes(int dtype, int64_t d, int64_t Hkv) {
  return 2 * 16 * kPagedUnit * dtype_size(dtype) * d * Hkv;
}

}  // namespace
}  // namespace ssa

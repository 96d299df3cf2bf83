// Selection over beams and vocabulary, and the states that follow it.
//
// The candidate (b, t) of a group is worth
//   v = S_b + L_bt                      or, with log-softmax,
//   v = S_b + (L_bt - max_t L_bt) - log(sum_t exp(L_bt - max_t L_bt)),
// compared in 64 bits; equal values go to the lower b * V + t. With log-softmax
// a beam's own candidates are ordered by S_b + L_bt in 64 bits, then t. Entries
// that are not finite are no candidates, neither are those of a beam whose S is
// not finite. A finished beam offers (b, end_token) alone, worth S_b.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gann_internal.hpp"

namespace gann {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kHits = 256;          // candidates that pass a block's threshold
constexpr float kNan = __builtin_nanf("");

template <typename T>
struct Raw;   // 16 bytes of logits
template <>
struct Raw<float> {
  static constexpr int n = 4;
  static constexpr uint32_t neg_inf = 0xff800000u;
  __device__ static float at(const uint4& v, int j) {
    return __uint_as_float(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w);
  }
  __device__ static float max(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  __device__ static float one(const float* p) { return *p; }
  __device__ static void put(uint4& v, int j, const float* p) {
    const uint32_t b = __float_as_uint(*p);
    if (j == 0) v.x = b;
    if (j == 1) v.y = b;
    if (j == 2) v.z = b;
    if (j == 3) v.w = b;
  }
};
__device__ __forceinline__ uint32_t word_of(const uint4& v, int w) {
  return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w;
}
template <typename T>
__device__ __forceinline__ void put16(uint4& v, int j, const T* p) {
  const uint32_t b = *reinterpret_cast<const uint16_t*>(p);
  const uint32_t keep = (j & 1) ? 0x0000ffffu : 0xffff0000u, set = (j & 1) ? b << 16 : b;
  if (j / 2 == 0) v.x = (v.x & keep) | set;
  if (j / 2 == 1) v.y = (v.y & keep) | set;
  if (j / 2 == 2) v.z = (v.z & keep) | set;
  if (j / 2 == 3) v.w = (v.w & keep) | set;
}
template <>
struct Raw<__half> {
  static constexpr int n = 8;
  static constexpr uint32_t neg_inf = 0xfc00fc00u;
  __device__ static __half2 h2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
  __device__ static float at(const uint4& v, int j) {
    const __half2 h = h2(word_of(v, j / 2));
    return (j & 1) ? __high2float(h) : __low2float(h);
  }
  __device__ static float max(const uint4& v) {
    const __half2 m = __hmax2(__hmax2(h2(v.x), h2(v.y)), __hmax2(h2(v.z), h2(v.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  __device__ static float one(const __half* p) { return __half2float(*p); }
  __device__ static void put(uint4& v, int j, const __half* p) { put16(v, j, p); }
};
template <>
struct Raw<__nv_bfloat16> {
  static constexpr int n = 8;
  static constexpr uint32_t neg_inf = 0xff80ff80u;
  __device__ static __nv_bfloat162 h2(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
  __device__ static float at(const uint4& v, int j) {
    const uint32_t w = word_of(v, j / 2);
    return __uint_as_float((j & 1) ? w & 0xffff0000u : w << 16);
  }
  __device__ static float max(const uint4& v) {
    const __nv_bfloat162 m = __hmax2(__hmax2(h2(v.x), h2(v.y)), __hmax2(h2(v.z), h2(v.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  __device__ static float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  __device__ static void put(uint4& v, int j, const __nv_bfloat16* p) { put16(v, j, p); }
};

// Floats as unsigned numbers of the same order (0 and -0 alike; no float is 0).
__device__ __forceinline__ uint32_t ord32(float f) {
  const uint32_t b = __float_as_uint(__fadd_rn(f, 0.f));
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unord32(uint32_t b) {
  return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}
__device__ __forceinline__ uint64_t ord64(double d) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(d + 0.0));
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double unord64(uint64_t b) {
  return __longlong_as_double(static_cast<int64_t>((b >> 63) ? (b & 0x7fffffffffffffffull) : ~b));
}

// Sort keys, largest first. Key1: a float's order and the complement of an
// index in one word; Key2: a double's order, then (see Place) what settles
// equal ones. The all-zero key stands behind every candidate.
struct Key1 {
  uint64_t a;
  __device__ bool above(const Key1& o) const { return a > o.a; }
  __device__ Key1 from(int lane_mask) const { return {__shfl_xor_sync(kFull, a, lane_mask)}; }
};
struct Key2 {
  uint64_t a, b;
  __device__ bool above(const Key2& o) const { return a > o.a || (a == o.a && b > o.b); }
  __device__ Key2 from(int lane_mask) const {
    return {__shfl_xor_sync(kFull, a, lane_mask), __shfl_xor_sync(kFull, b, lane_mask)};
  }
};

// Equal values: the lower beam first, within a beam the larger x (log-softmax
// can round the values of two x to one), then the lower token, packed so that
// the larger word comes first. beams * vocab < 2^31 leaves both numbers 32 bits.
struct Place {
  int token_bits;
  uint32_t last_beam;
  __device__ static Place of(int beams, int vocab) {
    return {32 - __clz(vocab - 1), static_cast<uint32_t>(beams) - 1};
  }
  __device__ uint64_t pack(uint32_t b, uint32_t x, uint32_t t) const {
    const uint64_t low = (static_cast<uint64_t>(1) << token_bits) - 1;
    return static_cast<uint64_t>(last_beam - b) << (32 + token_bits) | static_cast<uint64_t>(x) << token_bits | (low - t);
  }
  __device__ uint32_t beam(uint64_t p) const { return last_beam - static_cast<uint32_t>(p >> (32 + token_bits)); }
  __device__ uint32_t token(uint64_t p) const {
    const uint64_t low = (static_cast<uint64_t>(1) << token_bits) - 1;
    return static_cast<uint32_t>(low - (p & low));
  }
};

// One x for all that have the same sum with s in 64 bits: the sum less s. That
// is x itself unless s is so large that the sum rounds x to fewer bits, and
// float32 holds it either way (|x| >= |s|: off by 2^-52 of x, which rounds back;
// |x| < |s|: the difference is exact, a rounding of x). From |x| = 2^-27 |s| on
// the sum's step is at most x's and the sum exact.
// A call, not inlined: rows whose every element passes the threshold run the loop
// around it 16 to 32 times a tile (64 x 4 x 128000 equal bf16: rows 110 us
// without it, 118 with the call, 121 inlined).
__device__ __noinline__ float same_sum(float x, float s) {
  const double d = static_cast<double>(s);
  return static_cast<float>((d + static_cast<double>(x)) - d);
}
// A float that is not above any x with the same sum: those are within one step
// of the sum, which is at most 2^-52 of it.
__device__ __forceinline__ float below_same_sum(float x, float s) {
  const double d = static_cast<double>(x);
  return __double2float_rd(d - fabs(static_cast<double>(s) + d) * 0x1p-52);
}

// Whether a lane keeps the larger key at a step of a bitonic sort (largest
// first) over lanes: bit log2(size) of the lane equals bit log2(stride).
__device__ __forceinline__ bool keeps_larger(int lane, int size, int stride) {
  return size >= 32 ? (lane & stride) == 0 : ((lane ^ (lane / (size / stride))) & stride) == 0;
}

// Bitonic sort of 32 N keys by one warp, largest first; key n * 32 + lane is
// k[n] of the lane.
template <int N, typename K>
__device__ __forceinline__ void warp_sort(K (&k)[N], int lane) {
#pragma unroll
  for (int size = 2; size <= 32 * N; size <<= 1) {
#pragma unroll
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const bool down = size < 32 || ((n * 32) & size) == 0;
        if (stride >= 32) {
          const int o = n ^ (stride / 32);
          if (o > n && k[o].above(k[n]) == down) {
            const K t = k[n];
            k[n] = k[o];
            k[o] = t;
          }
        } else {
          const K o = k[n].from(stride);
          if (o.above(k[n]) == (keeps_larger(lane, size, stride) == down)) k[n] = o;
        }
      }
    }
  }
}

// The warp's 32 values sorted, largest first.
__device__ __forceinline__ float warp_sort32(float v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      const float o = __shfl_xor_sync(kFull, v, stride);
      v = keeps_larger(lane, size, stride) ? fmaxf(v, o) : fminf(v, o);
    }
  return v;
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;
// Row maxima of less than 2^17 have x log2e rounded by at most 2^-7, whose e^-d
// is 1 - d + d^2 / 2 to 3e-8. With larger ones the terms are exp(x - maximum),
// an instruction more each.
constexpr float kFarMax = 131072.f;

__device__ __forceinline__ bool live(float score) { return fabsf(score) < INFINITY; }

// Sorts the warp's keys get(0 .. total - 1) and stores the best `keep`.
template <int P, typename K, typename Get>
__device__ __forceinline__ void sort_keys(K* kept, int total, int keep, int lane, Get&& get) {
  K k[P];
#pragma unroll
  for (int n = 0; n < P; ++n) k[n] = n * kWarp + lane < total ? get(n * kWarp + lane) : K{};
  warp_sort<P>(k, lane);
  __syncwarp();
#pragma unroll
  for (int n = 0; n < P; ++n)
    if (n * kWarp + lane < min(total, keep)) kept[n * kWarp + lane] = k[n];
  __syncwarp();
}
// LONG: up to 256 keys, else up to 64.
template <bool LONG, typename K, typename Get>
__device__ __forceinline__ void sort_some(K* kept, int total, int keep, int lane, Get&& get) {
  __syncwarp();
  if (total <= 32) sort_keys<1>(kept, total, keep, lane, get);
  else if (!LONG || total <= 64) sort_keys<2>(kept, total, keep, lane, get);
  else if (total <= 128) sort_keys<4>(kept, total, keep, lane, get);
  else sort_keys<8>(kept, total, keep, lane, get);
}
// More than 128 (float, index) keys of which at most 128 are kept: the floats'
// order is bisected until between `keep` and 128 keys pass, which halves the
// sort. Returns how many are left, all of them if equal floats leave no such
// place.
__device__ __forceinline__ int trim_long(Key1* list, int total, int keep, int lane) {
  Key1 k[kHits / kWarp];
  uint32_t lo = 0xffffffffu, hi = 0;
  __syncwarp();
#pragma unroll
  for (int n = 0; n < kHits / kWarp; ++n) {
    k[n] = n * kWarp + lane < total ? list[n * kWarp + lane] : Key1{0};
    if (k[n].a) {
      lo = min(lo, static_cast<uint32_t>(k[n].a >> 32));
      hi = max(hi, static_cast<uint32_t>(k[n].a >> 32));
    }
  }
  lo = __reduce_min_sync(kFull, lo);
  hi = __reduce_max_sync(kFull, hi) + 1;
  int n_lo = total;
  while (n_lo > 128 && hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    int c = 0;
#pragma unroll
    for (int n = 0; n < kHits / kWarp; ++n) c += static_cast<uint32_t>(k[n].a >> 32) >= mid;
    c = __reduce_add_sync(kFull, c);
    if (c >= keep) {
      lo = mid;
      n_lo = c;
    } else {
      hi = mid;
    }
  }
  if (n_lo > 128) return total;
  int at = 0;
#pragma unroll
  for (int n = 0; n < kHits / kWarp; ++n) {
    const bool take = k[n].a && static_cast<uint32_t>(k[n].a >> 32) >= lo;
    const unsigned m = __ballot_sync(kFull, take);
    if (take) list[at + __popc(m & ((1u << lane) - 1u))] = k[n];
    at += __popc(m);
  }
  __syncwarp();
  return at;
}

// Candidates that a warp holds at a time, kept ones among them, in the two
// forms of the kernels below: keep <= 16, and more.
constexpr int kShortKeep = 16;
template <bool LONG>
struct Held {
  static constexpr int value = LONG ? kHits : 64;
};

// --------------------------------------------------------- segments of rows
// Large vocabularies, and every call with log-softmax: a warp streams a
// segment of one row, four 16-byte vectors a lane at a time with the next four
// on their way, and keeps, without any barrier,
//   - for each lane the running maximum and the sum of exp(x - maximum) (terms
//     in float32, at most 32 at a time, joined in 64 bits);
//   - the list of the best candidates. The first tile sets its threshold: of
//     the 32 lanes' maxima the keep-th largest (keep <= 16), or among the 128
//     vectors' maxima by bisection, has `keep` elements at or above it. Lanes
//     mark their elements at or above the threshold; the marked ones are
//     compared with the least kept key and listed, one a lane at a time. The
//     list is sorted and cut when it is full, which raises the threshold.
//     Listed is same_sum(x), so that the order is that of the 64-bit sums with
//     the score; the threshold lies at or below every x of an equal sum.
// A segment writes its `keep` best and its sum; merge_kernel joins them.
// 64 x 4 x 128000 bf16 with log-softmax takes 36 us with its join (reading alone
// would be 10): 25 us here, where 14 warp instructions for 32 elements (the
// exponential, its argument and sum are four of them) issue in 55 % of the slots:
// 16 warps an SM wait for their own last results, hardly for loads. The join
// takes 10 us.
// Where most elements pass the threshold they are listed one a lane a round:
// equal rows of that size take 139 us, rows masked but for four tokens by the
// type's lowest value 146 (by -inf 28), ascending rows 227.
constexpr int kRowWarps = 4, kRowVecs = 4;
constexpr int kRowTile = kRowVecs * kWarp;   // vectors

struct SegStat {
  double max, sum;
};

template <typename T, bool SOFTMAX, bool LONG>
__global__ void __launch_bounds__(kRowWarps* kWarp, 4) row_kernel(const T* __restrict__ logits, int64_t gstride,
                                                               int64_t bstride, const float* __restrict__ scores,
                                                               const uint8_t* __restrict__ finished, int64_t rows,
                                                               int beams, int vocab, int keep, int segs, int seg_tiles,
                                                               Key1* __restrict__ out, SegStat* __restrict__ stats) {
  constexpr int N = Raw<T>::n;
  constexpr uint32_t ninf = Raw<T>::neg_inf;
  constexpr int kCap = Held<LONG>::value;
  __shared__ Key1 lists[kRowWarps][kCap];
  const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kRowWarps + warp;
  if (item >= rows * segs) return;
  const int64_t rw = item / segs;
  const int seg = static_cast<int>(item - rw * segs);
  const float score = scores[rw];
  if (!live(score) || (finished && finished[rw])) return;
  const int64_t g = rw / beams;
  const T* row = logits + g * gstride + (rw - g * beams) * bstride;
  const int head = static_cast<int>((reinterpret_cast<uintptr_t>(row) % 16) / sizeof(T));
  // elements of the row before its first whole vector make a partial one; the
  // segment's first element, counted from that vector's start
  const int64_t first = static_cast<int64_t>(seg) * seg_tiles * kRowTile * N - head;

  auto load = [&](uint4 (&raw)[kRowVecs], int tile) {
    const int64_t p0 = first + static_cast<int64_t>(tile) * kRowTile * N;
    if (p0 >= 0 && p0 + kRowTile * N <= vocab) {
      const uint4* v = reinterpret_cast<const uint4*>(row + p0) + lane;
#pragma unroll
      for (int i = 0; i < kRowVecs; ++i) raw[i] = __ldcs(v + i * kWarp);
    } else {
#pragma unroll
      for (int i = 0; i < kRowVecs; ++i) {
        const int64_t p = p0 + (i * kWarp + lane) * N;
        raw[i] = make_uint4(ninf, ninf, ninf, ninf);
        if (p >= 0 && p + N <= vocab) {
          raw[i] = __ldcs(reinterpret_cast<const uint4*>(row + p));
        } else if (p + N > 0 && p < vocab) {
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (p + j >= 0 && p + j < vocab) Raw<T>::put(raw[i], j, row + p + j);
        }
      }
    }
  };

  Key1* list = lists[warp];
  Key1 floor{0};   // the least kept key once `keep` are known
  int cnt = 0;
  float thr = -INFINITY, m = -INFINITY, m2 = 0.f, fix = 1.f;
  auto cut = [&]() {
    if (LONG && cnt > 128) cnt = trim_long(list, cnt, keep, lane);
    sort_some<LONG>(list, cnt, keep, lane, [&](int i) { return list[i]; });
    cnt = min(cnt, keep);
    if (cnt < keep) return;
    floor = list[keep - 1];
    thr = fmaxf(below_same_sum(unord32(static_cast<uint32_t>(floor.a >> 32)), score), -3.402823466e+38f);
  };
  double sum = 0.0;
  const int64_t last = (vocab - first + static_cast<int64_t>(kRowTile) * N - 1) / (static_cast<int64_t>(kRowTile) * N);
  const int tiles = static_cast<int>(min(static_cast<int64_t>(seg_tiles), last));   // <= 0: nothing here
  uint4 cur[kRowVecs], nxt[kRowVecs];
  if (tiles > 0) load(cur, 0);
  for (int t = 0; t < tiles; ++t) {
    if (t + 1 < tiles) load(nxt, t + 1);
    float vm[kRowVecs], mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < kRowVecs; ++i) {
      vm[i] = Raw<T>::max(cur[i]);
      mx = fmaxf(mx, vm[i]);
    }
    if (mx == INFINITY) {   // infinite entries are masked: the maxima without them
      mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < kRowVecs; ++i) {
        vm[i] = -INFINITY;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float x = Raw<T>::at(cur[i], j);
          if (x < INFINITY) vm[i] = fmaxf(vm[i], x);
        }
        mx = fmaxf(mx, vm[i]);
      }
    }
    if (t == 0) {
      if (!LONG) {
        thr = __shfl_sync(kFull, warp_sort32(mx, lane), keep - 1);
      } else {
        uint32_t lo = 0x007fffffu, hi = __reduce_max_sync(kFull, ord32(mx)) + 1;   // lo: ord32(-inf)
        for (int r = 0; r < 32 && hi - lo > 1; ++r) {
          const uint32_t mid = lo + (hi - lo) / 2;
          const float x = unord32(mid);
          int n = 0;
#pragma unroll
          for (int i = 0; i < kRowVecs; ++i) n += __popc(__ballot_sync(kFull, vm[i] >= x));
          if (n >= keep) lo = mid;
          else hi = mid;
          if (n == keep) break;
        }
        thr = unord32(lo);
      }
      thr = fmaxf(below_same_sum(thr, score), -3.402823466e+38f);   // masked elements are below every float
    }
    const int64_t p0 = first + static_cast<int64_t>(t) * kRowTile * N;
    if (__any_sync(kFull, mx >= thr)) {
      uint32_t mark = 0;
#pragma unroll
      for (int i = 0; i < kRowVecs; ++i)
        if (vm[i] >= thr) {
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (Raw<T>::at(cur[i], j) >= thr) mark |= 1u << (i * N + j);
        }
      const bool exact = thr >= fabsf(score) * 0x1p-27f || score == 0.f;   // same_sum(x) = x from thr on
      while (__any_sync(kFull, mark)) {
        if (cnt > kCap - kWarp) cut();
        const int e = __ffs(mark) - 1;
        const int64_t p = p0 + ((e / N) * kWarp + lane) * N + e % N;
        float x = mark && p >= 0 && p < vocab ? Raw<T>::one(row + p) : kNan;
        if (!exact) x = same_sum(x, score);
        const Key1 k{(static_cast<uint64_t>(ord32(x)) << 32) | ~static_cast<uint32_t>(p)};
        const bool take = fabsf(x) < INFINITY && k.above(floor);
        const unsigned pass = __ballot_sync(kFull, take);
        if (take) list[cnt + __popc(pass & ((1u << lane) - 1u))] = k;
        cnt += __popc(pass);
        mark &= mark - 1;
      }
      // a higher threshold is worth a short sort
      if (cnt > max(16, 2 * keep)) cut();
    }
    if (SOFTMAX) {
      if (mx > m) {
        sum *= static_cast<double>(fast_exp2((m - mx) * kLog2e));
        m = mx;
        m2 = m * kLog2e;
        const float d = __fmaf_rn(m, kLog2e, -m2) * 0.6931471805599453f;
        fix = fabsf(m) < kFarMax ? __fmaf_rn(d, __fmaf_rn(0.5f, d, -1.f), 1.f) : kNan;
      }
      float part = 0.f;
      if (m > -INFINITY) {
        // 2^(x log2e - m2), one fused step an element; `fix` = e^-d makes up
        // for m2's rounding d
#pragma unroll
        for (int i = 0; i < kRowVecs; ++i)
#pragma unroll
          for (int j = 0; j < N; ++j) part += fast_exp2(__fmaf_rn(Raw<T>::at(cur[i], j), kLog2e, -m2));
        part *= fix;
        if (!(part >= 0.f && part < INFINITY)) {   // a NaN or infinite entry, or a maximum far from 0: again without
          part = 0.f;
#pragma unroll
          for (int i = 0; i < kRowVecs; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) {
              const float x = Raw<T>::at(cur[i], j);
              if (fabsf(x) < INFINITY) part += fast_exp2((x - m) * kLog2e);
            }
        }
      }
      sum += static_cast<double>(part);
    }
#pragma unroll
    for (int i = 0; i < kRowVecs; ++i) cur[i] = nxt[i];
  }
  if (cnt > keep) cut();
  __syncwarp();
  for (int j = lane; j < keep; j += kWarp) out[item * keep + j] = j < cnt ? list[j] : Key1{0};
  if (SOFTMAX) {
    const float mm = unord32(__reduce_max_sync(kFull, ord32(m)));
    sum = m > -INFINITY ? sum * static_cast<double>(fast_exp2((m - mm) * kLog2e)) : 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    if (lane == 0) stats[item] = {static_cast<double>(mm), sum};
  }
}

// ------------------------------------------------------------ whole groups
// Many groups, no softmax: a warp takes a whole group, in tiles of NV vectors a
// lane (16 bytes, or single elements when rows are not whole vectors), of which
// only the maxima stay in registers. f = fl32(x + S_b) orders candidates as
// their 64-bit values do, up to equality. The first tile sets a threshold of
// f: the keep-th largest of the lanes' maxima (keep <= 16), or of the vectors'
// by bisection, has `keep` elements at or above it. Vectors whose maximum
// passes are read again (from L1), one a lane at a time, and their elements at
// or above the threshold are listed as (f, index); the sort by that is looked
// over for equal f, which are put in the order of their 64-bit values.
// 100000 x 8 x 256 f32, keep 8: 182 us (4.6 TB/s; 17 warp instructions for 32
// elements would be 97), bound by the latency of one tile a warp, which is
// loaded, waited for and worked through; 10000 x 8 x 100, keep 100: 51 us, most
// of it the sort of 128. Groups of equal entries take 1260 us at the first size,
// four entries left 760 (the rest -inf) or 1110 (the type's lowest value).
constexpr int kGroupWarps = 4;

template <typename T, int VW>
struct Vec {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ float at(int j) const { return Raw<T>::at(v, j); }
  __device__ __forceinline__ float max() const { return Raw<T>::max(v); }
};
template <typename T>
struct Vec<T, 1> {
  float v;
  __device__ __forceinline__ void load(const T* p) { v = Raw<T>::one(p); }
  __device__ __forceinline__ float at(int) const { return v; }
  __device__ __forceinline__ float max() const { return v; }
};

template <typename T, int VW, int NV, bool LONG>
__global__ void __launch_bounds__(kGroupWarps* kWarp, NV * VW > 32 ? 5 : 7) group_kernel(
    const T* __restrict__ logits, int64_t gstride, int64_t bstride, const float* __restrict__ scores,
    const uint8_t* __restrict__ finished, int64_t groups, int beams, int vocab, int keep, int end_token, uint32_t magic,
    int shift, float* __restrict__ out_s, int32_t* __restrict__ out_p, int32_t* __restrict__ out_t) {
  constexpr int kCap = Held<LONG>::value;
  __shared__ Key1 lists[kGroupWarps][kCap];
  __shared__ float cs[kGroupWarps][kBeamMax];
  const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
  const int64_t g = static_cast<int64_t>(blockIdx.x) * kGroupWarps + warp;
  if (g >= groups) return;
  const T* base = logits + g * gstride;
  const float* sc = scores + g * beams;
  float* c = cs[warp];
  Key1* list = lists[warp];
  const uint32_t vr = static_cast<uint32_t>(vocab) / VW, nvec = vr * beams;
  // row of a vector: division by the row's length as a product (magic =
  // ceil(2^(32+shift) / vr), exact below 2^31)
  auto row_of = [&](uint32_t v) { return (magic ? __umulhi(v, magic) : v) >> shift; };
  auto where = [&](uint32_t v) {
    const uint32_t b = row_of(v);
    return base + b * bstride + static_cast<int64_t>(v - b * vr) * VW;
  };
  const bool joined = bstride == vocab;
  float f[NV];   // of the vectors' maxima; NaN: nothing there
  auto load = [&](uint32_t t0) {
    Vec<T, VW> raw[NV];
    if (joined && t0 + NV * kWarp <= nvec) {
      const T* p = base + static_cast<int64_t>(t0 + lane) * VW;
#pragma unroll
      for (int i = 0; i < NV; ++i) raw[i].load(p + i * kWarp * VW);
#pragma unroll
      for (int i = 0; i < NV; ++i) f[i] = raw[i].max();
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const uint32_t v = t0 + i * kWarp + lane;
        f[i] = kNan;
        if (v < nvec) {
          raw[i].load(where(v));
          f[i] = raw[i].max();
        }
      }
    }
  };
  load(0);
  for (int b = lane; b < beams; b += kWarp) {
    const float s = sc[b];
    c[b] = live(s) && !(finished && finished[g * beams + b]) ? s : kNan;
  }
  __syncwarp();

  int cnt = 0;
  bool full = false;       // `keep` candidates are known: the last one is the floor
  float thr = -INFINITY;   // candidates have f >= thr
  double floor_v = 0.0;
  uint32_t floor_id = 0;
  auto value = [&](uint32_t id) {
    const uint32_t b = row_of(id / VW);
    if (isnan(c[b])) return static_cast<double>(sc[b]);   // a finished beam's candidate
    return static_cast<double>(c[b]) + static_cast<double>(Raw<T>::one(base + b * bstride + (id - b * vocab)));
  };
  auto cut = [&]() {
    const int total = LONG && cnt > 128 ? trim_long(list, cnt, keep, lane) : cnt;
    sort_some<LONG>(list, total, total, lane, [&](int i) { return list[i]; });
    bool equal = false;
    for (int i = lane; i + 1 < total && i < keep; i += kWarp) equal |= (list[i].a >> 32) == (list[i + 1].a >> 32);
    if (__any_sync(kFull, equal)) {
      for (bool moved = true; moved;) {
        moved = false;
        for (int odd = 0; odd < 2; ++odd) {
          for (int i = odd + 2 * lane; i + 1 < total; i += 2 * kWarp) {
            const Key1 x = list[i], y = list[i + 1];
            if ((x.a >> 32) == (y.a >> 32) && value(~static_cast<uint32_t>(x.a)) < value(~static_cast<uint32_t>(y.a))) {
              list[i] = y;
              list[i + 1] = x;
              moved = true;
            }
          }
          __syncwarp();
        }
        moved = __any_sync(kFull, moved);
      }
    }
    cnt = min(total, keep);
    full = cnt == keep;
    if (!full) return;
    floor_id = ~static_cast<uint32_t>(list[keep - 1].a);
    floor_v = value(floor_id);
    thr = unord32(static_cast<uint32_t>(list[keep - 1].a >> 32));
  };

  for (uint32_t t0 = 0; t0 < nvec; t0 += NV * kWarp) {
    if (t0) load(t0);
    float mx = -INFINITY;
    bool inf = false;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      inf |= f[i] == INFINITY;
      const uint32_t v = t0 + i * kWarp + lane;
      f[i] = __fadd_rn(f[i], c[row_of(min(v, nvec - 1))]);
      mx = fmaxf(mx, f[i]);
    }
    if (__any_sync(kFull, inf)) {   // masked entries: maxima without them
      mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const uint32_t v = t0 + i * kWarp + lane;
        f[i] = kNan;
        if (v < nvec) {
          Vec<T, VW> w;
          w.load(where(v));
          float x = -INFINITY;
#pragma unroll
          for (int j = 0; j < VW; ++j)
            if (w.at(j) < INFINITY) x = fmaxf(x, w.at(j));
          f[i] = __fadd_rn(x, c[row_of(v)]);
          mx = fmaxf(mx, f[i]);
        }
      }
    }
    if (t0 == 0) {
      if (!LONG) {
        thr = __shfl_sync(kFull, warp_sort32(mx, lane), keep - 1);
      } else {
        // bisection by value, then (far from done) over the order of floats
        float lo = -INFINITY, low = INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (f[i] > -INFINITY) low = fminf(low, f[i]);
        float hi = unord32(__reduce_max_sync(kFull, ord32(mx)));
        float mid = -unord32(__reduce_max_sync(kFull, ord32(-low)));
        for (int r = 0; r < 24 && hi > mid; ++r) {
          int n = 0;
#pragma unroll
          for (int i = 0; i < NV; ++i) n += __popc(__ballot_sync(kFull, f[i] >= mid));
          if (n >= keep) {
            lo = mid;
            if (n <= keep + 4) break;
          } else {
            hi = mid;
          }
          const uint32_t a = ord32(lo), b = ord32(hi);
          if (b - a <= 1) break;
          mid = r < 10 && lo > -INFINITY ? 0.5f * lo + 0.5f * hi : unord32(a + (b - a) / 2);
          if (!(mid > lo && mid < hi)) mid = unord32(a + (b - a) / 2);
        }
        thr = lo;
      }
    }
    uint32_t vecs = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (f[i] >= thr) vecs |= 1u << i;
    // one element a lane a round; finished beams, one candidate each, behind
    // the first tile's
    Vec<T, VW> w;
    uint32_t elems = 0, id0 = 0;
    float cb = kNan;
    int b0 = finished && t0 == 0 ? 0 : beams;
    while (true) {
      bool take = false;
      float fx = kNan;
      uint32_t id = 0;
      if (__any_sync(kFull, vecs | elems)) {
        if (!elems && vecs) {
          const uint32_t v = t0 + (__ffs(vecs) - 1) * kWarp + lane;
          vecs &= vecs - 1;
          w.load(where(v));
          cb = c[row_of(v)];
          id0 = v * VW;
#pragma unroll
          for (int j = 0; j < VW; ++j)
            if (__fadd_rn(w.at(j), cb) >= thr && fabsf(w.at(j)) < INFINITY) elems |= 1u << j;
        }
        if (elems) {
          const int e = __ffs(elems) - 1;
          elems &= elems - 1;
          float x = w.at(0);
#pragma unroll
          for (int j = 1; j < VW; ++j)
            if (e == j) x = w.at(j);
          fx = __fadd_rn(x, cb);
          id = id0 + e;
          take = true;
        }
      } else if (b0 < beams) {
        const int b = b0 + lane;
        take = b < beams && isnan(c[b]) && live(sc[b]);
        if (take) {
          fx = sc[b];
          id = static_cast<uint32_t>(b) * vocab + end_token;
        }
        b0 += kWarp;
      } else {
        break;
      }
      if (cnt > kCap - kWarp) cut();
      take = take && fx >= thr;
      if (full && take && fx == thr) {
        const double v = value(id);
        take = v > floor_v || (v == floor_v && id < floor_id);
      }
      const unsigned pass = __ballot_sync(kFull, take);
      if (take) list[cnt + __popc(pass & ((1u << lane) - 1u))] = {(static_cast<uint64_t>(ord32(fx)) << 32) | ~id};
      cnt += __popc(pass);
    }
    if (t0 + NV * kWarp >= nvec || cnt > (LONG ? kCap / 2 : max(16, 2 * keep))) cut();
  }
  __syncwarp();
  for (int j = lane; j < keep; j += kWarp) {
    const bool ok = j < cnt;
    const uint32_t idx = ok ? ~static_cast<uint32_t>(list[j].a) : 0u, b = row_of(idx / VW);
    out_s[g * keep + j] = ok ? static_cast<float>(value(idx)) : -INFINITY;
    out_p[g * keep + j] = ok ? static_cast<int32_t>(b) : -1;
    out_t[g * keep + j] = ok ? static_cast<int32_t>(idx - b * vocab) : -1;
  }
}

// ------------------------------------------------------------------- join
// The segments' candidates of one group: a block a group. Warps join rows'
// sums, then each takes a part of the candidates, values them in 64 bits and
// keeps its best in a sorted list; a candidate's place in the result is its
// place in its own list plus, for every other list, the number of keys above
// it (binary search).
template <bool LONG>
struct Merge {
  static constexpr int warps = LONG ? 8 : 16;
};

template <bool LONG>
__global__ void __launch_bounds__(Merge<LONG>::warps* kWarp) merge_kernel(
    const Key1* __restrict__ cand, const SegStat* __restrict__ stats, const float* __restrict__ scores,
    const uint8_t* __restrict__ finished, int64_t groups, int beams, int vocab, int keep, int segs, int softmax,
    int end_token, float* __restrict__ out_s, int32_t* __restrict__ out_p, int32_t* __restrict__ out_t) {
  constexpr int kCap = Held<LONG>::value, kMergeWarps = Merge<LONG>::warps;
  __shared__ double offs[kBeamMax], tops[kBeamMax];   // v = offs + (x - tops)
  __shared__ uint8_t kind[kBeamMax];                  // 0 no candidates, 1 lists, 2 finished
  __shared__ Key2 lists[kMergeWarps][kCap];
  __shared__ int counts[kMergeWarps];
  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  const Place place = Place::of(beams, vocab);
  cudaGridDependencySynchronize();
  const int64_t per_beam = static_cast<int64_t>(segs) * keep, total = per_beam * beams;
  const bool small = total < (int64_t(1) << 31);
  for (int64_t g = blockIdx.x; g < groups; g += gridDim.x) {
    const float* sc = scores + g * beams;
    for (int b = warp; b < beams; b += kMergeWarps) {
      const float s = sc[b];
      const bool fin = finished && finished[g * beams + b];
      double mx = -INFINITY, sum = 0.0;
      if (softmax && !fin && live(s)) {
        const SegStat* st = stats + (g * beams + b) * segs;
        for (int i = lane; i < segs; i += kWarp) mx = fmax(mx, st[i].max);
#pragma unroll
        for (int o = 16; o; o >>= 1) mx = fmax(mx, __shfl_xor_sync(kFull, mx, o));
        if (mx > -INFINITY)
          for (int i = lane; i < segs; i += kWarp)
            if (st[i].sum > 0.0) sum += st[i].sum * exp(st[i].max - mx);
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
      }
      if (lane == 0) {
        kind[b] = !live(s) ? 0 : fin ? 2 : 1;
        offs[b] = static_cast<double>(s) - (sum > 0.0 ? log(sum) : 0.0);
        tops[b] = mx > -INFINITY ? mx : 0.0;
      }
    }
    __syncthreads();
    // at least 32 candidates a warp, and no more warps than that needs
    const int warps = static_cast<int>(min(static_cast<int64_t>(kMergeWarps), (total + kWarp - 1) / kWarp));
    const int64_t e0 = total * warp / warps, e1 = warp < warps ? total * (warp + 1) / warps : e0;
    Key2* list = lists[warp];
    Key2 floor{0, 0};
    int cnt = 0;
    int64_t e = e0;
    int b0 = warp == 0 && finished ? 0 : beams;
    while (true) {
      const bool more = e < e1 || b0 < beams;
      if (cnt > kCap - kWarp || (!more && cnt)) {
        sort_some<LONG>(list, cnt, keep, lane, [&](int i) { return list[i]; });
        cnt = min(cnt, keep);
        if (cnt == keep) floor = list[keep - 1];
      }
      if (!more) break;
      bool take = false;
      Key2 k{0, 0};
      if (e < e1) {
        const int64_t at = e + lane;
        if (at < e1) {
          const int b = small ? static_cast<int>(static_cast<uint32_t>(at) / static_cast<uint32_t>(per_beam))
                              : static_cast<int>(at / per_beam);
          if (kind[b] == 1) {   // rows without candidates have no lists
            const uint64_t x = cand[g * total + at].a;
            take = x != 0;
            const uint32_t o = static_cast<uint32_t>(x >> 32);
            if (take)
              k = {ord64(offs[b] + (static_cast<double>(unord32(o)) - tops[b])),
                   place.pack(b, o, ~static_cast<uint32_t>(x))};
          }
        }
        e += kWarp;
      } else {
        const int b = b0 + lane;
        take = b < beams && kind[b] == 2;
        if (take) k = {ord64(static_cast<double>(sc[b])), place.pack(b, 0, end_token)};
        b0 += kWarp;
      }
      take = take && k.above(floor);
      const unsigned pass = __ballot_sync(kFull, take);
      if (take) list[cnt + __popc(pass & ((1u << lane) - 1u))] = k;
      cnt += __popc(pass);
    }
    if (lane == 0) counts[warp] = cnt;
    __syncthreads();
    int found = 0;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) found += counts[w];
    for (int j = tid; j < kMergeWarps * keep; j += kMergeWarps * kWarp) {
      const int w = j / keep, i = j - w * keep;
      if (i >= counts[w]) continue;
      const Key2 k = lists[w][i];
      int rank = i;
      for (int o = 0; o < warps; ++o) {
        if (o == w) continue;
        int lo = 0, hi = counts[o];   // keys above k come first
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (lists[o][mid].above(k)) lo = mid + 1;
          else hi = mid;
        }
        rank += lo;
      }
      if (rank < keep) {
        out_s[g * keep + rank] = static_cast<float>(unord64(k.a));
        out_p[g * keep + rank] = static_cast<int32_t>(place.beam(k.b));
        out_t[g * keep + rank] = static_cast<int32_t>(place.token(k.b));
      }
    }
    for (int j = found + tid; j < keep; j += kMergeWarps * kWarp) {
      out_s[g * keep + j] = -INFINITY;
      out_p[g * keep + j] = -1;
      out_t[g * keep + j] = -1;
    }
    __syncthreads();
  }
}

struct StateTable {
  gann_state s[kStateBatch];
};

// A thread owns one unit of U bytes at one place of a group's blocks, in every
// beam. MAX > 0: it reads the unit of every kept row (at most MAX) before it
// writes any, so source and target may be the same rows; rows that stay where
// they are are not touched. MAX 0: source and target are apart, and eight rows
// at a time are on their way. Bound by memory: each kept row is written once
// and each distinct parent read once from DRAM (again from the caches); four
// caches of 16 x 4 beams, 0.9 GB, take 141 us (6.4 TB/s).
template <typename U, int MAX>
__global__ void __launch_bounds__(256) reorder_kernel(const __grid_constant__ StateTable tab,
                                                      const int32_t* __restrict__ parents, int beams, int keep) {
  const gann_state& s = tab.s[blockIdx.z];
  const int64_t g = blockIdx.y;
  __shared__ int32_t par[kBeamMax];
  for (int j = threadIdx.x; j < keep; j += blockDim.x) {
    const int b = parents[g * keep + j];
    par[j] = b >= 0 && b < beams ? b : -1;
  }
  __syncthreads();
  const int64_t units = s.row_bytes / static_cast<int64_t>(sizeof(U));
  const int64_t total = s.size[0] * s.size[1] * units;
  const uint8_t* src = static_cast<const uint8_t*>(s.src) + g * s.src_group;
  uint8_t* dst = static_cast<uint8_t*>(s.dst) + g * s.dst_group;
  const bool same = s.src == s.dst;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < total;
       e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    int64_t u, i0, i1;
    if (total < (int64_t(1) << 31)) {
      const uint32_t r = static_cast<uint32_t>(e) / static_cast<uint32_t>(units);
      u = static_cast<uint32_t>(e) - r * static_cast<uint32_t>(units);
      i0 = r / static_cast<uint32_t>(s.size[1]);
      i1 = r - static_cast<uint32_t>(i0) * static_cast<uint32_t>(s.size[1]);
    } else {
      const int64_t r = e / units;
      u = e - r * units;
      i0 = r / s.size[1];
      i1 = r - i0 * s.size[1];
    }
    const uint8_t* p = src + i0 * s.src_stride[0] + i1 * s.src_stride[1] + u * static_cast<int64_t>(sizeof(U));
    uint8_t* q = dst + i0 * s.dst_stride[0] + i1 * s.dst_stride[1] + u * static_cast<int64_t>(sizeof(U));
    constexpr int V = MAX ? MAX : 8;
    for (int j0 = 0; j0 < (MAX ? 1 : keep); j0 += V) {
      U v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[j] = U{};
        if (j0 + j < keep) {
          const int b = par[j0 + j];
          if (b >= 0 && !(MAX && same && b == j)) v[j] = *reinterpret_cast<const U*>(p + b * s.src_beam);
        }
      }
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j0 + j < keep && !(MAX && same && par[j0 + j] == j))
          *reinterpret_cast<U*>(q + (j0 + j) * s.dst_beam) = v[j];
    }
  }
}

}  // namespace

namespace {

// How a call is run. Without softmax a warp can take a whole group: one
// launch, nothing written but the result. That wants groups so small that a
// lone warp is done at once, or enough of them to fill the GPU and none so
// large that a warp's one tile at a time cannot keep the memory busy.
// Everything else is split: rows into segments, a warp each, as many as the
// GPU holds at a time, and joined by a second kernel. Sixteen warps an SM: more
// warps leave each fewer tiles to pay for its threshold with and the join more
// candidates (64 x 4 x 128000 bf16, keep 8: 34 us with 16, 35 with 20, 38 with
// 24, 45 with 32, before the segments compared 64-bit sums, which costs under a
// microsecond). The number of SMs is a constant because the workspace's size
// follows from it, and that is asked for without a device.
constexpr int kResidentWarps = 148 * 16;
constexpr int kSmallGroup = 4096, kLargeGroup = 65536;   // bytes of a group

struct SelectPlan {
  bool split = false;
  int segs = 0, seg_tiles = 0;
};

SelectPlan plan_select(int64_t groups, int beams, int vocab, int dtype, bool softmax) {
  SelectPlan p;
  const int elem = dtype == GANN_F32 ? 4 : 2, n = 16 / elem;
  const int64_t bytes = static_cast<int64_t>(beams) * vocab * elem;
  p.split = softmax || !(bytes <= kSmallGroup || (bytes <= kLargeGroup && groups >= kResidentWarps / 4));
  if (!p.split) return p;
  const int64_t rows = std::max<int64_t>(1, groups * beams);
  const int64_t tiles = (static_cast<int64_t>(vocab) + n - 1 + kRowTile * n - 1) / (kRowTile * n);   // a row may start inside a vector
  const int64_t want = std::max<int64_t>(1, kResidentWarps / rows);
  // at least four tiles a warp, or the join has more to do than is saved
  p.seg_tiles = static_cast<int>(std::min<int64_t>(tiles, std::max<int64_t>(4, (tiles + want - 1) / want)));
  p.segs = static_cast<int>((tiles + p.seg_tiles - 1) / p.seg_tiles);
  return p;
}

}  // namespace

size_t beam_select_workspace(int64_t groups, int beams, int vocab, int keep, int dtype, bool softmax) {
  const SelectPlan p = plan_select(groups, beams, vocab, dtype, softmax);
  if (!p.split) return 0;
  const size_t items = static_cast<size_t>(groups) * beams * p.segs;
  return items * (sizeof(SegStat) + sizeof(Key1) * keep);
}

namespace {

template <typename T>
cudaError_t run_group(const SelectArgs& a, cudaStream_t st) {
  constexpr int n = Raw<T>::n;
  const bool vec = a.vocab % n == 0 && a.group_stride % n == 0 && a.beam_stride % n == 0 &&
                   reinterpret_cast<uintptr_t>(a.logits) % 16 == 0;
  const uint32_t div = static_cast<uint32_t>(vec ? a.vocab / n : a.vocab);
  // magic and shift of a division by `div` that is exact below 2^31
  uint32_t magic = 0;
  int shift = 0;
  while ((1u << shift) < div) ++shift;
  if ((1u << shift) != div) {
    --shift;
    magic = static_cast<uint32_t>(((1ull << (32 + shift)) + div - 1) / div);
  }
  auto run = [&](auto fn) {
    fn<<<static_cast<unsigned>((a.groups + kGroupWarps - 1) / kGroupWarps), kGroupWarps * kWarp, 0, st>>>(
        static_cast<const T*>(a.logits), a.group_stride, a.beam_stride, a.scores, a.finished, a.groups, a.beams,
        a.vocab, a.keep, a.end_token, magic, shift, a.out_scores, a.out_parents, a.out_tokens);
    return cudaGetLastError();
  };
  const bool many = a.keep > kShortKeep;
  if (!vec) return many ? run(group_kernel<T, 1, 16, true>) : run(group_kernel<T, 1, 16, false>);
  // 16 vectors a lane when they hold the whole group
  const int64_t nvec = static_cast<int64_t>(div) * a.beams;
  if (nvec > 8 * kWarp && nvec <= 16 * kWarp)
    return many ? run(group_kernel<T, n, 16, true>) : run(group_kernel<T, n, 16, false>);
  return many ? run(group_kernel<T, n, 8, true>) : run(group_kernel<T, n, 8, false>);
}

template <typename T>
cudaError_t run_split(const SelectArgs& a, const SelectPlan& p, int sm_count, cudaStream_t st) {
  const int64_t rows = a.groups * a.beams, items = rows * p.segs;
  if ((items + kRowWarps - 1) / kRowWarps > INT32_MAX) return cudaErrorInvalidConfiguration;
  SegStat* stats = static_cast<SegStat*>(a.workspace);
  Key1* cand = reinterpret_cast<Key1*>(stats + items);
  auto run = [&](auto fn) {
    fn<<<static_cast<unsigned>((items + kRowWarps - 1) / kRowWarps), kRowWarps * kWarp, 0, st>>>(
        static_cast<const T*>(a.logits), a.group_stride, a.beam_stride, a.scores, a.finished, rows, a.beams, a.vocab,
        a.keep, p.segs, p.seg_tiles, cand, stats);
    return cudaGetLastError();
  };
  const bool many = a.keep > kShortKeep;
  const cudaError_t e = a.softmax ? many ? run(row_kernel<T, true, true>) : run(row_kernel<T, true, false>)
                        : many    ? run(row_kernel<T, false, true>)
                                  : run(row_kernel<T, false, false>);
  if (e != cudaSuccess) return e;
  // the join's launch is prepared while the segments run; its blocks start when
  // the last of theirs has ended, since none of them lets it start sooner
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(a.groups, static_cast<int64_t>(sm_count) * 64)));
  cfg.blockDim = dim3((many ? Merge<true>::warps : Merge<false>::warps) * kWarp);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, many ? merge_kernel<true> : merge_kernel<false>, static_cast<const Key1*>(cand),
                            static_cast<const SegStat*>(stats), a.scores, a.finished, a.groups, a.beams, a.vocab,
                            a.keep, p.segs, a.softmax, a.end_token, a.out_scores, a.out_parents, a.out_tokens);
}

template <typename T>
cudaError_t run_select(const SelectArgs& a, int sm_count, cudaStream_t st) {
  const SelectPlan p = plan_select(a.groups, a.beams, a.vocab, a.dtype, a.softmax != 0);
  return p.split ? run_split<T>(a, p, sm_count, st) : run_group<T>(a, st);
}

}  // namespace

cudaError_t launch_beam_select(const SelectArgs& a, int sm_count, cudaStream_t st) {
  if (a.groups <= 0) return cudaSuccess;
  if (a.dtype == GANN_F32) return run_select<float>(a, sm_count, st);
  if (a.dtype == GANN_F16) return run_select<__half>(a, sm_count, st);
  return run_select<__nv_bfloat16>(a, sm_count, st);
}

namespace {

// The widest unit that all addresses, strides and rows of the states allow.
int state_unit(const gann_state* s, int count) {
  int64_t bits = 16;
  for (int i = 0; i < count; ++i)
    bits |= static_cast<int64_t>(reinterpret_cast<uintptr_t>(s[i].src)) | static_cast<int64_t>(reinterpret_cast<uintptr_t>(s[i].dst)) |
            s[i].src_group | s[i].src_beam | s[i].dst_group | s[i].dst_beam | s[i].row_bytes | s[i].src_stride[0] |
            s[i].src_stride[1] | s[i].dst_stride[0] | s[i].dst_stride[1];
  return static_cast<int>(bits & -bits);
}

template <typename U>
cudaError_t run_reorder(const StateTable& t, bool in_place, const dim3& grid, const int32_t* parents, int beams,
                        int keep, cudaStream_t st) {
  if (!in_place) reorder_kernel<U, 0><<<grid, 256, 0, st>>>(t, parents, beams, keep);
  else if (keep <= 8) reorder_kernel<U, 8><<<grid, 256, 0, st>>>(t, parents, beams, keep);
  else if (keep <= 32) reorder_kernel<U, 32><<<grid, 256, 0, st>>>(t, parents, beams, keep);
  else if constexpr (sizeof(U) <= 4) reorder_kernel<U, kBeamMax><<<grid, 256, 0, st>>>(t, parents, beams, keep);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_reorder_states(const gann_state* states, int count, const int32_t* parents, int64_t groups,
                                  int beams, int keep, int sm_count, cudaStream_t st) {
  // states of the same kind (in place or not) and alignment share launches
  for (int kind = 0; kind < 10; ++kind) {
    const bool in_place = kind >= 5;
    const int unit = 1 << (kind % 5);
    for (int next = 0; next < count;) {
      StateTable tab{};
      int c = 0;
      int64_t most = 0;
      for (; next < count && c < kStateBatch; ++next) {
        const gann_state& s = states[next];
        const int64_t size = s.size[0] * s.size[1] * s.row_bytes;
        if (size == 0 || (s.src == s.dst) != in_place || state_unit(&s, 1) != unit) continue;
        tab.s[c++] = s;
        most = std::max(most, size);
      }
      if (c == 0) break;
      // 128 rows at a time in registers: at most 4 bytes of each
      const int width = in_place && keep > 32 ? std::min(unit, 4) : unit;
      const int64_t blocks = std::min<int64_t>((most / width + 255) / 256, static_cast<int64_t>(sm_count) * 1024);
      for (int64_t g0 = 0; g0 < groups; g0 += 65535) {
        StateTable t = tab;
        for (int i = 0; i < c; ++i) {
          t.s[i].src = static_cast<const uint8_t*>(tab.s[i].src) + g0 * tab.s[i].src_group;
          t.s[i].dst = static_cast<uint8_t*>(tab.s[i].dst) + g0 * tab.s[i].dst_group;
        }
        const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(std::min<int64_t>(65535, groups - g0)),
                        static_cast<unsigned>(c));
        const int32_t* par = parents + g0 * keep;
        const cudaError_t e = width == 16  ? run_reorder<uint4>(t, in_place, grid, par, beams, keep, st)
                              : width == 8 ? run_reorder<uint2>(t, in_place, grid, par, beams, keep, st)
                              : width == 4 ? run_reorder<uint32_t>(t, in_place, grid, par, beams, keep, st)
                              : width == 2 ? run_reorder<uint16_t>(t, in_place, grid, par, beams, keep, st)
                                           : run_reorder<uint8_t>(t, in_place, grid, par, beams, keep, st);
        if (e != cudaSuccess) return e;
      }
    }
  }
  return cudaSuccess;
}

}  // namespace gann

// Selection over beams and vocabulary, and the states that follow it.
//
// The candidate (b, t) of a group is worth
//   v = S_b + L_bt                      or, with log-softmax,
//   v = S_b + (L_bt - max_t L_bt) - log(sum_t exp(L_bt - max_t L_bt)),
// compared in 64 bits; equal values go to the lower b * V + t. Entries that
// are not finite are no candidates, neither are those of a beam whose S is
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
// index in one word; Key2: a double's order, then the complement of an index.
// The all-zero key stands behind every candidate.
struct Key1 {
  uint64_t a;
  __device__ bool above(const Key1& o) const { return a > o.a; }
  __device__ Key1 from(int lane_mask) const { return {__shfl_xor_sync(kFull, a, lane_mask)}; }
};
struct Key2 {
  uint64_t a;
  uint32_t b;
  __device__ bool above(const Key2& o) const { return a > o.a || (a == o.a && b > o.b); }
  __device__ Key2 from(int lane_mask) const {
    return {__shfl_xor_sync(kFull, a, lane_mask), __shfl_xor_sync(kFull, b, lane_mask)};
  }
};

// Bitonic sort of 32 N keys by one warp, largest first; key n * 32 + lane is
// k[n] of the lane.
template <int N, typename K>
__device__ __forceinline__ void warp_sort(K (&k)[N], int lane) {
#pragma unroll
  for (int size = 2; size <= 32 * N; size <<= 1) {
#pragma unroll
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      if (stride >= 32) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const int o = n ^ (stride / 32);
          if (o > n) {
            const bool down = ((n * 32) & size) == 0;
            if (k[o].above(k[n]) == down) {
              const K t = k[n];
              k[n] = k[o];
              k[o] = t;
            }
          }
        }
      } else {
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const K o = k[n].from(stride);
          const bool down = ((n * 32 + lane) & size) == 0, low = (lane & stride) == 0;
          if (o.above(k[n]) == (down == low)) k[n] = o;
        }
      }
    }
  }
}

// The r-th largest (r <= 32) of the warp's 32 values as ord32 keys (0: none).
__device__ __forceinline__ uint32_t warp_rth(uint32_t u, int r, int lane) {
  uint32_t w = __reduce_max_sync(kFull, u);
  for (int i = 1; i < r; ++i) {
    const unsigned m = __ballot_sync(kFull, u == w);
    if (lane == __ffs(m) - 1) u = 0;
    w = __reduce_max_sync(kFull, u);
  }
  return w;
}

// Sum of one int a thread over the block; `red` holds a word for each warp.
// The barriers around it make it safe to call in a loop.
template <int NW>
__device__ __forceinline__ int block_sum(int c, int* red) {
  c = __reduce_add_sync(kFull, c);
  if (NW == 1) return c;
  if (threadIdx.x % kWarp == 0) red[threadIdx.x / kWarp] = c;
  __syncthreads();
  int s = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) s += red[w];
  __syncthreads();
  return s;
}

__device__ __forceinline__ bool live(float score) { return fabsf(score) < INFINITY; }

// ------------------------------------------------------------ split rows
// Large vocabularies: a block takes a segment of one row, keeps it in
// registers, sums its exponentials against the segment's maximum and writes
// the segment's best candidates; merge_kernel joins the segments.
//
// Threshold: every warp finds the r-th largest of its 32 lanes' maxima, r =
// ceil(keep / 8); the least of the 8 warps' values has at least `keep`
// elements at or above it, so nothing below it can be kept. On data in no
// particular order a few dozen of 8192 elements pass it. More than kHits
// (equal values, sorted rows in the tail) are cut to exactly `keep` by
// bisection over the value and then the index.
constexpr int kSplitWarps = 8;
constexpr int kSplitThreads = kSplitWarps * kWarp;

struct SegStat {
  double max, sum;
};

template <typename T, int E>
__device__ __forceinline__ void load_segment(uint4 (&raw)[E / Raw<T>::n], const T* row, int vocab, int head, int64_t base) {
  constexpr int N = Raw<T>::n;
  constexpr uint32_t ninf = Raw<T>::neg_inf;
#pragma unroll
  for (int i = 0; i < E / N; ++i) {
    const int64_t p = base + (static_cast<int64_t>(i) * kSplitThreads + threadIdx.x) * N - head;   // first element
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

template <typename T, int E, bool SOFTMAX>
__global__ void __launch_bounds__(kSplitThreads, 4) split_kernel(const T* __restrict__ logits, int64_t gstride,
                                                                 int64_t bstride, const float* __restrict__ scores,
                                                                 const uint8_t* __restrict__ finished, int64_t rows,
                                                                 int beams, int vocab, int keep, int segs,
                                                                 Key1* __restrict__ out, SegStat* __restrict__ stats) {
  constexpr int N = Raw<T>::n, V = E / N;
  __shared__ uint64_t hits[kHits];
  __shared__ uint32_t rth[kSplitWarps], top[kSplitWarps];
  __shared__ double part[kSplitWarps];
  __shared__ int red[kSplitWarps], count;
  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  const int r = (keep + kSplitWarps - 1) / kSplitWarps;
  const int64_t total = rows * segs;
  for (int64_t item = blockIdx.x; item < total; item += gridDim.x) {
    const int64_t rw = item / segs;
    const int64_t g = rw / beams;
    const int b = static_cast<int>(rw - g * beams);
    if (!live(scores[rw]) || (finished && finished[rw])) continue;
    const T* row = logits + g * gstride + b * bstride;
    const int head = static_cast<int>((reinterpret_cast<uintptr_t>(row) % 16) / sizeof(T));
    const int64_t base = (item - rw * segs) * (static_cast<int64_t>(kSplitThreads) * E);
    uint4 raw[V];
    load_segment<T, E>(raw, row, vocab, head, base);
    float vm[V], mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      vm[i] = Raw<T>::max(raw[i]);
      mx = fmaxf(mx, vm[i]);
    }
    if (mx == INFINITY) {   // infinite entries are masked: the maximum without them
      mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        vm[i] = -INFINITY;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float x = Raw<T>::at(raw[i], j);
          if (x < INFINITY) vm[i] = fmaxf(vm[i], x);
        }
        mx = fmaxf(mx, vm[i]);
      }
    }
    const uint32_t u = ord32(mx);
    const uint32_t wm = __reduce_max_sync(kFull, u), wr = warp_rth(u, r, lane);
    if (lane == 0) {
      rth[warp] = wr;
      top[warp] = wm;
    }
    if (tid == 0) count = 0;
    __syncthreads();
    uint32_t lo = rth[0], hi = top[0];
#pragma unroll
    for (int w = 1; w < kSplitWarps; ++w) {
      lo = min(lo, rth[w]);
      hi = max(hi, top[w]);
    }
    const float m = unord32(hi);
    auto index_of = [&](int i, int j) {
      return static_cast<uint32_t>(base + (static_cast<int64_t>(i) * kSplitThreads + tid) * N + j - head);
    };
    auto collect = [&](float thr, uint32_t floor_key, uint32_t last_index) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (vm[i] >= thr) {
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const float x = Raw<T>::at(raw[i], j);
            if (x >= thr && fabsf(x) < INFINITY) {
              const uint32_t k = ord32(x), id = index_of(i, j);
              if (k > floor_key || id <= last_index) {
                const int at = atomicAdd(&count, 1);
                if (at < kHits) hits[at] = (static_cast<uint64_t>(k) << 32) | ~id;
              }
            }
          }
        }
    };
    collect(unord32(lo), 0, 0);
    if (SOFTMAX) {
      // sum of exp(x - m), at most 32 terms a thread; the maximum's term is 1
      float sum = 0.f;
      if (m > -INFINITY) {
        constexpr float kLog2e = 1.4426950408889634f;
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
          for (int j = 0; j < N; ++j) sum += exp2f((Raw<T>::at(raw[i], j) - m) * kLog2e);
        if (!(sum < INFINITY)) {   // a NaN or an infinite entry: again without them
          sum = 0.f;
#pragma unroll
          for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) {
              const float x = Raw<T>::at(raw[i], j);
              if (fabsf(x) < INFINITY) sum += exp2f((x - m) * kLog2e);
            }
        }
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
      if (lane == 0) part[warp] = sum;
    }
    __syncthreads();
    int c = count;
    if (c > kHits) {
      // exactly `keep`: the key of the keep-th largest value, then the index
      // up to which its equals are taken
      auto at_least = [&](uint32_t k) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const float x = Raw<T>::at(raw[i], j);
            n += fabsf(x) < INFINITY && ord32(x) >= k;
          }
        return block_sum<kSplitWarps>(n, red);
      };
      uint32_t top_key = hi + 1;   // fewer than keep at or above
      while (top_key - lo > 1) {
        const uint32_t mid = lo + (top_key - lo) / 2;
        if (at_least(mid) >= keep) lo = mid;
        else top_key = mid;
      }
      const int want = keep - at_least(lo + 1);
      int64_t i0 = base - N, i1 = base + static_cast<int64_t>(kSplitThreads) * E;   // want in (i0, i1]
      while (i1 - i0 > 1) {
        const int64_t mid = i0 + (i1 - i0) / 2;
        int n = 0;
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const float x = Raw<T>::at(raw[i], j);
            const int64_t p = base + (static_cast<int64_t>(i) * kSplitThreads + tid) * N + j - head;
            n += fabsf(x) < INFINITY && ord32(x) == lo && p <= mid;
          }
        if (block_sum<kSplitWarps>(n, red) >= want) i1 = mid;
        else i0 = mid;
      }
      if (tid == 0) count = 0;
      __syncthreads();
      collect(unord32(lo), lo, static_cast<uint32_t>(i1));
      __syncthreads();
      c = count;
    }
    Key1* o = out + item * keep;
    if (warp == 0) {
      auto sorted = [&](auto tag) {
        constexpr int P = decltype(tag)::value;
        Key1 k[P];
#pragma unroll
        for (int n = 0; n < P; ++n) k[n] = {n * kWarp + lane < c ? hits[n * kWarp + lane] : 0};
        warp_sort<P>(k, lane);
#pragma unroll
        for (int n = 0; n < P; ++n)
          if (n * kWarp + lane < keep) o[n * kWarp + lane] = k[n];
        for (int n = P * kWarp + lane; n < keep; n += kWarp) o[n] = {0};
      };
      if (c <= 32) sorted(std::integral_constant<int, 1>{});
      else if (c <= 64) sorted(std::integral_constant<int, 2>{});
      else if (c <= 128) sorted(std::integral_constant<int, 4>{});
      else sorted(std::integral_constant<int, 8>{});
    } else if (SOFTMAX && warp == 1 && lane == 0) {
      double s = 0.0;
#pragma unroll
      for (int w = 0; w < kSplitWarps; ++w) s += part[w];
      stats[item] = {m, s};
    }
    __syncthreads();
  }
}

// --------------------------------------------------- one block, many rows
// Selection among elements of several rows, each held as f = fl32(x + c_b)
// in registers (NaN: no candidate), c_b the row's offset rounded to float32.
// f is within 2^-24 (|c_b| + |f|) of the exact value v, so with F the keep-th
// largest f (or a lower bound of it) every kept candidate has
// f >= F - 2^-22 (max |c_b| + |F|): those are gathered, valued in 64 bits and
// sorted.
struct Picked {
  double v[kBeamMax];
  uint32_t i[kBeamMax];
  int n;
};

struct SelShared {
  double off[kBeamMax];     // S_b, less the log of the row's sum
  float top[kBeamMax];      // the row's maximum (log-softmax), else 0
  float c[kBeamMax];        // off - top, NaN for a row without elements
  uint8_t fin[kBeamMax];
  float cmax;
  uint32_t rth[8], hi[8];
  int red[8], count;
  uint32_t hits[kHits];     // element, or kHitFinished + beam, or kHitKept + slot
  Picked kept;
  double rv[8];
  uint32_t ri[8];
  double lv;
  uint32_t li;
};
constexpr uint32_t kHitFinished = 0xc0000000u, kHitKept = 0xd0000000u;

// offsets of the rows; SUM gives a row's maximum and sum of exponentials
__device__ __forceinline__ void set_row(SelShared& sh, int b, float score, bool fin, bool softmax, float mx,
                                        double sum) {
  const bool ok = live(score);
  sh.fin[b] = ok && fin;
  sh.off[b] = static_cast<double>(score) - (softmax && sum > 0.0 ? log(sum) : 0.0);
  sh.top[b] = softmax && fabsf(mx) < INFINITY ? mx : 0.f;
  sh.c[b] = ok && !fin ? static_cast<float>(sh.off[b] - static_cast<double>(sh.top[b])) : kNan;
}

__device__ __forceinline__ double row_value(const SelShared& sh, int b, float x) {
  return sh.off[b] + (static_cast<double>(x) - static_cast<double>(sh.top[b]));
}

// Src: f[E] a thread, and exact(i, v, idx) for the thread's i-th element.
// Elements are named by name(i); `value(name, v, idx)` gives any element's
// exact value. The result is left in sh.kept, sorted.
template <int NW, int E, typename Name, typename Value>
__device__ __forceinline__ void block_select(SelShared& sh, const float (&f)[E], int beams, int vocab, int keep,
                                             int end_token, bool first, Name&& name, Value&& value,
                                             const float* __restrict__ scores) {
  constexpr int NT = NW * kWarp;
  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  const int r = (keep + NW - 1) / NW;
  float mx = kNan;
#pragma unroll
  for (int i = 0; i < E; ++i) mx = fmaxf(mx, f[i]);
  const uint32_t u = isnan(mx) ? 0u : ord32(mx);
  const uint32_t wm = __reduce_max_sync(kFull, u), wr = r <= kWarp ? warp_rth(u, r, lane) : 0u;
  if (lane == 0) {
    sh.rth[warp] = wr;
    sh.hi[warp] = wm;
  }
  if (tid == 0) sh.count = 0;
  __syncthreads();
  uint32_t lo = sh.rth[0], hi = sh.hi[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    lo = min(lo, sh.rth[w]);
    hi = max(hi, sh.hi[w]);
  }
  const int kept = first ? 0 : sh.kept.n;
  // what is kept from the tiles before bounds this one from below
  float carry = -INFINITY;
  if (kept == keep) carry = static_cast<float>(sh.kept.v[keep - 1]);
  auto at_least = [&](uint32_t k) {
    const float t = unord32(k);
    int n = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) n += f[i] >= t;
    return block_sum<NW>(n, sh.red);
  };
  auto threshold = [&](uint32_t k) {
    const float t = fmaxf(k ? unord32(k) : -INFINITY, carry);
    const float thr = t - 0x1p-22f * (sh.cmax + fabsf(t));
    return isnan(thr) ? -INFINITY : thr;
  };
  auto collect = [&](float thr) {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (f[i] >= thr) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kHits) sh.hits[at] = name(i);
      }
    if (first)
      for (int b = tid; b < beams; b += NT)
        if (sh.fin[b] && scores[b] >= thr) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kHits) sh.hits[at] = kHitFinished + b;
        }
    for (int j = tid; j < kept; j += NT)
      if (sh.kept.v[j] >= static_cast<double>(thr)) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kHits) sh.hits[at] = kHitKept + j;
      }
  };
  // fewer survivors are cheaper to sort: bisect while there are more than the
  // power of two that holds `keep`
  int limit = 32;
  while (limit < keep) limit <<= 1;
  int rounds = keep > 32 ? 8 : 0, c;
  bool all = false;
  if (rounds && lo && at_least(lo) <= limit) rounds = 0;
  while (true) {
    uint32_t up = hi + 1;
    for (; rounds > 0 && up - lo > 1; --rounds) {
      const uint32_t mid = lo + (up - lo) / 2;
      const int n = at_least(mid);
      if (n >= keep) {
        lo = mid;
        if (n <= limit) break;
      } else {
        up = mid;
      }
    }
    collect(threshold(lo));
    __syncthreads();
    c = sh.count;
    if (c <= kHits || all) break;
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
    rounds = 34;
    all = true;
  }
  auto exact = [&](uint32_t h, double& v, uint32_t& idx) {
    if (h >= kHitKept) {
      v = sh.kept.v[h - kHitKept];
      idx = sh.kept.i[h - kHitKept];
    } else if (h >= kHitFinished) {
      const int b = h - kHitFinished;
      v = static_cast<double>(scores[b]);
      idx = static_cast<uint32_t>(b) * vocab + end_token;
    } else {
      value(h, v, idx);
    }
  };
  if (c <= kHits) {
    if (warp == 0) {
      auto sorted = [&](auto tag) {
        constexpr int P = decltype(tag)::value;
        Key2 k[P];
#pragma unroll
        for (int n = 0; n < P; ++n) {
          k[n] = {0, 0};
          if (n * kWarp + lane < c) {
            double v;
            uint32_t idx;
            exact(sh.hits[n * kWarp + lane], v, idx);
            k[n] = {ord64(v), ~idx};
          }
        }
        __syncwarp();
        warp_sort<P>(k, lane);
#pragma unroll
        for (int n = 0; n < P; ++n)
          if (n * kWarp + lane < keep) {
            sh.kept.v[n * kWarp + lane] = unord64(k[n].a);
            sh.kept.i[n * kWarp + lane] = ~k[n].b;
          }
      };
      if (c <= 32) sorted(std::integral_constant<int, 1>{});
      else if (c <= 64) sorted(std::integral_constant<int, 2>{});
      else if (c <= 128) sorted(std::integral_constant<int, 4>{});
      else sorted(std::integral_constant<int, 8>{});
      if (lane == 0) sh.kept.n = min(c, keep);
    }
    __syncthreads();
    return;
  }
  // Many equal values: one kept candidate a round, the best behind the last.
  // Results go to the hit list's place only when all are found, because the
  // kept ones of earlier tiles take part.
  double pv = INFINITY, tv[(kBeamMax + NT - 1) / NT];
  uint32_t pi = 0, ti[(kBeamMax + NT - 1) / NT];
  int found = 0;
  for (int j = 0; j < keep; ++j) {
    double v = -INFINITY;
    uint32_t vi = 0xffffffffu;
    auto offer = [&](double x, uint32_t idx) {
      if (j > 0 && (x > pv || (x == pv && idx <= pi))) return;
      if (vi == 0xffffffffu || x > v || (x == v && idx < vi)) {
        v = x;
        vi = idx;
      }
    };
    const float thr = threshold(lo);
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (f[i] >= thr) {
        double x;
        uint32_t idx;
        value(name(i), x, idx);
        offer(x, idx);
      }
    if (first)
      for (int b = tid; b < beams; b += NT)
        if (sh.fin[b]) offer(static_cast<double>(scores[b]), static_cast<uint32_t>(b) * vocab + end_token);
    for (int q = tid; q < kept; q += NT) offer(sh.kept.v[q], sh.kept.i[q]);
    auto join = [&](double v2, uint32_t i2) {
      if (i2 != 0xffffffffu && (vi == 0xffffffffu || v2 > v || (v2 == v && i2 < vi))) {
        v = v2;
        vi = i2;
      }
    };
    for (int o = 16; o; o >>= 1) {
      const double v2 = __shfl_xor_sync(kFull, v, o);
      const uint32_t i2 = __shfl_xor_sync(kFull, vi, o);
      join(v2, i2);
    }
    if (lane == 0) {
      sh.rv[warp] = v;
      sh.ri[warp] = vi;
    }
    __syncthreads();
    v = -INFINITY;
    vi = 0xffffffffu;
    for (int w = 0; w < NW; ++w) join(sh.rv[w], sh.ri[w]);
    __syncthreads();
    if (vi == 0xffffffffu) break;
    pv = v;
    pi = vi;
    if (j % NT == tid) {
#pragma unroll
      for (int q = 0; q < (kBeamMax + NT - 1) / NT; ++q)
        if (q == j / NT) {
          tv[q] = v;
          ti[q] = vi;
        }
    }
    found = j + 1;
  }
#pragma unroll
  for (int q = 0; q < (kBeamMax + NT - 1) / NT; ++q)
    if (q * NT + tid < found) {
      sh.kept.v[q * NT + tid] = tv[q];
      sh.kept.i[q * NT + tid] = ti[q];
    }
  if (tid == 0) sh.kept.n = found;
  __syncthreads();
}

template <int NW>
__device__ __forceinline__ void write_kept(const SelShared& sh, int64_t g, int vocab, int keep,
                                           float* __restrict__ out_s, int32_t* __restrict__ out_p,
                                           int32_t* __restrict__ out_t) {
  for (int j = threadIdx.x; j < keep; j += NW * kWarp) {
    const bool ok = j < sh.kept.n;
    const uint32_t idx = ok ? sh.kept.i[j] : 0u, b = idx / static_cast<uint32_t>(vocab);
    out_s[g * keep + j] = ok ? static_cast<float>(sh.kept.v[j]) : -INFINITY;
    out_p[g * keep + j] = ok ? static_cast<int32_t>(b) : -1;
    out_t[g * keep + j] = ok ? static_cast<int32_t>(idx - b * vocab) : -1;
  }
}

// the largest finite |c_b|: what c's own rounding can be off by
__device__ __forceinline__ void set_cmax(SelShared& sh, int beams) {
  if (threadIdx.x < kWarp) {
    float m = 0.f;
    for (int b = threadIdx.x; b < beams; b += kWarp) m = fmaxf(m, fabsf(sh.c[b]));
    m = __uint_as_float(__reduce_max_sync(kFull, __float_as_uint(m)));
    if (threadIdx.x == 0) sh.cmax = m;
  }
}

// Groups of at most 32 NW E elements: one block each, the group in registers.
template <typename T, int NW, int E>
__global__ void __launch_bounds__(NW* kWarp) group_kernel(const T* __restrict__ logits, int64_t gstride,
                                                          int64_t bstride, const float* __restrict__ scores,
                                                          const uint8_t* __restrict__ finished, int64_t groups,
                                                          int beams, int vocab, int keep, int softmax, int end_token,
                                                          int vec, uint32_t magic, float* __restrict__ out_s,
                                                          int32_t* __restrict__ out_p, int32_t* __restrict__ out_t) {
  constexpr int NT = NW * kWarp, N = Raw<T>::n;
  __shared__ SelShared sh;
  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  const int total = beams * vocab;
  for (int64_t g = blockIdx.x; g < groups; g += gridDim.x) {
    const T* base = logits + g * gstride;
    const float* sc = scores + g * beams;
    if (softmax) {
      for (int b = warp; b < beams; b += NW) {
        const T* row = base + b * bstride;
        float mx = -INFINITY;
        for (int t = lane; t < vocab; t += kWarp) {
          const float x = Raw<T>::one(row + t);
          if (x < INFINITY) mx = fmaxf(mx, x);
        }
        mx = unord32(__reduce_max_sync(kFull, ord32(mx)));
        double sum = 0.0;
        for (int t = lane; t < vocab; t += kWarp) {
          const float x = Raw<T>::one(row + t);
          if (fabsf(x) < INFINITY) sum += exp2f((x - mx) * 1.4426950408889634f);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
        if (lane == 0) set_row(sh, b, sc[b], finished && finished[g * beams + b], true, mx, sum);
      }
    } else {
      for (int b = tid; b < beams; b += NT) set_row(sh, b, sc[b], finished && finished[g * beams + b], false, 0.f, 0.0);
    }
    __syncthreads();
    set_cmax(sh, beams);
    // f[i]: with vec, elements are 16-byte vectors of the group's rows
    float f[E];
    auto name = [&](int i) {
      return vec ? static_cast<uint32_t>((i / N * NT + tid) * N + i % N) : static_cast<uint32_t>(i * NT + tid);
    };
    // row of an element or vector: division by the row's length as a product
    // (exact: e < 2^14, length <= 2^13)
    auto row_of = [&](uint32_t e) { return magic ? __umulhi(e, magic) : e; };
    if (vec) {
      const int vr = vocab / N;
#pragma unroll
      for (int i = 0; i < E / N; ++i) {
        const uint32_t v = i * NT + tid;
        uint4 raw = make_uint4(0, 0, 0, 0);
        float c = kNan;
        if (v * N < static_cast<uint32_t>(total)) {
          const uint32_t b = row_of(v);
          raw = __ldcs(reinterpret_cast<const uint4*>(base + b * bstride + (v - b * vr) * N));
          c = sh.c[b];
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float x = Raw<T>::at(raw, j);
          f[i * N + j] = __fmaf_rn(x, 0.f, __fadd_rn(x, c));   // NaN when x is not finite
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const uint32_t e = i * NT + tid;
        f[i] = kNan;
        if (e < static_cast<uint32_t>(total)) {
          const uint32_t b = row_of(e);
          const float x = Raw<T>::one(base + b * bstride + (e - b * vocab));
          f[i] = __fmaf_rn(x, 0.f, __fadd_rn(x, sh.c[b]));
        }
      }
    }
    auto value = [&](uint32_t e, double& v, uint32_t& idx) {
      const uint32_t b = e / static_cast<uint32_t>(vocab);
      v = row_value(sh, b, Raw<T>::one(base + b * bstride + (e - b * vocab)));
      idx = e;
    };
    block_select<NW, E>(sh, f, beams, vocab, keep, end_token, true, name, value, sc);
    write_kept<NW>(sh, g, vocab, keep, out_s, out_p, out_t);
    __syncthreads();
  }
}

// The segments' candidates of one group joined: one block a group, tiles of
// 32 x 8 x 16 candidates.
constexpr int kMergeWarps = 8, kMergeElems = 16;

__global__ void __launch_bounds__(kMergeWarps* kWarp) merge_kernel(
    const Key1* __restrict__ cand, const SegStat* __restrict__ stats, const float* __restrict__ scores,
    const uint8_t* __restrict__ finished, int64_t groups, int beams, int vocab, int keep, int segs, int softmax,
    int end_token, float* __restrict__ out_s, int32_t* __restrict__ out_p, int32_t* __restrict__ out_t) {
  constexpr int NT = kMergeWarps * kWarp, E = kMergeElems;
  __shared__ SelShared sh;
  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  cudaGridDependencySynchronize();
  const int64_t per_beam = static_cast<int64_t>(segs) * keep, total = per_beam * beams;
  for (int64_t g = blockIdx.x; g < groups; g += gridDim.x) {
    const float* sc = scores + g * beams;
    for (int b = warp; b < beams; b += kMergeWarps) {
      const bool fin = finished && finished[g * beams + b];
      double mx = -INFINITY, sum = 0.0;
      if (softmax && !fin && live(sc[b])) {
        const SegStat* st = stats + (g * beams + b) * segs;
        for (int s = lane; s < segs; s += kWarp) mx = fmax(mx, st[s].max);
#pragma unroll
        for (int o = 16; o; o >>= 1) mx = fmax(mx, __shfl_xor_sync(kFull, mx, o));
        if (mx > -INFINITY)
          for (int s = lane; s < segs; s += kWarp)
            if (st[s].sum > 0.0) sum += st[s].sum * exp(st[s].max - mx);
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
      }
      if (lane == 0) set_row(sh, b, sc[b], fin, softmax, static_cast<float>(mx), sum);
    }
    __syncthreads();
    set_cmax(sh, beams);
    const Key1* list = cand + g * total;
    for (int64_t t0 = 0; t0 < total; t0 += NT * E) {
      float f[E];
      auto name = [&](int i) { return static_cast<uint32_t>(i * NT + tid); };
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int64_t e = t0 + i * NT + tid;
        f[i] = kNan;
        if (e < total) {
          const float c = sh.c[e / per_beam];
          if (!isnan(c)) {   // rows without candidates have no lists
            const uint64_t k = list[e].a;
            if (k) f[i] = __fadd_rn(unord32(static_cast<uint32_t>(k >> 32)), c);
          }
        }
      }
      auto value = [&](uint32_t e, double& v, uint32_t& idx) {
        const uint64_t k = list[t0 + e].a;
        const int b = static_cast<int>((t0 + e) / per_beam);
        v = row_value(sh, b, unord32(static_cast<uint32_t>(k >> 32)));
        idx = static_cast<uint32_t>(b) * vocab + ~static_cast<uint32_t>(k);
      };
      block_select<kMergeWarps, E>(sh, f, beams, vocab, keep, end_token, t0 == 0, name, value, sc);
    }
    write_kept<kMergeWarps>(sh, g, vocab, keep, out_s, out_p, out_t);
    __syncthreads();
  }
}

struct StateTable {
  gann_state s[kStateBatch];
};

// One CTA per (state, group, slice of the row's bytes): a thread owns one unit
// of the row in every beam, reads all of them that a kept row needs and then
// writes them, so source and target may be the same rows.
template <typename U>
__global__ void __launch_bounds__(256) reorder_kernel(const __grid_constant__ StateTable tab,
                                                      const int32_t* __restrict__ parents, int beams, int keep) {
  const gann_state& s = tab.s[blockIdx.z];
  const int64_t g = blockIdx.y;
  const int32_t* par = parents + g * keep;
  const int64_t units = s.row_bytes / static_cast<int64_t>(sizeof(U));
  const int64_t total = s.size[0] * s.size[1] * units;
  const uint8_t* src = static_cast<const uint8_t*>(s.src) + g * s.src_group;
  uint8_t* dst = static_cast<uint8_t*>(s.dst) + g * s.dst_group;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < total;
       e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t u = e % units, r = e / units, i1 = r % s.size[1], i0 = r / s.size[1];
    const uint8_t* p = src + i0 * s.src_stride[0] + i1 * s.src_stride[1] + u * static_cast<int64_t>(sizeof(U));
    uint8_t* q = dst + i0 * s.dst_stride[0] + i1 * s.dst_stride[1] + u * static_cast<int64_t>(sizeof(U));
    U v[kBeamMax];
    for (int j = 0; j < keep; ++j) {
      const int b = par[j];
      v[j] = b >= 0 && b < beams ? *reinterpret_cast<const U*>(p + b * s.src_beam) : U{};
    }
    for (int j = 0; j < keep; ++j) *reinterpret_cast<U*>(q + j * s.dst_beam) = v[j];
  }
}

}  // namespace

namespace {

// How a call is run. A group of at most 8192 elements is one block's (group
// kernel: one launch, nothing written but the result); larger ones are split
// into rows' segments and joined. Elements a thread of the split kernel: as
// few as hold a row, and no fewer than 8.
struct SelectPlan {
  bool split = false;
  int elems = 32, segs = 0;
};

SelectPlan plan_select(int beams, int vocab, int dtype) {
  SelectPlan p;
  if (static_cast<int64_t>(beams) * vocab <= 8 * kWarp * 32) return p;
  p.split = true;
  const int64_t span = static_cast<int64_t>(vocab) + (dtype == GANN_F32 ? 3 : 7);   // a row may start inside a vector
  p.elems = span <= kSplitThreads * 8 ? 8 : span <= kSplitThreads * 16 ? 16 : 32;
  p.segs = static_cast<int>((span + kSplitThreads * p.elems - 1) / (kSplitThreads * p.elems));
  return p;
}

}  // namespace

size_t beam_select_workspace(int64_t groups, int beams, int vocab, int keep, int dtype) {
  const SelectPlan p = plan_select(beams, vocab, dtype);
  if (!p.split) return 0;
  const size_t items = static_cast<size_t>(groups) * beams * p.segs;
  return items * (sizeof(SegStat) + sizeof(Key1) * keep);
}

namespace {

template <typename T>
cudaError_t run_group(const SelectArgs& a, int sm_count, cudaStream_t st) {
  constexpr int n = Raw<T>::n;
  const int total = a.beams * a.vocab;
  const bool vec = a.vocab % n == 0 && a.group_stride % n == 0 && a.beam_stride % n == 0 &&
                   reinterpret_cast<uintptr_t>(a.logits) % 16 == 0;
  const uint32_t div = static_cast<uint32_t>(vec ? a.vocab / n : a.vocab);
  const uint32_t magic = div == 1 ? 0u : static_cast<uint32_t>(((1ull << 32) + div - 1) / div);
  auto run = [&](auto fn, int warps) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.groups, static_cast<int64_t>(sm_count) * 256));
    fn<<<grid, warps * kWarp, 0, st>>>(static_cast<const T*>(a.logits), a.group_stride, a.beam_stride, a.scores,
                                       a.finished, a.groups, a.beams, a.vocab, a.keep, a.softmax, a.end_token, vec,
                                       magic, a.out_scores, a.out_parents, a.out_tokens);
    return cudaGetLastError();
  };
  // the threshold wants keep <= 32 a warp; the smallest block that holds the
  // group
  if (total <= 256 && a.keep <= 32) return run(group_kernel<T, 1, 8>, 1);
  if (total <= 1024 && a.keep <= 32) return run(group_kernel<T, 1, 32>, 1);
  if (total <= 1024) return run(group_kernel<T, 4, 8>, 4);
  if (total <= 2048 && a.keep <= 64) return run(group_kernel<T, 2, 32>, 2);
  if (total <= 4096) return run(group_kernel<T, 4, 32>, 4);
  return run(group_kernel<T, 8, 32>, 8);
}

template <typename T>
cudaError_t run_split(const SelectArgs& a, const SelectPlan& p, int sm_count, cudaStream_t st) {
  const int64_t rows = a.groups * a.beams, items = rows * p.segs;
  SegStat* stats = static_cast<SegStat*>(a.workspace);
  Key1* cand = reinterpret_cast<Key1*>(stats + items);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(items, static_cast<int64_t>(1) << 30));
  auto run = [&](auto fn) {
    fn<<<grid, kSplitThreads, 0, st>>>(static_cast<const T*>(a.logits), a.group_stride, a.beam_stride, a.scores,
                                       a.finished, rows, a.beams, a.vocab, a.keep, p.segs, cand, stats);
    return cudaGetLastError();
  };
  cudaError_t e;
  if (a.softmax)
    e = p.elems == 8 ? run(split_kernel<T, 8, true>)
                     : p.elems == 16 ? run(split_kernel<T, 16, true>) : run(split_kernel<T, 32, true>);
  else
    e = p.elems == 8 ? run(split_kernel<T, 8, false>)
                     : p.elems == 16 ? run(split_kernel<T, 16, false>) : run(split_kernel<T, 32, false>);
  if (e != cudaSuccess) return e;
  // the join may be set up while the last segments still run; it waits for
  // them itself
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(a.groups, static_cast<int64_t>(sm_count) * 64)));
  cfg.blockDim = dim3(kMergeWarps * kWarp);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, merge_kernel, static_cast<const Key1*>(cand), static_cast<const SegStat*>(stats),
                            a.scores, a.finished, a.groups, a.beams, a.vocab, a.keep, p.segs, a.softmax, a.end_token,
                            a.out_scores, a.out_parents, a.out_tokens);
}

template <typename T>
cudaError_t run_select(const SelectArgs& a, int sm_count, cudaStream_t st) {
  const SelectPlan p = plan_select(a.beams, a.vocab, a.dtype);
  return p.split ? run_split<T>(a, p, sm_count, st) : run_group<T>(a, sm_count, st);
}

}  // namespace

cudaError_t launch_beam_select(const SelectArgs& a, int sm_count, cudaStream_t st) {
  if (a.groups <= 0) return cudaSuccess;
  if (a.dtype == GANN_F32) return run_select<float>(a, sm_count, st);
  if (a.dtype == GANN_F16) return run_select<__half>(a, sm_count, st);
  return run_select<__nv_bfloat16>(a, sm_count, st);
}

cudaError_t launch_reorder_states(const gann_state* states, int count, const int32_t* parents, int64_t groups,
                                  int beams, int keep, int sm_count, cudaStream_t st) {
  (void)sm_count;
  for (int lo = 0; lo < count; lo += kStateBatch) {
    const int c = std::min(kStateBatch, count - lo);
    StateTable tab{};
    int64_t most = 0;
    for (int i = 0; i < c; ++i) {
      tab.s[i] = states[lo + i];
      most = std::max(most, tab.s[i].size[0] * tab.s[i].size[1] * tab.s[i].row_bytes);
    }
    if (most == 0) continue;
    for (int64_t g0 = 0; g0 < groups; g0 += 65535) {
      const int64_t gn = std::min<int64_t>(65535, groups - g0);
      StateTable t = tab;
      for (int i = 0; i < c; ++i) {
        t.s[i].src = static_cast<const uint8_t*>(tab.s[i].src) + g0 * tab.s[i].src_group;
        t.s[i].dst = static_cast<uint8_t*>(tab.s[i].dst) + g0 * tab.s[i].dst_group;
      }
      const dim3 grid(static_cast<unsigned>(std::min<int64_t>((most + 255) / 256, 1024)), static_cast<unsigned>(gn),
                      static_cast<unsigned>(c));
      reorder_kernel<uint8_t><<<grid, 256, 0, st>>>(t, parents + g0 * keep, beams, keep);
      const cudaError_t e = cudaGetLastError();
      if (e != cudaSuccess) return e;
    }
  }
  return cudaSuccess;
}

}  // namespace gann

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
// A segment writes its `keep` best and its sum; merge_kernel joins them.
constexpr int kRowWarps = 4, kRowVecs = 4;
constexpr int kRowTile = kRowVecs * kWarp;   // vectors

struct SegStat {
  double max, sum;
};

template <typename T, bool SOFTMAX, bool LONG>
__global__ void __launch_bounds__(kRowWarps* kWarp, 5) row_kernel(const T* __restrict__ logits, int64_t gstride,
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
  if (!live(scores[rw]) || (finished && finished[rw])) return;
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
  float thr = -INFINITY, m = -INFINITY;
  auto cut = [&]() {
    sort_some<LONG>(list, cnt, keep, lane, [&](int i) { return list[i]; });
    cnt = min(cnt, keep);
    if (cnt < keep) return;
    floor = list[keep - 1];
    thr = unord32(static_cast<uint32_t>(floor.a >> 32));
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
    }
    const int64_t p0 = first + static_cast<int64_t>(t) * kRowTile * N;
    if (__any_sync(kFull, mx >= thr)) {
      uint32_t mark = 0;
#pragma unroll
      for (int i = 0; i < kRowVecs; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (Raw<T>::at(cur[i], j) >= thr) mark |= 1u << (i * N + j);
      while (__any_sync(kFull, mark)) {
        if (cnt > kCap - kWarp) cut();
        const int e = __ffs(mark) - 1;
        const int64_t p = p0 + ((e / N) * kWarp + lane) * N + e % N;
        const float x = mark && p >= 0 && p < vocab ? Raw<T>::one(row + p) : kNan;
        const Key1 k{(static_cast<uint64_t>(ord32(x)) << 32) | ~static_cast<uint32_t>(p)};
        const bool take = fabsf(x) < INFINITY && k.above(floor);
        const unsigned pass = __ballot_sync(kFull, take);
        if (take) list[cnt + __popc(pass & ((1u << lane) - 1u))] = k;
        cnt += __popc(pass);
        mark &= mark - 1;
      }
    }
    if (SOFTMAX) {
      if (mx > m) {
        sum *= static_cast<double>(fast_exp2((m - mx) * kLog2e));
        m = mx;
      }
      float part = 0.f;
      if (m > -INFINITY) {
#pragma unroll
        for (int i = 0; i < kRowVecs; ++i)
#pragma unroll
          for (int j = 0; j < N; ++j) part += fast_exp2((Raw<T>::at(cur[i], j) - m) * kLog2e);
        if (!(part < INFINITY)) {   // a NaN or an infinite entry: again without them
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
// Many groups, no softmax: a warp takes a whole group, in tiles of 16 to
// 64 elements a lane in registers, vectors of 16 bytes (single elements when rows
// are not whole vectors). f = fl32(x + S_b) orders candidates as their 64-bit
// values do, up to equality. The first tile sets a threshold of f: the keep-th
// largest of the lanes' maxima (keep <= 16), or one bisected until between
// `keep` and 128 elements pass. Lanes mark the elements with x >= thr - S_b (a
// little less, so none with f >= thr is missed); the marked ones are valued
// in 64 bits, compared with the least kept key and listed.
constexpr int kGroupWarps = 4;

template <typename T, int VW>
struct Vec {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = __ldcs(reinterpret_cast<const uint4*>(p)); }
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

template <typename T, int VW, int ELEMS, bool LONG>
__global__ void __launch_bounds__(kGroupWarps* kWarp, LONG || ELEMS > 32 ? 4 : 6) group_kernel(
    const T* __restrict__ logits, int64_t gstride, int64_t bstride, const float* __restrict__ scores,
    const uint8_t* __restrict__ finished, int64_t groups, int beams, int vocab, int keep, int end_token, uint32_t magic,
    int shift, float* __restrict__ out_s, int32_t* __restrict__ out_p, int32_t* __restrict__ out_t) {
  constexpr int NV = ELEMS / VW, kCap = Held<LONG>::value;
  using Mark = typename std::conditional<(ELEMS > 32), unsigned long long, uint32_t>::type;
  __shared__ Key2 lists[kGroupWarps][kCap];
  __shared__ float cs[kGroupWarps][kBeamMax];
  const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
  const int64_t g = static_cast<int64_t>(blockIdx.x) * kGroupWarps + warp;
  if (g >= groups) return;
  const T* base = logits + g * gstride;
  const float* sc = scores + g * beams;
  float* c = cs[warp];
  Key2* list = lists[warp];
  const uint32_t vr = static_cast<uint32_t>(vocab) / VW, nvec = vr * beams;
  const bool joined = bstride == vocab;
  // row of a vector: division by the row's length as a product (magic =
  // ceil(2^(32+shift) / vr), exact below 2^31)
  auto row_of = [&](uint32_t v) { return (magic ? __umulhi(v, magic) : v) >> shift; };
  Vec<T, VW> raw[NV];
  auto load = [&](uint32_t t0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t v = t0 + i * kWarp + lane;
      if (v < nvec) {
        if (joined) {
          raw[i].load(base + static_cast<int64_t>(v) * VW);
        } else {
          const uint32_t b = row_of(v);
          raw[i].load(base + b * bstride + static_cast<int64_t>(v - b * vr) * VW);
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
  Key2 floor{0, 0};   // the least kept key once `keep` are known
  float thr = -INFINITY;
  auto cut = [&]() {
    sort_some<LONG>(list, cnt, keep, lane, [&](int i) { return list[i]; });
    cnt = min(cnt, keep);
    if (cnt < keep) return;
    floor = list[keep - 1];
    thr = static_cast<float>(unord64(floor.a));
  };
  for (uint32_t t0 = 0; t0 < nvec; t0 += NV * kWarp) {
    if (t0) load(t0);
    float cb[NV];   // NaN: a row without elements, or nothing there
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t v = t0 + i * kWarp + lane;
      cb[i] = v < nvec ? c[row_of(v)] : kNan;
    }
    if (t0 == 0) {
      if (!LONG) {
        // rounding keeps order, so one sum a vector; masked entries that are
        // +infinity have to be left out
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i) mx = fmaxf(mx, __fadd_rn(raw[i].max(), cb[i]));
        if (mx == INFINITY) {
          mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VW; ++j)
              if (raw[i].at(j) < INFINITY) mx = fmaxf(mx, __fadd_rn(raw[i].at(j), cb[i]));
        }
        thr = __shfl_sync(kFull, warp_sort32(mx, lane), keep - 1);
      } else {
        // bisection by value, then (far from done) over the order of floats
        float hi = -INFINITY, lo = -INFINITY, low = INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < VW; ++j) {
            const float x = raw[i].at(j), f = __fadd_rn(x, cb[i]);
            if (fabsf(x) < INFINITY && fabsf(f) < INFINITY) {
              hi = fmaxf(hi, f);
              low = fminf(low, f);
            }
          }
        hi = unord32(__reduce_max_sync(kFull, ord32(hi)));
        float mid = -unord32(__reduce_max_sync(kFull, ord32(-low)));
        for (int r = 0; r < 24 && hi > mid; ++r) {
          int n = 0;
#pragma unroll
          for (int i = 0; i < NV; ++i)
            if (i * kWarp < nvec) {
#pragma unroll
              for (int j = 0; j < VW; ++j) n += __fadd_rn(raw[i].at(j), cb[i]) >= mid && raw[i].at(j) < INFINITY;
            }
          n = __reduce_add_sync(kFull, n);
          if (n >= keep) {
            lo = mid;
            if (n <= 128) break;
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
    Mark mark = 0;
    const float below = thr - fabsf(thr) * 0x1p-23f;   // by half a step of thr at least
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float least = __fadd_rd(below, -cb[i]);
#pragma unroll
      for (int j = 0; j < VW; ++j)
        if (raw[i].at(j) >= least) mark |= Mark(1) << (i * VW + j);
    }
    int b0 = 0;
    while (true) {
      bool take = mark != 0;
      double v = 0.0;
      uint32_t id = 0;
      if (__any_sync(kFull, take)) {
        if (take) {
          const int e = (ELEMS > 32 ? __ffsll(mark) : __ffs(static_cast<uint32_t>(mark))) - 1;
          id = (t0 + (e / VW) * kWarp + lane) * VW + e % VW;
          const uint32_t b = row_of(id / VW);
          const float x = Raw<T>::one(base + b * bstride + (id - b * vocab));
          take = fabsf(x) < INFINITY;
          v = static_cast<double>(c[b]) + static_cast<double>(x);
          mark &= mark - 1;
        }
      } else {
        if (!finished || t0 || b0 >= beams) break;
        const int b = b0 + lane;
        take = b < beams && isnan(c[b]) && live(sc[b]);
        if (take) {
          v = static_cast<double>(sc[b]);
          id = static_cast<uint32_t>(b) * vocab + end_token;
        }
        b0 += kWarp;
      }
      if (cnt > kCap - kWarp) cut();
      const Key2 k{ord64(v), ~id};
      take = take && k.above(floor);
      const unsigned pass = __ballot_sync(kFull, take);
      if (take) list[cnt + __popc(pass & ((1u << lane) - 1u))] = k;
      cnt += __popc(pass);
    }
  }
  if (cnt) cut();
  const int nkept = cnt;
  for (int j = lane; j < keep; j += kWarp) {
    const bool ok = j < nkept;
    const Key2 k = ok ? list[j] : Key2{0, 0};
    const uint32_t idx = ~k.b, b = ok ? idx / static_cast<uint32_t>(vocab) : 0u;
    out_s[g * keep + j] = ok ? static_cast<float>(unord64(k.a)) : -INFINITY;
    out_p[g * keep + j] = ok ? static_cast<int32_t>(b) : -1;
    out_t[g * keep + j] = ok ? static_cast<int32_t>(idx - b * vocab) : -1;
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

// A thread owns one unit of U bytes at one place of a group's blocks, in every
// beam. MAX > 0: it reads the unit of every kept row (at most MAX) before it
// writes any, so source and target may be the same rows; rows that stay where
// they are are not touched. MAX 0: source and target are apart, and eight rows
// at a time are on their way. Bound by memory: each kept row is written once
// and each distinct parent read once from DRAM (again from the caches).
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
// launch, nothing written but the result. That needs enough groups to fill the
// GPU, or groups so small that one warp is done at once. Everything else is
// split: rows into segments, a warp each, as many as the GPU holds at a time,
// and joined by a second kernel.
constexpr int kResidentWarps = 148 * 20;
constexpr int kSmallGroup = 4096;      // bytes of a group that a lone warp reads in one tile

struct SelectPlan {
  bool split = false;
  int segs = 0, seg_tiles = 0;
};

SelectPlan plan_select(int64_t groups, int beams, int vocab, int dtype, bool softmax) {
  SelectPlan p;
  const int elem = dtype == GANN_F32 ? 4 : 2, n = 16 / elem;
  const int64_t bytes = static_cast<int64_t>(beams) * vocab * elem;
  p.split = softmax || !(bytes <= kSmallGroup || groups >= kResidentWarps / 4);
  if (!p.split) return p;
  const int64_t rows = std::max<int64_t>(1, groups * beams);
  const int64_t tiles = (static_cast<int64_t>(vocab) + n - 1 + kRowTile * n - 1) / (kRowTile * n);   // a row may start inside a vector
  const int64_t want = std::max<int64_t>(1, kResidentWarps / rows);
  p.seg_tiles = static_cast<int>((tiles + want - 1) / want);
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
  if (many) return run(group_kernel<T, n, 32, true>);
  const int64_t total = static_cast<int64_t>(a.beams) * a.vocab;
  return total > 32 * kWarp && total <= 64 * kWarp ? run(group_kernel<T, n, 64, false>)
                                                    : run(group_kernel<T, n, 32, false>);
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

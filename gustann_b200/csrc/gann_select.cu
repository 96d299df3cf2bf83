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

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gann_internal.hpp"

namespace gann {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kSelThreads = 256;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// The larger of two candidates, the lower index among equal values.
__device__ __forceinline__ void better(double& v, int32_t& i, double v2, int32_t i2) {
  if (i2 >= 0 && (i < 0 || v2 > v || (v2 == v && i2 < i))) {
    v = v2;
    i = i2;
  }
}

// One CTA per group: the rows' log-sums first, then `keep` rounds, each of
// which finds the best candidate behind the last one.
template <typename T>
__global__ void __launch_bounds__(kSelThreads) select_kernel(const T* __restrict__ logits, int64_t gstride,
                                                             int64_t bstride, const float* __restrict__ scores,
                                                             const uint8_t* __restrict__ finished, int beams, int vocab,
                                                             int keep, int softmax, int end_token,
                                                             float* __restrict__ out_s, int32_t* __restrict__ out_p,
                                                             int32_t* __restrict__ out_t) {
  __shared__ double off[kBeamMax], red_v[kSelThreads / kWarp], last_v;
  __shared__ float top[kBeamMax];
  __shared__ int32_t red_i[kSelThreads / kWarp], last_i;
  const int64_t g = blockIdx.x;
  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  for (int b = warp; b < beams; b += kSelThreads / kWarp) {
    const T* row = logits + g * gstride + b * bstride;
    float mx = -INFINITY;
    double sum = 0.0;
    if (softmax) {
      for (int t = lane; t < vocab; t += kWarp) {
        const float x = to_f32(row[t]);
        if (isfinite(x)) mx = fmaxf(mx, x);
      }
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, o));
      for (int t = lane; t < vocab; t += kWarp) {
        const float x = to_f32(row[t]);
        if (isfinite(x)) sum += expf(x - mx);
      }
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    }
    if (lane == 0) {
      off[b] = static_cast<double>(scores[g * beams + b]) - (softmax && sum > 0.0 ? log(sum) : 0.0);
      top[b] = softmax && isfinite(mx) ? mx : 0.f;
    }
  }
  __syncthreads();
  double pv = INFINITY;
  int32_t pi = -1;
  const int total = beams * vocab;
  for (int j = 0; j < keep; ++j) {
    double v = -INFINITY;
    int32_t vi = -1;
    for (int e = tid; e < total; e += kSelThreads) {
      const int b = e / vocab, t = e - b * vocab;
      double c;
      if (finished && finished[g * beams + b]) {
        if (t != end_token) continue;
        c = scores[g * beams + b];
      } else {
        const float x = to_f32(logits[g * gstride + b * bstride + t]);
        if (!isfinite(x)) continue;
        c = off[b] + (static_cast<double>(x) - static_cast<double>(top[b]));
      }
      if (!isfinite(c) || c > pv || (c == pv && e <= pi)) continue;
      better(v, vi, c, e);
    }
    for (int o = 16; o; o >>= 1) {
      const double v2 = __shfl_xor_sync(kFull, v, o);
      const int32_t i2 = __shfl_xor_sync(kFull, vi, o);
      better(v, vi, v2, i2);
    }
    if (lane == 0) {
      red_v[warp] = v;
      red_i[warp] = vi;
    }
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kSelThreads / kWarp; ++w) better(v, vi, red_v[w], red_i[w]);
      out_s[g * keep + j] = vi >= 0 ? static_cast<float>(v) : -INFINITY;
      out_p[g * keep + j] = vi >= 0 ? vi / vocab : -1;
      out_t[g * keep + j] = vi >= 0 ? vi % vocab : -1;
      last_v = vi >= 0 ? v : -INFINITY;
      last_i = vi >= 0 ? vi : INT32_MAX;
    }
    __syncthreads();
    pv = last_v;
    pi = last_i;
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

size_t beam_select_workspace(int64_t, int, int, int, int) { return 0; }

cudaError_t launch_beam_select(const SelectArgs& a, int sm_count, cudaStream_t st) {
  (void)sm_count;
  if (a.groups <= 0) return cudaSuccess;
  auto run = [&](auto fn, auto* l) {
    fn<<<static_cast<unsigned>(a.groups), kSelThreads, 0, st>>>(l, a.group_stride, a.beam_stride, a.scores, a.finished,
                                                                a.beams, a.vocab, a.keep, a.softmax, a.end_token,
                                                                a.out_scores, a.out_parents, a.out_tokens);
    return cudaGetLastError();
  };
  if (a.dtype == GANN_F32) return run(select_kernel<float>, static_cast<const float*>(a.logits));
  if (a.dtype == GANN_F16) return run(select_kernel<__half>, static_cast<const __half*>(a.logits));
  return run(select_kernel<__nv_bfloat16>, static_cast<const __nv_bfloat16*>(a.logits));
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

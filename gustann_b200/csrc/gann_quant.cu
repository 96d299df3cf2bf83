// 8-bit rows with one scale each, and products of such rows.
//
//   quantize_rows   s_i = max_j |x_ij| * (1/127) in float32,  c_ij = x_ij / s_i
//                   rounded to the nearest integer (ties to even)
//   matmul_i8       y_ij = (sum_k a_ik b_jk) sa_i sb_j + bias_j
#include <algorithm>
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gann_internal.hpp"

namespace gann {
namespace {

constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// The scale of a row and what its entries are multiplied by. A tiny scale
// (its reciprocal could overflow) is worked with 2^64 times larger, which
// changes no quotient.
struct RowScale {
  float scale;   // stored
  float up;      // 1 or 2^64
  float s;       // scale * up
  float inv;     // about 1 / s
};

__device__ __forceinline__ RowScale row_scale(float amax) {
  RowScale r;
  r.scale = isfinite(amax) ? __fmul_rn(amax, 1.f / 127.f) : __int_as_float(0x7fc00000);
  r.up = r.scale < 0x1p-60f ? 0x1p64f : 1.f;
  r.s = r.scale * r.up;
  r.inv = r.s > 0.f ? __frcp_rn(r.s) : 0.f;   // 0 and NaN scales: every code 0
  return r;
}

// Nearest integer to x / s, ties to even, exactly: the product with the
// reciprocal gives one of the two integers beside the quotient, and the
// remainder x - r s (exact in one fma: |r| <= 127, and near a tie it is a
// multiple of 2^-25 times the power of two at s, below s in size) says which
// one is nearer.
__device__ __forceinline__ int quant_code(float x, const RowScale& rs) {
  const float xs = x * rs.up;
  float r = rintf(xs * rs.inv);
  const float e = __fmaf_rn(-r, rs.s, xs);
  const float e2 = 2.f * fabsf(e);
  const bool odd = static_cast<int>(r) & 1;
  if (e2 > rs.s || (e2 == rs.s && odd)) r += e > 0.f ? 1.f : -1.f;
  return rs.inv > 0.f ? static_cast<int>(fminf(fmaxf(r, -127.f), 127.f)) : 0;
}

// |x| for the maximum: a NaN becomes infinity, so it is not lost in fmaxf.
__device__ __forceinline__ float mag(float x) { return isnan(x) ? INFINITY : fabsf(x); }

// One warp per row.
template <typename T>
__global__ void __launch_bounds__(256) quantize_kernel(const uint8_t* __restrict__ x, int64_t rows, int64_t stride,
                                                       int dim, int8_t* __restrict__ codes, int64_t cstride,
                                                       float* __restrict__ scales) {
  const int lane = threadIdx.x % kWarp;
  const int64_t wpg = static_cast<int64_t>(gridDim.x) * (blockDim.x / kWarp);
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * (blockDim.x / kWarp) + threadIdx.x / kWarp; r < rows; r += wpg) {
    const T* row = reinterpret_cast<const T*>(x + r * stride);
    float a = 0.f;
    for (int j = lane; j < dim; j += kWarp) a = fmaxf(a, mag(to_f32(row[j])));
#pragma unroll
    for (int o = 16; o; o >>= 1) a = fmaxf(a, __shfl_xor_sync(kFull, a, o));
    const RowScale rs = row_scale(a);
    for (int j = lane; j < dim; j += kWarp)
      codes[r * cstride + j] = static_cast<int8_t>(quant_code(to_f32(row[j]), rs));
    if (lane == 0) scales[r] = rs.scale;
  }
}

// 16 bytes of a row from column b, zero past k.
__device__ __forceinline__ uint4 load16(const int8_t* row, int b, int k) {
  if (b + 16 <= k) return __ldg(reinterpret_cast<const uint4*>(row + b));
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; i < 16 && b + i < k; ++i)
    w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(row[b + i])) << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// y = acc sa sb (+ bias): the sum is an exact integer; it is rounded to 24
// bits when it needs more, then once at each product and sum.
__device__ __forceinline__ float i8_value(int acc, float sa, float sb, bool has_bias, float bias) {
  const float y = static_cast<float>(acc) * sa;
  return has_bias ? __fmaf_rn(y, sb, bias) : y * sb;
}

constexpr int kMmTile = 64;
constexpr int kMmRow = 64 + 16;

// A 64 x 64 tile a CTA, 4 x 4 products a thread by dp4a.
template <typename T>
__global__ void __launch_bounds__(256) matmul_tile_kernel(
    const int8_t* __restrict__ a, int64_t m, int64_t as, const float* __restrict__ sa, const int8_t* __restrict__ b,
    int64_t n, int64_t bs, const float* __restrict__ sb, const float* __restrict__ bias, int k, T* __restrict__ out,
    int64_t os, int64_t ntn) {
  __shared__ __align__(16) int8_t ta[kMmTile * kMmRow], tb[kMmTile * kMmRow];
  const int64_t i0 = (blockIdx.x / ntn) * kMmTile, j0 = (blockIdx.x % ntn) * kMmTile;
  const int tid = threadIdx.x, lr = tid >> 2, lc = (tid & 3) * 16, tx = tid & 15, ty = tid >> 4;
  int acc[4][4] = {};
  for (int c = 0; c < k; c += 64) {
    const uint4 z = make_uint4(0, 0, 0, 0);
    const uint4 va = i0 + lr < m ? load16(a + (i0 + lr) * as, c + lc, k) : z;
    const uint4 vb = j0 + lr < n ? load16(b + (j0 + lr) * bs, c + lc, k) : z;
    __syncthreads();
    *reinterpret_cast<uint4*>(ta + lr * kMmRow + lc) = va;
    *reinterpret_cast<uint4*>(tb + lr * kMmRow + lc) = vb;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      int x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const int*>(ta + (ty + 16 * i) * kMmRow + 4 * q);
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const int*>(tb + (tx + 16 * j) * kMmRow + 4 * q);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(x[i], y[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = i0 + ty + 16 * i, c = j0 + tx + 16 * j;
      if (r < m && c < n)
        out[r * os + c] = from_f32<T>(i8_value(acc[i][j], sa[r], sb[c], bias != nullptr, bias ? bias[c] : 0.f));
    }
}

}  // namespace

cudaError_t launch_quantize_rows(const void* x, int64_t rows, int64_t stride, int dim, int dtype, int8_t* codes,
                                 int64_t code_stride, float* scales, int sm_count, cudaStream_t st) {
  if (rows <= 0) return cudaSuccess;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((rows + 7) / 8, static_cast<int64_t>(sm_count) * 32));
  auto run = [&](auto fn) {
    fn<<<grid, 256, 0, st>>>(static_cast<const uint8_t*>(x), rows, stride, dim, codes, code_stride, scales);
    return cudaGetLastError();
  };
  if (dtype == GANN_F32) return run(quantize_kernel<float>);
  if (dtype == GANN_F16) return run(quantize_kernel<__half>);
  return run(quantize_kernel<__nv_bfloat16>);
}

cudaError_t launch_matmul_i8(const int8_t* a, int64_t m, int64_t as, const float* sa, const int8_t* b, int64_t n,
                             int64_t bs, const float* sb, const float* bias, int k, void* out, int64_t os, int dtype,
                             int sm_count, cudaStream_t st) {
  if (m <= 0 || n <= 0) return cudaSuccess;
  const int64_t ntm = (m + kMmTile - 1) / kMmTile, ntn = (n + kMmTile - 1) / kMmTile;
  if (ntm * ntn > INT32_MAX) return cudaErrorInvalidConfiguration;
  auto run = [&](auto fn, auto* o) {
    fn<<<static_cast<unsigned>(ntm * ntn), 256, 0, st>>>(a, m, as, sa, b, n, bs, sb, bias, k, o, os, ntn);
    return cudaGetLastError();
  };
  if (dtype == GANN_F32) return run(matmul_tile_kernel<float>, static_cast<float*>(out));
  if (dtype == GANN_F16) return run(matmul_tile_kernel<__half>, static_cast<__half*>(out));
  return run(matmul_tile_kernel<__nv_bfloat16>, static_cast<__nv_bfloat16*>(out));
}

}  // namespace gann

// 8-bit rows with one scale each, and products of such rows.
//
//   quantize_rows   s_i = max_j |x_ij| * (1/127) in float32,  c_ij = x_ij / s_i
//                   rounded to the nearest integer (ties to even)
//   matmul_i8       y_ij = (sum_k a_ik b_jk) sa_i sb_j + bias_j
#include <algorithm>
#include <cstdint>

#include <cuda.h>
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

// The scale of a row and what its entries are multiplied by. The maximum times
// 1/127 in float32 is off by 0.56 of a step at most (the quotient would be by
// 0.5); the codes refer to the scale as it is stored. A tiny scale
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

template <typename T>
struct Row16 {   // 16 bytes of a row
  static constexpr int n = 16 / sizeof(T);
  uint4 v;
  __device__ __forceinline__ float at(int j) const {
    const uint32_t w = j * static_cast<int>(sizeof(T)) / 4 == 0   ? v.x
                       : j * static_cast<int>(sizeof(T)) / 4 == 1 ? v.y
                       : j * static_cast<int>(sizeof(T)) / 4 == 2 ? v.z
                                                                  : v.w;
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w);
    } else {
      const uint16_t h = static_cast<uint16_t>((j & 1) ? w >> 16 : w);
      return to_f32(*reinterpret_cast<const T*>(&h));
    }
  }
};

// Four codes of a word. With an ordinary scale the sum x / s + 1.5 * 2^23 holds
// the rounded quotient in its low byte (|x / s| < 127.5); only an element whose
// remainder is half a scale or more, where the product with the reciprocal may
// have gone to the wrong side, takes the exact form above.
__device__ __forceinline__ uint32_t quant_word(float x0, float x1, float x2, float x3, const RowScale& rs, bool plain) {
  if (plain) {
    constexpr float kMagic = 12582912.f;
    const float a = __fadd_rn(__fmul_rn(x0, rs.inv), kMagic), b = __fadd_rn(__fmul_rn(x1, rs.inv), kMagic);
    const float c = __fadd_rn(__fmul_rn(x2, rs.inv), kMagic), d = __fadd_rn(__fmul_rn(x3, rs.inv), kMagic);
    const float ea = __fmaf_rn(kMagic - a, rs.s, x0), eb = __fmaf_rn(kMagic - b, rs.s, x1);
    const float ec = __fmaf_rn(kMagic - c, rs.s, x2), ed = __fmaf_rn(kMagic - d, rs.s, x3);
    const float e = fmaxf(fmaxf(fabsf(ea), fabsf(eb)), fmaxf(fabsf(ec), fabsf(ed)));
    if (2.f * e < rs.s) {
      const uint32_t lo = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040);
      const uint32_t hi = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
      return __byte_perm(lo, hi, 0x5410);
    }
  }
  return (quant_code(x0, rs) & 0xff) | (quant_code(x1, rs) & 0xff) << 8 | (quant_code(x2, rs) & 0xff) << 16 |
         static_cast<uint32_t>(quant_code(x3, rs) & 0xff) << 24;
}

// A row by a group of threads: one warp, or (rows longer than a warp's
// registers hold) a whole block. Bound by memory: 5 bytes move per float32
// element, and the codes take about seven instructions each. The row's 16-byte
// vectors (VEC: rows start on 16-byte boundaries) stay in registers between
// the maximum and the codes, up to kRowHeld a thread; longer rows are read
// again, which the caches serve. 500000 x 768 f32: 305 to 330 us (5.8 TB/s and
// more), bf16 298 us (3.9 TB/s: the instructions of a code are the same). Rows off
// 16-byte boundaries are read element by element, and twice: 500000 x 769 f32 459
// us, bf16 458. Rows of zeros take the codes' exact form: 442 us.
constexpr int kRowHeld = 8;

template <typename T, bool VEC, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 256 : WARPS * kWarp, WARPS == 1 ? 4 : 1) quantize_kernel(
    const uint8_t* __restrict__ x, int64_t rows, int64_t stride, int dim, int8_t* __restrict__ codes, int64_t cstride,
    float* __restrict__ scales) {
  constexpr int N = VEC ? Row16<T>::n : 1, NT = WARPS * kWarp;
  __shared__ float red[WARPS];
  const int t = WARPS == 1 ? threadIdx.x % kWarp : threadIdx.x;
  const int per = WARPS == 1 ? 256 / kWarp : 1;   // rows of a block at a time
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * per + (WARPS == 1 ? threadIdx.x / kWarp : 0); r < rows;
       r += static_cast<int64_t>(gridDim.x) * per) {
    const T* row = reinterpret_cast<const T*>(x + r * stride);
    int8_t* out = codes + r * cstride;
    const int nv = VEC ? dim / N : 0;   // whole vectors; the rest one by one
    Row16<T> held[VEC ? kRowHeld : 1];
    float a = 0.f;
    bool bad = false;
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < kRowHeld; ++i)
        if (t + i * NT < nv) held[i].v = __ldcs(reinterpret_cast<const uint4*>(row) + t + i * NT);
#pragma unroll
      for (int i = 0; i < kRowHeld; ++i)
        if (t + i * NT < nv) {
#pragma unroll
          for (int j = 0; j < N; ++j) {
            a = fmaxf(a, fabsf(held[i].at(j)));
            bad |= isnan(held[i].at(j));
          }
        }
      for (int v = t + kRowHeld * NT; v < nv; v += NT) {
        Row16<T> w;
        w.v = __ldg(reinterpret_cast<const uint4*>(row) + v);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          a = fmaxf(a, fabsf(w.at(j)));
          bad |= isnan(w.at(j));
        }
      }
    }
    for (int j = nv * N + t; j < dim; j += NT) {
      const float e = to_f32(row[j]);
      a = fmaxf(a, fabsf(e));
      bad |= isnan(e);
    }
    if (bad) a = INFINITY;
    a = __uint_as_float(__reduce_max_sync(kFull, __float_as_uint(a)));   // not negative: bits are ordered
    if constexpr (WARPS > 1) {
      __syncthreads();
      if (t % kWarp == 0) red[t / kWarp] = a;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WARPS; ++w) a = fmaxf(a, red[w]);
    }
    const RowScale rs = row_scale(a);
    const bool plain = rs.scale >= 0x1p-60f;   // not for tiny, zero and NaN scales
    if constexpr (VEC) {
      auto put = [&](const Row16<T>& w, int v) {
        if constexpr (N == 4) {
          reinterpret_cast<uint32_t*>(out)[v] = quant_word(w.at(0), w.at(1), w.at(2), w.at(3), rs, plain);
        } else {
          reinterpret_cast<uint2*>(out)[v] = make_uint2(quant_word(w.at(0), w.at(1), w.at(2), w.at(3), rs, plain),
                                                        quant_word(w.at(4), w.at(5), w.at(6), w.at(7), rs, plain));
        }
      };
#pragma unroll
      for (int i = 0; i < kRowHeld; ++i)
        if (t + i * NT < nv) put(held[i], t + i * NT);
      for (int v = t + kRowHeld * NT; v < nv; v += NT) {
        Row16<T> w;
        w.v = __ldg(reinterpret_cast<const uint4*>(row) + v);
        put(w, v);
      }
    }
    for (int j = nv * N + t; j < dim; j += NT) out[j] = static_cast<int8_t>(quant_code(to_f32(row[j]), rs));
    if (t == 0) scales[r] = rs.scale;
  }
}

// y = acc sa sb + bias (0 when there is none): the sum is an exact integer; it
// is rounded to 24 bits when it needs more, then after the first product and
// after the second with its sum.
__device__ __forceinline__ float i8_value(int acc, float sa, float sb, float bias) {
  return __fmaf_rn(static_cast<float>(acc) * sa, sb, bias);
}

// ------------------------------------------------------------ one to four rows
// With one to four rows of a the product only reads b: bound by memory, dp4a
// keeps up with it. A group of `lanes` lanes (as few as its vectors of 16 codes
// need, at least 8) takes R rows of b at a time, so a's vector is read from
// shared memory once for R of b's and R loads are on their way; the R sums are
// folded into the lanes while they are added up. 1 x 100000 x 768: 14 us (5.4
// TB/s), on the tensor cores 21.6 us.
constexpr int kThinRows = 4, kThinThreads = 256, kThinBytes = 48 * 1024;

__device__ __forceinline__ int dot16(const uint4& x, const uint4& y, int acc) {
  acc = __dp4a(static_cast<int>(x.x), static_cast<int>(y.x), acc);
  acc = __dp4a(static_cast<int>(x.y), static_cast<int>(y.y), acc);
  acc = __dp4a(static_cast<int>(x.z), static_cast<int>(y.z), acc);
  return __dp4a(static_cast<int>(x.w), static_cast<int>(y.w), acc);
}

template <typename T, int M, int R>
__global__ void __launch_bounds__(kThinThreads) thin_kernel(const int8_t* __restrict__ a, int m, int64_t as,
                                                            const float* __restrict__ sa, const int8_t* __restrict__ b,
                                                            int64_t n, int64_t bs, const float* __restrict__ sb,
                                                            const float* __restrict__ bias, int k, int lanes,
                                                            T* __restrict__ out, int64_t os) {
  extern __shared__ uint4 rows_a[];   // [M][nv], zeros past k and m
  const int nv = (k + 15) / 16, tid = threadIdx.x;
  for (int e = tid; e < M * nv; e += kThinThreads) {
    const int i = e / nv, v = e - i * nv;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (i < m) {
      const int8_t* p = a + i * as + v * 16;
      if (v * 16 + 16 <= k) {
        w = *reinterpret_cast<const uint4*>(p);
      } else {
        uint32_t q[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (v * 16 + j < k) q[j / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(p[j])) << (8 * (j % 4));
        w = make_uint4(q[0], q[1], q[2], q[3]);
      }
    }
    rows_a[e] = w;
  }
  __syncthreads();
  const int lane = tid & (lanes - 1);
  const int64_t per = kThinThreads / lanes, groups = (n + R - 1) / R;
  // every lane of a warp takes part in the folding, so loops run whole
  const int64_t first = static_cast<int64_t>(blockIdx.x) * per;
  for (int64_t q0 = first; q0 < groups; q0 += static_cast<int64_t>(gridDim.x) * per) {
    const int64_t r0 = (q0 + tid / lanes) * R;
    int acc[M][R];
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r) acc[i][r] = 0;
#pragma unroll(R == 1 ? 4 : 2)
    for (int v = lane; v < nv; v += lanes) {
      uint4 w[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t row = min(r0 + r, n - 1);
        const int8_t* p = b + row * bs + static_cast<int64_t>(v) * 16;
        // the last vector's codes past k meet zeros; behind the last row there
        // may be no memory for them
        if (v * 16 + 16 <= k || row < n - 1) {
          w[r] = __ldcs(reinterpret_cast<const uint4*>(p));
        } else {
          uint32_t z[4] = {0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (v * 16 + j < k) z[j / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(p[j])) << (8 * (j % 4));
          w[r] = make_uint4(z[0], z[1], z[2], z[3]);
        }
      }
#pragma unroll
      for (int i = 0; i < M; ++i) {
        const uint4 x = rows_a[i * nv + v];
#pragma unroll
        for (int r = 0; r < R; ++r) acc[i][r] = dot16(w[r], x, acc[i][r]);
      }
    }
#pragma unroll
    for (int i = 0; i < M; ++i) {
      int sum;
      int64_t row = r0;
      if (R == 4) {
        // lanes 0..3 of every four end up with rows 0..3
        const bool hi = lane & 2, odd = lane & 1;
        const int x0 = hi ? acc[i][2 % R] : acc[i][0], y0 = hi ? acc[i][0] : acc[i][2 % R];
        const int x1 = hi ? acc[i][3 % R] : acc[i][1 % R], y1 = hi ? acc[i][1 % R] : acc[i][3 % R];
        const int s0 = x0 + __shfl_xor_sync(kFull, y0, 2), s1 = x1 + __shfl_xor_sync(kFull, y1, 2);
        sum = (odd ? s1 : s0) + __shfl_xor_sync(kFull, odd ? s0 : s1, 1);
        for (int o = 4; o < lanes; o <<= 1) sum += __shfl_xor_sync(kFull, sum, o);
        row += lane & 3;
      } else {
        sum = acc[i][0];
        for (int o = 1; o < lanes; o <<= 1) sum += __shfl_xor_sync(kFull, sum, o);
      }
      if (lane < R && row < n && i < m)
        out[i * os + row] = from_f32<T>(i8_value(sum, sa[i], sb[row], bias ? bias[row] : 0.f));
    }
  }
}

// ------------------------------------------------------- tensor-core product
// The 5th-generation tensor cores multiply signed bytes with 32-bit sums
// (tcgen05.mma, kind::i8): 128 rows of b by `tn` rows of a, 128 bytes of k a
// step. b is the side with the 128 TMEM lanes, so a lane's results lie in one
// column of the output and 32 lanes store 32 neighbours of an output row: any
// output alignment is coalesced without staging. A persistent block per SM:
//   warp 0      TMA loads of both sides' 128-byte columns into a ring of stages
//   warp 1      issues the products; sums in TMEM, two buffers of tn columns
//   the others  read a finished buffer, scale and store it while the next fills
// Rows and columns past the matrices are zeros (TMA fills them), k need not be
// a multiple of anything; tn shrinks to the rows of a that are left.
// Large products use pairs of blocks (cta_group::2): 256 rows of b by tn rows of
// a, each block loading its 128 rows of b and half of a's rows, so a step
// moves 32 KB instead of 48 KB into an SM for the same work (8192^3: 416 us with
// single blocks, 396 us with pairs).
// With few tiles and a long k, the blocks of a cluster share a tile: each sums
// a part of k, then each gets the others' sums of a part of the columns
// through distributed shared memory (integers: the order does not matter).
//
// Measured: 8192^3 395 us (2.8 PFLOP/s; the power limit holds the tensor pipe
// there), 4097 x 4096 x 4096 to bf16 57 to 68 us, 4096 x 131072 x 768 to f32 500
// us alone and up to 600 in a long run at the power limit (the output is 330 us
// of writes; the epilogue stores 4 bytes a lane), 24 x 32001 x 1024 11 us.
//
// Waits for copies, products and buffers end: after kWaitClocks the block gives
// up, and the tiles it has not finished are filled with NaN (there is no other
// sign of it). The allocation of TMEM and the clusters' barriers have no limit of
// their own. A lone block waits for TMEM while it holds none, so whoever has it
// goes on and frees it. The blocks of a cluster need theirs all at once, and two
// clusters on the same SMs could each hold what the other waits for: a block of a
// cluster therefore asks for all of an SM's shared memory, which leaves no room
// for any other block, of this kernel or another, until it ends. The barriers
// wait only for the cluster's own blocks, each of which gets there.
constexpr int kEpiWarps = 8, kEpiThreads = kEpiWarps * kWarp;
constexpr int kMmaThreads = kEpiThreads + 2 * kWarp;
constexpr int kMmaRows = 128, kMmaK = 128;
constexpr int kMmaMaxTn = 256, kMmaMaxStages = 12;
constexpr int64_t kWaitClocks = 8000000000ll;   // about 4 s

struct MmaArgs {
  const float* sa;
  const float* sb;
  const float* bias;
  void* out;
  int64_t m, n, os;
  int k, tn, stages, split, pairs;
  int tiles_m, tiles_n, group_m;
};

struct MmaShared {
  uint64_t full[kMmaMaxStages], empty[kMmaMaxStages];
  uint64_t sum_full[2], sum_empty[2], drain;
  uint32_t tmem, dead;
  __align__(16) float sa[2][kMmaMaxTn];
};

// The most dynamic shared memory that a block may ask for beside MmaShared, and
// the kernels' limit: one value for every call, for a limit that followed the
// call's own size could fall below another thread's before that one launches.
constexpr size_t kMmaSmem = (227 * 1024 - sizeof(MmaShared)) / 128 * 128;
// With the 1 KB that every block is charged, an SM of 228 KB has less than that left.
static_assert(228 * 1024 - 1024 - kMmaSmem - sizeof(MmaShared) < 1024, "another block would fit beside a cluster's");

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint64_t* b, int n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\n"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(b)), "r"(parity)
      : "memory");
  return ok != 0;
}
// False when the block has given up. The clock is looked at once in 256 tries
// (each of which the hardware may suspend for a while).
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, uint32_t* dead) {
  for (int i = 0; i < 256; ++i)
    if (mbar_try(b, parity)) return true;
  const int64_t t0 = clock64();
  while (true) {
    for (int i = 0; i < 256; ++i)
      if (mbar_try(b, parity)) return true;
    if (*reinterpret_cast<volatile uint32_t*>(dead)) return false;
    if (clock64() - t0 > kWaitClocks) {
      *reinterpret_cast<volatile uint32_t*>(dead) = 1;
      return false;
    }
  }
}
// The same without a word to the others: for what is still in flight then.
__device__ __forceinline__ void mbar_drain(uint64_t* b, uint32_t parity) {
  const int64_t t0 = clock64();
  while (!mbar_try(b, parity) && clock64() - t0 < kWaitClocks) {
  }
}
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
// The same within a pair of blocks, counted by the first block's barrier.
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ uint32_t in_block(const void* p, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Operand tile of rows of 128 bytes, 128-byte swizzle: groups of 8 rows are
// 1024 bytes apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// s32 += s8 x s8, both operands K-major.
template <bool PAIR>
__device__ __forceinline__ uint32_t i8_instr(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>((PAIR ? 2 : 1) * kMmaRows >> 4) << 24);
}
template <bool PAIR>
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool add) {
  if (PAIR)
    asm volatile(
        "{\n.reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(instr), "r"(static_cast<uint32_t>(add))
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(instr), "r"(static_cast<uint32_t>(add))
        : "memory");
}
// An arrival, once the products issued so far are done, at this block's
// barrier, or at both of a pair's.
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  if (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t addr, int (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
      "%13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_load(uint32_t addr, int (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
      "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, "
      "[%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]),
        "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]),
        "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]),
        "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kEpiThreads) : "memory"); }

// Tiles in groups of group_m rows of tiles: within a group the tiles that
// share rows of b come one after another, and a's rows of the group stay in L2.
__device__ __forceinline__ void tile_at(const MmaArgs& p, int64_t t, int& im, int& in) {
  const int64_t per = static_cast<int64_t>(p.group_m) * p.tiles_n;
  const int gi = static_cast<int>(t / per);
  const int m0 = gi * p.group_m, gm = min(p.tiles_m - m0, p.group_m);
  const int64_t r = t - gi * per;
  in = static_cast<int>(r / gm);
  im = m0 + static_cast<int>(r - static_cast<int64_t>(in) * gm);
}

// A warp's 32 neighbours of 32 output rows: o is the lane's element of the first.
__device__ __forceinline__ void store_columns(float* o, int64_t os, const float (&y)[32], int, bool) {
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    *o = y[j];
    o += os;
  }
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, const __half*) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 16-bit results: with rows of 4-byte multiples (pairs), lanes 2i and 2i + 1
// trade values so that one stores both of an even row, the other both of the
// odd one: half the stores.
template <typename T>
__device__ __forceinline__ void store_columns(T* o, int64_t os, const float (&y)[32], int lane, bool pairs) {
  if (pairs) {
    const bool odd = lane & 1;
    T* q = odd ? o - 1 + os : o;
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      const float got = __shfl_xor_sync(kFull, odd ? y[j] : y[j + 1], 1);
      *reinterpret_cast<uint32_t*>(q) = odd ? pack2(got, y[j + 1], q) : pack2(y[j], got, q);
      q += 2 * os;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      *o = from_f32<T>(y[j]);
      o += os;
    }
  }
}

template <typename T, bool PAIR>
__global__ void __launch_bounds__(kMmaThreads, 1) mma_kernel(const __grid_constant__ CUtensorMap map_a,
                                                             const __grid_constant__ CUtensorMap map_b,
                                                             const __grid_constant__ MmaArgs p) {
  extern __shared__ uint8_t dyn[];
  __shared__ MmaShared sh;
  uint8_t* ring = dyn + (1024 - smem_u32(dyn) % 1024) % 1024;
  const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
  const int stage_bytes = kMmaRows * kMmaK + p.tn / (PAIR ? 2 : 1) * kMmaK;
  const int steps = (p.k + kMmaK - 1) / kMmaK;
  // a cluster is a pair, the parts of k, or one block
  const int cluster = PAIR ? 2 : p.split, rank = static_cast<int>(blockIdx.x) % cluster;
  const int k0 = PAIR ? 0 : static_cast<int>(static_cast<int64_t>(steps) * rank / p.split);
  const int k1 = PAIR ? steps : static_cast<int>(static_cast<int64_t>(steps) * (rank + 1) / p.split);
  const int64_t total = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  const int64_t t0 = blockIdx.x / cluster, dt = gridDim.x / cluster;
  // rows of a in a tile, as many as the products' granularity makes of them
  auto rows_of = [&](int im) {
    const int left = static_cast<int>(min(static_cast<int64_t>(p.tn), p.m - static_cast<int64_t>(im) * p.tn));
    return PAIR ? (left + 31) / 32 * 32 : (left + 15) / 16 * 16;
  };
  auto first_row_of = [&](int in) { return PAIR ? in * 2 * kMmaRows + rank * kMmaRows : in * kMmaRows; };
  int columns = 32;   // TMEM columns: two buffers, a power of two
  while (columns < 2 * p.tn) columns <<= 1;

  // the loading lane's place: tile, step, stage
  int64_t lt = t0;
  int lk = k0, ls = 0, lm = 0, ln = 0, loaded = 0;
  uint32_t lphase = 0;
  bool lok = true;
  auto load_steps = [&]() {
    while (lt < total && lok) {
      if (lk == k0) tile_at(p, lt, lm, ln);
      if (!mbar_wait(&sh.empty[ls], lphase ^ 1u, &sh.dead)) {
        lok = false;
        break;
      }
      uint8_t* dst = ring + ls * stage_bytes;
      if (PAIR) {
        const uint32_t bar = in_block(&sh.full[ls], 0);
        if (rank == 0) mbar_expect(&sh.full[ls], 2 * stage_bytes);
        tma_load_pair(dst, &map_b, lk * kMmaK, first_row_of(ln), bar);
        tma_load_pair(dst + kMmaRows * kMmaK, &map_a, lk * kMmaK, lm * p.tn + rank * (rows_of(lm) / 2), bar);
      } else {
        mbar_expect(&sh.full[ls], stage_bytes);
        tma_load(dst, &map_b, lk * kMmaK, first_row_of(ln), &sh.full[ls]);
        tma_load(dst + kMmaRows * kMmaK, &map_a, lk * kMmaK, lm * p.tn, &sh.full[ls]);
      }
      loaded = min(loaded + 1, p.stages);
      if (++ls == p.stages) {
        ls = 0;
        lphase ^= 1u;
      }
      if (++lk == k1) {
        lk = k0;
        lt += dt;
      }
    }
  };
  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < p.stages; ++i) {
        mbar_init(&sh.full[i], 1);
        mbar_init(&sh.empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sh.sum_full[i], 1);
        mbar_init(&sh.sum_empty[i], (PAIR ? 2 : 1) * kEpiWarps);
      }
      mbar_init(&sh.drain, 1);
      sh.dead = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
  } else if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                   "r"(columns)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                   "r"(columns)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_fence_before();
  }
  __syncthreads();
  if (PAIR) cluster_sync();   // the other block's barriers are ready
  tmem_fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp == 0) {
    if (lane == 0) {
      load_steps();
      // on giving up, copies may still be in flight: see each stage's last one
      // through (a stage whose copy was consumed long ago has passed its phase);
      // a pair's are counted by the first block, and the other ends after it
      if (!lok && !(PAIR && rank))
        for (int i = 0; i < loaded; ++i) {
          const int st = (ls - 1 - i + 2 * p.stages) % p.stages;
          mbar_drain(&sh.full[st], st < ls ? lphase : lphase ^ 1u);
        }
    }
  } else if (warp == 1) {
    if (lane == 0 && !(PAIR && rank)) {
      int s = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int64_t t = t0; t < total && ok; t += dt, ++it) {
        int im, in;
        tile_at(p, t, im, in);
        const uint32_t instr = i8_instr<PAIR>(rows_of(im));
        const uint32_t d = tmem + static_cast<uint32_t>((it & 1) * p.tn);
        if (!mbar_wait(&sh.sum_empty[it & 1], ((it >> 1) & 1) ^ 1u, &sh.dead)) {
          ok = false;
          break;
        }
        tmem_fence_after();
        for (int kb = k0; kb < k1; ++kb) {
          if (!mbar_wait(&sh.full[s], phase, &sh.dead)) {
            ok = false;
            break;
          }
          tmem_fence_after();
          const uint32_t at = smem_u32(ring + s * stage_bytes);
          const uint64_t db = operand_desc(at), da = operand_desc(at + kMmaRows * kMmaK);
#pragma unroll
          for (int q = 0; q < kMmaK / 32; ++q)   // 32 bytes of k an instruction
            if (kb * kMmaK + q * 32 < p.k) mma_i8<PAIR>(d, db + 2 * q, da + 2 * q, instr, kb > k0 || q > 0);
          mma_commit<PAIR>(&sh.empty[s]);
          if (++s == p.stages) {
            s = 0;
            phase ^= 1u;
          }
        }
        if (ok) mma_commit<PAIR>(&sh.sum_full[it & 1]);
      }
      if (!ok) {   // products that are still running
        mma_commit<PAIR>(&sh.drain);
        mbar_drain(&sh.drain, 0);
      }
    }
  } else if (PAIR || p.split == 1) {
    const int quarter = warp % 4, etid = tid - 2 * kWarp;
    const int cols = max(p.tn / (kEpiWarps / 4), 16), c0 = (warp - 2) / 4 * cols;
    // scales of the next tile are fetched while this one is stored
    float sa_next = 0.f, sb_next = 0.f, bias_next = 0.f;
    auto fetch = [&](int64_t t) {
      if (t >= total) return;
      int im, in;
      tile_at(p, t, im, in);
      const int64_t mm = static_cast<int64_t>(im) * p.tn + etid;
      const int64_t nn = static_cast<int64_t>(first_row_of(in)) + quarter * kWarp + lane;
      sa_next = etid < p.tn && mm < p.m ? p.sa[mm] : 0.f;
      sb_next = nn < p.n ? p.sb[nn] : 0.f;
      bias_next = nn < p.n && p.bias ? p.bias[nn] : 0.f;
    };
    fetch(t0);
    int it = 0;
    for (int64_t t = t0; t < total; t += dt, ++it) {
      int im, in;
      tile_at(p, t, im, in);
      const int64_t m0 = static_cast<int64_t>(im) * p.tn;
      const int64_t nn = static_cast<int64_t>(first_row_of(in)) + quarter * kWarp + lane;
      const int buf = it & 1;
      if (etid < p.tn) sh.sa[buf][etid] = sa_next;
      const bool inside = nn < p.n, whole = __all_sync(kFull, inside);
      float sb = sb_next;
      const float bias = bias_next;
      epilogue_sync();
      fetch(t + dt);
      // a block that gave up: NaN
      if (!__all_sync(kFull, mbar_wait(&sh.sum_full[buf], (it >> 1) & 1, &sh.dead))) sb = __int_as_float(0x7fc00000);
      tmem_fence_after();
      const uint32_t at = tmem + (static_cast<uint32_t>(quarter * kWarp) << 16) + static_cast<uint32_t>(buf * p.tn + c0);
      T* o = static_cast<T*>(p.out) + (m0 + c0) * p.os + nn;
      const int end = static_cast<int>(min(static_cast<int64_t>(cols), min(static_cast<int64_t>(p.tn), p.m - m0) - c0));
      const float* sa = sh.sa[buf] + c0;
      int c = 0;
      if (whole && end >= 32) {
        // 32 columns at a time, the next 32 on their way
        int v[32];
        tmem_load(at, v);
        for (; c + 32 <= end; c += 32) {
          tmem_wait_load();
          float y[32];
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 s4 = *reinterpret_cast<const float4*>(sa + c + j);
            y[j] = i8_value(v[j], s4.x, sb, bias);
            y[j + 1] = i8_value(v[j + 1], s4.y, sb, bias);
            y[j + 2] = i8_value(v[j + 2], s4.z, sb, bias);
            y[j + 3] = i8_value(v[j + 3], s4.w, sb, bias);
          }
          if (c + 64 <= end) tmem_load(at + c + 32, v);
          store_columns(o, p.os, y, lane, p.pairs);
          o += 32 * p.os;
        }
        tmem_wait_load();
      }
      for (; c < end; c += 16) {
        int acc[16];
        tmem_load(at + c, acc);
        tmem_wait_load();
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c + j < end && inside) o[j * p.os] = from_f32<T>(i8_value(acc[j], sa[c + j], sb, bias));
        o += 16 * p.os;
      }
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) mbar_arrive_at(in_block(&sh.sum_empty[buf], 0));
        else mbar_arrive(&sh.sum_empty[buf]);
      }
    }
  } else {
    mbar_wait(&sh.sum_full[0], 0, &sh.dead);
  }

  if (!PAIR && p.split > 1) {
    // one tile a cluster; this block has summed its part of k
    __syncwarp();
    tmem_fence_after();
    cluster_sync();   // no block's ring is in use any more
    int im, in;
    tile_at(p, t0, im, in);
    const int64_t m0 = static_cast<int64_t>(im) * p.tn;
    const int share = p.tn / p.split;   // columns of each block
    if (warp >= 2) {
      const int quarter = warp % 4, part = (warp - 2) / 4;
      const int cols = max(p.tn / (kEpiWarps / 4), 16);
      const uint32_t at = tmem + (static_cast<uint32_t>(quarter * kWarp) << 16);
      for (int c = part * cols; c < min(p.tn, (part + 1) * cols); c += 16) {
        int acc[16];
        tmem_load(at + c, acc);
        tmem_wait_load();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int owner = (c + j) / share, slot = rank * share + (c + j) % share;
          const int local = (slot * kMmaRows + quarter * kWarp + lane) * 4;
          asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(in_block(ring + local, owner)), "r"(acc[j]) : "memory");
        }
      }
    }
    uint32_t bad = *reinterpret_cast<volatile uint32_t*>(&sh.dead);
    cluster_sync();
    // a block that gave up has spoilt the sums of all of them
    for (int r = 0; r < p.split; ++r) {
      uint32_t v;
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(in_block(&sh.dead, r)) : "memory");
      bad |= v;
    }
    const int* recv = reinterpret_cast<const int*>(ring);
    for (int e = tid; e < share * kMmaRows; e += kMmaThreads) {
      const int c = e / kMmaRows, r = e % kMmaRows;
      const int64_t mm = m0 + rank * share + c, nn = static_cast<int64_t>(in) * kMmaRows + r;
      if (mm >= p.m || nn >= p.n) continue;
      int acc = 0;
      for (int q = 0; q < p.split; ++q) acc += recv[(q * share + c) * kMmaRows + r];
      const float y = i8_value(acc, p.sa[mm], p.sb[nn], p.bias ? p.bias[nn] : 0.f);
      static_cast<T*>(p.out)[mm * p.os + nn] = from_f32<T>(bad ? __int_as_float(0x7fc00000) : y);
    }
    cluster_sync();   // the flags of this block are not read any more
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();   // neither block uses the other's memory any more
  if (warp == 1) {
    tmem_fence_after();
    if (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
  }
}

}  // namespace

cudaError_t launch_quantize_rows(const void* x, int64_t rows, int64_t stride, int dim, int dtype, int8_t* codes,
                                 int64_t code_stride, float* scales, int sm_count, cudaStream_t st) {
  if (rows <= 0) return cudaSuccess;
  const bool vec = stride % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  // one warp a row while its registers hold it, or there are rows enough to
  // fill the GPU with single warps
  const int held = kRowHeld * kWarp * (dtype == GANN_F32 ? 4 : 8);
  const bool block = dim > held && rows < static_cast<int64_t>(sm_count) * 64;
  auto run = [&](auto one, auto many) {
    const int64_t grid = block ? std::min<int64_t>(rows, static_cast<int64_t>(sm_count) * 16)
                               : std::min<int64_t>((rows + 7) / 8, static_cast<int64_t>(sm_count) * 32);
    auto fn = block ? many : one;
    fn<<<static_cast<unsigned>(grid), block ? 512 : 256, 0, st>>>(static_cast<const uint8_t*>(x), rows, stride, dim,
                                                                  codes, code_stride, scales);
    return cudaGetLastError();
  };
  if (dtype == GANN_F32)
    return vec ? run(quantize_kernel<float, true, 1>, quantize_kernel<float, true, 16>)
               : run(quantize_kernel<float, false, 1>, quantize_kernel<float, false, 16>);
  if (dtype == GANN_F16)
    return vec ? run(quantize_kernel<__half, true, 1>, quantize_kernel<__half, true, 16>)
               : run(quantize_kernel<__half, false, 1>, quantize_kernel<__half, false, 16>);
  return vec ? run(quantize_kernel<__nv_bfloat16, true, 1>, quantize_kernel<__nv_bfloat16, true, 16>)
             : run(quantize_kernel<__nv_bfloat16, false, 1>, quantize_kernel<__nv_bfloat16, false, 16>);
}

namespace {

// Rows of a that the kernel is made for: 1, 2 or 4.
int thin_rows(int64_t m) { return m <= 2 ? static_cast<int>(m) : 4; }

// Four rows of b at a time when that leaves 16 warps and more for every SM.
template <typename T>
cudaError_t run_thin(const int8_t* a, int64_t m, int64_t as, const float* sa, const int8_t* b, int64_t n, int64_t bs,
                     const float* sb, const float* bias, int k, T* out, int64_t os, int sm_count, cudaStream_t st) {
  const int nv = (k + 15) / 16;
  const int lanes = nv <= 16 ? 8 : nv <= 64 ? 16 : 32;
  const bool four = n * lanes / 4 >= static_cast<int64_t>(sm_count) * 16 * kWarp;
  const size_t smem = static_cast<size_t>(thin_rows(m)) * nv * 16;
  auto run = [&](auto fn, int r) {
    const int64_t per = kThinThreads / lanes * r;
    const int64_t grid = std::min<int64_t>((n + per - 1) / per, static_cast<int64_t>(sm_count) * 8);
    fn<<<static_cast<unsigned>(grid), kThinThreads, smem, st>>>(a, static_cast<int>(m), as, sa, b, n, bs, sb, bias, k,
                                                                lanes, out, os);
    return cudaGetLastError();
  };
  if (m == 1) return four ? run(thin_kernel<T, 1, 4>, 4) : run(thin_kernel<T, 1, 1>, 1);
  if (m == 2) return four ? run(thin_kernel<T, 2, 4>, 4) : run(thin_kernel<T, 2, 1>, 1);
  return four ? run(thin_kernel<T, 4, 4>, 4) : run(thin_kernel<T, 4, 1>, 1);
}

// cuTensorMapEncodeTiled from the driver that the runtime has loaded.
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

// Rows of k bytes in boxes of 128 bytes by `box` rows, zeros outside.
cudaError_t encode_rows(CUtensorMap* map, const int8_t* p, int64_t rows, int64_t stride, int k, int box) {
  const EncodeTiled fn = encode_tiled();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
  const cuuint32_t boxes[2] = {kMmaK, static_cast<cuuint32_t>(box)};
  const cuuint32_t steps[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(p), dims, strides, boxes, steps,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

struct MmaPlan {
  int tn, split;
  bool pair;
};

// Rows of a in a tile: all of them up to 256, in steps that the two output
// halves share; with more, 256, halved while the tiles do not fill the GPU.
// A tile's k is split over 2, 4 or 8 blocks while blocks are idle, if that
// saves more than it costs: a step of 128 takes a lone block about 0.36 us, the
// exchange of the parts' sums 2.8 us and 0.05 us a column (16 x 4096 x 4096:
// 12.9 us in two parts, 10.5 in four; 64 x 8192 x 1024: 11.6 in two, 7.1 in
// one). Full-width tiles are made by pairs.
MmaPlan plan_mma(int64_t m, int64_t n, int k, int sm_count) {
  MmaPlan p{16, 1, false};
  while (p.tn < m && p.tn < kMmaMaxTn) p.tn <<= 1;
  const int64_t tn_tiles = (n + kMmaRows - 1) / kMmaRows;
  while (m > p.tn / 2 && p.tn > 64 && tn_tiles * ((m + p.tn - 1) / p.tn) * 2 <= sm_count) p.tn >>= 1;
  const int64_t tiles = tn_tiles * ((m + p.tn - 1) / p.tn);
  const int steps = (k + kMmaK - 1) / kMmaK;
  while (p.split < 8 && tiles * p.split * 2 <= sm_count && steps >= p.split * 4) p.split <<= 1;
  if (steps * (p.split - 1) * 36 < (280 + 5 * p.tn) * p.split) p.split = 1;
  p.pair = p.tn == kMmaMaxTn && p.split == 1 && n > kMmaRows;
  return p;
}

}  // namespace

cudaError_t launch_matmul_i8(const int8_t* a, int64_t m, int64_t as, const float* sa, const int8_t* b, int64_t n,
                             int64_t bs, const float* sb, const float* bias, int k, void* out, int64_t os, int dtype,
                             int sm_count, cudaStream_t st) {
  if (m <= 0 || n <= 0) return cudaSuccess;
  if (m <= kThinRows && thin_rows(m) * ((k + 15) / 16) * 16 <= kThinBytes) {
    if (dtype == GANN_F32) return run_thin(a, m, as, sa, b, n, bs, sb, bias, k, static_cast<float*>(out), os, sm_count, st);
    if (dtype == GANN_F16) return run_thin(a, m, as, sa, b, n, bs, sb, bias, k, static_cast<__half*>(out), os, sm_count, st);
    return run_thin(a, m, as, sa, b, n, bs, sb, bias, k, static_cast<__nv_bfloat16*>(out), os, sm_count, st);
  }
  const MmaPlan plan = plan_mma(m, n, k, sm_count);
  MmaArgs p{};
  p.sa = sa;
  p.sb = sb;
  p.bias = bias;
  p.out = out;
  p.m = m;
  p.n = n;
  p.os = os;
  p.k = k;
  p.tn = plan.tn;
  p.split = plan.split;
  p.pairs = os % 2 == 0 && reinterpret_cast<uintptr_t>(out) % 4 == 0;
  const int64_t rows = plan.pair ? 2 * kMmaRows : kMmaRows;
  const int64_t tiles_m = (m + p.tn - 1) / p.tn, tiles_n = (n + rows - 1) / rows;
  p.tiles_m = static_cast<int>(tiles_m);
  p.tiles_n = static_cast<int>(tiles_n);
  // rows of a that stay in L2 beside the stream of b: about 32 MB
  p.group_m = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(tiles_m, (32 << 20) / (static_cast<int64_t>(k) * p.tn + 1))));
  const int a_rows = plan.pair ? p.tn / 2 : p.tn, cluster = plan.pair ? 2 : p.split;
  const int stage = (kMmaRows + a_rows) * kMmaK;
  p.stages = std::min({kMmaMaxStages, (200 * 1024) / stage, std::max(2, (k + kMmaK - 1) / kMmaK * 2)});
  const size_t ring = std::max<size_t>(static_cast<size_t>(p.stages) * stage,
                                       p.split > 1 ? static_cast<size_t>(p.tn) * kMmaRows * 4 : 0);
  const size_t smem = cluster > 1 ? kMmaSmem : ring + 1024;   // a cluster's blocks have their SMs to themselves
  if (ring + 1024 > kMmaSmem) return cudaErrorInvalidConfiguration;
  const int64_t blocks = cluster * (p.split > 1 ? tiles_m * tiles_n : std::min<int64_t>(tiles_m * tiles_n, sm_count / cluster));
  auto run = [&](auto fn) -> cudaError_t {
    cudaError_t r = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMmaSmem));
    // the driver's call wants a context, which the one before has made current
    // if this is the host thread's first
    CUtensorMap ma, mb;
    if (r == cudaSuccess) r = encode_rows(&ma, a, m, as, k, a_rows);
    if (r == cudaSuccess) r = encode_rows(&mb, b, n, bs, k, kMmaRows);
    if (r != cudaSuccess) return r;
    if (cluster == 1) {
      fn<<<static_cast<unsigned>(blocks), kMmaThreads, smem, st>>>(ma, mb, p);
      return cudaGetLastError();
    }
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(cluster);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks));
    cfg.blockDim = dim3(kMmaThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fn, ma, mb, p);
  };
  if (dtype == GANN_F32) return plan.pair ? run(mma_kernel<float, true>) : run(mma_kernel<float, false>);
  if (dtype == GANN_F16) return plan.pair ? run(mma_kernel<__half, true>) : run(mma_kernel<__half, false>);
  return plan.pair ? run(mma_kernel<__nv_bfloat16, true>) : run(mma_kernel<__nv_bfloat16, false>);
}

}  // namespace gann

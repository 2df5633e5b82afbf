// The gated activation between an expert's two products, as an operator of its own:
//   y[r, i]  = w[r] * SiLU(g[r, i]) * u[r, i]        g = gu[:, :I], u = gu[:, I:], w optional (1)
// with its gradients, s = sigmoid(g):
//   dg = w dy u s (1 + g (1 - s)),  du = w dy g s,  dw[r] = sum_i dy g s u
// and a form that leaves y as e4m3 rows with 1x128 scales, the operand of a block-scaled product.
//
// All of them are bound by memory: 6 bytes a cell forward (16-bit types), 10 backward, 5 with the
// e4m3 result.  Every thread moves 16-byte vectors (8 cells) of the gate half and of the up half.
// Measured on a B200, 16384 x 2048 bf16: forward 31 us = 6460 GB/s, the rate of a copy; backward 51 us =
// 6600 GB/s, with row weights 53 to 56 us = 6000 to 6340 GB/s (a block of 256 threads to a row, one vector
// each, took 63); to e4m3 36 us = 4650 GB/s with f32 scales and 37 with power-of-two scales (38 and 39 with row
// weights), 8192 x 14336 126 and 130 us: the maximum of a group is a chain of four shuffles between the loads
// and the stores, and the stores are half as wide.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "host.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "scales.cuh"

namespace fmoe {
namespace {

constexpr int kSiluThreads = 256;
constexpr int kSiluHeld = 2;          // vectors per thread: both halves of each are in flight together
// A launch covers at most this many 16-byte vectors, so that vector indices stay in 31 bits.
constexpr int64_t kSiluMaxVec = int64_t{1} << 30;

// Division of a 31-bit number by a constant: n / d == mulhi(n, mul) >> shift.
struct FastDiv {
  uint32_t d, mul, shift;
};
FastDiv make_fast_div(uint32_t d) {
  // l = ceil(log2 d); mul = floor(2^32 (2^l - d) / d) + 1 is the round-up multiplier of the
  // 33-bit form; restricted to n < 2^31 the plain form with 2^(31 + l) is exact.
  uint32_t l = 0;
  while (l < 31 && (1u << l) < d) ++l;
  const uint64_t m = ((uint64_t{1} << (31 + l)) + d - 1) / d;
  return FastDiv{d, static_cast<uint32_t>(m), l == 0 ? 0u : l - 1};
}
__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv& f) {
  return f.d == 1 ? n : __umulhi(n, f.mul) >> f.shift;
}

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float2 load(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t store(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <> struct Pair<__half> {
  static __device__ __forceinline__ float2 load(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ uint32_t store(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = Pair<T>::load(w[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&f)[8]) {
  return make_uint4(Pair<T>::store(f[0], f[1]), Pair<T>::store(f[2], f[3]), Pair<T>::store(f[4], f[5]),
                    Pair<T>::store(f[6], f[7]));
}

// 1 / (1 + exp(-g)) by the two special-function instructions.  __expf is off by at most 2 + 1.173 |g| units
// in the last place (2^-23), the sum and the reciprocal by one each, so the relative error is below
// (4 + 1.173 |g|) 2^-23: 2^-20 up to |g| = 3, 2^-16 at -80, far inside a rounding to 16 bits.  Below -88.7
// the exponential is infinite and the result zero (the approximate reciprocal takes every finite input
// and infinity, which the approximate division does not).
__device__ __forceinline__ float sigmoid(float g) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + __expf(-g)));
  return r;
}

template <typename T, bool kWeighted>
__global__ void __launch_bounds__(kSiluThreads)
silu_mul_kernel(const uint4* __restrict__ gu, const float* __restrict__ row_weight, uint4* __restrict__ out,
                uint32_t n_vec, FastDiv row_vec) {
  ptx::pdl_wait();
  ptx::pdl_release();
  const uint32_t i0 = blockIdx.x * (kSiluThreads * kSiluHeld) + threadIdx.x;
  uint4 g[kSiluHeld], u[kSiluHeld];
  float w[kSiluHeld];
#pragma unroll
  for (int j = 0; j < kSiluHeld; ++j) {
    const uint32_t i = i0 + j * kSiluThreads;
    if (i < n_vec) {
      const uint32_t row = fast_div(i, row_vec);
      const uint4* s = gu + (static_cast<size_t>(i) + static_cast<size_t>(row) * row_vec.d);
      g[j] = __ldcs(s);
      u[j] = __ldcs(s + row_vec.d);
      w[j] = kWeighted ? __ldg(row_weight + row) : 1.0f;
    }
  }
#pragma unroll
  for (int j = 0; j < kSiluHeld; ++j) {
    const uint32_t i = i0 + j * kSiluThreads;
    if (i < n_vec) {
      float gf[8], uf[8];
      unpack<T>(g[j], gf);
      unpack<T>(u[j], uf);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = gf[e] * sigmoid(gf[e]) * uf[e];
        gf[e] = kWeighted ? y * w[j] : y;
      }
      out[i] = pack<T>(gf);
    }
  }
}

// y rounded to T, then quantised per 128 columns as quantise_rows does it (16 lanes hold a group).
template <typename T, bool kWeighted, bool kHw>
__global__ void __launch_bounds__(kSiluThreads)
silu_mul_quantise_kernel(const uint4* __restrict__ gu, const float* __restrict__ row_weight, uint2* __restrict__ q,
                         void* __restrict__ scales, uint32_t n_vec, FastDiv row_vec) {
  ptx::pdl_wait();
  ptx::pdl_release();
  const uint32_t i0 = blockIdx.x * (kSiluThreads * kSiluHeld) + threadIdx.x;
  uint4 g[kSiluHeld], u[kSiluHeld];
  float w[kSiluHeld];
  uint32_t rows[kSiluHeld];
#pragma unroll
  for (int j = 0; j < kSiluHeld; ++j) {
    const uint32_t i = i0 + j * kSiluThreads;
    g[j] = u[j] = make_uint4(0, 0, 0, 0);
    w[j] = 1.0f;
    rows[j] = 0;
    if (i < n_vec) {
      rows[j] = fast_div(i, row_vec);
      const uint4* s = gu + (static_cast<size_t>(i) + static_cast<size_t>(rows[j]) * row_vec.d);
      g[j] = __ldcs(s);
      u[j] = __ldcs(s + row_vec.d);
      if (kWeighted) w[j] = __ldg(row_weight + rows[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < kSiluHeld; ++j) {
    const uint32_t i = i0 + j * kSiluThreads;
    float gf[8], uf[8];
    unpack<T>(g[j], gf);
    unpack<T>(u[j], uf);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = gf[e] * sigmoid(gf[e]) * uf[e];
      gf[e] = kWeighted ? y * w[j] : y;
    }
    unpack<T>(pack<T>(gf), gf);          // the rounding point of the arithmetic contract
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(gf[e]));
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    uint32_t sbyte;
    const float sc = group_scale<kHw>(amax, sbyte);
    const float inv = 1.0f / sc;
    if (i < n_vec) {
      const uint32_t col = i - rows[j] * row_vec.d;
      if ((col & 15u) == 0) {
        const uint32_t groups = row_vec.d >> 4;
        if (kHw)
          static_cast<uint8_t*>(scales)[static_cast<size_t>(rows[j]) * scale_pitch(groups) + (col >> 4)] =
              static_cast<uint8_t>(sbyte);
        else
          static_cast<float*>(scales)[static_cast<size_t>(rows[j]) * groups + (col >> 4)] = sc;
      }
      uint32_t half[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        half[e] = __nv_cvt_float2_to_fp8x2(make_float2(gf[2 * e] * inv, gf[2 * e + 1] * inv), __NV_SATFINITE, __NV_E4M3);
      q[i] = make_uint2(half[0] | (half[1] << 16), half[2] | (half[3] << 16));
    }
  }
}

template <typename T, bool kWeighted>
__device__ __forceinline__ float silu_grad8(const uint4& gv, const uint4& uv, const uint4& dv, float w, uint4& dg,
                                            uint4& du) {
  float g[8], u[8], d[8], a[8], b[8];
  unpack<T>(gv, g);
  unpack<T>(uv, u);
  unpack<T>(dv, d);
  float dot = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float s = sigmoid(g[e]);
    const float act = g[e] * s;
    if (kWeighted) dot += d[e] * (act * u[e]);
    const float dy = kWeighted ? d[e] * w : d[e];
    a[e] = dy * u[e] * s * (1.0f + g[e] * (1.0f - s));
    b[e] = dy * act;
  }
  dg = pack<T>(a);
  du = pack<T>(b);
  return dot;
}

template <typename T>
__global__ void __launch_bounds__(kSiluThreads)
silu_mul_backward_kernel(const uint4* __restrict__ gu, const uint4* __restrict__ dy, uint4* __restrict__ dgu,
                         uint32_t n_vec, FastDiv row_vec) {
  ptx::pdl_wait();
  ptx::pdl_release();
  const uint32_t i = blockIdx.x * kSiluThreads + threadIdx.x;
  if (i >= n_vec) return;
  const uint32_t row = fast_div(i, row_vec);
  const size_t at = static_cast<size_t>(i) + static_cast<size_t>(row) * row_vec.d;
  uint4 dg, du;
  silu_grad8<T, false>(__ldcs(gu + at), __ldcs(gu + at + row_vec.d), __ldcs(dy + i), 1.0f, dg, du);
  dgu[at] = dg;
  dgu[at + row_vec.d] = du;
}

// With row weights a row's gradient of its weight is a sum over the whole row: kTeam threads (one warp
// or four) own a row and add up in a fixed order, so no atomics and the same result every time.  A
// thread has the loads of two vectors in flight.
template <typename T, int kTeam>
__global__ void __launch_bounds__(kSiluThreads)
silu_mul_backward_weighted_kernel(const uint4* __restrict__ gu, const float* __restrict__ row_weight,
                                  const uint4* __restrict__ dy, uint4* __restrict__ dgu, float* __restrict__ dweight,
                                  int64_t rows, int row_vec) {
  ptx::pdl_wait();
  ptx::pdl_release();
  constexpr int kRows = kSiluThreads / kTeam;
  __shared__ float part[kSiluThreads / 32];
  const int t = threadIdx.x % kTeam;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kTeam;
  const bool live = row < rows;
  float dot = 0.0f;
  if (live) {
    const float w = __ldg(row_weight + row);
    const uint4* g = gu + row * (2 * static_cast<int64_t>(row_vec));
    const uint4* d = dy + row * row_vec;
    uint4* o = dgu + row * (2 * static_cast<int64_t>(row_vec));
    for (int i = t; i < row_vec; i += 2 * kTeam) {
      const int i2 = i + kTeam;
      const bool two = i2 < row_vec;
      const uint4 g0 = __ldcs(g + i), u0 = __ldcs(g + row_vec + i), d0 = __ldcs(d + i);
      uint4 g1, u1, d1;
      if (two) { g1 = __ldcs(g + i2); u1 = __ldcs(g + row_vec + i2); d1 = __ldcs(d + i2); }
      uint4 dg, du;
      dot += silu_grad8<T, true>(g0, u0, d0, w, dg, du);
      __stcs(o + i, dg);
      __stcs(o + row_vec + i, du);
      if (two) {
        dot += silu_grad8<T, true>(g1, u1, d1, w, dg, du);
        __stcs(o + i2, dg);
        __stcs(o + row_vec + i2, du);
      }
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
  if (kTeam == 32) {
    if (live && t == 0) dweight[row] = dot;
    return;
  }
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = dot;
  __syncthreads();
  if (live && t == 0) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kTeam / 32; ++i) sum += part[(threadIdx.x >> 5) + i];
    dweight[row] = sum;
  }
}

int check_silu(const char* name, const void* gu, const float* row_weight, int64_t rows, int32_t width, int32_t dtype) {
  if (!gu) return fail(FMOE_ERR_INVALID_ARG, "%s: gu is required", name);
  if (reinterpret_cast<uintptr_t>(row_weight) & 3) return fail(FMOE_ERR_INVALID_ARG, "%s: row_weight must be 4-byte aligned", name);
  if (rows < 0 || width <= 0) return fail(FMOE_ERR_INVALID_ARG, "%s: bad dimensions (rows=%lld width=%d)", name, (long long)rows, width);
  if (dtype != FMOE_BF16 && dtype != FMOE_F16) return fail(FMOE_ERR_UNSUPPORTED, "%s: bf16 and f16 only", name);
  if (width % 8) return fail(FMOE_ERR_UNSUPPORTED, "%s: width must be a multiple of 8", name);
  return FMOE_OK;
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows per launch, so that a launch's vector indices fit 31 bits.
int64_t rows_per_launch(int32_t width) {
  const int64_t r = kSiluMaxVec / (width / 8);
  return r > 0 ? r : 1;
}
unsigned blocks(int64_t n, int per) { return static_cast<unsigned>((n + per - 1) / per); }

template <typename T>
int run_forward(const void* gu, const float* rw, int64_t rows, int width, void* out, cudaStream_t stream) {
  const int rv = width / 8;
  const FastDiv fd = make_fast_div(static_cast<uint32_t>(rv));
  for (int64_t r0 = 0; r0 < rows; r0 += rows_per_launch(width)) {
    const int64_t n = (rows - r0 < rows_per_launch(width) ? rows - r0 : rows_per_launch(width)) * rv;
    const uint4* in = static_cast<const uint4*>(gu) + r0 * 2 * rv;
    uint4* o = static_cast<uint4*>(out) + r0 * rv;
    const dim3 grid(blocks(n, kSiluThreads * kSiluHeld));
    FMOE_CUDA(rw ? launch_pdl(silu_mul_kernel<T, true>, grid, dim3(kSiluThreads), 0, stream, in, rw + r0, o, static_cast<uint32_t>(n), fd)
                 : launch_pdl(silu_mul_kernel<T, false>, grid, dim3(kSiluThreads), 0, stream, in, rw, o, static_cast<uint32_t>(n), fd));
  }
  return FMOE_OK;
}

template <typename T>
int run_quantise(const void* gu, const float* rw, int64_t rows, int width, bool hw, void* q, void* scales, cudaStream_t stream) {
  const int rv = width / 8;
  const FastDiv fd = make_fast_div(static_cast<uint32_t>(rv));
  const int64_t scale_row = hw ? scale_pitch(width / 128) : 4 * (width / 128);
  for (int64_t r0 = 0; r0 < rows; r0 += rows_per_launch(width)) {
    const int64_t n = (rows - r0 < rows_per_launch(width) ? rows - r0 : rows_per_launch(width)) * rv;
    const uint4* in = static_cast<const uint4*>(gu) + r0 * 2 * rv;
    uint2* o = static_cast<uint2*>(q) + r0 * rv;
    void* sc = static_cast<uint8_t*>(scales) + r0 * scale_row;
    const dim3 grid(blocks(n, kSiluThreads * kSiluHeld));
    auto launch = [&](auto kernel) {
      return launch_pdl(kernel, grid, dim3(kSiluThreads), 0, stream, in, rw ? rw + r0 : nullptr, o, sc, static_cast<uint32_t>(n), fd);
    };
    FMOE_CUDA(rw ? (hw ? launch(silu_mul_quantise_kernel<T, true, true>) : launch(silu_mul_quantise_kernel<T, true, false>))
                 : (hw ? launch(silu_mul_quantise_kernel<T, false, true>) : launch(silu_mul_quantise_kernel<T, false, false>)));
  }
  return FMOE_OK;
}

template <typename T>
int run_backward(const void* gu, const float* rw, const void* dy, int64_t rows, int width, void* dgu, float* dweight,
                 cudaStream_t stream) {
  const int rv = width / 8;
  const FastDiv fd = make_fast_div(static_cast<uint32_t>(rv));
  for (int64_t r0 = 0; r0 < rows; r0 += rows_per_launch(width)) {
    const int64_t nr = rows - r0 < rows_per_launch(width) ? rows - r0 : rows_per_launch(width);
    const uint4* in = static_cast<const uint4*>(gu) + r0 * 2 * rv;
    const uint4* d = static_cast<const uint4*>(dy) + r0 * rv;
    uint4* o = static_cast<uint4*>(dgu) + r0 * 2 * rv;
    if (!rw) {
      FMOE_CUDA(launch_pdl(silu_mul_backward_kernel<T>, dim3(blocks(nr * rv, kSiluThreads)), dim3(kSiluThreads), 0, stream,
                           in, d, o, static_cast<uint32_t>(nr * rv), fd));
    } else if (rv <= 64) {
      FMOE_CUDA(launch_pdl(silu_mul_backward_weighted_kernel<T, 32>, dim3(blocks(nr, kSiluThreads / 32)), dim3(kSiluThreads), 0,
                           stream, in, rw + r0, d, o, dweight + r0, nr, rv));
    } else {
      FMOE_CUDA(launch_pdl(silu_mul_backward_weighted_kernel<T, 128>, dim3(blocks(nr, kSiluThreads / 128)), dim3(kSiluThreads), 0,
                           stream, in, rw + r0, d, o, dweight + r0, nr, rv));
    }
  }
  return FMOE_OK;
}

}  // namespace
}  // namespace fmoe

extern "C" int fmoe_silu_mul(const void* gu, const float* row_weight, int64_t rows, int32_t width, int32_t dtype, void* out,
                             void* stream) {
  using namespace fmoe;
  if (rows == 0 && width > 0) return FMOE_OK;
  int rc = check_silu("fmoe_silu_mul", gu, row_weight, rows, width, dtype);
  if (rc != FMOE_OK) return rc;
  if (!out) return fail(FMOE_ERR_INVALID_ARG, "fmoe_silu_mul: out is required");
  if (!aligned16(gu) || !aligned16(out)) return fail(FMOE_ERR_INVALID_ARG, "fmoe_silu_mul: gu and out must be 16-byte aligned");
  DeviceGuard guard(gu);
  if (guard.rc() != FMOE_OK) return guard.rc();
  NvtxRange range("fmoe_silu_mul");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == FMOE_BF16 ? run_forward<__nv_bfloat16>(gu, row_weight, rows, width, out, s)
                            : run_forward<__half>(gu, row_weight, rows, width, out, s);
}

extern "C" int fmoe_silu_mul_quantise(const void* gu, const float* row_weight, int64_t rows, int32_t width, int32_t dtype,
                                      int32_t quant, void* q, void* scales, void* stream) {
  using namespace fmoe;
  if (quant != FMOE_QUANT_BLOCK128 && quant != FMOE_QUANT_BLOCK128_UE8M0)
    return fail(FMOE_ERR_INVALID_ARG, "fmoe_silu_mul_quantise: quant must be a block mode");
  if (rows == 0 && width > 0) return FMOE_OK;
  int rc = check_silu("fmoe_silu_mul_quantise", gu, row_weight, rows, width, dtype);
  if (rc != FMOE_OK) return rc;
  if (width % 128) return fail(FMOE_ERR_UNSUPPORTED, "fmoe_silu_mul_quantise: width must be a multiple of 128");
  if (!q || !scales) return fail(FMOE_ERR_INVALID_ARG, "fmoe_silu_mul_quantise: q and scales are required");
  if (!aligned16(gu) || (reinterpret_cast<uintptr_t>(q) & 7) || (reinterpret_cast<uintptr_t>(scales) & 3))
    return fail(FMOE_ERR_INVALID_ARG, "fmoe_silu_mul_quantise: gu, q and scales must be aligned to 16, 8 and 4 bytes");
  DeviceGuard guard(gu);
  if (guard.rc() != FMOE_OK) return guard.rc();
  NvtxRange range("fmoe_silu_mul_quantise");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool hw = quant == FMOE_QUANT_BLOCK128_UE8M0;
  return dtype == FMOE_BF16 ? run_quantise<__nv_bfloat16>(gu, row_weight, rows, width, hw, q, scales, s)
                            : run_quantise<__half>(gu, row_weight, rows, width, hw, q, scales, s);
}

extern "C" int fmoe_silu_mul_backward(const void* gu, const float* row_weight, const void* dy, int64_t rows, int32_t width,
                                      int32_t dtype, void* dgu, float* dweight, void* stream) {
  using namespace fmoe;
  if (rows == 0 && width > 0) return FMOE_OK;
  int rc = check_silu("fmoe_silu_mul_backward", gu, row_weight, rows, width, dtype);
  if (rc != FMOE_OK) return rc;
  if (!dy || !dgu) return fail(FMOE_ERR_INVALID_ARG, "fmoe_silu_mul_backward: dy and dgu are required");
  if ((row_weight != nullptr) != (dweight != nullptr))
    return fail(FMOE_ERR_INVALID_ARG, "fmoe_silu_mul_backward: row_weight and dweight come together");
  if (!aligned16(gu) || !aligned16(dy) || !aligned16(dgu) || (reinterpret_cast<uintptr_t>(dweight) & 3))
    return fail(FMOE_ERR_INVALID_ARG, "fmoe_silu_mul_backward: gu, dy and dgu must be 16-byte aligned, dweight 4-byte aligned");
  DeviceGuard guard(gu);
  if (guard.rc() != FMOE_OK) return guard.rc();
  NvtxRange range("fmoe_silu_mul_backward");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == FMOE_BF16 ? run_backward<__nv_bfloat16>(gu, row_weight, dy, rows, width, dgu, dweight, s)
                            : run_backward<__half>(gu, row_weight, dy, rows, width, dgu, dweight, s);
}

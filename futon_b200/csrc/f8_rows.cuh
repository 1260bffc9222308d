// f8_rows.cuh — HBM-bound row kernels of the 8-bit float operators.
//
//   rms_norm_f8_kernel   (x + residual) · 1/rms · w, quantised per row and
//                        block of 128 columns
//   quant_rows_f8_kernel activation, then the same quantisation
//   quant_tiles_f8_kernel weights, quantised per 128 × 128 block
//
// A block's scale is amax / 448 with amax = max(|y|, 2^-100), its codes
// e4m3(y · (448 / amax)) rounded to nearest even: the largest magnitude maps
// to the largest code, and the bound keeps an all-zero block finite. amax is
// the maximum of the bit patterns of |y|, in which NaN stands above infinity
// above every number: a block with a NaN gets a NaN scale and NaN codes.
//
// 16 consecutive lanes hold one block of 128 columns, 8 per lane: one
// 16-byte load of 16-bit values, one 8-byte store of codes, and four
// shuffles for the maximum. Everything is read once and written once; sums
// and maxima are f32.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "mathf32.cuh"

namespace futon {

constexpr float kF8Top = 448.0f;
constexpr uint32_t kF8LeastBits = 0x0D800000u;  // 2^-100

enum QuantAct : int { kQuantNone = 0, kQuantGelu = 1, kQuantSwiglu = 2 };

// Whether rows of the operands start at multiples of 16 bytes (8 for codes).
struct RowVec {
  bool src, q;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}

// Eight columns of a row; columns past n read as 0.
template <typename T>
__device__ __forceinline__ void load8(const T* p, long long n, bool vec, float (&v)[8]) {
  if (vec && n >= 8) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = reinterpret_cast<const float4*>(p)[0];
      const float4 b = reinterpret_cast<const float4*>(p)[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32<T>(p[i]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, long long n, bool vec, const float (&v)[8]) {
  if (vec && n >= 8) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint4 a;
      T* e = reinterpret_cast<T*>(&a);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
      *reinterpret_cast<uint4*>(p) = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = from_f32<T>(v[i]);
  }
}

__device__ __forceinline__ uint32_t abs_bits_max8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}

// Two f32 as e4m3 codes, the first in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ void store_codes8(uint8_t* p, long long n, bool vec,
                                             const float (&v)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = e4m3x2(v[4 * i] * inv, v[4 * i + 1] * inv) |
           (e4m3x2(v[4 * i + 2] * inv, v[4 * i + 3] * inv) << 16);
  if (vec && n >= 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
  }
}

// Quantises the block that 16 consecutive lanes hold (all 32 lanes call).
__device__ __forceinline__ void quant_block16(const float (&v)[8], uint8_t* q, float* scale,
                                              long long n, bool vec, int lane) {
  uint32_t bits = max(abs_bits_max8(v), kF8LeastBits);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
  const float amax = __uint_as_float(bits);
  if (n > 0) {
    store_codes8(q, n, vec, v, __fdiv_rn(kF8Top, amax));
    if ((lane & 15) == 0) *scale = __fdiv_rn(amax, kF8Top);
  }
}

// Exact-erf GELU through erfc: no cancellation in the negative tail, whose
// blocks are scaled by their own maximum.
__device__ __forceinline__ float gelu_erfc(float x) {
  return 0.5f * x * erfcf(x * -0.70710678118654752f);
}
// g / (1 + e^-g); e^-g overflowing to +inf gives 0, the limit.
__device__ __forceinline__ float silu_div(float g) {
  return g * rcp_approx(1.0f + exp2_approx(g * -1.4426950408889634f));
}

// One half-warp per (row, block of 128 columns), U blocks at a time so that
// their loads are in flight together.
template <typename T, int ACT>
__global__ void __launch_bounds__(256)
    quant_rows_f8_kernel(const T* __restrict__ src, long long lds, int rows, int k,
                         uint8_t* __restrict__ q, long long ldq, float* __restrict__ scales,
                         RowVec vec) {
  constexpr int U = (sizeof(T) == 4 || ACT == kQuantSwiglu) ? 2 : 4;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, part = lane & 15;
  const int nb = (k + 127) / 128;
  const long long total = (long long)rows * nb;
  const long long half0 = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 4;
  const long long halves = ((long long)gridDim.x * blockDim.x) >> 4;
  // Both halves of a warp make the same number of rounds (shuffles).
  for (long long base = half0 - (half0 & 1); base < total; base += halves * U) {
    float v[U][8], g[ACT == kQuantSwiglu ? U : 1][8];
    long long row[U];
    int col[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long item = base + (half0 & 1) + u * halves;
      const bool in = item < total;
      const long long it = in ? item : 0;
      row[u] = total <= 0x7fffffff ? (long long)((uint32_t)it / (uint32_t)nb) : it / nb;
      const int blk = (int)(it - row[u] * nb);
      col[u] = in ? blk * 128 + part * 8 : k + 128;
      const T* p = src + row[u] * lds + col[u];
      load8<T>(p, (long long)k - col[u], vec.src, v[u]);
      if constexpr (ACT == kQuantSwiglu) load8<T>(p + k, (long long)k - col[u], vec.src && k % 8 == 0, g[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (ACT == kQuantGelu) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = gelu_erfc(v[u][i]);
      } else if constexpr (ACT == kQuantSwiglu) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] *= silu_div(g[u][i]);
      }
      quant_block16(v[u], q + row[u] * ldq + col[u], scales + row[u] * nb + (col[u] >> 7),
                    (long long)k - col[u], vec.q, lane);
    }
  }
}

// One CTA per 128 × 128 block: 16 half-warps hold 8 rows each.
template <typename T>
__global__ void __launch_bounds__(256)
    quant_tiles_f8_kernel(const T* __restrict__ src, long long lds, int rows, int k,
                          uint8_t* __restrict__ q, long long ldq, float* __restrict__ scales,
                          RowVec vec) {
  __shared__ uint32_t red[8];
  pdl_wait();
  pdl_trigger();
  const int nb = (k + 127) / 128;
  const long long total = (long long)((rows + 127LL) / 128) * nb;
  const int part = threadIdx.x & 15, half = threadIdx.x >> 4;
  for (long long tile = blockIdx.x; tile < total; tile += gridDim.x) {
    const long long rb = tile / nb;
    const int col = (int)(tile - rb * nb) * 128 + part * 8;
    float v[8][8];
    uint32_t bits = kF8LeastBits;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long row = rb * 128 + half + 16 * j;
      load8<T>(src + row * lds + col, row < rows ? (long long)k - col : 0, vec.src, v[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) bits = max(bits, abs_bits_max8(v[j]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = bits;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) bits = max(bits, red[w]);
    const float amax = __uint_as_float(bits);
    const float inv = __fdiv_rn(kF8Top, amax);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long long row = rb * 128 + half + 16 * j;
      if (row < rows) store_codes8(q + row * ldq + col, (long long)k - col, vec.q, v[j], inv);
    }
    if (threadIdx.x == 0) scales[tile] = __fdiv_rn(amax, kF8Top);
  }
}

// Sum over the TPR threads that share a row.
template <int TPR>
__device__ __forceinline__ float row_sum(float s, float* red) {
  s = warp_sum(s);
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    const int warp = threadIdx.x >> 5, first = warp / kWarps * kWarps;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[warp] = s;
    __syncthreads();
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += red[first + w];
  }
  return s;
}

// TPR threads per row. NV > 0: the row (k ≤ TPR · 8 · NV) stays in
// registers between the sum of squares and the quantisation. NV = 0: any k,
// x and the residual are read a second time; the sum is stored in that
// second pass, so that residual_out may be the residual or x itself.
template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256)
    rms_norm_f8_kernel(const T* x, long long ldx, const T* residual, long long ldr,
                       T* residual_out, long long ldo, const float* __restrict__ w, int rows,
                       int k, float eps, uint8_t* __restrict__ q, long long ldq,
                       float* __restrict__ scales, RowVec vec) {
  __shared__ float red[32];
  constexpr int kRows = (TPR > 256 ? TPR : 256) / TPR;  // rows per CTA
  pdl_wait();
  pdl_trigger();
  const int t = threadIdx.x % TPR, lane = threadIdx.x & 31;
  const int nb = (k + 127) / 128;
  const bool wvec = (reinterpret_cast<uintptr_t>(w) & 15) == 0;
  const long long rounds = (rows + (long long)kRows - 1) / kRows;
  for (long long r = blockIdx.x; r < rounds; r += gridDim.x) {
    const long long row = r * kRows + threadIdx.x / TPR;
    const bool in = row < rows;
    const T* xr = x + (in ? row : 0) * ldx;
    const T* rr = residual ? residual + (in ? row : 0) * ldr : nullptr;
    auto load = [&](int col, float (&h)[8]) {
      const long long n = in ? (long long)k - col : 0;
      load8<T>(xr + col, n, vec.src, h);
      if (rr) {
        float b[8];
        load8<T>(rr + col, n, vec.src, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] += b[i];
      }
    };
    auto finish = [&](int col, float (&h)[8], float inv) {
      const long long n = in ? (long long)k - col : 0;
      if (residual_out) store8<T>(residual_out + (in ? row : 0) * ldo + col, n, vec.src, h);
      float g[8];
      load8<float>(w + col, n, wvec, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = h[i] * inv * g[i];
      quant_block16(h, q + (in ? row : 0) * ldq + col, scales + (in ? row : 0) * nb + (col >> 7),
                    n, vec.q, lane);
    };
    float s = 0.0f;
    if constexpr (NV > 0) {
      float h[NV][8];
#pragma unroll
      for (int j = 0; j < NV; ++j) load((j * TPR + t) * 8, h[j]);
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(h[j][i], h[j][i], s);
      s = row_sum<TPR>(s, red);
      const float inv = 1.0f / sqrtf(s / (float)k + eps);
#pragma unroll
      for (int j = 0; j < NV; ++j) finish((j * TPR + t) * 8, h[j], inv);
    } else {
      const int steps = (int)(((long long)k + TPR * 8 - 1) / (TPR * 8));
      for (int j = 0; j < steps; ++j) {
        float h[8], a = 0.0f;
        load((j * TPR + t) * 8, h);
#pragma unroll
        for (int i = 0; i < 8; ++i) a = fmaf(h[i], h[i], a);
        s += a;
      }
      s = row_sum<TPR>(s, red);
      const float inv = 1.0f / sqrtf(s / (float)k + eps);
      for (int j = 0; j < steps; ++j) {
        float h[8];
        load((j * TPR + t) * 8, h);
        finish((j * TPR + t) * 8, h, inv);
      }
    }
  }
}

}  // namespace futon

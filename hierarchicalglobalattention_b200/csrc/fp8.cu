// 8-bit block-scaled operators: quantisation of activations and the product with an e4m3 weight.
//
//   scale[m][kb] = max |x[m][k]|, k in block kb of 128, / 448        (1 where that maximum is <= 1e-30)
//   q[m][k]      = e4m3(x[m][k] / scale[m][k / 128])                  round to nearest, ties to even
//   y[m][n]      = sum_kb scale[m][kb] * w_scale[n / 128][kb] * sum_{k in kb} q[m][k] * w[n][k]  (+ bias[n])
//
// The division is the IEEE one: a reciprocal's last-bit error would move values that lie on a rounding
// boundary of e4m3 (about one in a thousand: quotients of two bf16 numbers meet the boundaries exactly).
// A block that holds an infinity or a NaN gets a non-finite scale, so its products are NaN.
#include <cuda_fp8.h>

#include "fp8_common.cuh"

namespace hga {

// largest magnitude as an integer of the float's bits without its sign: NaN is larger than infinity,
// which is larger than every finite value, so a NaN is never lost
__device__ __forceinline__ uint32_t mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ float fp8_scale(uint32_t amax_bits) {
  const float amax = __uint_as_float(amax_bits);
  return amax <= 1e-30f ? 1.0f : __fdiv_rn(amax, 448.0f);  // NaN compares false: the scale is NaN
}

__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = Num<T>::to_f(h[i]);
  }
}

// One block of 128 channels of one row per 16 lanes, 8 channels a lane.  Bound by HBM: 2 bytes read
// and 1 written per 16-bit channel.  VEC: rows and base are 16-byte aligned (8-byte for q).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) fp8_quantize_kernel(const T* __restrict__ x, int64_t x_stride, int64_t m,
                                                           int64_t k, int kb, uint8_t* __restrict__ q, int64_t q_stride,
                                                           int64_t q_cols, float* __restrict__ scale) {
  const int lane16 = threadIdx.x & 15;
  const int64_t nblk = m * kb;
  const int64_t step = (int64_t)gridDim.x * (blockDim.x / 16);
  // every lane of a warp runs the same number of rounds (the shuffles below are warp-wide)
  const int64_t first = (int64_t)blockIdx.x * (blockDim.x / 16) + threadIdx.x / 16;
  const int64_t first0 = (int64_t)blockIdx.x * (blockDim.x / 16) + (threadIdx.x / 32) * 2;
  for (int64_t i0 = first0, i = first; i0 < nblk; i0 += step, i += step) {
    const bool live = i < nblk;
    const int64_t row = live ? i / kb : 0;
    const int64_t c0 = (live ? i - row * kb : 0) * 128 + lane16 * 8;
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 0.f;
    if (live) {
      const T* src = x + row * x_stride + c0;
      if (VEC && c0 + 8 <= k) {
        load8<T>(src, f);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + e < k) f[e] = Num<T>::to_f(src[e]);
      }
    }
    uint32_t a = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = max(a, mag_bits(f[e]));
#pragma unroll
    for (int o = 8; o; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
    if (!live) continue;
    const float s = fp8_scale(a);
    if (lane16 == 0) scale[i] = s;
    uint16_t h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = e4m3x2(__fdiv_rn(f[2 * e], s), __fdiv_rn(f[2 * e + 1], s));
    uint8_t* dst = q + row * q_stride + c0;
    if (VEC && c0 + 8 <= q_cols) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c0 + e < q_cols) dst[e] = (uint8_t)(h[e / 2] >> (8 * (e & 1)));
    }
  }
}

template <typename T>
static cudaError_t quantize_t(const void* x, int64_t x_stride, int64_t m, int64_t k, void* q, int64_t q_stride,
                              int64_t q_cols, float* scale, cudaStream_t st) {
  const int kb = (int)((k + 127) / 128);
  const int64_t nblk = m * kb;
  int64_t grid = (nblk + 15) / 16;
  if (grid > 148 * 8) grid = 148 * 8;
  const bool vec = ((uintptr_t)x % 16) == 0 && (x_stride * (int64_t)sizeof(T)) % 16 == 0 && ((uintptr_t)q % 8) == 0 &&
                   q_stride % 8 == 0;
  if (vec)
    fp8_quantize_kernel<T, true><<<(unsigned)grid, 256, 0, st>>>((const T*)x, x_stride, m, k, kb, (uint8_t*)q, q_stride,
                                                                 q_cols, scale);
  else
    fp8_quantize_kernel<T, false><<<(unsigned)grid, 256, 0, st>>>((const T*)x, x_stride, m, k, kb, (uint8_t*)q,
                                                                  q_stride, q_cols, scale);
  return cudaGetLastError();
}

// q_cols >= k columns are written: channels past k are zeros
cudaError_t launch_fp8_quantize(int dtype, const void* x, int64_t x_stride, int64_t m, int64_t k, void* q,
                                int64_t q_stride, int64_t q_cols, float* scale, cudaStream_t st) {
  switch (dtype) {
    case HGA_DTYPE_F32: return quantize_t<float>(x, x_stride, m, k, q, q_stride, q_cols, scale, st);
    case HGA_DTYPE_BF16: return quantize_t<__nv_bfloat16>(x, x_stride, m, k, q, q_stride, q_cols, scale, st);
    case HGA_DTYPE_F16: return quantize_t<__half>(x, x_stride, m, k, q, q_stride, q_cols, scale, st);
  }
  return cudaErrorInvalidValue;
}

// ---- product ------------------------------------------------------------------------------------
__device__ __forceinline__ float e4m3_f(uint8_t v) {
  __nv_fp8_e4m3 h;
  h.__x = v;
  return (float)h;
}

// 64 tokens x 64 output features per CTA, one block of 128 channels at a time through shared memory,
// 4 x 4 outputs a thread.
template <typename T>
__global__ void __launch_bounds__(256) fp8_product_kernel(const uint8_t* __restrict__ q, int64_t q_stride,
                                                          const float* __restrict__ xs, const uint8_t* __restrict__ w,
                                                          int64_t w_stride, const float* __restrict__ ws, int64_t ws_stride,
                                                          const T* __restrict__ bias, T* __restrict__ out,
                                                          int64_t out_stride, int64_t m, int64_t n, int64_t k, int kb) {
  __shared__ float sa[64][33], sb[64][33];
  const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int b = 0; b < kb; ++b) {
    float part[4][4] = {};
    for (int k0 = b * 128; k0 < (b + 1) * 128; k0 += 32) {
      for (int i = threadIdx.x; i < 64 * 32; i += 256) {
        const int r = i / 32, c = i % 32;
        sa[r][c] = (m0 + r < m && k0 + c < k) ? e4m3_f(q[(m0 + r) * q_stride + k0 + c]) : 0.f;
        sb[r][c] = (n0 + r < n && k0 + c < k) ? e4m3_f(w[(n0 + r) * w_stride + k0 + c]) : 0.f;
      }
      __syncthreads();
      for (int c = 0; c < 32; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[i][j] = fmaf(sa[ty * 4 + i][c], sb[tx + 16 * j][c], part[i][j]);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t r = m0 + ty * 4 + i, c = n0 + tx + 16 * j;
        if (r < m && c < n) acc[i][j] = fmaf(part[i][j], xs[r * kb + b] * ws[c / 128 * ws_stride + b], acc[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = m0 + ty * 4 + i, c = n0 + tx + 16 * j;
      if (r < m && c < n) out[r * out_stride + c] = Num<T>::from_f(acc[i][j] + (bias ? Num<T>::to_f(bias[c]) : 0.f));
    }
}

int64_t fp8_linear_workspace(const Fp8Linear& a) {
  const int64_t kb = (a.k + 127) / 128;
  return a.x_dtype == HGA_DTYPE_E4M3 ? 0 : a.m * kb * 128 + a.m * kb * 4;
}

template <typename T>
static cudaError_t product_t(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, cudaStream_t st) {
  const int kb = (int)((a.k + 127) / 128);
  fp8_product_kernel<T><<<dim3((unsigned)((a.n + 63) / 64), (unsigned)((a.m + 63) / 64)), 256, 0, st>>>(
      (const uint8_t*)q, q_stride, xs, (const uint8_t*)a.w, a.w_stride, a.w_scale, a.ws_stride, (const T*)a.bias,
      (T*)a.out, a.out_stride, a.m, a.n, a.k, kb);
  return cudaGetLastError();
}

cudaError_t launch_fp8_linear(const Fp8Linear& a, cudaStream_t st) {
  const void* q = a.x;
  int64_t q_stride = a.x_stride;
  const float* xs = a.x_scale;
  if (a.x_dtype != HGA_DTYPE_E4M3) {
    const int64_t kb = (a.k + 127) / 128;
    q_stride = kb * 128;
    float* s = (float*)((char*)a.workspace + a.m * q_stride);
    cudaError_t e = launch_fp8_quantize(a.x_dtype, a.x, a.x_stride, a.m, a.k, a.workspace, q_stride, q_stride, s, st);
    if (e != cudaSuccess) return e;
    q = a.workspace;
    xs = s;
  }
  switch (a.out_dtype) {
    case HGA_DTYPE_F32: return product_t<float>(a, q, q_stride, xs, st);
    case HGA_DTYPE_BF16: return product_t<__nv_bfloat16>(a, q, q_stride, xs, st);
    case HGA_DTYPE_F16: return product_t<__half>(a, q, q_stride, xs, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace hga

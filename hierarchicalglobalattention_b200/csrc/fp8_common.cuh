// Shared by the 8-bit block-scaled kernels: the call's arguments, and the quantisation of one value block.
#pragma once

#include "hga_common.cuh"

namespace hga {

// Arguments of one hga_fp8_linear call.
struct Fp8Linear {
  int64_t m, n, k;
  const void* x;
  int64_t x_stride;
  int x_dtype;
  const float* x_scale;
  const void* w;
  int64_t w_stride;
  const float* w_scale;
  int64_t ws_stride;
  const void* bias;
  void* out;
  int64_t out_stride;
  int out_dtype;
  void* workspace;
};

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

// 8 consecutive elements as fp32; p 16-byte aligned
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

// The scale of a block of 128 channels held 8 a lane by 16 neighbouring lanes (all 32 lanes call), and the
// lane's 8 e4m3 values.
__device__ __forceinline__ float fp8_block(const float (&f)[8], uint2& v) {
  uint32_t a = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) a = max(a, mag_bits(f[e]));
#pragma unroll
  for (int o = 8; o; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
  const float s = fp8_scale(a);
  uint16_t h[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = e4m3x2(__fdiv_rn(f[2 * e], s), __fdiv_rn(f[2 * e + 1], s));
  v = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
  return s;
}

cudaError_t launch_fp8_quantize(int dtype, const void* x, int64_t x_stride, int64_t m, int64_t k, void* q,
                                int64_t q_stride, int64_t q_cols, float* scale, cudaStream_t st);

// The products on the tensor cores.  q [m][k] e4m3 and w: 16-byte aligned bases and row strides.
cudaError_t launch_fp8_tiles(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, const void* w,
                             int64_t w_stride, cudaStream_t st);
// Few rows: quantises x itself (x_dtype not E4M3) or takes q / xs.
bool fp8_rows_fused(const Fp8Linear& a);
bool fp8_rows_better(const Fp8Linear& a);
cudaError_t launch_fp8_rows(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, const void* w,
                            int64_t w_stride, cudaStream_t st);

}  // namespace hga

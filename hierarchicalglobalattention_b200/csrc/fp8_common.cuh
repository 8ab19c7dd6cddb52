// Shared by the 8-bit block-scaled kernels: the call's arguments, and the quantisation of one value block.
#pragma once

#include "fp32x2.cuh"
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

__device__ __forceinline__ float fp8_scale(float amax) {
  return amax <= 1e-30f ? 1.0f : __fdiv_rn(amax, 448.0f);  // NaN compares false: the scale is NaN
}

__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// 8 consecutive channels of a row as they are in memory.
template <typename T> struct Raw8 {
  uint4 u;
};
template <> struct Raw8<float> {
  float4 a, b;
};
template <typename T>
__device__ __forceinline__ Raw8<T> raw_zero() {
  Raw8<T> r;
  if constexpr (sizeof(T) == 4) r.a = r.b = make_float4(0.f, 0.f, 0.f, 0.f);
  else r.u = make_uint4(0u, 0u, 0u, 0u);
  return r;
}
// vec: p is 16-byte aligned; n of the 8 channels exist
template <typename T>
__device__ __forceinline__ Raw8<T> raw_load(const T* p, bool vec, int64_t n) {
  Raw8<T> r = raw_zero<T>();
  if (vec && n >= 8) {
    if constexpr (sizeof(T) == 4) {
      r.a = reinterpret_cast<const float4*>(p)[0];
      r.b = reinterpret_cast<const float4*>(p)[1];
    } else {
      r.u = *reinterpret_cast<const uint4*>(p);
    }
  } else {
    T t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = e < n ? p[e] : Num<T>::from_f(0.f);
    if constexpr (sizeof(T) == 4) {
      r.a = make_float4(t[0], t[1], t[2], t[3]);
      r.b = make_float4(t[4], t[5], t[6], t[7]);
    } else {
      r.u = *reinterpret_cast<const uint4*>(t);
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void raw_floats(const Raw8<T>& r, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = r.a.x; f[1] = r.a.y; f[2] = r.a.z; f[3] = r.a.w;
    f[4] = r.b.x; f[5] = r.b.y; f[6] = r.b.z; f[7] = r.b.w;
  } else {
    const T* h = reinterpret_cast<const T*>(&r.u);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = Num<T>::to_f(h[i]);
  }
}
// Largest magnitude of the 16 lanes' channels as an integer (fp32 bits, or 16-bit bits), see mag_bits.
template <typename T>
__device__ __forceinline__ float raw_amax(const Raw8<T>& r) {
  if constexpr (sizeof(T) == 4) {
    uint32_t a = max(max(max(mag_bits(r.a.x), mag_bits(r.a.y)), max(mag_bits(r.a.z), mag_bits(r.a.w))),
                     max(max(mag_bits(r.b.x), mag_bits(r.b.y)), max(mag_bits(r.b.z), mag_bits(r.b.w))));
#pragma unroll
    for (int o = 8; o; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
    return __uint_as_float(a);
  } else {
    uint32_t a = __vmaxu2(__vmaxu2(r.u.x & 0x7fff7fffu, r.u.y & 0x7fff7fffu),
                          __vmaxu2(r.u.z & 0x7fff7fffu, r.u.w & 0x7fff7fffu));
#pragma unroll
    for (int o = 8; o; o >>= 1) a = __vmaxu2(a, __shfl_xor_sync(0xffffffffu, a, o));
    const uint16_t h = (uint16_t)max(a & 0xffffu, a >> 16);
    return Num<T>::to_f(*reinterpret_cast<const T*>(&h));
  }
}

// e4m3 of the quotients f / s.  A quotient from the correctly rounded reciprocal by one exact remainder
// (Markstein 1990: y = f r, q = y + (f - y s) r), three paired operations for two channels, where a plain
// division takes about ten each.  It may differ from the IEEE quotient only where that lies within 2^-46
// (relative) of the middle between two neighbouring floats; a quotient that is exactly on a boundary of
// e4m3 comes out exactly.
__device__ __forceinline__ uint2 fp8_quotients(const float (&f)[8], float s, float inv) {
  uint16_t h[4];
  const uint64_t r2 = f32x2(inv, inv), ns2 = f32x2(-s, -s);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint64_t f2 = f32x2(f[2 * e], f[2 * e + 1]);
    const uint64_t y = f32x2_mul(f2, r2);
    float lo, hi;
    f32x2_get(f32x2_fma(f32x2_fma(y, ns2, f2), r2, y), lo, hi);
    h[e] = e4m3x2(lo, hi);
  }
  return make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
}
// The same by divisions: for a scale that is not finite, where the remainder is no number.
static __device__ __noinline__ uint2 fp8_divisions(float a, float b, float c, float d, float e, float f, float g, float h,
                                                   float s) {
  return make_uint2(e4m3x2(__fdiv_rn(a, s), __fdiv_rn(b, s)) | (uint32_t)e4m3x2(__fdiv_rn(c, s), __fdiv_rn(d, s)) << 16,
                    e4m3x2(__fdiv_rn(e, s), __fdiv_rn(f, s)) | (uint32_t)e4m3x2(__fdiv_rn(g, s), __fdiv_rn(h, s)) << 16);
}
__device__ __forceinline__ uint2 fp8_divisions(const float (&f)[8], float s) {
  return fp8_divisions(f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7], s);
}

// The scale of a block of 128 channels held 8 a lane by 16 neighbouring lanes (all 32 lanes call), and the
// lane's 8 e4m3 values.
template <typename T>
__device__ __forceinline__ float fp8_block(const Raw8<T>& r, uint2& v) {
  const float s = fp8_scale(raw_amax<T>(r));
  float f[8];
  raw_floats<T>(r, f);
  v = s < INFINITY ? fp8_quotients(f, s, __frcp_rn(s)) : fp8_divisions(f, s);
  return s;
}

cudaError_t launch_fp8_quantize(int dtype, const void* x, int64_t x_stride, int64_t m, int64_t k, void* q,
                                int64_t q_stride, int64_t q_cols, float* scale, int64_t scale_stride, cudaStream_t st);

// The products on the tensor cores.  q [m][k] e4m3 and w: 16-byte aligned bases and row strides.
cudaError_t launch_fp8_tiles(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, int64_t xs_stride,
                             const void* w, int64_t w_stride, cudaStream_t st);
// Few rows: quantises x itself (x_dtype not E4M3) or takes q / xs.
bool fp8_rows_fused(const Fp8Linear& a);
bool fp8_rows_better(const Fp8Linear& a);
cudaError_t launch_fp8_rows(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, int64_t xs_stride,
                            const void* w, int64_t w_stride, cudaStream_t st);

}  // namespace hga

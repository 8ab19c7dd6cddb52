// 4-bit KV record: pack, unpack, and the portable attention over it (any type, head_dim a multiple of 64).
// The record's format is in kv4_common.cuh.
#include <cooperative_groups.h>

#include <type_traits>

#include "fp32x2.cuh"
#include "kv4_common.cuh"

namespace hga {

namespace cg = cooperative_groups;

HGA_DEVICE_ERROR_WORD(g_kv4_error, kv4_error_status)

// ---- pack and unpack ------------------------------------------------------------------------------
// 16 channels of one token as they are in memory, their extremes, and their values as pairs of fp32.
template <typename T> struct Row16 {
  uint4 u[2];
};
template <> struct Row16<float> {
  uint4 u[4];
};
template <typename T>
__device__ __forceinline__ Row16<T> row16_load(const T* p, bool live) {
  Row16<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) r.u[i] = live ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0u, 0u, 0u, 0u);
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// a NaN among the channels makes both extremes NaN
template <typename T>
__device__ __forceinline__ void row16_extremes(const Row16<T>& r, float& lo, float& hi) {
  if constexpr (sizeof(T) == 4) {
    const float* f = reinterpret_cast<const float*>(r.u);
    lo = hi = f[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) {
      lo = min_nan(lo, f[i]);
      hi = max_nan(hi, f[i]);
    }
  } else {
    using V2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const V2* v = reinterpret_cast<const V2*>(r.u);
    V2 l = v[0], h = v[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      l = __hmin2_nan(l, v[i]);
      h = __hmax2_nan(h, v[i]);
    }
    lo = min_nan(Num<T>::to_f(l.x), Num<T>::to_f(l.y));
    hi = max_nan(Num<T>::to_f(h.x), Num<T>::to_f(h.y));
  }
}
template <typename T>
__device__ __forceinline__ void row16_pair(const Row16<T>& r, int i, float& a, float& b) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(r.u);
  if constexpr (sizeof(T) == 4) {
    a = __uint_as_float(w[2 * i]);
    b = __uint_as_float(w[2 * i + 1]);
  } else if constexpr (std::is_same<T, __half>::value) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(w + i));
    a = f.x;
    b = f.y;
  } else {
    a = __uint_as_float(w[i] << 16);
    b = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// What quantising one token's block needs: minimum, scale and its reciprocal; the (scale, min) word.
struct Kv4Block {
  float m, s, inv;
  uint32_t word;
};
template <typename T>
__device__ __forceinline__ Kv4Block kv4_block(float lo, float hi) {
  using MT = typename Kv4Meta<T>::type;
  const float odd = (lo - lo) + (hi - hi);  // 0, or NaN for a block with an infinity or a NaN
  const MT pair[2] = {Num<MT>::from_f(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f) + odd), Num<MT>::from_f(lo + odd)};
  Kv4Block b;
  b.s = Num<MT>::to_f(pair[0]);
  b.m = Num<MT>::to_f(pair[1]);
  b.inv = __frcp_rn(b.s);
  b.word = *reinterpret_cast<const uint32_t*>(pair);
  return b;
}
// The codes of 16 channels, two to a word: codes[i] = n(2i) | n(2i + 1) << 16.  The quotient (x - m) / s comes
// from the reciprocal and one exact remainder (Markstein 1990); adding 1.5 * 2^23 rounds it to an integer,
// ties to even, in the low bits of the float.
template <typename T>
__device__ __forceinline__ void kv4_codes(const Row16<T>& r, const Kv4Block& b, uint32_t (&codes)[8]) {
  // a scale that is normal in its type is within 2^-9 of the exact one and the minimum of a 16-bit cache is
  // exact, so its quotients round to 0..15 by themselves
  const bool plain = sizeof(T) == 2 && b.s >= (std::is_same<T, __half>::value ? 6.104e-5f : 1e-30f) && b.s < INFINITY;
  const uint64_t nm = f32x2(-b.m, -b.m), inv = f32x2(b.inv, b.inv), ns = f32x2(-b.s, -b.s);
  const uint64_t big = f32x2(12582912.f, 12582912.f), one = f32x2(1.f, 1.f);
  if (plain) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x0, x1;
      row16_pair<T>(r, i, x0, x1);
      const uint64_t d = f32x2_fma(f32x2(x0, x1), one, nm);
      const uint64_t y = f32x2_mul(d, inv);
      const uint64_t q = f32x2_fma(f32x2_fma(f32x2_fma(y, ns, d), inv, y), one, big);
      float q0, q1;
      f32x2_get(q, q0, q1);
      codes[i] = __byte_perm(__float_as_uint(q0), __float_as_uint(q1), 0x5410);
    }
  } else {
    const bool usable = b.s > 0.f && b.s < INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x0, x1;
      row16_pair<T>(r, i, x0, x1);
      const float n0 = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x0, b.m), b.s)), 0.f), 15.f);
      const float n1 = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x1, b.m), b.s)), 0.f), 15.f);
      codes[i] = usable ? (uint32_t)(int)n0 | (uint32_t)(int)n1 << 16 : 0u;
    }
  }
}
// 4 x 4 transposition between 4 neighbouring lanes: w[k] of lane j becomes w[j] of lane k.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4], int j) {
#pragma unroll
  for (int s = 1; s < 4; s <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i & s) continue;
      const bool up = j & s;
      const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? w[i] : w[i + s], s);
      if (up) w[i] = got; else w[i + s] = got;
    }
}

constexpr int kPackWarps = 8;

// K: a warp takes a unit, four 16 x 16 tiles (64 channels) at a time; lane 4 g + j reads tokens g and g + 8
// of tile j (two times 32 bytes), which is all that the words of lanes 4 g .. 4 g + 3 of that tile hold, and a
// 4 x 4 transposition between neighbours brings each lane the four words that it stores as 16 bytes.
// V: a half warp takes 64 channels of a unit; lane 4 c + j reads tokens 2c, 2c + 1, 2c + 8, 2c + 9 of tile j.
// A block of 32 channels is two neighbouring lanes.  Bound by HBM; codes never pass through shared memory
// (byte stores and nibble gathers there took three times as long).  131069 rows of 4 KV heads, K and V: 75 us
// for 268 MB read and 84 written, 4.7 TB/s.
template <typename T, int DH>
__global__ void __launch_bounds__(kPackWarps * 32) kv4_pack_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                                   int64_t bk, int64_t rows, int64_t cap,
                                                                   uint8_t* __restrict__ rec_k, uint8_t* __restrict__ rec_v,
                                                                   int64_t unit_cap, int64_t unit0) {
  constexpr int QUADS = DH / 64, NB = DH / 32;
  const int lane = threadIdx.x & 31, j = lane & 3;
  const int64_t units = (rows + 15) / 16, n_k = bk * units, items_v = bk * units * QUADS, n_v = (items_v + 1) / 2;
  for (int64_t w = (int64_t)blockIdx.x * kPackWarps + (threadIdx.x >> 5); w < n_k + n_v; w += (int64_t)gridDim.x * kPackWarps) {
    if (w < n_k) {
      const int64_t head = w / units, u = w - head * units;
      const T* src = k + (head * cap + u * 16) * DH + j * 16;
      uint8_t* dst = rec_k + (head * unit_cap + unit0 + u) * kv4_unit_bytes(DH);
      uint32_t* meta = reinterpret_cast<uint32_t*>(dst + 8 * DH);
      const int64_t left = rows - u * 16;
      const int g = lane >> 2;
      Row16<T> x[QUADS][2];
#pragma unroll
      for (int quad = 0; quad < QUADS; ++quad)
#pragma unroll
        for (int r = 0; r < 2; ++r) x[quad][r] = row16_load<T>(src + (int64_t)(g + 8 * r) * DH + quad * 64, g + 8 * r < left);
#pragma unroll
      for (int quad = 0; quad < QUADS; ++quad) {
        uint32_t word[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float lo, hi;
          row16_extremes<T>(x[quad][r], lo, hi);
          lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, 1));
          hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, 1));
          const Kv4Block b = kv4_block<T>(lo, hi);
          if ((j & 1) == r) meta[(g + 8 * r) * NB + quad * 2 + (j >> 1)] = b.word;
          uint32_t n[8];
          kv4_codes<T>(x[quad][r], b, n);
          // channels 2c, 2c + 1 (pair c) and 8 + 2c, 9 + 2c (pair 4 + c): nibbles r, r + 4 and r + 2, r + 6
#pragma unroll
          for (int c = 0; c < 4; ++c) word[c] += ((n[c] & 0x000f000fu) << (4 * r)) + ((n[4 + c] & 0x000f000fu) << (4 * r + 8));
        }
        transpose4(word, j);
        *reinterpret_cast<uint4*>(dst + (quad * 32 + lane) * 16) = make_uint4(word[0], word[1], word[2], word[3]);
      }
    } else {
      const int64_t item = (w - n_k) * 2 + (lane >> 4);
      const bool on = item < items_v;
      const int64_t it = on ? item : 0, unit = it / QUADS;
      const int quad = (int)(it - unit * QUADS), c = (lane >> 2) & 3;
      const int64_t head = unit / units, u = unit - head * units;
      const T* src = v + (head * cap + u * 16) * DH + quad * 64 + j * 16;
      uint8_t* dst = rec_v + (head * unit_cap + unit0 + u) * kv4_unit_bytes(DH);
      uint32_t* meta = reinterpret_cast<uint32_t*>(dst + 8 * DH);
      const int64_t left = rows - u * 16;
      Row16<T> x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = 2 * c + (i & 1) + 8 * (i >> 1);
        x[i] = row16_load<T>(src + (int64_t)tok * DH, on && tok < left);
      }
      uint32_t word[8];
#pragma unroll
      for (int g = 0; g < 8; ++g) word[g] = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = 2 * c + (i & 1) + 8 * (i >> 1);
        float lo, hi;
        row16_extremes<T>(x[i], lo, hi);
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, 1));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, 1));
        const Kv4Block b = kv4_block<T>(lo, hi);
        if (on && (j & 1) == (i & 1)) meta[tok * NB + quad * 2 + (j >> 1)] = b.word;
        uint32_t n[8];
        kv4_codes<T>(x[i], b, n);
        // token: nibble 4 * (tok % 2) + 2 * (tok / 8); channel g and g + 8 (pairs g / 2 and 4 + g / 2): + 0, + 1
        constexpr uint32_t kLow = 0xfu;
        const int sh = 16 * (i & 1) + 8 * (i >> 1);
#pragma unroll
        for (int g = 0; g < 8; ++g)
          word[g] += ((n[g >> 1] >> (16 * (g & 1)) & kLow) << sh) + ((n[4 + (g >> 1)] >> (16 * (g & 1)) & kLow) << (sh + 4));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t t[4] = {word[4 * h], word[4 * h + 1], word[4 * h + 2], word[4 * h + 3]};
        transpose4(t, j);  // channel row g = 4 h + j, tiles 0..3
        if (on) *reinterpret_cast<uint4*>(dst + (quad * 32 + 4 * (4 * h + j) + c) * 16) = make_uint4(t[0], t[1], t[2], t[3]);
      }
    }
  }
}

// 16 channels of a token from their codes as fp32 (scale * code + min: the product is exact).
template <typename T>
__device__ __forceinline__ void row16_store(T* p, const float (&n)[16], uint32_t word) {
  using MT = typename Kv4Meta<T>::type;
  const MT* pair = reinterpret_cast<const MT*>(&word);
  const float s = Num<MT>::to_f(pair[0]), m = Num<MT>::to_f(pair[1]);
  const uint64_t s2 = f32x2(s, s), m2 = f32x2(m, m);
  T y[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float a, b;
    f32x2_get(f32x2_fma(f32x2(n[2 * i], n[2 * i + 1]), s2, m2), a, b);
    y[2 * i] = Num<T>::from_f(a);
    y[2 * i + 1] = Num<T>::from_f(b);
  }
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(y)[i];
}
__device__ __forceinline__ float nibble(uint32_t w, int i) {
  return __uint_as_float((w >> (4 * i) & 15u) | 0x4b000000u) - 8388608.f;
}

// The values of rows [0, rows): kv4_pack_kernel backwards.  The same rows back: 60 us, 5.9 TB/s.
template <typename T, int DH>
__global__ void __launch_bounds__(kPackWarps * 32) kv4_unpack_kernel(const uint8_t* __restrict__ rec_k,
                                                                     const uint8_t* __restrict__ rec_v, int64_t unit_cap,
                                                                     int64_t unit0, int64_t bk, int64_t rows,
                                                                     T* __restrict__ k, T* __restrict__ v, int64_t cap) {
  constexpr int QUADS = DH / 64, NB = DH / 32;
  const int lane = threadIdx.x & 31, j = lane & 3;
  const int64_t units = (rows + 15) / 16, n_k = bk * units, items_v = bk * units * QUADS, n_v = (items_v + 1) / 2;
  for (int64_t w = (int64_t)blockIdx.x * kPackWarps + (threadIdx.x >> 5); w < n_k + n_v; w += (int64_t)gridDim.x * kPackWarps) {
    if (w < n_k) {
      const int64_t head = w / units, u = w - head * units;
      const uint8_t* src = rec_k + (head * unit_cap + unit0 + u) * kv4_unit_bytes(DH);
      const uint32_t* meta = reinterpret_cast<const uint32_t*>(src + 8 * DH);
      T* dst = k + (head * cap + u * 16) * DH + j * 16;
      const int64_t left = rows - u * 16;
      const int g = lane >> 2;
      uint4 q4[QUADS];
      uint32_t mw[QUADS][2];
#pragma unroll
      for (int quad = 0; quad < QUADS; ++quad) {
        q4[quad] = *reinterpret_cast<const uint4*>(src + (quad * 32 + lane) * 16);
#pragma unroll
        for (int r = 0; r < 2; ++r) mw[quad][r] = meta[(g + 8 * r) * NB + quad * 2 + (j >> 1)];
      }
#pragma unroll
      for (int quad = 0; quad < QUADS; ++quad) {
        uint32_t word[4] = {q4[quad].x, q4[quad].y, q4[quad].z, q4[quad].w};
        transpose4(word, j);  // tile j: the words of lanes 4 g + c
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float n[16];
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              n[2 * c + e] = nibble(word[c], r + 4 * e);
              n[8 + 2 * c + e] = nibble(word[c], r + 2 + 4 * e);
            }
          if (g + 8 * r < left) row16_store<T>(dst + (int64_t)(g + 8 * r) * DH + quad * 64, n, mw[quad][r]);
        }
      }
    } else {
      const int64_t item = (w - n_k) * 2 + (lane >> 4);
      const bool on = item < items_v;
      const int64_t it = on ? item : 0, unit = it / QUADS;
      const int quad = (int)(it - unit * QUADS), c = (lane >> 2) & 3;
      const int64_t head = unit / units, u = unit - head * units;
      const uint8_t* src = rec_v + (head * unit_cap + unit0 + u) * kv4_unit_bytes(DH);
      const uint32_t* meta = reinterpret_cast<const uint32_t*>(src + 8 * DH);
      T* dst = v + (head * cap + u * 16) * DH + quad * 64 + j * 16;
      const int64_t left = rows - u * 16;
      uint32_t word[8], mw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) mw[i] = meta[(2 * c + (i & 1) + 8 * (i >> 1)) * NB + quad * 2 + (j >> 1)];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 q4 = *reinterpret_cast<const uint4*>(src + (quad * 32 + 4 * (4 * h + j) + c) * 16);
        uint32_t t[4] = {q4.x, q4.y, q4.z, q4.w};
        transpose4(t, j);  // tile j: channel rows 4 h + 0..3
#pragma unroll
        for (int e = 0; e < 4; ++e) word[4 * h + e] = t[e];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = 2 * c + (i & 1) + 8 * (i >> 1), nib = 4 * (i & 1) + 2 * (i >> 1);
        float n[16];
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          n[g] = nibble(word[g], nib);
          n[8 + g] = nibble(word[g], nib + 1);
        }
        if (on && tok < left) row16_store<T>(dst + (int64_t)tok * DH, n, mw[i]);
      }
    }
  }
}

static unsigned pack_grid(int64_t units, int dh) {
  const int64_t ctas = (units + (units * (dh / 64) + 1) / 2 + kPackWarps - 1) / kPackWarps;
  return (unsigned)(ctas < 148 * 64 ? ctas : 148 * 64);
}

#define HGA_KV4_DH(TT, CALL)                       \
  switch (dh) {                                    \
    case 64: { constexpr int DH = 64; using T = TT; CALL; } break;   \
    case 128: { constexpr int DH = 128; using T = TT; CALL; } break; \
    case 192: { constexpr int DH = 192; using T = TT; CALL; } break; \
    case 256: { constexpr int DH = 256; using T = TT; CALL; } break; \
    default: return cudaErrorInvalidValue;         \
  }
#define HGA_KV4_DISPATCH(CALL)                                \
  switch (dtype) {                                            \
    case HGA_DTYPE_F32: HGA_KV4_DH(float, CALL) break;        \
    case HGA_DTYPE_BF16: HGA_KV4_DH(__nv_bfloat16, CALL) break; \
    case HGA_DTYPE_F16: HGA_KV4_DH(__half, CALL) break;       \
    default: return cudaErrorInvalidValue;                    \
  }

cudaError_t launch_kv4_pack(int dtype, int dh, int64_t bk, int64_t rows, const void* k, const void* v, int64_t cap,
                            void* rec_k, void* rec_v, int64_t unit_cap, int64_t unit0, cudaStream_t st) {
  const unsigned grid = pack_grid(bk * ((rows + 15) / 16), dh);
  HGA_KV4_DISPATCH((kv4_pack_kernel<T, DH><<<grid, kPackWarps * 32, 0, st>>>(
      (const T*)k, (const T*)v, bk, rows, cap, (uint8_t*)rec_k, (uint8_t*)rec_v, unit_cap, unit0)))
  return cudaGetLastError();
}

cudaError_t launch_kv4_unpack(int dtype, int dh, int64_t bk, int64_t rows, const void* rec_k, const void* rec_v,
                              int64_t unit_cap, int64_t unit0, void* k, void* v, int64_t cap, cudaStream_t st) {
  const unsigned grid = pack_grid(bk * ((rows + 15) / 16), dh);
  HGA_KV4_DISPATCH((kv4_unpack_kernel<T, DH><<<grid, kPackWarps * 32, 0, st>>>(
      (const uint8_t*)rec_k, (const uint8_t*)rec_v, unit_cap, unit0, bk, rows, (T*)k, (T*)v, cap)))
  return cudaGetLastError();
}

// ---- attention, portable ------------------------------------------------------------------------
constexpr int kPortWarps = 4;

// The rows of a CTA, its units in shared memory as fp32 (K and V, a warp's own), the rows' queries (afterwards the
// CTA's result) and softmax states.
template <int DH, int R> struct PortSmem {
  static constexpr int LD = DH + 4;
  static constexpr int kUnit = 2 * kKv4Unit * LD;             // floats of a warp
  static constexpr int kRows = kPortWarps * kUnit;            // [R][DH]
  static constexpr int kMax = kRows + R * DH, kSum = kMax + (kPortWarps + 1) * R;  // [warps, then the CTA][R]
  static constexpr int kTotal = (kSum + (kPortWarps + 1) * R) * 4;
};

template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const T* t = reinterpret_cast<const T*>(&w);
    return make_float4(Num<T>::to_f(t[0]), Num<T>::to_f(t[1]), Num<T>::to_f(t[2]), Num<T>::to_f(t[3]));
  }
}
template <typename MT>
__device__ __forceinline__ float2 scale_min(const uint8_t* meta, int pair) {
  const uint32_t w = reinterpret_cast<const uint32_t*>(meta)[pair];
  const MT* t = reinterpret_cast<const MT*>(&w);
  return make_float2(Num<MT>::to_f(t[0]), Num<MT>::to_f(t[1]));
}

// Any type and head_dim, fp32 throughout.  A cluster serves up to R rows of one query head; the units of 16 keys
// (slots and the head's own opened groups) are dealt to its warps, each of which decodes a unit into
// shared memory, scores a key with a lane pair and keeps its own online softmax of all R rows in registers.
// The partial results are joined as in the matrix kernel: warps, then CTAs, in a fixed order.
// Bound by issue (decoding into fp32 and plain FMAs) and, for one sequence, by latency: one token of 32 heads
// over 4 at 32768 in fp32 13.6 us, a block of 64 rows 262 us; with the units one after the other in one CTA per
// head and bytes decoded one by one 409 and 835.
template <typename T, int DH, int R>
__global__ void __launch_bounds__(kPortWarps * 32) attend_kv4_kernel(
    hga_params p, int L, const T* __restrict__ q, const int32_t* __restrict__ seq_pos, const T* __restrict__ hot_k,
    const T* __restrict__ hot_v, int64_t hot_cap, const uint8_t* rec_k, const uint8_t* rec_v, int64_t unit_cap,
    const int32_t* __restrict__ open_gid, const int32_t* __restrict__ open_t0, int Kg, T* __restrict__ out) {
  using MT = typename Kv4Meta<T>::type;
  using S = PortSmem<DH, R>;
  constexpr int LD = S::LD, VD = DH / 32;
  extern __shared__ __align__(16) float port_smem[];
  const int tiles = (L + R - 1) / R;
  const int rank = blockIdx.x, splits = gridDim.x, h = blockIdx.y, b = blockIdx.z / tiles, row0 = blockIdx.z % tiles * R;
  const int H = p.nhead, KVH = p.kv_heads, C = p.chunk_size, U = p.group_size / kKv4Unit;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nrows = L - row0 < R ? L - row0 : R;
  const int pos = seq_pos[b];
  const int kf = p.keep_first > 0 ? p.keep_first : 0, kl = p.keep_last > 0 ? p.keep_last : 0;
  const size_t bh = (size_t)b * H + h, bk = (size_t)b * KVH + h / (H / KVH);
  T* o_base = out + (bh * L + row0) * DH;
  const int n_closed = pos / C, c0 = pos % C;
  if (pos < 0 || c0 + L > C || (int64_t)(kf + kl + 1) * C > hot_cap) {
    if (tid == 0) atomicCAS(&g_kv4_error, 0, kErrBoundsAttendKv4);
    if (rank == 0)
      for (int i = tid; i < nrows * DH; i += blockDim.x) o_base[i] = Num<T>::from_f(0.f);
    return;  // the whole cluster
  }
  float* qs = port_smem + S::kRows;
  float* ks = port_smem + warp * S::kUnit;
  float* vs = ks + kKv4Unit * LD;
  for (int i = tid; i < R * DH; i += blockDim.x) qs[i] = i / DH < nrows ? Num<T>::to_f(q[(bh * L + row0) * DH + i]) : 0.f;
  __syncthreads();
  float o[R][VD], m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int d = 0; d < VD; ++d) o[r][d] = 0.f;
  }
  int f_hi, l_lo;
  windows(n_closed, kf, kl, f_hi, l_lo);
  const int wu = C / kKv4Unit, n_first = f_hi * wu, n_win = n_first + (n_closed - l_lo) * wu;
  const int nact = c0 + row0 + nrows, n_hot = n_win + (nact + kKv4Unit - 1) / kKv4Unit, n_all = n_hot + Kg * U;
  for (int i = rank * kPortWarps + warp; i < n_all; i += splits * kPortWarps) {
    // key j of the unit is visible to row t iff j < count and t >= tmin + causal * j
    int tmin = 0, causal = 0, count = kKv4Unit;
    __syncwarp();  // the last unit has been read
    if (i < n_hot) {
      int64_t row;
      if (i < n_first) {
        row = (int64_t)i * kKv4Unit;
      } else if (i < n_win) {
        row = (int64_t)(kf + (l_lo + (i - n_first) / wu) % (kl > 0 ? kl : 1)) * C + (i - n_first) % wu * kKv4Unit;
      } else {
        const int act = (i - n_win) * kKv4Unit;
        row = (int64_t)(kf + kl) * C + act;
        tmin = act - c0;
        causal = 1;
        if (nact - act < count) count = nact - act;
      }
      const size_t base = (bk * hot_cap + row) * DH;
#pragma unroll 4
      for (int x = lane; x < kKv4Unit * DH / 4; x += 32) {
        const int tok = x / (DH / 4), c4 = x % (DH / 4) * 4;
        const bool in = tok < count;  // rows past the block hold an earlier sequence's values
        *reinterpret_cast<float4*>(ks + tok * LD + c4) = in ? load4<T>(hot_k + base + x * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
        *reinterpret_cast<float4*>(vs + tok * LD + c4) = in ? load4<T>(hot_v + base + x * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    } else {
      const int j = (i - n_hot) / U, gid = open_gid[bh * Kg + j];
      tmin = open_t0[bh * Kg + j];
      if (gid < 0 || tmin < 0 || tmin >= row0 + nrows) continue;
      if (((int64_t)gid + 1) * U > unit_cap) {
        if (lane == 0) atomicCAS(&g_kv4_error, 0, kErrBoundsAttendKv4);
        continue;
      }
      const size_t base = (bk * unit_cap + (int64_t)gid * U + (i - n_hot) % U) * kv4_unit_bytes(DH);
      // a lane's words hold rows g, g + 8 and columns 2c, 2c + 1, 2c + 8, 2c + 9 of their tiles
      const int g = lane >> 2, c = 2 * (lane & 3);
      const uint8_t *uk = rec_k + base, *uv = rec_v + base;
#pragma unroll
      for (int quad = 0; quad < DH / 64; ++quad) {
        const uint4 k4 = *reinterpret_cast<const uint4*>(uk + (quad * 32 + lane) * 16);
        const uint4 v4 = *reinterpret_cast<const uint4*>(uv + (quad * 32 + lane) * 16);
        const uint32_t kw[4] = {k4.x, k4.y, k4.z, k4.w}, vw[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
          const int blk = quad * 2 + t2;  // 32 channels: two tiles
          float2 km[2], vm[4];
#pragma unroll
          for (int r = 0; r < 2; ++r) km[r] = scale_min<MT>(uk + 8 * DH, (g + 8 * r) * VD + blk);
#pragma unroll
          for (int e = 0; e < 4; ++e) vm[e] = scale_min<MT>(uv + 8 * DH, (c + (e & 1) + 8 * (e >> 1)) * VD + blk);
#pragma unroll
          for (int t1 = 0; t1 < 2; ++t1) {
            const int ch = blk * 32 + t1 * 16;
            const uint32_t wk = kw[t2 * 2 + t1], wv = vw[t2 * 2 + t1];
#pragma unroll
            for (int n = 0; n < 4; ++n) {  // row half n & 1, column half n >> 1; the pair's second column 4 nibbles on
              const int r = n & 1, e = n >> 1;
              *reinterpret_cast<float2*>(ks + (g + 8 * r) * LD + ch + c + 8 * e) =
                  make_float2(fmaf((float)(wk >> (4 * n) & 15u), km[r].x, km[r].y),
                              fmaf((float)(wk >> (4 * n + 16) & 15u), km[r].x, km[r].y));
              vs[(c + 8 * e) * LD + ch + g + 8 * r] = fmaf((float)(wv >> (4 * n) & 15u), vm[2 * e].x, vm[2 * e].y);
              vs[(c + 1 + 8 * e) * LD + ch + g + 8 * r] = fmaf((float)(wv >> (4 * n + 16) & 15u), vm[2 * e + 1].x, vm[2 * e + 1].y);
            }
          }
        }
      }
    }
    __syncwarp();
    const int key = lane >> 1, half = 2 * (lane & 1);
    float dot[R];
#pragma unroll
    for (int r = 0; r < R; ++r) dot[r] = 0.f;
#pragma unroll 8
    for (int d = half; d < DH; d += 4) {
      const float2 kv = *reinterpret_cast<const float2*>(ks + key * LD + d);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float2 qv = *reinterpret_cast<const float2*>(qs + r * DH + d);
        dot[r] = fmaf(qv.y, kv.y, fmaf(qv.x, kv.x, dot[r]));
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r >= nrows) break;
      const float x = dot[r] + __shfl_xor_sync(0xffffffffu, dot[r], 1);
      const bool vis = key < count && row0 + r >= tmin + causal * key;
      const unsigned mask = __ballot_sync(0xffffffffu, vis);
      if (!mask) continue;
      const float s = vis ? x * p.scale * 1.4426950408889634f : -INFINITY;
      float mx = s;
#pragma unroll
      for (int w = 16; w >= 2; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float m_new = fmaxf(m[r], mx);
      const float base = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = exp2f(m[r] - base), pe = vis ? exp2f(s - base) : 0.f;
      float ps = pe;
#pragma unroll
      for (int w = 16; w >= 2; w >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, w);
      l[r] = l[r] * alpha + ps;
      m[r] = m_new;
#pragma unroll
      for (int d = 0; d < VD; ++d) o[r][d] *= alpha;
#pragma unroll
      for (int j = 0; j < kKv4Unit; ++j) {
        const float pj = __shfl_sync(0xffffffffu, pe, 2 * j);
        if (!(mask >> (2 * j) & 1)) continue;  // what an invisible key holds does not count, NaN included
#pragma unroll
        for (int d = 0; d < VD; ++d) o[r][d] = fmaf(pj, vs[j * LD + lane + 32 * d], o[r][d]);
      }
    }
  }
  __syncthreads();
  float *pm = port_smem + S::kMax, *pl = port_smem + S::kSum;
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int d = 0; d < VD; ++d) ks[r * DH + lane + 32 * d] = o[r][d];
    if (lane == 0) {
      pm[warp * R + r] = m[r];
      pl[warp * R + r] = l[r];
    }
  }
  __syncthreads();
  if (tid < R) {
    float mx = -INFINITY, sum = 0.f;
    for (int w = 0; w < kPortWarps; ++w) mx = fmaxf(mx, pm[w * R + tid]);
    for (int w = 0; w < kPortWarps; ++w) {
      // a maximum of -infinity: nothing seen (sum 0), or only scores that are NaN (sum NaN)
      const float mw = pm[w * R + tid], lw = pl[w * R + tid], f = mw == -INFINITY ? lw : exp2f(mw - mx);
      sum += f * lw;
      pm[w * R + tid] = f;
    }
    pm[kPortWarps * R + tid] = mx;
    pl[kPortWarps * R + tid] = sum;
  }
  __syncthreads();
  for (int i = tid; i < nrows * DH; i += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kPortWarps; ++w) {
      const float f = pm[w * R + i / DH];
      s += f == 0.f ? 0.f : f * port_smem[w * S::kUnit + i];
    }
    qs[i] = s;
  }
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  const int lo = DH * rank / splits, width = DH * (rank + 1) / splits - lo;
  for (int i = tid; i < width * nrows; i += blockDim.x) {
    const int r = i / width, ch = lo + i % width;
    float mr[8], lr[8], vr[8], mx = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k >= splits) break;
      const float* other = cl.map_shared_rank(port_smem, k);
      mr[k] = other[S::kMax + kPortWarps * R + r];
      lr[k] = other[S::kSum + kPortWarps * R + r];
      vr[k] = other[S::kRows + r * DH + ch];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < splits) mx = fmaxf(mx, mr[k]);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k >= splits) break;
      const float f = mr[k] == -INFINITY ? lr[k] : exp2f(mr[k] - mx);
      sum += f * lr[k];  // with a factor of 0 too: a sum that is NaN is not lost
      if (f == 0.f) continue;
      acc += f * vr[k];
    }
    o_base[(size_t)r * DH + ch] = Num<T>::from_f(acc / sum);
  }
  cl.sync();  // no CTA leaves while another still reads its result
}

template <typename T, int DH, int R>
static cudaError_t port_t(const hga_params& p, int L, const void* q, const int32_t* seq_pos, const void* hk,
                          const void* hv, int64_t hot_cap, const void* rec_k, const void* rec_v, int64_t unit_cap,
                          const int32_t* og, const int32_t* ot, int Kg, void* out, cudaStream_t st) {
  constexpr int smem = PortSmem<DH, R>::kTotal;
  auto kern = attend_kv4_kernel<T, DH, R>;
  static unsigned long long raised = 0;
  cudaError_t e = raise_smem_limit((const void*)kern, smem, &raised);
  if (e != cudaSuccess) return e;
  // CTAs along the units: as many as are resident, at most 8 (clusters leave about a tenth of the places empty)
  const int64_t ctas = (int64_t)p.nhead * p.batch * ((L + R - 1) / R);
  int64_t splits = 132 * (200 * 1024 / smem < 4 ? 200 * 1024 / smem : 4) / ctas;
  splits = splits < 1 ? 1 : splits > 8 ? 8 : splits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)splits, p.nhead, (unsigned)((int64_t)p.batch * ((L + R - 1) / R)));
  cfg.blockDim = dim3(kPortWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p, L, (const T*)q, seq_pos, (const T*)hk, (const T*)hv, hot_cap,
                            (const uint8_t*)rec_k, (const uint8_t*)rec_v, unit_cap, og, ot, Kg, (T*)out);
}

cudaError_t launch_attend_kv4(const hga_params& p, int L, const void* q, const int32_t* seq_pos, const void* hk,
                              const void* hv, int64_t hot_cap, const void* rec_k, const void* rec_v, int64_t unit_cap,
                              const int32_t* og, const int32_t* ot, int Kg, void* out, cudaStream_t st) {
  const int dtype = p.dtype, dh = p.head_dim;
#define HGA_KV4_PORT(RR) port_t<T, DH, RR>(p, L, q, seq_pos, hk, hv, hot_cap, rec_k, rec_v, unit_cap, og, ot, Kg, out, st)
  cudaError_t e = cudaSuccess;
  HGA_KV4_DISPATCH((e = L == 1 ? HGA_KV4_PORT(1) : HGA_KV4_PORT(8)))
#undef HGA_KV4_PORT
  return e;
}

}  // namespace hga

// 8-bit block-scaled operators: quantisation of activations, and the dispatch of the product with an e4m3
// weight (its kernels are in fp8_tiles.cu, for many rows, and fp8_rows.cu, for few).
//
//   scale[m][kb] = max |x[m][k]|, k in block kb of 128, / 448        (1 where that maximum is <= 1e-30)
//   q[m][k]      = e4m3(x[m][k] / scale[m][k / 128])                  round to nearest, ties to even
//   y[m][n]      = sum_kb scale[m][kb] * w_scale[n / 128][kb] * sum_{k in kb} q[m][k] * w[n][k]  (+ bias[n])
//
// The division is the IEEE one: a reciprocal's last-bit error would move values that lie on a rounding
// boundary of e4m3 (about one in a thousand: quotients of two bf16 numbers meet the boundaries exactly).
// A block that holds an infinity or a NaN gets a non-finite scale, so its products are NaN.
#include "fp8_common.cuh"

namespace hga {

// A warp takes 8 neighbouring blocks of a row, two at a time (16 lanes a block, 8 channels a lane), their
// four loads in flight together.  The four rounds' scales and reciprocals are worked out side by side, one
// round a lane, and handed out by shuffles: computed per round they were a third of the instructions.
// Bound by HBM (2 bytes read and 1 written per 16-bit channel) and nearly so by issue: 32768 x 4096 bf16 in 75 us,
// 5.4 TB/s, 83 % of the measured copy (plain divisions, a scale a block and one block in flight a warp: 160 us).
// Five CTAs an SM: 78 us with four, 80 with six (its registers spill).  VEC: rows and base are 16-byte
// aligned (8-byte for q).
constexpr int kQuantWarps = 8;

template <typename T, bool VEC>
__global__ void __launch_bounds__(kQuantWarps * 32, 5) fp8_quantize_kernel(const T* __restrict__ x, int64_t x_stride,
                                                                        int64_t m, int64_t k, int kb, int segs,
                                                                        uint8_t* __restrict__ q, int64_t q_stride,
                                                                        int64_t q_cols, float* __restrict__ scale,
                                                                        int64_t scale_stride) {
  const int lane = threadIdx.x & 31, sub = lane & 15, half = lane >> 4;
  const int64_t tasks = m * segs, step = (int64_t)gridDim.x * kQuantWarps;
  for (int64_t task = (int64_t)blockIdx.x * kQuantWarps + (threadIdx.x >> 5); task < tasks; task += step) {
    const int64_t row = (uint64_t)task >> 32 ? task / segs : (int64_t)((uint32_t)task / (uint32_t)segs);
    const int blk0 = (int)(task - row * segs) * 8 + half;  // of round 0
    const T* src = x + row * x_stride + (int64_t)blk0 * 128 + sub * 8;
    const int64_t c0 = (int64_t)blk0 * 128 + sub * 8;
    Raw8<T> raw[4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      raw[r] = blk0 + 2 * r < kb ? raw_load<T>(src + r * 256, VEC, k - (c0 + r * 256)) : raw_zero<T>();
    float mine = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float a = raw_amax<T>(raw[r]);
      if ((lane & 3) == r) mine = a;
    }
    const float my_s = fp8_scale(mine), my_inv = __frcp_rn(my_s);
    const bool odd = __any_sync(0xffffffffu, !(my_s < INFINITY));
    if (sub < 4 && blk0 + 2 * sub < kb) scale[row * scale_stride + blk0 + 2 * sub] = my_s;
    uint8_t* dst = q + row * q_stride + c0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float s = __shfl_sync(0xffffffffu, my_s, half * 16 + r), inv = __shfl_sync(0xffffffffu, my_inv, half * 16 + r);
      float f[8];
      raw_floats<T>(raw[r], f);
      uint2 v = fp8_quotients(f, s, inv);
      if (odd) {
        if (!(s < INFINITY)) v = fp8_divisions(f, s);
      }
      if (blk0 + 2 * r >= kb) continue;
      if (VEC && c0 + r * 256 + 8 <= q_cols) {
        *reinterpret_cast<uint2*>(dst + r * 256) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + r * 256 + e < q_cols) dst[r * 256 + e] = (uint8_t)((e < 4 ? v.x : v.y) >> (8 * (e & 3)));
      }
    }
  }
}

template <typename T>
static cudaError_t quantize_t(const void* x, int64_t x_stride, int64_t m, int64_t k, void* q, int64_t q_stride,
                              int64_t q_cols, float* scale, int64_t scale_stride, cudaStream_t st) {
  const int kb = (int)((k + 127) / 128), segs = (kb + 7) / 8;
  int64_t grid = (m * segs + kQuantWarps - 1) / kQuantWarps;
  if (grid > 148 * 32) grid = 148 * 32;
  const bool vec = ((uintptr_t)x % 16) == 0 && (x_stride * (int64_t)sizeof(T)) % 16 == 0 && ((uintptr_t)q % 8) == 0 &&
                   q_stride % 8 == 0;
  if (vec)
    fp8_quantize_kernel<T, true><<<(unsigned)grid, kQuantWarps * 32, 0, st>>>(
        (const T*)x, x_stride, m, k, kb, segs, (uint8_t*)q, q_stride, q_cols, scale, scale_stride);
  else
    fp8_quantize_kernel<T, false><<<(unsigned)grid, kQuantWarps * 32, 0, st>>>(
        (const T*)x, x_stride, m, k, kb, segs, (uint8_t*)q, q_stride, q_cols, scale, scale_stride);
  return cudaGetLastError();
}

// q_cols >= k columns are written: channels past k are zeros
cudaError_t launch_fp8_quantize(int dtype, const void* x, int64_t x_stride, int64_t m, int64_t k, void* q,
                                int64_t q_stride, int64_t q_cols, float* scale, int64_t scale_stride, cudaStream_t st) {
  switch (dtype) {
    case HGA_DTYPE_F32: return quantize_t<float>(x, x_stride, m, k, q, q_stride, q_cols, scale, scale_stride, st);
    case HGA_DTYPE_BF16: return quantize_t<__nv_bfloat16>(x, x_stride, m, k, q, q_stride, q_cols, scale, scale_stride, st);
    case HGA_DTYPE_F16: return quantize_t<__half>(x, x_stride, m, k, q, q_stride, q_cols, scale, scale_stride, st);
  }
  return cudaErrorInvalidValue;
}

// Rows of k bytes to rows of `cols` bytes (zeros behind k), 16-byte aligned: operands that TMA cannot
// address where they are (a base or a row stride off the 16-byte grid).
__global__ void __launch_bounds__(256) fp8_realign_kernel(const uint8_t* __restrict__ src, int64_t src_stride,
                                                          int64_t rows, int64_t k, uint4* __restrict__ dst, int64_t cols) {
  const int64_t per = cols / 16, total = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / per, c = (i - r * per) * 16;
    uint32_t w[4] = {0, 0, 0, 0};
    const uint8_t* p = src + r * src_stride + c;
    const int sh = (int)((uintptr_t)p & 3);
    if (c - sh >= 0 && c + 20 <= k) {  // five aligned words, all inside the row
      const uint32_t* q = reinterpret_cast<const uint32_t*>(p - sh);
      uint32_t v[5];
#pragma unroll
      for (int e = 0; e < 5; ++e) v[e] = q[e];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = __funnelshift_r(v[e], v[e + 1], 8 * sh);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (c + e < k) w[e >> 2] |= (uint32_t)p[e] << (8 * (e & 3));
    }
    dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

static cudaError_t realign(const void* src, int64_t stride, int64_t rows, int64_t k, void* dst, int64_t cols,
                           cudaStream_t st) {
  int64_t grid = (rows * (cols / 16) + 255) / 256;
  if (grid > 148 * 8) grid = 148 * 8;
  fp8_realign_kernel<<<(unsigned)grid, 256, 0, st>>>((const uint8_t*)src, stride, rows, k, (uint4*)dst, cols);
  return cudaGetLastError();
}

static bool off_grid(const void* p, int64_t stride) { return ((uintptr_t)p & 15) || (stride & 15); }

// Floats between the scales of two rows in the workspace: whole 16-byte pieces.
static int64_t scale_stride(int64_t kb) { return (kb + 3) / 4 * 4; }

// Workspace: [quantised or realigned x][its scales][realigned w], each part present only where needed.
static void parts(const Fp8Linear& a, int64_t& xq, int64_t& xs, int64_t& w) {
  const int64_t kb = (a.k + 127) / 128;
  xq = xs = w = 0;
  if (a.x_dtype != HGA_DTYPE_E4M3) {
    if (!fp8_rows_fused(a)) {
      xq = a.m * kb * 128;
      xs = a.m * scale_stride(kb) * 4;
    }
  } else if (off_grid(a.x, a.x_stride)) {
    xq = a.m * kb * 128;
  }
  if (off_grid(a.w, a.w_stride)) w = a.n * kb * 128;
}

int64_t fp8_linear_workspace(const Fp8Linear& a) {
  int64_t xq, xs, w;
  parts(a, xq, xs, w);
  return xq + xs + w;
}

cudaError_t launch_fp8_linear(const Fp8Linear& a, cudaStream_t st) {
  const int64_t cols = (a.k + 127) / 128 * 128;
  int64_t xqb, xsb, wb;
  parts(a, xqb, xsb, wb);
  char* ws = (char*)a.workspace;
  const void* q = a.x;
  int64_t q_stride = a.x_stride;
  const float* xs = a.x_scale;
  int64_t xs_stride = cols / 128;
  const void* w = a.w;
  int64_t w_stride = a.w_stride;
  cudaError_t e = cudaSuccess;
  if (xqb) {
    q = ws;
    q_stride = cols;
    if (xsb) {
      xs = (const float*)(ws + xqb);
      xs_stride = scale_stride(cols / 128);
      e = launch_fp8_quantize(a.x_dtype, a.x, a.x_stride, a.m, a.k, ws, cols, cols, (float*)(ws + xqb), xs_stride, st);
    } else {
      e = realign(a.x, a.x_stride, a.m, a.k, ws, cols, st);
    }
    if (e != cudaSuccess) return e;
  }
  if (wb) {
    w = ws + xqb + xsb;
    w_stride = cols;
    e = realign(a.w, a.w_stride, a.n, a.k, ws + xqb + xsb, cols, st);
    if (e != cudaSuccess) return e;
  }
  if (fp8_rows_better(a)) return launch_fp8_rows(a, q, q_stride, xs, xs_stride, w, w_stride, st);
  return launch_fp8_tiles(a, q, q_stride, xs, xs_stride, w, w_stride, st);
}

}  // namespace hga

// Product of many rows with an e4m3 weight on the tensor cores (tcgen05 kind::f8f6f4, TMA, TMEM).
//
//   y[m][n] = sum_kb xs[m][kb] * ws[n / 128][kb] * (sum over the block's 128 channels of q[m][k] w[n][k])
//
// The scales change every 128 channels, so a block's products cannot stay in the accumulator: each
// block is one MMA group of four K = 32 steps into one of two TMEM buffers, and eight epilogue warps
// add it, scaled, to fp32 sums in registers (one fp32 FMA per output and block) while the tensor cores
// work on the next block in the other buffer.  Persistent CTAs, one per SM, walk the output tiles with
// neighbouring feature tiles first (their rows of x are then read from L2).
//   warp 0      TMA producer: 128 x 128 bytes of x and BN x 128 bytes of w per block, STAGES deep, SW128
//   warp 1      MMA issuer (one lane), TMEM owner
//   warps 2-9   each reads 32 TMEM lanes (rows) x BN / 2 columns: one row a thread, one weight block a
//               warp, so a block's scale is one product per thread
// Results go through 4 KB of swizzled shared memory per warp to whole-line TMA stores (plain stores where
// the output's rows are off the 16-byte grid).  Waits are bounded as in tc_common.cuh.
#include "fp8_common.cuh"
#include "tc_common.cuh"

namespace hga {
namespace tc {

constexpr int kTileThreads = 320;
constexpr int kErrFp8 = 0x40;  // codes 0x40..0x47 of the bounded waits

struct TileArgs {
  int m, n, kb, tiles_n, tiles;
  const float* xs;
  const float* ws;
  int64_t ws_stride;
  const void* bias;
  void* out;
  int64_t out_stride;
  int tma_out;
};

template <int BN, int STAGES> struct TileSmem {
  static constexpr int kA = 128 * 128, kB = BN * 128;
  static constexpr int kStage = kA + kB;
  static constexpr int kOut = STAGES * kStage;       // 8 x 4 KB
  static constexpr int kBars = kOut + 8 * 4096;
  static constexpr int kMisc = kBars + (2 * STAGES + 5) * 8;
  static constexpr int kTotal = kMisc + 32;
};

__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t ffma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
               "r"(smem_u32(src))
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
  if constexpr (sizeof(T) == 2) {
    const T h[2] = {Num<T>::from_f(a), Num<T>::from_f(b)};
    return *reinterpret_cast<const uint32_t*>(h);
  } else {
    return 0;
  }
}

template <typename T, int BN, int STAGES>
__global__ void __launch_bounds__(kTileThreads, 1)
    fp8_tiles_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ CUtensorMap tm_o, const TileArgs a) {
  using S = TileSmem<BN, STAGES>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* full = bars;
  uint64_t* empty = bars + STAGES;
  uint64_t* d_full = bars + 2 * STAGES;       // [2]
  uint64_t* d_empty = bars + 2 * STAGES + 2;  // [2]
  uint64_t* drain = bars + 2 * STAGES + 4;
  int* misc = reinterpret_cast<int*>(smem + S::kMisc);
  volatile int* abort_flag = misc;
  uint32_t* tmem_s = reinterpret_cast<uint32_t*>(misc + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(d_full + i, 1);
      mbar_init(d_empty + i, 8);
    }
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *abort_flag = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_s)),
                 "r"(2u * BN));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_s;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x) {
        const int m0 = tile / a.tiles_n * 128, n0 = tile % a.tiles_n * BN;
        for (int kb = 0; kb < a.kb; ++kb, ++it) {
          const int st = it % STAGES;
          if (it >= STAGES && !mbar_wait(empty + st, (it / STAGES - 1) & 1, abort_flag, kErrFp8)) { ok = false; break; }
          unsigned char* s = smem + st * S::kStage;
          mbar_expect_tx(full + st, S::kStage);
          tma_load_2d(s, &tm_x, kb * 128, m0, full + st);
          tma_load_2d(s + S::kA, &tm_w, kb * 128, n0, full + st);
        }
      }
      // every load that was issued has landed before the shared memory is given up
      for (int i = it > STAGES ? it - STAGES : 0; i < it; ++i) mbar_drain(full + i % STAGES, (i / STAGES) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t id = idesc_e4m3(BN);
      int it = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x) {
        for (int kb = 0; kb < a.kb; ++kb, ++it) {
          const int st = it % STAGES, buf = it & 1;
          if (!mbar_wait(full + st, (it / STAGES) & 1, abort_flag, kErrFp8 + 1) ||
              (it >= 2 && !mbar_wait(d_empty + buf, (it / 2 - 1) & 1, abort_flag, kErrFp8 + 2))) {
            ok = false;
            break;
          }
          fence_after();
          const uint32_t xa = smem_u32(smem + st * S::kStage), wa = xa + S::kA;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_ss_f8(tmem + buf * BN, sdesc(xa + k * 32, 16, 1024), sdesc(wa + k * 32, 16, 1024), id, k != 0);
          mma_commit(empty + st);
          mma_commit(d_full + buf);
        }
      }
      mma_commit(drain);
      mbar_drain(drain, 0);
    }
  } else {
    constexpr int COLS = BN / 2;                // columns of this warp
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    unsigned char* stage = smem + S::kOut + (warp - 2) * 4096;
    int it = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < a.tiles && ok; tile += gridDim.x) {
      const int m0 = tile / a.tiles_n * 128 + quarter * 32, n0 = tile % a.tiles_n * BN + half * COLS;
      const int row = m0 + lane;
      const float* xs = a.xs + (int64_t)(row < a.m ? row : a.m - 1) * a.kb;
      const float* ws = a.ws + (int64_t)((n0 < a.n ? n0 : a.n - 1) / 128) * a.ws_stride;
      uint64_t acc[COLS / 2];
#pragma unroll
      for (int i = 0; i < COLS / 2; ++i) acc[i] = 0ull;
      float s_next = xs[0] * ws[0];
      for (int kb = 0; kb < a.kb; ++kb, ++it) {
        const int buf = it & 1;
        const float s = s_next;
        if (kb + 1 < a.kb) s_next = xs[kb + 1] * ws[kb + 1];
        const uint64_t s2 = pack2(s, s);
        ok = __all_sync(0xffffffffu, mbar_wait(d_full + buf, (it / 2) & 1, abort_flag, kErrFp8 + 3));
        if (!ok) break;
        fence_after();
#pragma unroll
        for (int c = 0; c < COLS; c += 32) {
          uint32_t r[32];
          HGA_LD32(tmem + lane_addr + buf * BN + half * COLS + c, r);
          tmem_wait_ld();
          if (c + 32 == COLS) {
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(d_empty + buf);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i)
            acc[c / 2 + i] = ffma2(pack2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), s2, acc[c / 2 + i]);
        }
      }
      if (!ok) break;
      constexpr int PC = 128 / (int)sizeof(T);  // columns per 128-byte pass
      const T* bias = static_cast<const T*>(a.bias);
#pragma unroll
      for (int c = 0; c < COLS; c += PC) {
        if (n0 + c >= a.n || m0 >= a.m) break;  // warp-uniform
        if (a.tma_out) {
          if (lane == 0) bulk_wait_read();
          __syncwarp();
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {           // 16-byte pieces of the row's 128 bytes
          uint32_t w[4];
          if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float lo, hi;
              unpack2(acc[c / 2 + j * 4 + e], lo, hi);
              if (bias) {
                const int col = n0 + c + j * 8 + e * 2;
                lo += col < a.n ? Num<T>::to_f(bias[col]) : 0.f;
                hi += col + 1 < a.n ? Num<T>::to_f(bias[col + 1]) : 0.f;
              }
              w[e] = pack_out<T>(lo, hi);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float lo, hi;
              unpack2(acc[c / 2 + j * 2 + e], lo, hi);
              if (bias) {
                const int col = n0 + c + j * 4 + e * 2;
                lo += col < a.n ? Num<T>::to_f(bias[col]) : 0.f;
                hi += col + 1 < a.n ? Num<T>::to_f(bias[col + 1]) : 0.f;
              }
              w[2 * e] = __float_as_uint(lo);
              w[2 * e + 1] = __float_as_uint(hi);
            }
          }
          if (a.tma_out) {
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          } else if (row < a.m) {
            T* o = static_cast<T*>(a.out) + (int64_t)row * a.out_stride + n0 + c + j * (16 / (int)sizeof(T));
            const T* v = reinterpret_cast<const T*>(w);
#pragma unroll
            for (int e = 0; e < 16 / (int)sizeof(T); ++e)
              if (n0 + c + j * (16 / (int)sizeof(T)) + e < a.n) o[e] = v[e];
          }
        }
        if (a.tma_out) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tm_o, stage, n0 + c, m0);
            bulk_commit();
          }
        }
      }
    }
    if (lane == 0) bulk_wait_all();
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2u * BN));
}

template <typename T, int BN, int STAGES>
static cudaError_t tiles_t(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, const void* w,
                           int64_t w_stride, cudaStream_t st) {
  CUtensorMap mx, mw, mo;
  const cuuint64_t dx[2] = {(cuuint64_t)a.k, (cuuint64_t)a.m}, sx[1] = {(cuuint64_t)q_stride};
  const cuuint64_t dw[2] = {(cuuint64_t)a.k, (cuuint64_t)a.n}, sw[1] = {(cuuint64_t)w_stride};
  const cuuint32_t bx[2] = {128, 128}, bw[2] = {128, BN};
  if (!make_map_typed(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, q, 2, dx, sx, bx, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_map_typed(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, 2, dw, sw, bw, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  const int64_t ostr = a.out_stride * (int64_t)sizeof(T);
  const bool tma_out = ((uintptr_t)a.out & 15) == 0 && ostr % 16 == 0;
  mo = mx;
  if (tma_out) {
    const cuuint64_t d[2] = {(cuuint64_t)a.n, (cuuint64_t)a.m}, s[1] = {(cuuint64_t)ostr};
    const cuuint32_t b[2] = {128 / sizeof(T), 32};
    const CUtensorMapDataType ty = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    if (!make_map_typed(&mo, ty, a.out, 2, d, s, b, CU_TENSOR_MAP_SWIZZLE_128B)) return cudaErrorInvalidValue;
  }
  TileArgs t;
  t.m = (int)a.m; t.n = (int)a.n; t.kb = (int)((a.k + 127) / 128);
  t.tiles_n = (int)((a.n + BN - 1) / BN);
  const int64_t tiles = (a.m + 127) / 128 * t.tiles_n;
  if (tiles > 0x7fffffff) return cudaErrorInvalidValue;
  t.tiles = (int)tiles;
  t.xs = xs; t.ws = a.w_scale; t.ws_stride = a.ws_stride;
  t.bias = a.bias; t.out = a.out; t.out_stride = a.out_stride; t.tma_out = tma_out;
  constexpr int smem = TileSmem<BN, STAGES>::kTotal + 1024;
  auto kern = fp8_tiles_kernel<T, BN, STAGES>;
  static unsigned long long raised = 0;
  cudaError_t e = raise_smem_limit((const void*)kern, smem, &raised);
  if (e != cudaSuccess) return e;
  kern<<<t.tiles < 148 ? t.tiles : 148, kTileThreads, smem, st>>>(mx, mw, mo, t);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t tiles_n(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, const void* w,
                           int64_t w_stride, cudaStream_t st) {
  // 128 x 256 tiles read the operands from shared memory fewer times; where they would leave SMs
  // without a tile, 128 x 128 ones
  const int64_t rows = (a.m + 127) / 128;
  if (rows * ((a.n + 255) / 256) >= 148) return tiles_t<T, 256, 4>(a, q, q_stride, xs, w, w_stride, st);
  return tiles_t<T, 128, 5>(a, q, q_stride, xs, w, w_stride, st);
}

}  // namespace tc

cudaError_t launch_fp8_tiles(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, const void* w,
                             int64_t w_stride, cudaStream_t st) {
  switch (a.out_dtype) {
    case HGA_DTYPE_F32: return tc::tiles_n<float>(a, q, q_stride, xs, w, w_stride, st);
    case HGA_DTYPE_BF16: return tc::tiles_n<__nv_bfloat16>(a, q, q_stride, xs, w, w_stride, st);
    case HGA_DTYPE_F16: return tc::tiles_n<__half>(a, q, q_stride, xs, w, w_stride, st);
  }
  return cudaErrorInvalidValue;
}

HGA_DEFINE_ERROR_READER(fp8_tiles_error_status)

}  // namespace hga

// Product of few rows (a decode step's tokens) with an e4m3 weight.  The weight is what has to be read, so
// it is the 128-row operand of the tensor cores (D^T[feature][token] = w q^T) and every SM streams a part
// of it: a CTA takes 128 features x TN tokens x a slice of the channels, and a cluster of up to 8 CTAs
// shares one output tile along the channels, joining the partial sums through distributed shared memory in
// a fixed order (no atomics, no second launch).
//   warp 0     TMA producer of the weight's (and, when x comes quantised, the tokens') 128-channel blocks
//   warp 1     MMA issuer, TMEM owner: one group of four K = 32 steps per block into its own TMEM columns
//   warps 2-9  FUSED: quantise the CTA's slice of x straight into the swizzled shared operand while the
//              weight is on its way (each slice is small and comes from L2)
//   warps 2-5  then one feature a thread: sum[token] += D * (ws * xs[token]) per block
// FUSED saves the quantisation's launch and its round trip through memory; past some 64 blocks a CTA its
// repetition in every CTA costs more than that (16 x 8192 into 8192 features: 27.2 us against 19.7).
// One token of 2048 channels into 5120 features: 7.6 us (the launch of a cluster and the chain of loads, product
// and join bound it; the weight alone is 1.6 us of HBM); 16 rows of 8192 channels, already quantised, into 8192
// features: 16.7 us with the weight in HBM (4.0 TB/s), 11.9 with it in L2.
#include <cooperative_groups.h>

#include "fp8_common.cuh"
#include "tc_common.cuh"

namespace hga {
namespace tc {

namespace cg = cooperative_groups;

__host__ __device__ constexpr int rows_threads(bool fused) { return fused ? 320 : 192; }
constexpr int kErrFp8Rows = 0x48;
constexpr int kMaxSlice = 16;  // channel blocks per CTA

struct RowsArgs {
  int m, n, k, kb, splits;
  const void* x;      // FUSED: the activations
  int64_t x_stride;
  int x_vec;          // 16-byte loads are possible
  const float* xs;    // not FUSED: their scales
  int64_t xs_stride;
  const float* ws;
  int64_t ws_stride;
  const void* bias;
  void* out;
  int64_t out_stride;
};

template <int TN, bool FUSED> struct RowsSmem {
  static constexpr int kStages = FUSED || TN == 64 ? 4 : 5;  // two CTAs fit an SM
  static constexpr int kBufs = TN == 64 ? 4 : 8;               // TMEM buffers of TN columns
  static constexpr int kW = 128 * 128, kX = TN * 128;
  static constexpr int kStage = kW + (FUSED ? 0 : kX);
  static constexpr int kScale = kStages * kStage;               // [kMaxSlice][TN]
  static constexpr int kBars = kScale + kMaxSlice * TN * 4;
  static constexpr int kNumBars = 2 * kStages + 2 * kBufs + 2;
  static constexpr int kMisc = kBars + kNumBars * 8;
  static constexpr int kXs = (kMisc + 32 + 1023) / 1024 * 1024;  // FUSED: the quantised slice, as long as it is
  static constexpr int total(int slice) { return FUSED ? kXs + slice * kX : kMisc + 32; }
  static constexpr uint32_t kCols = kBufs * TN;                 // 128 or 256
  static_assert(kStages * kStage >= 128 * TN * 4, "the partial sums reuse the ring");
};

template <typename TX, typename TO, int TN, bool FUSED>
__global__ void __launch_bounds__(rows_threads(FUSED))
    fp8_rows_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const RowsArgs a) {
  using S = RowsSmem<TN, FUSED>;
  constexpr int kRowsThreads = rows_threads(FUSED), kWork = kRowsThreads - 64;  // threads of warps 2 on
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  // every CTA of a cluster places its parts at the same offset (the distributed reads need that): the
  // dynamic base is the same in all of them
  unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* full = bars;
  uint64_t* empty = full + S::kStages;
  uint64_t* d_full = empty + S::kStages;
  uint64_t* d_empty = d_full + S::kBufs;
  uint64_t* x_ready = d_empty + S::kBufs;
  uint64_t* drain = x_ready + 1;
  int* misc = reinterpret_cast<int*>(smem + S::kMisc);
  volatile int* abort_flag = misc;
  uint32_t* tmem_s = reinterpret_cast<uint32_t*>(misc + 1);
  float* scale_s = reinterpret_cast<float*>(smem + S::kScale);  // token's scale x weight block's scale
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x, n0 = blockIdx.y * 128, t0 = blockIdx.z * TN;
  const int kb0 = (int)((int64_t)a.kb * rank / a.splits), kb1 = (int)((int64_t)a.kb * (rank + 1) / a.splits);
  const int nkb = kb1 - kb0;

  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < S::kBufs; ++i) {
      mbar_init(d_full + i, 1);
      mbar_init(d_empty + i, 4);
    }
    mbar_init(x_ready, kWork);
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *abort_flag = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_s)),
                 "r"(S::kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_s;

  float acc[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) acc[j] = 0.f;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (; it < nkb; ++it) {
        const int st = it % S::kStages;
        if (it >= S::kStages && !mbar_wait(empty + st, (it / S::kStages - 1) & 1, abort_flag, kErrFp8Rows)) break;
        unsigned char* s = smem + st * S::kStage;
        mbar_expect_tx(full + st, S::kStage);
        tma_load_2d(s, &tm_w, (kb0 + it) * 128, n0, full + st);
        if constexpr (!FUSED) tma_load_2d(s + S::kW, &tm_x, (kb0 + it) * 128, t0, full + st);
      }
      for (int i = it > S::kStages ? it - S::kStages : 0; i < it; ++i)
        mbar_drain(full + i % S::kStages, (i / S::kStages) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t id = idesc_e4m3(TN);
      bool ok = mbar_wait(x_ready, 0, abort_flag, kErrFp8Rows + 1);
      for (int it = 0; it < nkb && ok; ++it) {
        const int st = it % S::kStages, buf = it % S::kBufs;
        if (!mbar_wait(full + st, (it / S::kStages) & 1, abort_flag, kErrFp8Rows + 2) ||
            (it >= S::kBufs && !mbar_wait(d_empty + buf, (it / S::kBufs - 1) & 1, abort_flag, kErrFp8Rows + 3)))
          break;
        fence_after();
        const uint32_t wa = smem_u32(smem + st * S::kStage);
        const uint32_t xa = FUSED ? smem_u32(smem + S::kXs + it * S::kX) : wa + S::kW;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_ss_f8(tmem + buf * TN, sdesc(wa + k * 32, 16, 1024), sdesc(xa + k * 32, 16, 1024), id, k != 0);
        mma_commit(empty + st);
        mma_commit(d_full + buf);
      }
      mma_commit(drain);
      mbar_drain(drain, 0);
    }
  } else {
    const int e = tid - 64;  // 0..kWork-1
    if constexpr (FUSED) {
      // 16 lanes a block of 128 channels; the (block, row) pairs of the CTA's slice are dealt to the 16 half
      // warps, two side by side each.  The operand's 128-byte swizzle: 16-byte piece p of row r sits at
      // p ^ (r & 7).  Rows past m are zeros with scale 0.
      const TX* x = static_cast<const TX*>(a.x);
      const float* ws = a.ws + (int64_t)blockIdx.y * a.ws_stride + kb0;
      const int sub = e & 15, live = a.m - t0 < TN ? a.m - t0 : TN, pairs = nkb * live;
      constexpr int R = 2;
      for (int i = e; i < nkb * (TN - live) * 8; i += kWork) {
        const int blk = i / ((TN - live) * 8), pc = i % ((TN - live) * 8);
        *reinterpret_cast<uint4*>(smem + S::kXs + blk * S::kX + live * 128 + pc * 16) = make_uint4(0u, 0u, 0u, 0u);
      }
      for (int i = e; i < nkb * TN; i += kWork) {
        if (i % TN >= live) scale_s[i] = 0.f;
      }
      for (int base = (e >> 5) * 2; base < pairs; base += 16 * R) {
        Raw8<TX> f[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int pr = base + r * 16 + ((e >> 4) & 1);
          const int c0 = (kb0 + pr / live) * 128 + sub * 8;
          f[r] = pr < pairs ? raw_load<TX>(x + (int64_t)(t0 + pr % live) * a.x_stride + c0, a.x_vec, a.k - c0)
                            : raw_zero<TX>();
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int pr = base + r * 16 + ((e >> 4) & 1);
          uint2 v;
          const float s = fp8_block<TX>(f[r], v);
          if (pr < pairs) {
            const int blk = pr / live, row = pr % live;
            *reinterpret_cast<uint2*>(smem + S::kXs + blk * S::kX + row * 128 + (((sub >> 1) ^ (row & 7)) << 4) +
                                      (sub & 1) * 8) = v;
            if (sub == 0) scale_s[blk * TN + row] = s * ws[blk];
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    } else {
      for (int i = e; i < nkb * TN; i += kWork) {
        const int r = t0 + i % TN;
        scale_s[i] = r < a.m ? a.xs[(int64_t)r * a.xs_stride + kb0 + i / TN] *
                                   a.ws[(int64_t)blockIdx.y * a.ws_stride + kb0 + i / TN]
                             : 0.f;
      }
    }
    mbar_arrive(x_ready);
    asm volatile("bar.sync 1, %0;" ::"n"(kWork) : "memory");  // the scales are in shared memory
    const int quarter = warp & 3;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    for (int it = 0; it < nkb && warp < 6; ++it) {
      const int buf = it % S::kBufs;
      if (!__all_sync(0xffffffffu, mbar_wait(d_full + buf, (it / S::kBufs) & 1, abort_flag, kErrFp8Rows + 4))) break;
      fence_after();
      uint32_t r[TN];
      if constexpr (TN == 16) {
        HGA_LD16(tmem + lane_addr + buf * TN, r);
      } else {
#pragma unroll
        for (int c = 0; c < TN; c += 32) {
          uint32_t(&rr)[32] = *reinterpret_cast<uint32_t(*)[32]>(r + c);
          HGA_LD32(tmem + lane_addr + buf * TN + c, rr);
        }
      }
      tmem_wait_ld();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(d_empty + buf);
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[j] = fmaf(__uint_as_float(r[j]), scale_s[it * TN + j], acc[j]);
    }
  }

  const int feat = (warp >= 2 ? ((warp & 3) * 32 + lane) : 0);
  TO* out = static_cast<TO*>(a.out);
  const TO* bias = static_cast<const TO*>(a.bias);
  if (a.splits == 1) {
    if (warp >= 2 && warp < 6 && n0 + feat < a.n) {
      const float add = bias ? Num<TO>::to_f(bias[n0 + feat]) : 0.f;
#pragma unroll
      for (int j = 0; j < TN; ++j)
        if (t0 + j < a.m) out[(int64_t)(t0 + j) * a.out_stride + n0 + feat] = Num<TO>::from_f(acc[j] + add);
    }
  } else {
    // the ring is free: the last block's MMAs (which read it) have completed and no load is outstanding
    float* part = reinterpret_cast<float*>(smem);  // [TN][128]
    __syncthreads();
    if (warp >= 2 && warp < 6) {
#pragma unroll
      for (int j = 0; j < TN; ++j) part[j * 128 + feat] = acc[j];
    }
    cg::cluster_group cl = cg::this_cluster();
    __syncwarp();
    cl.sync();
    // this CTA's share of the tile, four features of a token at a time, the CTAs' sums in rank order
    const int lo = TN * rank / a.splits, hi = TN * (rank + 1) / a.splits;
    for (int i = lo * 32 + tid; i < hi * 32; i += kRowsThreads) {
      const int j = i >> 5, f = (i & 31) * 4;
      if (t0 + j >= a.m || n0 + f >= a.n) continue;
      float4 v[8];
#pragma unroll
      for (int p = 0; p < 8; ++p)
        if (p < a.splits) v[p] = *cl.map_shared_rank(reinterpret_cast<float4*>(part) + i, p);
      float o[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
      for (int p = 1; p < 8; ++p)
        if (p < a.splits) {
          o[0] += v[p].x;
          o[1] += v[p].y;
          o[2] += v[p].z;
          o[3] += v[p].w;
        }
      TO* dst = out + (int64_t)(t0 + j) * a.out_stride + n0 + f;
      TO y[4];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        y[c] = Num<TO>::from_f(o[c] + (bias && n0 + f + c < a.n ? Num<TO>::to_f(bias[n0 + f + c]) : 0.f));
      if (n0 + f + 4 <= a.n && ((uintptr_t)dst & (4 * sizeof(TO) - 1)) == 0) {
        if constexpr (sizeof(TO) == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(y);
        else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(y);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (n0 + f + c < a.n) dst[c] = y[c];
      }
    }
    cl.sync();  // no CTA leaves while another still reads its sums
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kCols));
}

// CTAs along the channels: as many as are resident at once (two an SM less what clusters leave empty), at least two
// blocks each, at most 8 (a portable cluster) and kMaxSlice blocks a CTA.
static int rows_splits(int64_t m, int64_t n, int64_t kb, int tn) {
  const int64_t tiles = (n + 127) / 128 * ((m + tn - 1) / tn);
  int s = 1;
  while (s < 8 && ((tiles * s * 2 <= 264 && kb >= 4 * s) || kb > (int64_t)s * kMaxSlice)) s *= 2;
  return s;
}

static int rows_tn(int64_t m) { return m <= 16 ? 16 : m <= 32 ? 32 : 64; }

template <typename TX, typename TO, int TN, bool FUSED>
static cudaError_t rows_t(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, int64_t xs_stride,
                          const void* w, int64_t w_stride, cudaStream_t st) {
  CUtensorMap mx, mw;
  const cuuint64_t dw[2] = {(cuuint64_t)a.k, (cuuint64_t)a.n}, sw[1] = {(cuuint64_t)w_stride};
  const cuuint32_t bw[2] = {128, 128};
  if (!make_map_typed(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, 2, dw, sw, bw, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  mx = mw;
  if (!FUSED) {
    const cuuint64_t dx[2] = {(cuuint64_t)a.k, (cuuint64_t)a.m}, sx[1] = {(cuuint64_t)q_stride};
    const cuuint32_t bx[2] = {128, TN};
    if (!make_map_typed(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, q, 2, dx, sx, bx, CU_TENSOR_MAP_SWIZZLE_128B))
      return cudaErrorInvalidValue;
  }
  RowsArgs r;
  r.m = (int)a.m; r.n = (int)a.n; r.k = (int)a.k; r.kb = (int)((a.k + 127) / 128);
  r.splits = rows_splits(a.m, a.n, r.kb, TN);
  r.x = a.x; r.x_stride = a.x_stride;
  r.x_vec = ((uintptr_t)a.x & 15) == 0 && (a.x_stride * (int64_t)sizeof(TX)) % 16 == 0;
  r.xs = xs; r.xs_stride = xs_stride; r.ws = a.w_scale; r.ws_stride = a.ws_stride;
  r.bias = a.bias; r.out = a.out; r.out_stride = a.out_stride;
  const int smem = RowsSmem<TN, FUSED>::total((r.kb + r.splits - 1) / r.splits) + 1024;
  auto kern = fp8_rows_kernel<TX, TO, TN, FUSED>;
  static unsigned long long raised = 0;
  cudaError_t e = raise_smem_limit((const void*)kern, RowsSmem<TN, FUSED>::total(kMaxSlice) + 1024, &raised);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(r.splits, (unsigned)((a.n + 127) / 128), (unsigned)((a.m + TN - 1) / TN));
  cfg.blockDim = dim3(rows_threads(FUSED));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = r.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, mw, mx, r);
}

template <typename TX, typename TO, bool FUSED>
static cudaError_t rows_m(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, int64_t xs_stride,
                          const void* w, int64_t w_stride, cudaStream_t st) {
  const int tn = rows_tn(a.m);
  if (tn == 16) return rows_t<TX, TO, 16, FUSED>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
  if constexpr (!FUSED) {
    if (tn == 32) return rows_t<TX, TO, 32, false>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
    return rows_t<TX, TO, 64, false>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
  }
  return cudaErrorInvalidValue;
}

template <typename TO>
static cudaError_t rows_o(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, int64_t xs_stride,
                          const void* w, int64_t w_stride, cudaStream_t st) {
  if (!fp8_rows_fused(a)) return rows_m<TO, TO, false>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
  switch (a.x_dtype) {
    case HGA_DTYPE_F32: return rows_m<float, TO, true>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
    case HGA_DTYPE_BF16: return rows_m<__nv_bfloat16, TO, true>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
    case HGA_DTYPE_F16: return rows_m<__half, TO, true>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace tc

static bool rows_fit(const Fp8Linear& a) {
  const int64_t kb = (a.k + 127) / 128;
  return kb <= 8 * tc::kMaxSlice && (a.n + 127) / 128 <= 65535;
}

// Where the weight is read by CTAs that are all resident at once (two an SM, four along the channels) this
// kernel is ahead of the 128-row tiles, which have fewer CTAs and walk all channels in each: 128 rows of 4096
// channels into 2048 features 13.4 against 19.1 us, 64 of 2048 into 5120 11.7 against 12.9; past that
// behind: 128 of 2048 into 5120 14.9 against 13.4.
bool fp8_rows_better(const Fp8Linear& a) {
  const int tn = tc::rows_tn(a.m);
  return rows_fit(a) && (a.m <= 64 || (a.n + 127) / 128 * ((a.m + tn - 1) / tn) <= 64);
}

// Quantising inside pays as long as a CTA has no more than about 64 (row, block) pairs of its own.  Inside against
// apart: 1 x 2048 -> 5120 (4 pairs) 7.8 and 8.8 us, 8 x 4096 -> 2048 (32) 8.3 and 9.4, 4 x 8192 -> 8192 (64) 18.5 and
// 19.2, 16 x 2048 -> 5120 (64) 9.7 and 9.6, 16 x 8192 -> 1024 (128) 11.9 and 10.2, 8 x 8192 -> 8192 (128) 21.3 and 19.3,
// 16 x 8192 -> 8192 (256) 27.2 and 19.7.
bool fp8_rows_fused(const Fp8Linear& a) {
  if (a.x_dtype == HGA_DTYPE_E4M3 || a.m > 16 || !rows_fit(a)) return false;
  const int64_t kb = (a.k + 127) / 128, splits = tc::rows_splits(a.m, a.n, kb, 16);
  return a.m * ((kb + splits - 1) / splits) <= 64;
}

cudaError_t launch_fp8_rows(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, int64_t xs_stride,
                            const void* w, int64_t w_stride, cudaStream_t st) {
  switch (a.out_dtype) {
    case HGA_DTYPE_F32: return tc::rows_o<float>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
    case HGA_DTYPE_BF16: return tc::rows_o<__nv_bfloat16>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
    case HGA_DTYPE_F16: return tc::rows_o<__half>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
  }
  return cudaErrorInvalidValue;
}

HGA_DEFINE_ERROR_READER(fp8_rows_error_status)

}  // namespace hga

// Product of many rows with an e4m3 weight on the tensor cores (tcgen05 kind::f8f6f4, TMA, TMEM).
//
//   y[m][n] = sum_kb xs[m][kb] * ws[n / 128][kb] * (sum over the block's 128 channels of q[m][k] w[n][k])
//
// The scales change every 128 channels, so a block's products cannot stay in the accumulator: each
// block is one MMA group of four K = 32 steps into one of two TMEM buffers, and eight epilogue warps
// add it, scaled, to fp32 sums in registers (one fp32 FMA per output and block) while the tensor cores
// work on the next block in the other buffer.  Persistent CTAs walk the output tiles with neighbouring
// feature tiles first (their rows of x are then read from L2).  Large products run as pairs of CTAs on
// 256 x 256 tiles (cta_group::2): every CTA loads its own 128 rows and half of the features, 32 KB a block
// where a single CTA's 128 x 256 tile needs 48.
//   warp 0      TMA producer: x and w of one block per stage, STAGES deep, SW128
//   warp 1      MMA issuer (of the even CTA), TMEM owner
//   warps 4-11  each reads 32 TMEM lanes (rows) x BN / 2 columns: one row a thread, one weight block a
//               warp, so a block's scale is one product per thread
// 32768 x 2048 into 5120 features: 335 us, 2.05 PFLOP/s in a burst, the tensor pipe busy 49 % of the time.  A block
// of a 256 x 256 tile takes about 1100 cycles, its MMAs 512 of them; what the rest is spent on is not known.  It is
// not the loads (three stages instead of five, or every load from the same tile, changed nothing), mostly not the
// epilogue's reads and sums (290 us with them left out), and not a hand-over latency that more buffers would hide:
// 256 x 128 tiles in four TMEM buffers took 570 us, about 1000 cycles for half the block.
// Measured and not kept: one CTA on 128 x 256 tiles (48 KB of loads a block) 470 us, sixteen epilogue warps of 64
// columns 370 (440 with scales ahead, which spill; 395 with two more warps bringing the scales into shared
// memory), reads 32 columns ahead of the sums 400, a block's two halves of 128 features as MMAs and hand-overs of
// their own 375, arrivals with cluster-scope release 690 (a memory barrier each).
// Results go through two 4 KB pieces of swizzled shared memory per warp to whole-line TMA stores (plain stores where
// the output's rows are off the 16-byte grid).  Waits are bounded as in tc_common.cuh.
#include "fp8_common.cuh"
#include "tc_common.cuh"

namespace hga {
namespace tc {

constexpr int kEpiWarps = 8;
constexpr int kTileThreads = 128 + 32 * kEpiWarps;
constexpr int kErrFp8 = 0x40;      // codes 0x40..0x47 of the bounded waits

struct TileArgs {
  int m, n, kb, tiles_n, tiles;
  const float* xs;
  int64_t xs_stride;  // floats between rows
  int xs_vec;         // rows are 16-byte aligned and padded to whole float4
  const float* ws;
  int64_t ws_stride;
  const void* bias;
  void* out;
  int64_t out_stride;
  int tma_out;
};

// The scales of 4 blocks from block kb on (0 past the end).
__device__ __forceinline__ float4 scales4(const float* p, int kb, int n, bool vec) {
  if (vec) return kb < n ? *reinterpret_cast<const float4*>(p + kb) : make_float4(0.f, 0.f, 0.f, 0.f);
  float4 v;
  v.x = kb < n ? p[kb] : 0.f;
  v.y = kb + 1 < n ? p[kb + 1] : 0.f;
  v.z = kb + 2 < n ? p[kb + 2] : 0.f;
  v.w = kb + 3 < n ? p[kb + 3] : 0.f;
  return v;
}

// PAIR CTAs make one tile of 128 * PAIR rows x BN features; each loads its 128 rows of x and BN / PAIR
// features of w per block.
template <int BN, int PAIR, int STAGES> struct TileSmem {
  static constexpr int kA = 128 * 128, kB = BN / PAIR * 128;
  static constexpr int kStage = kA + kB;
  static constexpr int kOut = STAGES * kStage;       // 2 x 4 KB per epilogue warp
  static constexpr int kBars = kOut + kEpiWarps * 8192;
  static constexpr int kMisc = kBars + (2 * STAGES + 3) * 8;
  static constexpr int kTotal = kMisc + 32;
};

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
               "r"(smem_u32(src))
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// until the sources of all but the latest N stores of this thread have been read
template <int N> __device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// One lane of the warp, the same one every time; all lanes call.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
  if constexpr (sizeof(T) == 2) {
    const T h[2] = {Num<T>::from_f(a), Num<T>::from_f(b)};
    return *reinterpret_cast<const uint32_t*>(h);
  } else {
    return 0;
  }
}

template <typename T, int BN, int PAIR, int STAGES>
__global__ void __launch_bounds__(kTileThreads, 1)
    fp8_tiles_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ CUtensorMap tm_o, const TileArgs a) {
  using S = TileSmem<BN, PAIR, STAGES>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* full = bars;                      // the even CTA's counts the bytes of both
  uint64_t* done = bars + STAGES;             // the MMAs of a stage: its operands are free and its block is in TMEM
  uint64_t* d_empty = bars + 2 * STAGES;      // [2] the even CTA's counts the epilogue warps of both
  uint64_t* drain = bars + 2 * STAGES + 2;
  int* misc = reinterpret_cast<int*>(smem + S::kMisc);
  volatile int* abort_flag = misc;
  uint32_t* tmem_s = reinterpret_cast<uint32_t*>(misc + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = PAIR == 2 ? blockIdx.x & 1 : 0, group = blockIdx.x / PAIR, groups = gridDim.x / PAIR;

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(full + i, 1);
      mbar_init(done + i, 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(d_empty + i, kEpiWarps * PAIR);
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *abort_flag = 0;
  }
  if (warp == 1) {
    if constexpr (PAIR == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_s)),
                   "r"(2u * BN));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_s)),
                   "r"(2u * BN));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  fence_before();
  __syncthreads();
  if constexpr (PAIR == 2) cluster_sync();
  fence_after();
  const uint32_t tmem = *tmem_s;

  // registers: 384 threads x 168 at launch = 128 x 40 (the producers' group) + 256 x 232 (the epilogue: 128
  // sums, a 64-column read, the scales ahead; a spilled register would come from L2).  In the branches
  // themselves: after a join the compiler would hold every role to the smaller count.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    // The producer and MMA warps run their loops as whole warps with one elected lane issuing: the loop
    // state, addresses and descriptors are then uniform.  (From a single-lane branch every operand of an
    // MMA was moved to a uniform register first, 90 cycles an instruction.)
    const bool leader = elect_one();
    if (warp == 0) {
      int st = 0, it = 0;
      uint32_t phase = 1;  // the first round finds the stages empty
      bool ok = true;
      for (int tile = group; tile < a.tiles && ok; tile += groups) {
        const int m0 = tile / a.tiles_n * (128 * PAIR) + rank * 128, n0 = tile % a.tiles_n * BN + rank * (BN / PAIR);
        for (int kb = 0; kb < a.kb; ++kb, ++it) {
          if (it >= STAGES) ok = __all_sync(0xffffffffu, mbar_wait(done + st, phase, abort_flag, kErrFp8));
          if (!ok) break;
          if (leader) {
            unsigned char* s = smem + st * S::kStage;
            if (rank == 0) mbar_expect_tx(full + st, S::kStage * PAIR);
            if constexpr (PAIR == 2) {
              const uint32_t bar = peer_addr(full + st, 0);
              tma_load_2d_pair(s, &tm_x, kb * 128, m0, bar);
              tma_load_2d_pair(s + S::kA, &tm_w, kb * 128, n0, bar);
            } else {
              tma_load_2d(s, &tm_x, kb * 128, m0, full + st);
              tma_load_2d(s + S::kA, &tm_w, kb * 128, n0, full + st);
            }
          }
          __syncwarp();
          if (++st == STAGES) { st = 0; phase ^= 1; }
        }
      }
      // every load that was issued has landed before the shared memory is given up (the even CTA's barriers
      // count both CTAs' bytes, and no CTA leaves before the cluster's last barrier)
      if (rank == 0 && leader)
        for (int i = it > STAGES ? it - STAGES : 0; i < it; ++i) mbar_drain(full + i % STAGES, (i / STAGES) & 1);
    }
    if (warp == 1 && rank == 0) {
      constexpr uint32_t id = idesc_e4m3(BN, 128 * PAIR);
      const uint64_t dx0 = sdesc(smem_u32(smem), 16, 1024), dw0 = sdesc(smem_u32(smem) + S::kA, 16, 1024);
      int st = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = group; tile < a.tiles && ok; tile += groups) {
        for (int kb = 0; kb < a.kb; ++kb, ++it) {
          const int buf = it & 1;
          // the buffer's release comes last: it is what the loop turns on (with it first 379 against 374 us)
          ok = __all_sync(0xffffffffu, mbar_wait(full + st, phase, abort_flag, kErrFp8 + 1));
          if (it >= 2) ok = ok && __all_sync(0xffffffffu, mbar_wait(d_empty + buf, (it / 2 - 1) & 1, abort_flag, kErrFp8 + 2));
          if (!ok) break;
          fence_after();
          const uint64_t dx = dx0 + (uint64_t)(st * (S::kStage >> 4)), dw = dw0 + (uint64_t)(st * (S::kStage >> 4));
          const uint32_t d = tmem + buf * BN;
          if (leader) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // 32 bytes along the channels: 2 in the descriptor's 16-byte units
              if constexpr (PAIR == 2) mma_ss_f8_pair(d, dx + 2 * k, dw + 2 * k, id, k != 0);
              else mma_ss_f8(d, dx + 2 * k, dw + 2 * k, id, k != 0);
            }
            if constexpr (PAIR == 2) mma_commit_pair(done + st, 3); else mma_commit(done + st);
          }
          __syncwarp();
          if (++st == STAGES) { st = 0; phase ^= 1; }
        }
      }
      if (leader) {
        if constexpr (PAIR == 2) mma_commit_pair(drain, 1); else mma_commit(drain);
        mbar_drain(drain, 0);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    constexpr int COLS = BN / 2;  // columns of this warp
    const int quarter = warp & 3, part = (warp - 4) >> 2;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    unsigned char* stage = smem + S::kOut + (warp - 4) * 8192;
    const uint32_t free0 = peer_addr(d_empty, 0);
    int it = 0, st = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = group; tile < a.tiles && ok; tile += groups) {
      const int m0 = tile / a.tiles_n * (128 * PAIR) + rank * 128 + quarter * 32, n0 = tile % a.tiles_n * BN + part * COLS;
      const int row = m0 + lane;
      const float* xs = a.xs + (int64_t)(row < a.m ? row : a.m - 1) * a.xs_stride;
      const float* ws = a.ws + (int64_t)((n0 < a.n ? n0 : a.n - 1) / 128) * a.ws_stride;
      uint64_t acc[COLS / 2];
#pragma unroll
      for (int i = 0; i < COLS / 2; ++i) acc[i] = 0ull;
      // the scales of four blocks at a time, loaded four blocks before they are multiplied: with nearly all of
      // the SM's memory taken as shared memory they come from L2, and a distance of one block was too short
      float4 xn = scales4(xs, 0, a.kb, a.xs_vec), wn = scales4(ws, 0, a.kb, false), s4 = xn;
      for (int kb = 0; kb < a.kb; ++kb, ++it) {
        const int buf = it & 1;
        if ((kb & 3) == 0) {
          s4 = make_float4(xn.x * wn.x, xn.y * wn.y, xn.z * wn.z, xn.w * wn.w);
          xn = scales4(xs, kb + 4, a.kb, a.xs_vec);
          wn = scales4(ws, kb + 4, a.kb, false);
        }
        const uint64_t s2 = f32x2(s4.x, s4.x);
        s4 = make_float4(s4.y, s4.z, s4.w, s4.x);
        ok = __all_sync(0xffffffffu, mbar_wait(done + st, phase, abort_flag, kErrFp8 + 3));
        if (!ok) break;
        if (++st == STAGES) { st = 0; phase ^= 1; }
        fence_after();
        const uint32_t at = tmem + lane_addr + buf * BN + part * COLS;
#pragma unroll
        for (int c = 0; c < COLS; c += 64) {
          uint32_t r[2][32];  // two reads under way together
          HGA_LD32(at + c, r[0]);
          HGA_LD32(at + c + 32, r[1]);
          tmem_wait_ld();
          if (c + 64 == COLS) {
            fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (PAIR == 2) mbar_arrive_peer(free0 + 8 * buf); else mbar_arrive(d_empty + buf);
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              acc[c / 2 + h * 16 + i] = f32x2_fma(f32x2(__uint_as_float(r[h][2 * i]), __uint_as_float(r[h][2 * i + 1])), s2,
                                                  acc[c / 2 + h * 16 + i]);
        }
      }
      if (!ok) break;
      constexpr int PC = 128 / (int)sizeof(T);  // columns per 128-byte pass
      const T* bias = static_cast<const T*>(a.bias);
#pragma unroll
      for (int c = 0; c < COLS; c += PC) {
        if (n0 + c >= a.n || m0 >= a.m) break;  // warp-uniform
        unsigned char* stg = stage + ((c / PC) & 1) * 4096;
        if (PAIR == 2 || a.tma_out) {
          // The store that used this piece before has been read out.  Within a tile that is the store before
          // the last; a tile begins with piece 0 whichever the last tile ended with (one pass of 16-bit results in a
          // 64-column part, an odd number at a ragged edge), so its first pass waits for every store.
          if (lane == 0) {
            if (c == 0) bulk_wait_read<0>(); else bulk_wait_read<1>();
          }
          __syncwarp();
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {           // 16-byte pieces of the row's 128 bytes
          uint32_t w[4];
          if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float lo, hi;
              f32x2_get(acc[c / 2 + j * 4 + e], lo, hi);
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
              f32x2_get(acc[c / 2 + j * 2 + e], lo, hi);
              if (bias) {
                const int col = n0 + c + j * 4 + e * 2;
                lo += col < a.n ? Num<T>::to_f(bias[col]) : 0.f;
                hi += col + 1 < a.n ? Num<T>::to_f(bias[col + 1]) : 0.f;
              }
              w[2 * e] = __float_as_uint(lo);
              w[2 * e + 1] = __float_as_uint(hi);
            }
          }
          *reinterpret_cast<uint4*>(stg + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (PAIR == 2 || a.tma_out) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tm_o, stg, n0 + c, m0);
            bulk_commit();
          }
        } else {
          // rows off the 16-byte grid: whole rows of the piece, neighbouring lanes neighbouring columns
          __syncwarp();
          const int rows = a.m - m0 < 32 ? a.m - m0 : 32;
#pragma unroll
          for (int h = 0; h < PC; h += 32) {
            const int at = (h + lane) * (int)sizeof(T);
            if (n0 + c + h + lane >= a.n) break;
            T* o = static_cast<T*>(a.out) + (int64_t)m0 * a.out_stride + n0 + c + h + lane;
            for (int r = 0; r < rows; ++r, o += a.out_stride)
              *o = *reinterpret_cast<const T*>(stg + r * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 15));
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) bulk_wait_all();
  }
  fence_before();
  __syncthreads();
  if constexpr (PAIR == 2) cluster_sync();  // the pair's MMAs read both CTAs' shared memory and write both TMEMs
  fence_after();
  if (warp == 1) {
    if constexpr (PAIR == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2u * BN));
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2u * BN));
  }
}

static bool rows_on_grid(const void* p, int64_t stride) { return ((uintptr_t)p & 15) == 0 && stride % 16 == 0; }

template <typename T, int BN, int PAIR, int STAGES>
static cudaError_t tiles_t(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, int64_t xs_stride,
                           const void* w, int64_t w_stride, cudaStream_t st) {
  CUtensorMap mx, mw, mo;
  const cuuint64_t dx[2] = {(cuuint64_t)a.k, (cuuint64_t)a.m}, sx[1] = {(cuuint64_t)q_stride};
  const cuuint64_t dw[2] = {(cuuint64_t)a.k, (cuuint64_t)a.n}, sw[1] = {(cuuint64_t)w_stride};
  const cuuint32_t bx[2] = {128, 128}, bw[2] = {128, BN / PAIR};
  if (!make_map_typed(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, q, 2, dx, sx, bx, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_map_typed(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, 2, dw, sw, bw, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  const int64_t ostr = a.out_stride * (int64_t)sizeof(T);
  const bool tma_out = rows_on_grid(a.out, ostr);
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
  const int64_t tiles = (a.m + 128 * PAIR - 1) / (128 * PAIR) * t.tiles_n;
  if (tiles > 0x7fffffff) return cudaErrorInvalidValue;
  t.tiles = (int)tiles;
  t.xs = xs; t.xs_stride = xs_stride; t.xs_vec = xs_stride % 4 == 0 && ((uintptr_t)xs & 15) == 0 && xs_stride >= (t.kb + 3) / 4 * 4; t.ws = a.w_scale; t.ws_stride = a.ws_stride;
  t.bias = a.bias; t.out = a.out; t.out_stride = a.out_stride; t.tma_out = tma_out;
  constexpr int smem = TileSmem<BN, PAIR, STAGES>::kTotal + 1024;
  auto kern = fp8_tiles_kernel<T, BN, PAIR, STAGES>;
  static unsigned long long raised = 0;
  cudaError_t e = raise_smem_limit((const void*)kern, smem, &raised);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((t.tiles < 148 / PAIR ? t.tiles : 148 / PAIR) * PAIR);
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PAIR;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, mx, mw, mo, t);
}

template <typename T>
static cudaError_t tiles_n(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, int64_t xs_stride,
                           const void* w, int64_t w_stride, cudaStream_t st) {
  // 256 x 256 tiles of CTA pairs or 128 x 128 tiles of single CTAs, by the waves that the GPU's SMs take over them: a
  // wave of pairs (74 tiles) takes about 4/3 of a wave of single tiles (148, half the area), 9 against 6.7 us at
  // 2048 channels.  Measured at 2048 channels, pairs against single: 4096 x 2304 (2 waves, 4) 23.5 and 32.4 us,
  // 2304 x 2304 (2, 3) 22.3 and 24.9, 2048 x 2048 (1, 2) 14.0 and 17.9; 2432 x 1920 (2, 2) 22.2 and 18.5, 1408 x 1664
  // (1, 1) 13.3 and 10.7.  At 512 and 8192 channels the order is the same except for 2560 x 2048 x 512 (2, 3), 10.9
  // and 10.3.
  const int64_t pairs = (a.m + 255) / 256 * ((a.n + 255) / 256), singles = (a.m + 127) / 128 * ((a.n + 127) / 128);
  // (the pairs' results leave by TMA only: the plain stores' registers would spill the sums)
  if ((pairs + 73) / 74 * 4 < (singles + 147) / 148 * 3 && rows_on_grid(a.out, a.out_stride * (int64_t)sizeof(T)))
    return tiles_t<T, 256, 2, 5>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
  return tiles_t<T, 128, 1, 4>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
}

}  // namespace tc

cudaError_t launch_fp8_tiles(const Fp8Linear& a, const void* q, int64_t q_stride, const float* xs, int64_t xs_stride,
                             const void* w, int64_t w_stride, cudaStream_t st) {
  switch (a.out_dtype) {
    case HGA_DTYPE_F32: return tc::tiles_n<float>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
    case HGA_DTYPE_BF16: return tc::tiles_n<__nv_bfloat16>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
    case HGA_DTYPE_F16: return tc::tiles_n<__half>(a, q, q_stride, xs, xs_stride, w, w_stride, st);
  }
  return cudaErrorInvalidValue;
}

HGA_DEFINE_ERROR_READER(fp8_tiles_error_status)

}  // namespace hga

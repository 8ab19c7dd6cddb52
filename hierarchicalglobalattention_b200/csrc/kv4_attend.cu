// Decode attention over the 4-bit record for 16-bit caches (head_dim 64 / 128), all query heads of a KV head
// at once.
//
// A CTA serves up to 8 query heads of one KV head, 8 * NT columns of (head, new row) pairs.  It forms the
// union of the groups those heads opened, so a group is read and decoded once for all of them, and works
// in units of 16 keys on m16n8k16 matrix instructions with the keys as the 16 rows:
//   S^T [16 keys][8 columns]  = K_unit Q^T           O^T [dims][8 columns] += V_unit^T P^T
// The 8 query heads of a KV head fill the instruction's 8 columns, so decoding (not the products) is
// what a unit costs; tcgen05's 128-row tiles would be 94 % padding here.
// The record's codes are used as integers.  With n the code, (word >> 4 i) & 0x000f000f | magic is a register
// of two values 128 + n (bf16; 1024 + n in fp16), and one packed subtraction makes them n - 8, exactly:
//   q . k = sum_blocks  scale_b (sum q (n - 8)) + mid_b sum_b q,     mid_b = min_b + 8 scale_b
//   o     = sum_keys    w (n - 8) + p mid_b,                         w = p scale_b
// so keys enter the scores unrounded.  A weight's product with its block's scale is two bf16 terms, 16 bits together
// (fp16 would lose small scales to its range), as are the weights of the exact rows in the cache's type: with one
// bf16 term the results of bf16 caches were up to 38 % further from 64 bits than fp32 arithmetic's, at 26.4 us
// against 28.0 for 16 sequences of 32768 and 30.7 against 32.4 for a block of 64 rows.  The mid terms are fp32 sums
// beside the products.  bf16 scores leave the 128 in the products and take 128 sum q off instead; with fp16's 1024
// that cost up to 1 % of a score (the instruction truncates its sums relative to their largest term), and in the
// output, whose sum runs over all keys, a bf16 ulp.
//
// Units are dealt to the warps of the `splits` CTAs of a cluster (windows and the active chunk first,
// then the union); every warp keeps its own online softmax and copies its next units with cp.async (plain
// loads for records in pinned host memory, where asynchronous copies are slower).  Warps join in shared
// memory, CTAs through distributed shared memory, in a fixed order: no atomics on results, one launch.
// One token for each of 16 sequences of 32768 (32 heads over 4): 28 us for 63 MB (2.25 TB/s).  No single limit is
// near: 24 % of DRAM's rate, 40 % of the SMs' issue.  While warps are resident half of the issue slots are empty; the
// four warps a scheduler has at most wait for fixed latencies, the math pipes, loads and barriers in turn (1.2, 0.8,
// 0.7 and 0.6 cycles an issued instruction).  One sequence is set-up and the two cluster barriers (9 us together): 10.5 us at
// 4100 tokens.  One pass over keys per query head with plain FMAs took 566 and 398 us.
#include <cooperative_groups.h>

#include "fp32x2.cuh"
#include "kv4_common.cuh"

namespace hga {

HGA_DEVICE_ERROR_WORD(g_kv4_mma_error, kv4_attend_error_status)

namespace kv4 {

namespace cg = cooperative_groups;

// warps of a CTA and CTAs an SM: with 8 columns a warp's state fits 128 registers, with 16 it takes 168
__host__ __device__ constexpr int warps_of(int nt) { return nt == 1 ? 8 : 4; }
__host__ __device__ constexpr int ctas_of(int nt) { return nt == 1 ? 2 : 3; }
constexpr int kStages = 4;          // record units in flight per warp
constexpr int kNever = 255;         // t0 of a (unit, head) that does not see the unit

template <int DH> struct Buf {
  static constexpr int kUnit = 20 * DH;                                          // K and V of a record unit
  static constexpr int kHot = 2 * 16 * DH * 2;                                   // K and V rows of a slot unit
  // the last stage lies behind the slot unit's rows: the first record unit is on its way while those are attended
  static constexpr int kRing = kHot - (kStages - 1) * kUnit;                     // offset of stage 0
  static constexpr int kWarp = kRing + kStages * kUnit;
  static_assert(kRing >= 0 && kRing % 16 == 0 && kWarp - kUnit >= kHot, "stage kStages - 1 is clear of the slot rows");
};

struct Args {
  int L, Kg, splits, rep, hpc, tiles, hash_bits, direct;  // hpc: query heads of a CTA
  const void *q, *hot_k, *hot_v;
  const uint8_t *rec_k, *rec_v;
  const int32_t *seq_pos, *open_gid, *open_t0;
  int64_t hot_cap, unit_cap;
  void* out;
};

template <typename T> struct Half2;
template <> struct Half2<__nv_bfloat16> {
  using V2 = __nv_bfloat162;
  static constexpr uint32_t kMagic = 0x43004300u, kMid = 0x43084308u;  // 128 and 136 twice
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
  }
  static __device__ __forceinline__ uint32_t pack_down(float a, float b) {  // towards zero
    uint32_t r;
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
  }
  static constexpr float kTiny = 1.17549435e-38f;  // 2^-126, the smallest normal
  static constexpr uint32_t kInf = 0x7f80u;
};
template <> struct Half2<__half> {
  using V2 = __half2;
  static constexpr uint32_t kMagic = 0x64006400u, kMid = 0x64086408u;  // 1024 and 1032 twice
  static __device__ __forceinline__ float lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)w)); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
  }
  static __device__ __forceinline__ uint32_t pack_down(float a, float b) {  // towards zero
    uint32_t r;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
  }
  static constexpr float kTiny = 5.9604645e-8f;  // 2^-24, the smallest subnormal
  static constexpr uint32_t kInf = 0x7c00u;
};
using BF = Half2<__nv_bfloat16>;

// the i-th operand register (codes - 8) of a word of the record
template <typename H>
__device__ __forceinline__ uint32_t codes(uint32_t word, int i) {
  const uint32_t a = (word >> (4 * i) & 0x000f000fu) | H::kMagic, mid = H::kMid;
  const typename H::V2 v = __hsub2(*reinterpret_cast<const typename H::V2*>(&a),
                                   *reinterpret_cast<const typename H::V2*>(&mid));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// whether the scale or the minimum of a word is not finite
template <typename H>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  return ((w >> 16) & H::kInf) == H::kInf || (w & H::kInf) == H::kInf;
}

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (Half2<T>::kInf == 0x7f80u)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void copy16(void* dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(read ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// Shared memory: the warps' copy buffers (afterwards their partial results), then the union's tables.
template <int DH, int NT> struct Layout {
  static constexpr int kWarps = warps_of(NT);
  static constexpr int kOut = DH * 8 * NT * 4;                       // one partial O^T, fp32
  static constexpr int kRing = kWarps * Buf<DH>::kWarp;
  static constexpr int kPart = kWarps * kOut + 8 * NT * (DH + 4) * 4 + (kWarps + 1) * 2 * 8 * NT * 4;
  static constexpr int kQ = kRing > kPart ? kRing : kPart;           // [NT][DH/16][32] uint2: Q as B fragments
  static constexpr int kScratch = kQ + NT * (DH / 16) * 32 * 8;      // [warps][16][8 NT] fp32 weights (rare path)
  static constexpr int kMisc = kScratch + kWarps * 16 * 8 * NT * 4;
  static constexpr int kTables = kMisc + 64;
};

static size_t table_bytes(int hr, int Kg, int hash_bits) {
  const size_t n = (size_t)hr * Kg;
  return (size_t)3 * (4u << hash_bits) + n * 4 + n * 4 + n * hr + 16;
}

template <typename T, int DH, int NT>
__global__ void __launch_bounds__(warps_of(NT) * 32, ctas_of(NT)) attend_kv4_mma_kernel(const hga_params p, const Args a) {
  using H = Half2<T>;
  using LY = Layout<DH, NT>;
  constexpr int kWarps = LY::kWarps;
  constexpr int KS = DH / 16, NB = DH / 32, COLS = 8 * NT;
  // what the keys' codes have in the products besides themselves: 8 off (n - 8), or 128 on (bf16 keeps it:
  // 128 sum q is taken off in fp32 with an error of 1e-5 of a score)
  constexpr bool FP16 = H::kInf != 0x7f80u;
  constexpr float kOffK = FP16 ? 8.f : -128.f;
  extern __shared__ __align__(128) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int rank = blockIdx.x, bk = blockIdx.y, b = bk / p.kv_heads, kvh = bk % p.kv_heads;
  const int hb = blockIdx.z / a.tiles, tile = blockIdx.z % a.tiles;
  const int hr = a.rep - hb * a.hpc < a.hpc ? a.rep - hb * a.hpc : a.hpc;  // heads of this CTA
  const int h0 = kvh * a.rep + hb * a.hpc;
  const int x0 = tile * COLS, ncols = hr * a.L - x0 < COLS ? hr * a.L - x0 : COLS;
  const int C = p.chunk_size, U = p.group_size / kKv4Unit, L = a.L, Kg = a.Kg;
  const int kf = p.keep_first > 0 ? p.keep_first : 0, kl = p.keep_last > 0 ? p.keep_last : 0;
  int* misc = reinterpret_cast<int*>(smem + LY::kMisc);

  cg::cluster_group cl = cg::this_cluster();
  // the first entries of the heads' lists (all of them for 64 groups and 8 heads), asked
  // for before anything waits for the sequence's position
  const int N = hr * Kg, hsize = 1 << a.hash_bits;
  const size_t list0 = ((size_t)b * p.nhead + h0) * Kg;
  constexpr int kEarly = 512 / (kWarps * 32);
  int e_gid[kEarly], e_t0[kEarly];
#pragma unroll
  for (int j = 0; j < kEarly; ++j) {
    const int i = tid + j * kWarps * 32;
    e_gid[j] = ncols > 0 && i < N ? a.open_gid[list0 + i] : -1;
    e_t0[j] = ncols > 0 && i < N ? a.open_t0[list0 + i] : -1;
  }
  if (ncols <= 0) return;  // the whole cluster: a smaller last head block has fewer tiles
  const int pos = a.seq_pos[b];
  const int n_closed = pos / C, c0 = pos % C;
  T* out = static_cast<T*>(a.out);
  if (pos < 0 || c0 + L > C || (int64_t)(kf + kl + 1) * C > a.hot_cap) {
    if (tid == 0) atomicCAS(&g_kv4_mma_error, 0, kErrBoundsAttendKv4);
    if (rank == 0)
      for (int i = tid; i < ncols * DH; i += kWarps * 32) {
        const int x = x0 + i / DH;
        out[(((size_t)b * p.nhead + h0 + x % hr) * L + x / hr) * DH + i % DH] = Num<T>::from_f(0.f);
      }
    return;  // cluster-uniform
  }
  int f_hi, l_lo;
  windows(n_closed, kf, kl, f_hi, l_lo);
  const int wu = C / kKv4Unit;
  const int t_last = (x0 + ncols - 1) / hr;
  const int n_first = f_hi * wu, n_last = (n_closed - l_lo) * wu;
  const int nact = c0 + t_last + 1, n_hot = n_first + n_last + (nact + kKv4Unit - 1) / kKv4Unit;
  const int me = rank * kWarps + warp, stride = a.splits * kWarps;

  unsigned char* buf = smem + warp * Buf<DH>::kWarp;
  const size_t hot_base = (size_t)bk * a.hot_cap * DH;
  const T* hk = static_cast<const T*>(a.hot_k) + hot_base;
  const T* hv = static_cast<const T*>(a.hot_v) + hot_base;

  // slot unit i: first row and number of rows that some column sees
  auto hot_unit = [&](int i, int& rows, int& act) -> int64_t {
    rows = kKv4Unit;
    act = -1;
    if (i < n_first) return (int64_t)i * kKv4Unit;
    i -= n_first;
    if (i < n_last) return (int64_t)(kf + (l_lo + i / wu) % (kl > 0 ? kl : 1)) * C + (i % wu) * kKv4Unit;
    act = (i - n_last) * kKv4Unit;
    if (nact - act < rows) rows = nact - act;
    return (int64_t)(kf + kl) * C + act;
  };
  // 16-byte piece j of row r at piece j ^ (r & 7): conflict-free ldmatrix
  auto issue_hot = [&](int i) {
    int rows, act;
    const int64_t row = hot_unit(i, rows, act);
    constexpr int PR = DH / 8;
#pragma unroll
    for (int j = lane; j < 16 * PR; j += 32) {
      const int r = j / PR, pc = j % PR, dst = r * DH * 2 + ((pc ^ (r & 7)) << 4);
      const bool read = r < rows;  // rows past the block hold an earlier sequence's values: zeros instead
      const int64_t at = (row + (read ? r : 0)) * DH + pc * 8;
      copy16(buf + dst, hk + at, read);
      copy16(buf + 16 * DH * 2 + dst, hv + at, read);
    }
    copy_commit();
  };
  if (me < n_hot) issue_hot(me);

  // ---- Q as B fragments -------------------------------------------------------------------------
  uint2* qf = reinterpret_cast<uint2*>(smem + LY::kQ);
  const T* q = static_cast<const T*>(a.q);
  for (int i = tid; i < NT * KS * 32; i += kWarps * 32) {
    const int ln = i & 31, ks = (i >> 5) % KS, nt = (i >> 5) / KS;
    const int x = nt * 8 + (ln >> 2);
    uint2 v = make_uint2(0u, 0u);
    if (x < ncols) {
      const int xx = x0 + x;
      const T* row = q + (((size_t)b * p.nhead + h0 + xx % hr) * L + xx / hr) * DH + ks * 16 + 2 * (ln & 3);
      v.x = *reinterpret_cast<const uint32_t*>(row);
      v.y = *reinterpret_cast<const uint32_t*>(row + 8);
    }
    qf[i] = v;
  }

  // ---- union of the heads' opened groups --------------------------------------------------------
  int* keys = reinterpret_cast<int*>(smem + LY::kTables);  // [hsize] group, -1 empty
  int* own = keys + hsize;                                 // [hsize] first entry that names it
  int* rnk = own + hsize;                                  // [hsize] its place in the union
  int* slot = rnk + hsize;                                 // [N] hash slot of an entry, -1 skipped
  int* ugid = slot + N;                                    // [N] the union's groups
  uint8_t* ut0 = reinterpret_cast<uint8_t*>(ugid + N);     // [N][hr] first row that sees it
  int* wcnt = misc;                                        // [2][warps]
  for (int i = tid; i < hsize; i += kWarps * 32) {
    keys[i] = -1;
    own[i] = 0x7fffffff;
  }
  for (int i = tid; i < N * hr; i += kWarps * 32) ut0[i] = kNever;
  __syncthreads();
  auto insert = [&](int i, int gid, int t0) {
    int s = -1;
    if (gid >= 0 && t0 >= 0 && t0 <= t_last) {
      if (((int64_t)gid + 1) * U > a.unit_cap) {
        atomicCAS(&g_kv4_mma_error, 0, kErrBoundsAttendKv4);
      } else {
        s = (int)((uint32_t)gid * 2654435761u >> (32 - a.hash_bits));
        while (true) {  // at most N of the hsize >= 2 N slots are taken: an empty one is met
          const int old = atomicCAS(&keys[s], -1, gid);
          if (old == -1 || old == gid) break;
          s = (s + 1) & (hsize - 1);
        }
        atomicMin(&own[s], i);
      }
    }
    slot[i] = s;
  };
#pragma unroll
  for (int j = 0; j < kEarly; ++j)
    if (tid + j * kWarps * 32 < N) insert(tid + j * kWarps * 32, e_gid[j], e_t0[j]);
  for (int i = tid + kEarly * kWarps * 32; i < N; i += kWarps * 32) insert(i, a.open_gid[list0 + i], a.open_t0[list0 + i]);
  __syncthreads();
  // places in the order of the first entries (the same in every run, whatever slot the hash gave)
  int n_open = 0;
  for (int base = 0; base < N; base += 2 * kWarps * 32) {  // two entries a thread and round
    bool first[2];
    unsigned bal[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = base + j * kWarps * 32 + tid;
      first[j] = i < N && slot[i] >= 0 && own[slot[i]] == i;
      bal[j] = __ballot_sync(0xffffffffu, first[j]);
      if (lane == 0) wcnt[j * kWarps + warp] = __popc(bal[j]);
    }
    __syncthreads();
    int before[2] = {n_open, n_open};
#pragma unroll
    for (int w = 0; w < 2 * kWarps; ++w) {
      const int x = wcnt[w];
      if (w < warp) before[0] += x;
      if (w < kWarps + warp) before[1] += x;
      n_open += x;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (first[j]) {
        const int sl = slot[base + j * kWarps * 32 + tid], r = before[j] + __popc(bal[j] & ((1u << lane) - 1u));
        rnk[sl] = r;
        ugid[r] = keys[sl];
      }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < kEarly; ++j) {
    const int i = tid + j * kWarps * 32;
    if (i < N && slot[i] >= 0) ut0[rnk[slot[i]] * hr + i / Kg] = (uint8_t)e_t0[j];
  }
  for (int i = tid + kEarly * kWarps * 32; i < N; i += kWarps * 32)
    if (slot[i] >= 0) ut0[rnk[slot[i]] * hr + i / Kg] = (uint8_t)a.open_t0[list0 + i];
  __syncthreads();

  // ---- this lane's columns ------------------------------------------------------------------------
  int col_h[NT][2], col_t[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      int x = nt * 8 + 2 * c + e;
      if (x >= ncols) x = ncols - 1;  // a padding column: its query is zero and its result is not written
      col_h[nt][e] = (x0 + x) % hr;
      col_t[nt][e] = (x0 + x) / hr;
    }
  float o[KS][NT][4], m[NT][2], l[NT][2], corr[NB][NT][2], qsum[NB][NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[nt][e] = -INFINITY;
      l[nt][e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      corr[i][nt][0] = corr[i][nt][1] = 0.f;
      // sums of q over a block's channels, in the layout of the scores: a product with ones
      const uint32_t one = H::pack(1.f, 1.f);
      const uint32_t ones[4] = {one, one, one, one};
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint2 v = qf[(nt * KS + 2 * i + k) * 32 + lane];
        mma<T>(s, ones, v.x, v.y);
      }
      qsum[i][nt][0] = s[0];
      qsum[i][nt][1] = s[1];
    }
  }
  const float sl2 = p.scale * 1.4426950408889634f;

  // Scores s[nt][4] (keys g, g, g + 8, g + 8; columns 2c, 2c + 1) to weights against the running maxima;
  // vis: bit i for s[nt][i].  The maximum is raised, and the sums rescaled, only when a weight could
  // pass 2^8.
  auto soften = [&](float (&s)[NT][4], const unsigned (&vis)[NT]) {
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[nt][e] *= sl2;
        if ((vis[nt] >> e & 1) && s[nt][e] > m[nt][e & 1] + 8.f) grow = true;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(vis[nt] >> e & 1 ? s[nt][e] : -INFINITY, vis[nt] >> (e + 2) & 1 ? s[nt][e + 2] : -INFINITY);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
          x = fmaxf(x, m[nt][e]);
          const float f = m[nt][e] == -INFINITY ? 0.f : ex2(m[nt][e] - x);
          m[nt][e] = x;
          l[nt][e] *= f;
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            o[i][nt][e] *= f;
            o[i][nt][e + 2] *= f;
          }
#pragma unroll
          for (int i = 0; i < NB; ++i) corr[i][nt][e] *= f;
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // a maximum of -infinity: only such scores so far, whose weight is 0 (a NaN stays one)
        s[nt][e] = vis[nt] >> e & 1 ? ex2(s[nt][e] - (m[nt][e & 1] == -INFINITY ? 0.f : m[nt][e & 1])) : 0.f;
        l[nt][e & 1] += s[nt][e];
      }
  };

  // ---- copies of opened groups ---------------------------------------------------------------------------------
  // the warps go on where the slot units' deal ended, so that one extra slot unit is paid back here
  const int n_units = n_open * U;
  const int start = (me + stride - n_hot % stride) % stride;
  const size_t rec_base = (size_t)bk * a.unit_cap * kv4_unit_bytes(DH);
  constexpr int QUADS = DH / 64;
  // a lane copies the code words that it will read itself, and one 16-byte piece of the (scale, min) pairs
  auto issue_rec = [&](int u, int st) {
    const int64_t unit = U == 1 ? (int64_t)ugid[u] : (int64_t)ugid[u / U] * U + u % U;
    const uint8_t* ks = a.rec_k + rec_base + unit * kv4_unit_bytes(DH);
    const uint8_t* vs = a.rec_v + rec_base + unit * kv4_unit_bytes(DH);
    unsigned char* d = buf + Buf<DH>::kRing + st * Buf<DH>::kUnit;
    constexpr int MP = DH / 8;  // 16-byte pieces of one operand's pairs
    const uint8_t* ms = lane < MP ? ks + 8 * DH + lane * 16 : vs + 8 * DH + (lane - MP) * 16;
    unsigned char* md = lane < MP ? d + 8 * DH + lane * 16 : d + 18 * DH + (lane - MP) * 16;
    if (!a.direct) {
#pragma unroll
      for (int j = 0; j < QUADS; ++j) {
        copy16(d + (j * 32 + lane) * 16, ks + (j * 32 + lane) * 16, true);
        copy16(d + 10 * DH + (j * 32 + lane) * 16, vs + (j * 32 + lane) * 16, true);
      }
      if (lane < 2 * MP) copy16(md, ms, true);
    } else {
      uint4 x[2 * QUADS + 1];
#pragma unroll
      for (int j = 0; j < QUADS; ++j) {
        x[2 * j] = load16(ks + (j * 32 + lane) * 16);
        x[2 * j + 1] = load16(vs + (j * 32 + lane) * 16);
      }
      if (lane < 2 * MP) x[2 * QUADS] = load16(ms);
#pragma unroll
      for (int j = 0; j < QUADS; ++j) {
        *reinterpret_cast<uint4*>(d + (j * 32 + lane) * 16) = x[2 * j];
        *reinterpret_cast<uint4*>(d + 10 * DH + (j * 32 + lane) * 16) = x[2 * j + 1];
      }
      if (lane < 2 * MP) *reinterpret_cast<uint4*>(md) = x[2 * QUADS];
    }
  };
  if (start < n_units) issue_rec(start, kStages - 1);
  copy_commit();

  // ---- windows and the active chunk -----------------------------------------------------------------
  for (int i = me; i < n_hot; i += stride) {
    if (i == me) copy_wait<1>(); else copy_wait<0>();  // the first was issued before the record's first unit
    __syncwarp();
    int rows, act;
    hot_unit(i, rows, act);
    const uint32_t kb = smem_addr(buf), vb = kb + 16 * DH * 2;
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
    const int kr = lane & 15;                               // K: rows 0-15, then the same rows 8 channels on
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t f[4];
      ldmatrix4<false>(f, kb + kr * DH * 2 + (((ks * 2 + (lane >> 4)) ^ (kr & 7)) << 4));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint2 v = qf[(nt * KS + ks) * 32 + lane];
        mma<T>(s[nt], f, v.x, v.y);
      }
    }
    unsigned vis[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      vis[nt] = 15u;
      if (act >= 0) {
        vis[nt] = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (act + g + 8 * (e >> 1) <= c0 + col_t[nt][e & 1]) vis[nt] |= 1u << e;
      }
    }
    soften(s, vis);
    // The weights as two 16-bit terms: these rows are exact, and one term alone would keep 8 significant bits
    // (bf16) of every weight.  The first is rounded towards zero and the second is kept above zero, so that
    // a value of infinity meets two positive factors (infinity - infinity is not what it stands for).  With one term
    // the 64-row block took 30.0 us instead of 30.7, 16 sequences of 32768 26.2 instead of 26.4.
    uint32_t pb[NT][2], pl[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float s0 = s[nt][2 * r], s1 = s[nt][2 * r + 1];
        const uint32_t w = H::pack_down(s0, s1);
        pl[nt][r] = transpose8(H::pack(fmaxf(s0 - H::lo(w), fminf(s0, H::kTiny)), fmaxf(s1 - H::hi(w), fminf(s1, H::kTiny))));
        pb[nt][r] = transpose8(w);
      }
    // V^T: tokens 0-7 (lanes 0-15) and 8-15, channels 0-7 and 8-15 of each 16
    const int vr = (lane & 7) + ((lane >> 4) << 3);
    bool odd = false;
    if (act >= 0 && L > 1) {
      // a row that some columns do not see yet: a weight of 0 times an infinity or a NaN is not 0
      for (int j = lane; j < 16 * DH / 2; j += 32) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(buf + 16 * DH * 2)[j];
        odd |= (w & H::kInf) == H::kInf || (w >> 16 & H::kInf) == H::kInf;
      }
      odd = __any_sync(0xffffffffu, odd);
    }
    if (odd) {
      // such values by plain sums for the columns that see their rows, then zeros in their place: a product of 0
      // either way for the other columns, whose bits do not change
      float* w = reinterpret_cast<float*>(smem + LY::kScratch) + warp * 16 * COLS;  // [16 keys][COLS], -1 = unseen
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[(g + 8 * (e >> 1)) * COLS + nt * 8 + 2 * c + (e & 1)] = vis[nt] >> e & 1 ? s[nt][e] : -1.f;
      __syncwarp();
      for (int key = 0; key < rows; ++key)
#pragma unroll
        for (int mt = 0; mt < KS; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int ch = mt * 16 + g + 8 * (e >> 1);
            const float v = Num<T>::to_f(*reinterpret_cast<const T*>(buf + 16 * DH * 2 + key * DH * 2 +
                                                                      (((ch >> 3) ^ (key & 7)) << 4) + (ch & 7) * 2));
            if (fabsf(v) < INFINITY) continue;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float x = w[key * COLS + nt * 8 + 2 * c + (e & 1)];
              if (!(x < 0.f)) o[mt][nt][e] = fmaf(x, v, o[mt][nt][e]);
            }
          }
      __syncwarp();
      for (int j = lane; j < 16 * DH / 2; j += 32) {
        uint32_t* at = reinterpret_cast<uint32_t*>(buf + 16 * DH * 2) + j;
        const uint32_t v = *at;
        *at = ((v & H::kInf) == H::kInf ? 0u : v & 0xffffu) | ((v >> 16 & H::kInf) == H::kInf ? 0u : v & 0xffff0000u);
      }
      __syncwarp();
    }
#pragma unroll
    for (int mt = 0; mt < KS; ++mt) {
      uint32_t f[4];
      ldmatrix4<true>(f, vb + vr * DH * 2 + (((mt * 2 + (lane >> 3 & 1)) ^ (vr & 7)) << 4));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma<T>(o[mt][nt], f, pb[nt][0], pb[nt][1]);
        mma<T>(o[mt][nt], f, pl[nt][0], pl[nt][1]);
      }
    }
    __syncwarp();
    if (i + stride < n_hot) issue_hot(i + stride);
  }

  // ---- opened groups ---------------------------------------------------------------------------------
#pragma unroll
  for (int i = 1; i < kStages - 1; ++i) {
    if (start + i * stride < n_units) issue_rec(start + i * stride, i - 1);
    copy_commit();
  }
  int st = kStages - 1;
  for (int u = start; u < n_units; u += stride) {
    copy_wait<kStages - 2>();
    __syncwarp();
    const unsigned char* d = buf + Buf<DH>::kRing + st * Buf<DH>::kUnit;
    {
      const int un = u + (kStages - 1) * stride;
      if (un < n_units) issue_rec(un, (st + kStages - 1) % kStages);
      copy_commit();
    }
    st = (st + 1) % kStages;
    // scores
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
    uint32_t km[2][NB];  // (scale, min) of keys g and g + 8
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int j = 0; j < NB; j += 2) {
        const uint2 w = *reinterpret_cast<const uint2*>(d + 8 * DH + ((g + 8 * r) * NB + j) * 4);
        km[r][j] = w.x;
        km[r][j + 1] = w.y;
      }
#pragma unroll
    for (int quad = 0; quad < QUADS; ++quad) {
      const uint4 w4 = *reinterpret_cast<const uint4*>(d + (quad * 32 + lane) * 16);
      const uint32_t word[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int hb2 = 0; hb2 < 2; ++hb2) {
        const int blk = quad * 2 + hb2;
        float acc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[nt][e] = 0.f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t f[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] = FP16 ? codes<H>(word[hb2 * 2 + k], e) : (word[hb2 * 2 + k] >> (4 * e) & 0x000f000fu) | H::kMagic;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint2 v = qf[(nt * KS + blk * 2 + k) * 32 + lane];
            mma<T>(acc[nt], f, v.x, v.y);
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float sc = H::lo(km[r][blk]), mid = fmaf(kOffK, sc, H::hi(km[r][blk]));
          const uint64_t sc2 = f32x2(sc, sc), mid2 = f32x2(mid, mid);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint64_t q2 = f32x2(qsum[blk][nt][0], qsum[blk][nt][1]);
            f32x2_get(f32x2_fma(sc2, f32x2(acc[nt][2 * r], acc[nt][2 * r + 1]),
                                f32x2_fma(mid2, q2, f32x2(s[nt][2 * r], s[nt][2 * r + 1]))),
                      s[nt][2 * r], s[nt][2 * r + 1]);
          }
        }
      }
    }
    unsigned vis[NT];
    const uint8_t* t0 = ut0 + (U == 1 ? u : u / U) * hr;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      vis[nt] = (col_t[nt][0] >= t0[col_h[nt][0]] ? 5u : 0u) | (col_t[nt][1] >= t0[col_h[nt][1]] ? 10u : 0u);
    soften(s, vis);
    // values; odd: a block of the unit reads back as NaN, which columns that do not see the unit must not meet
    const unsigned char* dv = d + 10 * DH;
    bool odd = false;
    if (lane < NB * 4) {
      const uint4 m4 = *reinterpret_cast<const uint4*>(dv + 8 * DH + lane * 16);
      odd = not_finite<H>(m4.x) | not_finite<H>(m4.y) | not_finite<H>(m4.z) | not_finite<H>(m4.w);
    }
    odd = __any_sync(0xffffffffu, odd);
#pragma unroll
    for (int quad = 0; quad < QUADS; ++quad) {
      const uint4 w4 = *reinterpret_cast<const uint4*>(dv + (quad * 32 + lane) * 16);
      const uint32_t word[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int hb2 = 0; hb2 < 2; ++hb2) {
        const int blk = quad * 2 + hb2;
        uint32_t wb[NT][2], wl[NT][2];  // weight x scale as two bf16 terms
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t vm = *reinterpret_cast<const uint32_t*>(dv + 8 * DH + ((g + 8 * r) * NB + blk) * 4);
          const float sc = H::lo(vm), mid = fmaf(8.f, sc, H::hi(vm));
          const uint64_t sc2 = f32x2(sc, sc), mid2 = f32x2(mid, mid);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint64_t p2 = f32x2(s[nt][2 * r], s[nt][2 * r + 1]);
            float w0, w1, d0, d1;
            f32x2_get(f32x2_mul(p2, sc2), w0, w1);
            f32x2_get(f32x2_fma(p2, mid2, f32x2(corr[blk][nt][0], corr[blk][nt][1])), d0, d1);
            if (odd) {  // an unseen key's scale and minimum do not count, whatever they hold
              const bool v0 = vis[nt] & 1u, v1 = vis[nt] & 2u;
              w0 = v0 ? w0 : 0.f;
              w1 = v1 ? w1 : 0.f;
              d0 = v0 ? d0 : corr[blk][nt][0];
              d1 = v1 ? d1 : corr[blk][nt][1];
            }
            corr[blk][nt][0] = d0;
            corr[blk][nt][1] = d1;
            const uint32_t w = BF::pack(w0, w1);
            wl[nt][r] = transpose8(BF::pack(w0 - BF::lo(w), w1 - BF::hi(w)));
            wb[nt][r] = transpose8(w);
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t f[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] = codes<BF>(word[hb2 * 2 + k], e);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma<__nv_bfloat16>(o[blk * 2 + k][nt], f, wb[nt][0], wb[nt][1]);
            mma<__nv_bfloat16>(o[blk * 2 + k][nt], f, wl[nt][0], wl[nt][1]);
          }
        }
      }
    }
    __syncwarp();
  }
  copy_wait<0>();

  // ---- join the warps, then the cluster's CTAs ---------------------------------------------------------
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], d);
#pragma unroll
        for (int i = 0; i < NB; ++i) corr[i][nt][e] += __shfl_xor_sync(0xffffffffu, corr[i][nt][e], d);
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        o[i][nt][e] += corr[i / 2][nt][e];
        o[i][nt][e + 2] += corr[i / 2][nt][e];
      }
    }
  __syncthreads();  // the copy buffers become the partial results
  float* part = reinterpret_cast<float*>(smem);                 // [warps][DH][COLS], then the CTA's [COLS][DH + 4]
  float* pm = part + kWarps * DH * COLS + COLS * (DH + 4);       // [warps + 1][COLS] maxima
  float* pl = pm + (kWarps + 1) * COLS;                         // [warps + 1][COLS] sums
#pragma unroll
  for (int i = 0; i < KS; ++i)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        *reinterpret_cast<float2*>(part + (warp * DH + i * 16 + g + 8 * r) * COLS + nt * 8 + 2 * c) =
            make_float2(o[i][nt][2 * r], o[i][nt][2 * r + 1]);
  if (g == 0)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        pm[warp * COLS + nt * 8 + 2 * c + e] = m[nt][e];
        pl[warp * COLS + nt * 8 + 2 * c + e] = l[nt][e];
      }
  __syncthreads();
  if (tid < COLS) {
    float mx = -INFINITY, sum = 0.f;
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, pm[w * COLS + tid]);
    for (int w = 0; w < kWarps; ++w) {
      // a maximum of -infinity: nothing seen (sum 0), or only scores that are NaN (sum NaN)
      const float mw = pm[w * COLS + tid], lw = pl[w * COLS + tid], f = mw == -INFINITY ? lw : ex2(mw - mx);
      sum += f * lw;
      pm[w * COLS + tid] = f;  // the warp's factor
    }
    pm[kWarps * COLS + tid] = mx;
    pl[kWarps * COLS + tid] = sum;
  }
  __syncthreads();
  constexpr int MS = DH + 4;  // the CTA's result, [COLS][MS]: channels next to one another
  float* mine = part + kWarps * DH * COLS;
  for (int i = tid; i < DH * COLS; i += kWarps * 32) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = pm[w * COLS + i % COLS];
      s += f == 0.f ? 0.f : f * part[w * DH * COLS + i];
    }
    mine[(i % COLS) * MS + i / COLS] = s;
  }
  if (a.splits > 1) cl.sync(); else __syncthreads();
  // this CTA's share of the channels, the CTAs' results in rank order (all of an element's reads in flight
  // together: one after the other they took as long as the attention of a short context)
  const int lo = DH * rank / a.splits, width = DH * (rank + 1) / a.splits - lo;
  for (int i = tid; i < width * ncols; i += kWarps * 32) {
    const int col = i / width, ch = lo + i % width;
    float mr[8], lr[8], vr[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (r >= a.splits) break;
      const float* rm = a.splits > 1 ? cl.map_shared_rank(pm, r) : pm;
      mr[r] = rm[kWarps * COLS + col];
      lr[r] = rm[(2 * kWarps + 1) * COLS + col];  // pl follows pm
      vr[r] = (a.splits > 1 ? cl.map_shared_rank(mine, r) : mine)[col * MS + ch];
    }
    float mx = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < a.splits) mx = fmaxf(mx, mr[r]);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (r >= a.splits) break;
      const float f = mr[r] == -INFINITY ? lr[r] : ex2(mr[r] - mx);
      sum += f * lr[r];  // with a factor of 0 too: a sum that is NaN is not lost
      if (f == 0.f) continue;
      acc += f * vr[r];
    }
    const int x = x0 + col;
    out[(((size_t)b * p.nhead + h0 + x % hr) * L + x / hr) * DH + ch] = Num<T>::from_f(acc / sum);
  }
  if (a.splits > 1) cl.sync();  // no CTA leaves while another still reads its sums
}

template <typename T, int DH, int NT>
static cudaError_t launch_t(const hga_params& p, Args a, cudaStream_t st) {
  const int hr = a.hpc, heads_blk = (a.rep + hr - 1) / hr;
  a.tiles = (hr * a.L + 8 * NT - 1) / (8 * NT);
  a.hash_bits = 5;
  while ((1 << a.hash_bits) < 2 * hr * a.Kg) ++a.hash_bits;
  const size_t smem = Layout<DH, NT>::kTables + table_bytes(hr, a.Kg, a.hash_bits);
  if (smem > 227 * 1024) return cudaErrorNotSupported;
  const int64_t z = (int64_t)heads_blk * a.tiles;
  if (z > 65535 || (int64_t)p.batch * p.kv_heads > 65535) return cudaErrorNotSupported;
  auto kern = attend_kv4_mma_kernel<T, DH, NT>;
  static unsigned long long raised = 0;
  cudaError_t e = raise_smem_limit((const void*)kern, 227 * 1024, &raised);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.splits, p.batch * p.kv_heads, (unsigned)z);
  cfg.blockDim = dim3(warps_of(NT) * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p, a);
}

}  // namespace kv4

// cudaErrorNotSupported: the shape is the portable kernel's
cudaError_t launch_attend_kv4_mma(const hga_params& p, int L, const void* q, const int32_t* seq_pos, const void* hk,
                                  const void* hv, int64_t hot_cap, const void* rec_k, const void* rec_v,
                                  int64_t unit_cap, const int32_t* og, const int32_t* ot, int Kg, void* out,
                                  cudaStream_t st) {
  if ((p.dtype != HGA_DTYPE_BF16 && p.dtype != HGA_DTYPE_F16) || (p.head_dim != 64 && p.head_dim != 128))
    return cudaErrorNotSupported;
  kv4::Args a = {};
  a.L = L; a.Kg = Kg; a.rep = p.nhead / p.kv_heads;
  a.q = q; a.hot_k = hk; a.hot_v = hv; a.rec_k = (const uint8_t*)rec_k; a.rec_v = (const uint8_t*)rec_v;
  a.seq_pos = seq_pos; a.open_gid = og; a.open_t0 = ot; a.hot_cap = hot_cap; a.unit_cap = unit_cap; a.out = out;
  cudaPointerAttributes pa;
  if (Kg > 0 && cudaPointerGetAttributes(&pa, rec_k) == cudaSuccess) a.direct = pa.type == cudaMemoryTypeHost;
  else (void)cudaGetLastError();
  // Heads of a CTA: as many as fill 8 columns with their rows.  More heads mean a longer union that every tile
  // of columns decodes anew, fewer leave columns empty: 64 rows of one sequence, 64 groups opened by each of 8
  // heads, take 32 us with one head a CTA and 92 with 8 where the heads opened different groups (33 and 31
  // where all opened the same), 2 rows of each of 16 sequences 48 with 4 and 65 with 8 (22 and 24).
  a.hpc = L >= 8 ? 1 : 8 / L;
  if (a.hpc > a.rep) a.hpc = a.rep;
  // One row of few sequences: half as many heads where twice the CTAs are still resident (4 sequences 14.3
  // against 18.4 us, or 11.5 either way with the same groups for all heads).
  if (L == 1 && (int64_t)p.batch * p.kv_heads * ((a.rep + a.hpc - 1) / a.hpc) * 16 <= 132 * kv4::ctas_of(1))
    a.hpc = (a.hpc + 1) / 2;
  const int cols = a.hpc * L;
  const bool wide = cols > 8;
  const int64_t ctas = (int64_t)p.batch * p.kv_heads * ((a.rep + a.hpc - 1) / a.hpc) * ((cols + (wide ? 15 : 7)) / (wide ? 16 : 8));
  // CTAs per tile: as many as are resident at once, at most 8 (a portable cluster).  Clusters of 4 to 8 leave
  // about a tenth of the places empty (33 of 8 CTAs fit where 37 would): a 36th of 8 would wait for a second round.
  const int64_t room = 132 * kv4::ctas_of(wide ? 2 : 1);
  a.splits = (int)(room / ctas < 1 ? 1 : room / ctas > 8 ? 8 : room / ctas);
#define HGA_KV4_L(TT)                                                                              \
  if (p.head_dim == 128) return wide ? kv4::launch_t<TT, 128, 2>(p, a, st) : kv4::launch_t<TT, 128, 1>(p, a, st); \
  return wide ? kv4::launch_t<TT, 64, 2>(p, a, st) : kv4::launch_t<TT, 64, 1>(p, a, st);
  if (p.dtype == HGA_DTYPE_BF16) { HGA_KV4_L(__nv_bfloat16) }
  HGA_KV4_L(__half)
#undef HGA_KV4_L
}

}  // namespace hga

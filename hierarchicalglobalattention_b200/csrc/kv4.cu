// 4-bit KV record: pack, unpack, and the portable attention over it (any type, head_dim a multiple of 64).
// The record's format is in kv4_common.cuh.
#include "kv4_common.cuh"

namespace hga {

HGA_DEVICE_ERROR_WORD(g_kv4_error, kv4_error_status)

template <typename T>
__device__ __forceinline__ void kv4_load8(const T* p, float (&f)[8]) {
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

constexpr int kPackWarps = 4;

// One warp per unit of K or of V.  The rows are read in their natural order (16-byte loads, 8 channels a
// lane, a block of 32 channels in 4 neighbouring lanes), quantised, and their codes put as bytes in
// shared memory, from which each lane assembles its words.  Bound by HBM.
template <typename T, int DH>
__global__ void __launch_bounds__(kPackWarps * 32) kv4_pack_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                                   int64_t bk, int64_t rows, int64_t cap,
                                                                   uint8_t* __restrict__ rec_k, uint8_t* __restrict__ rec_v,
                                                                   int64_t unit_cap, int64_t unit0) {
  using MT = typename Kv4Meta<T>::type;
  constexpr int LD = DH + 8;                 // bytes per staged code row
  constexpr int LPR = DH / 8;                // lanes per row
  __shared__ __align__(8) uint8_t stage[kPackWarps][16 * LD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t units = (rows + 15) / 16;
  const int64_t total = 2 * bk * units;
  uint8_t* sc = stage[warp];
  for (int64_t w = (int64_t)blockIdx.x * kPackWarps + warp; w < total; w += (int64_t)gridDim.x * kPackWarps) {
    const bool is_v = w >= bk * units;
    const int64_t x = is_v ? w - bk * units : w;
    const int64_t head = x / units, u = x - head * units;
    const T* src = (is_v ? v : k) + (head * cap + u * 16) * DH;
    uint8_t* dst = (is_v ? rec_v : rec_k) + (head * unit_cap + unit0 + u) * kv4_unit_bytes(DH);
    uint32_t* meta = reinterpret_cast<uint32_t*>(dst + 8 * DH);
    const int valid = rows - u * 16 < 16 ? (int)(rows - u * 16) : 16;
#pragma unroll
    for (int i = lane; i < 16 * LPR; i += 32) {
      const int r = i / LPR, c8 = i % LPR;
      float f[8];
      if (r < valid) {
        kv4_load8<T>(src + (int64_t)r * DH + c8 * 8, f);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 0.f;
      }
      float lo = f[0], hi = f[0], odd = 0.f;  // odd: NaN as soon as one value is not finite
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo = fminf(lo, f[e]);
        hi = fmaxf(hi, f[e]);
        odd += f[e] * 0.f;
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        odd += __shfl_xor_sync(0xffffffffu, odd, o);
      }
      const MT mt = Num<MT>::from_f(lo + odd), st = Num<MT>::from_f(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f) + odd);
      const float m = Num<MT>::to_f(mt), s = Num<MT>::to_f(st);
      uint32_t codes[2] = {0u, 0u};
      if (s > 0.f && s < INFINITY) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float n = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(f[e], m), s)), 0.f), 15.f);
          codes[e >> 2] |= (uint32_t)(int)n << (8 * (e & 3));
        }
      }
      *reinterpret_cast<uint2*>(sc + r * LD + c8 * 8) = make_uint2(codes[0], codes[1]);
      if ((c8 & 3) == 0) {
        const MT pair[2] = {st, mt};
        meta[r * (DH / 32) + c8 / 4] = *reinterpret_cast<const uint32_t*>(pair);
      }
    }
    __syncwarp();
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int quad = 0; quad < DH / 64; ++quad) {
      uint32_t word[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = quad * 4 + j;
        uint32_t a = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int row = g + 8 * (e & 1), col = 2 * c + 8 * ((e >> 1) & 1) + (e >> 2);
          const uint32_t n = is_v ? sc[col * LD + t * 16 + row] : sc[row * LD + t * 16 + col];
          a |= n << (4 * e);
        }
        word[j] = a;
      }
      *reinterpret_cast<uint4*>(dst + (quad * 32 + lane) * 16) = make_uint4(word[0], word[1], word[2], word[3]);
    }
    __syncwarp();
  }
}

// The values of rows [0, rows): the mirror of kv4_pack_kernel.
template <typename T, int DH>
__global__ void __launch_bounds__(kPackWarps * 32) kv4_unpack_kernel(const uint8_t* __restrict__ rec_k,
                                                                     const uint8_t* __restrict__ rec_v, int64_t unit_cap,
                                                                     int64_t unit0, int64_t bk, int64_t rows,
                                                                     T* __restrict__ k, T* __restrict__ v, int64_t cap) {
  using MT = typename Kv4Meta<T>::type;
  constexpr int LD = DH + 8;
  constexpr int LPR = DH / 8;
  __shared__ __align__(8) uint8_t stage[kPackWarps][16 * LD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t units = (rows + 15) / 16;
  const int64_t total = 2 * bk * units;
  uint8_t* sc = stage[warp];
  for (int64_t w = (int64_t)blockIdx.x * kPackWarps + warp; w < total; w += (int64_t)gridDim.x * kPackWarps) {
    const bool is_v = w >= bk * units;
    const int64_t x = is_v ? w - bk * units : w;
    const int64_t head = x / units, u = x - head * units;
    const uint8_t* src = (is_v ? rec_v : rec_k) + (head * unit_cap + unit0 + u) * kv4_unit_bytes(DH);
    T* dst = (is_v ? v : k) + (head * cap + u * 16) * DH;
    const uint32_t* meta = reinterpret_cast<const uint32_t*>(src + 8 * DH);
    const int valid = rows - u * 16 < 16 ? (int)(rows - u * 16) : 16;
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int quad = 0; quad < DH / 64; ++quad) {
      const uint4 q4 = *reinterpret_cast<const uint4*>(src + (quad * 32 + lane) * 16);
      const uint32_t word[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = quad * 4 + j;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int row = g + 8 * (e & 1), col = 2 * c + 8 * ((e >> 1) & 1) + (e >> 2);
          sc[is_v ? col * LD + t * 16 + row : row * LD + t * 16 + col] = (uint8_t)((word[j] >> (4 * e)) & 15u);
        }
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = lane; i < 16 * LPR; i += 32) {
      const int r = i / LPR, c8 = i % LPR;
      const uint2 n8 = *reinterpret_cast<const uint2*>(sc + r * LD + c8 * 8);
      const uint32_t mw = meta[r * (DH / 32) + c8 / 4];
      const MT* pair = reinterpret_cast<const MT*>(&mw);
      const float s = Num<MT>::to_f(pair[0]), m = Num<MT>::to_f(pair[1]);
      if (r < valid) {
        T y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t n = ((e < 4 ? n8.x : n8.y) >> (8 * (e & 3))) & 255u;
          y[e] = Num<T>::from_f(__fadd_rn(__fmul_rn((float)n, s), m));
        }
        uint4* o = reinterpret_cast<uint4*>(dst + (int64_t)r * DH + c8 * 8);
        o[0] = reinterpret_cast<const uint4*>(y)[0];
        if constexpr (sizeof(T) == 4) o[1] = reinterpret_cast<const uint4*>(y)[1];
      }
    }
    __syncwarp();
  }
}

static unsigned pack_grid(int64_t total) {
  const int64_t ctas = (total + kPackWarps - 1) / kPackWarps;
  return (unsigned)(ctas < 148 * 16 ? ctas : 148 * 16);
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
  const unsigned grid = pack_grid(2 * bk * ((rows + 15) / 16));
  HGA_KV4_DISPATCH((kv4_pack_kernel<T, DH><<<grid, kPackWarps * 32, 0, st>>>(
      (const T*)k, (const T*)v, bk, rows, cap, (uint8_t*)rec_k, (uint8_t*)rec_v, unit_cap, unit0)))
  return cudaGetLastError();
}

cudaError_t launch_kv4_unpack(int dtype, int dh, int64_t bk, int64_t rows, const void* rec_k, const void* rec_v,
                              int64_t unit_cap, int64_t unit0, void* k, void* v, int64_t cap, cudaStream_t st) {
  const unsigned grid = pack_grid(2 * bk * ((rows + 15) / 16));
  HGA_KV4_DISPATCH((kv4_unpack_kernel<T, DH><<<grid, kPackWarps * 32, 0, st>>>(
      (const uint8_t*)rec_k, (const uint8_t*)rec_v, unit_cap, unit0, bk, rows, (T*)k, (T*)v, cap)))
  return cudaGetLastError();
}

// ---- attention, portable ------------------------------------------------------------------------
constexpr int kPortRows = 8;    // query rows per CTA, two per warp
constexpr int kPortWarps = 4;

// One CTA per (query head, sequence, 8 query rows); units of 16 keys pass through shared memory as fp32,
// a lane pair scores one key, and every warp keeps its rows' online softmax in registers.
template <typename T, int DH>
__global__ void __launch_bounds__(kPortWarps * 32) attend_kv4_kernel(
    hga_params p, int L, const T* __restrict__ q, const int32_t* __restrict__ seq_pos, const T* __restrict__ hot_k,
    const T* __restrict__ hot_v, int64_t hot_cap, const uint8_t* rec_k, const uint8_t* rec_v, int64_t unit_cap,
    const int32_t* __restrict__ open_gid, const int32_t* __restrict__ open_t0, int Kg, T* __restrict__ out) {
  using MT = typename Kv4Meta<T>::type;
  constexpr int LD = DH + 2, VD = DH / 32;
  __shared__ float qs[kPortRows][LD], ks[kKv4Unit][LD], vs[kKv4Unit][LD];
  const int h = blockIdx.x, b = blockIdx.y, row0 = blockIdx.z * kPortRows;
  const int H = p.nhead, KVH = p.kv_heads, C = p.chunk_size, gs = p.group_size, U = gs / kKv4Unit;
  const int kvh = h / (H / KVH);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nrows = L - row0 < kPortRows ? L - row0 : kPortRows;
  const int pos = seq_pos[b];
  const int kf = p.keep_first > 0 ? p.keep_first : 0, kl = p.keep_last > 0 ? p.keep_last : 0;
  const size_t bh = (size_t)b * H + h;
  T* o_base = out + (bh * L + row0) * DH;
  const int n_closed = pos / C, c0 = pos % C;
  if (pos < 0 || c0 + L > C || (int64_t)(kf + kl + 1) * C > hot_cap) {
    if (tid == 0) atomicCAS(&g_kv4_error, 0, kErrBoundsAttendKv4);
    for (int i = tid; i < nrows * DH; i += blockDim.x) o_base[i] = Num<T>::from_f(0.f);
    return;
  }
  int f_hi, l_lo;
  windows(n_closed, kf, kl, f_hi, l_lo);
  for (int i = tid; i < kPortRows * DH; i += blockDim.x)
    qs[i / DH][i % DH] = i / DH < nrows ? Num<T>::to_f(q[(bh * L + row0) * DH + i]) : 0.f;
  float o[2][VD], m[2], l[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < VD; ++d) o[i][d] = 0.f;
  }
  // one unit: from the slots (chunk >= 0) or the record (unit number), key j visible to row t iff
  // t >= tmin + causal * j
  auto take = [&](int64_t hot_row, int64_t unit, int tmin, int causal, int count) {
    __syncthreads();
    if (unit < 0) {
      const size_t base = (((size_t)b * KVH + kvh) * hot_cap + hot_row) * DH;
      for (int i = tid; i < kKv4Unit * DH; i += blockDim.x) {
        const bool in = i / DH < count;  // rows past the block hold an earlier sequence's values
        ks[i / DH][i % DH] = in ? Num<T>::to_f(hot_k[base + i]) : 0.f;
        vs[i / DH][i % DH] = in ? Num<T>::to_f(hot_v[base + i]) : 0.f;
      }
    } else {
      const size_t base = (((size_t)b * KVH + kvh) * unit_cap + unit) * kv4_unit_bytes(DH);
      for (int i = tid; i < 2 * kKv4Unit * DH; i += blockDim.x) {
        const bool is_v = i >= kKv4Unit * DH;
        const int x = is_v ? i - kKv4Unit * DH : i, tok = x / DH, ch = x % DH;
        const uint8_t* u = (is_v ? rec_v : rec_k) + base;
        const int r = is_v ? ch & 15 : tok, c = is_v ? tok : ch & 15, nib = kv4_nibble(r, c);
        const uint32_t n = (u[kv4_word_byte(ch >> 4, r, c) + nib / 2] >> (4 * (nib & 1))) & 15u;
        const MT* pair = reinterpret_cast<const MT*>(u + 8 * DH) + 2 * (tok * (DH / 32) + ch / 32);
        const float y = fmaf((float)n, Num<MT>::to_f(pair[0]), Num<MT>::to_f(pair[1]));
        if (is_v) vs[tok][ch] = y; else ks[tok][ch] = y;
      }
    }
    __syncthreads();
    const int key = lane >> 1, half = lane & 1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = warp * 2 + i, t = row0 + r;
      if (r >= nrows) continue;  // warp-uniform
      float dot = 0.f;
      for (int d = half; d < DH; d += 2) dot = fmaf(qs[r][d], ks[key][d], dot);
      dot += __shfl_xor_sync(0xffffffffu, dot, 1);
      const bool vis = key < count && t >= tmin + causal * key;
      const unsigned mask = __ballot_sync(0xffffffffu, vis);
      if (!mask) continue;
      const float s = vis ? dot * p.scale * 1.4426950408889634f : -INFINITY;
      float mx = s;
#pragma unroll
      for (int w = 16; w >= 2; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float m_new = fmaxf(m[i], mx);
      const float base = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = exp2f(m[i] - base), pe = vis ? exp2f(s - base) : 0.f;
      float ps = half ? 0.f : pe;
#pragma unroll
      for (int w = 16; w; w >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, w);
      l[i] = l[i] * alpha + ps;
      m[i] = m_new;
#pragma unroll
      for (int d = 0; d < VD; ++d) o[i][d] *= alpha;
      for (int j = 0; j < kKv4Unit; ++j) {
        const float pj = __shfl_sync(0xffffffffu, pe, 2 * j);
        if (!(mask >> (2 * j) & 1)) continue;  // what an invisible key holds does not count, NaN included
#pragma unroll
        for (int d = 0; d < VD; ++d) o[i][d] = fmaf(pj, vs[j][lane + 32 * d], o[i][d]);
      }
    }
  };
  const int wu = C / kKv4Unit;
  for (int u = 0; u < f_hi * wu; ++u) take((int64_t)u * kKv4Unit, -1, 0, 0, kKv4Unit);
  for (int n = l_lo; n < n_closed; ++n)
    for (int u = 0; u < wu; ++u) take((int64_t)(kf + n % (kl > 0 ? kl : 1)) * C + u * kKv4Unit, -1, 0, 0, kKv4Unit);
  for (int j = 0; j < Kg; ++j) {
    const int gid = open_gid[bh * Kg + j], t0 = open_t0[bh * Kg + j];
    if (gid < 0 || t0 < 0) continue;
    if ((int64_t)(gid + 1) * U > unit_cap) {
      if (tid == 0) atomicCAS(&g_kv4_error, 0, kErrBoundsAttendKv4);
      continue;
    }
    for (int u = 0; u < U; ++u) take(0, (int64_t)gid * U + u, t0, 0, kKv4Unit);
  }
  const int nact = c0 + row0 + nrows;
  for (int u = 0; u * kKv4Unit < nact; ++u)
    take((int64_t)(kf + kl) * C + u * kKv4Unit, -1, u * kKv4Unit - c0, 1,
         nact - u * kKv4Unit < kKv4Unit ? nact - u * kKv4Unit : kKv4Unit);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = warp * 2 + i;
    if (r >= nrows) continue;
#pragma unroll
    for (int d = 0; d < VD; ++d) o_base[(size_t)r * DH + lane + 32 * d] = Num<T>::from_f(l[i] == 0.f ? 0.f : o[i][d] / l[i]);
  }
}

cudaError_t launch_attend_kv4(const hga_params& p, int L, const void* q, const int32_t* seq_pos, const void* hk,
                              const void* hv, int64_t hot_cap, const void* rec_k, const void* rec_v, int64_t unit_cap,
                              const int32_t* og, const int32_t* ot, int Kg, void* out, cudaStream_t st) {
  const int dtype = p.dtype, dh = p.head_dim;
  const dim3 grid(p.nhead, p.batch, (L + kPortRows - 1) / kPortRows);
  HGA_KV4_DISPATCH((attend_kv4_kernel<T, DH><<<grid, kPortWarps * 32, 0, st>>>(
      p, L, (const T*)q, seq_pos, (const T*)hk, (const T*)hv, hot_cap, (const uint8_t*)rec_k, (const uint8_t*)rec_v,
      unit_cap, og, ot, Kg, (T*)out)))
  return cudaGetLastError();
}

}  // namespace hga

// The 4-bit KV record, shared by its pack / unpack kernels and the attention that reads it.
//
// A record holds units of 16 token rows of one (sequence, KV head).  Each token's channels are cut into
// blocks of 32:  min = smallest value, scale = (largest - smallest) * (1 / 15), both held in 16 bits (the
// cache's type; bf16 for an fp32 cache), and a channel's code n = clamp(rint((x - min) / scale), 0, 15)
// stands for scale * n + min.  A block of equal values has scale 0 and reads back as its minimum; a block
// that holds an infinity or a NaN reads back as NaN throughout.
//
// Bytes of a unit (10 * Dh; 5 bits a value):
//   [0, 8 Dh)       codes, in 16 x 16 tiles along the channels, each in the register order of the
//                   16-row A operand of mma.m16n8k16: lane l = 4 g + c holds rows g and g + 8, columns
//                   2c, 2c + 1, 2c + 8, 2c + 9 as one 32-bit word, nibble (row / 8) + 2 (col / 8) + 4
//                   (col % 2), so (word >> 4 i) & 0x000f000f is the operand's i-th register (two 16-bit
//                   halves).  Four tiles' words of a lane are neighbours: a warp reads a unit with
//                   16-byte loads, whole lines, and no shuffles.  K tiles have the token as row (S^T =
//                   K Q^T), V tiles the channel as row (O^T = V^T P^T).
//   [8 Dh, 10 Dh)   (scale, min) pairs [16 tokens][Dh / 32]
#pragma once

#include "hga_common.cuh"

namespace hga {

constexpr int kKv4Unit = 16;
constexpr int kErrBoundsAttendKv4 = 0x104;

template <typename T> struct Kv4Meta { using type = T; };
template <> struct Kv4Meta<float> { using type = __nv_bfloat16; };

__host__ __device__ constexpr int kv4_unit_bytes(int dh) { return 10 * dh; }

}  // namespace hga

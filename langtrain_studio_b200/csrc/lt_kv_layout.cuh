// Device-side cell layout of the f16 block pool and the f32 -> f16
// conversion of its rows, shared by every kernel that writes or reads pool
// cells (the K/V write, attention, and the Llama decode step), so they agree
// bit for bit.
//
// Pool layout (per layer): f16 [block][kv_head][2 (K,V)][D/64][16 slots][64].
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "lt_kv_internal.h"

namespace ltkv {

// f32 -> f16 with the bit semantics of half 2.7.1's f16::from_f32: IEEE
// round-to-nearest-even (the hardware cvt.rn), and NaN -> quiet NaN that
// keeps the top 10 payload bits (the hardware returns a canonical NaN).
__device__ __forceinline__ uint16_t f32_to_f16_ref(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7F800000u) == 0x7F800000u && (u & 0x007FFFFFu))
        return static_cast<uint16_t>(((u >> 16) & 0x8000u) | 0x7E00u | ((u & 0x007FFFFFu) >> 13));
    return __half_as_ushort(__float2half_rn(x));
}

// Element offset of 16-byte chunk c (8 f16) of slot s inside the K (or V)
// part of a (block, head) tile: the part is head_dim/64 sub-tiles of 16 rows
// x 128 bytes, chunk c in sub-tile c/8, at chunk position (c%8) ^ (s%8).
// Each sub-tile is the 128-byte-swizzled row-major layout of the tensor-core
// operand descriptors, and ldmatrix over it is bank-conflict free.
__device__ __forceinline__ int chunk_off(int c, int slot) {
    return (c >> 3) * (kBlock * 64) + slot * 64 + (((c & 7) ^ (slot & 7)) << 3);
}

__host__ __device__ constexpr int q8_tile_bytes(int D) { return 34 * D; }

// Position of entry i (0..15) inside a 16-byte run: the order
// 0,1,8,9, 2,3,10,11, 4,5,12,13, 6,7,14,15, so bytes 4t..4t+3 of a run hold
// entries 2t, 2t+1, 2t+8, 2t+9 -- one lane's part of an m16n8k16 B fragment.
__device__ __forceinline__ int q8_pos(int i) { return ((i & 7) >> 1) * 4 + ((i >> 3) << 1) + (i & 1); }

// Byte offset of the 16-byte run of K values 16k..16k+15 of slot s: run
// L = s*D/16 + k of the row-major K part, 128-byte lines swizzled by line.
template <int D>
__device__ __forceinline__ int q8_krun(int s, int k) {
    const int L = s * (D / 16) + k;
    return ((L >> 3) << 7) + (((L & 7) ^ ((L >> 3) & 7)) << 4);
}

// Q4_0 tile (LT_KV_Q4_0), 18*D bytes per (block, head): K codes, V codes,
// then the f16 scales of K and of V.  The 4-bit codes are stored as 32-bit
// words, one word per lane and 16x16 step of the mma.sync A fragment
// (m16n8k16): the word of step i of lane (g = lane / 4, t = lane % 4) is
// word lane*4 + i%4 of the 512-byte run i/4, so a lane's four steps are one
// 16-byte load and a warp's are 512 contiguous bytes.  Every byte belongs to
// one slot, so rows are stored without touching their neighbours:
//   K (rows = slots, columns = dims 16i..): byte 0 = slot g, dims 2t (low
//     nibble) and 2t+8 (high); byte 1 = slot g+8, the same dims; bytes 2, 3 =
//     slots g, g+8, dims 2t+1 and 2t+9;
//   V (rows = dims 16i.., columns = slots): byte 0 = slot 2t, dims g (low)
//     and g+8 (high); byte 1 = slot 2t+8; bytes 2, 3 = slots 2t+1, 2t+9.
// Scales: K [slot%8][slot/8][D/32] f16; V [(slot%8)/2][D/32][4] f16, the four
// being slots 2t, 2t+1, 2t+8, 2t+9.
__host__ __device__ constexpr int q4_tile_bytes(int D) { return 18 * D; }

// Byte of word (step i, lane g*4 + t) inside the K or V part.
__device__ __forceinline__ int q4_word(int i, int g, int t) { return ((i >> 2) << 9) + ((g * 4 + t) << 4) + ((i & 3) << 2); }

// Byte of the codes of dim e (0..D-1) of a slot in the K (V) part; e's code
// is the low nibble when e % 16 < 8, else the high one.
__device__ __forceinline__ int q4_kbyte(int slot, int e) {
    return q4_word(e >> 4, slot & 7, (e & 7) >> 1) + ((e & 1) << 1) + (slot >> 3);
}
__device__ __forceinline__ int q4_vbyte(int slot, int e) {
    return q4_word(e >> 4, e & 7, (slot & 7) >> 1) + ((slot & 1) << 1) + (slot >> 3);
}

// Byte of the scale of group c (dims 32c..32c+31) of a slot inside the tile.
template <int D>
__device__ __forceinline__ int q4_kscale(int slot, int c) {
    return 16 * D + (((slot & 7) * 2 + (slot >> 3)) * (D / 32) + c) * 2;
}
template <int D>
__device__ __forceinline__ int q4_vscale(int slot, int c) {
    return 17 * D + ((((slot & 7) >> 1) * (D / 32) + c) * 4 + ((slot >> 3) << 1) + (slot & 1)) * 2;
}

}  // namespace ltkv

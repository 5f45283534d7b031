// sm_100a kernels of the 4-bit cache (LT_KV_Q4_0): K/V write, read-back of
// cells and rows, and stream-K attention over 4-bit tiles.
//
// Format.  A group of 32 values shares one scale d; a value reads back as
// (code - 8) * d with code in 0..15.  d = +-max|x| / 8, signed so that the
// largest magnitude takes code 0 (-8 * d), rounded to 8 significant bits and
// held as f16.  With 8 bits in d and 4 in code - 8, every (code - 8) * d is an
// f16 exactly: rows() rounds nothing, and attention multiplies the same values
// on the f16 tensor cores with no rounding of its own.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "lt_kv_device.cuh"
#include "lt_kv_internal.h"
#include "lt_kv_layout.cuh"

namespace ltkv {
namespace {

constexpr float kQ4MaxScale = 2720.0f;  // 8 significant bits, and 24 * d is still an f16

// ------------------------------------------------------------ quantise ----
// The scale of a 32-value group from its extremes top = max(x, 0) and low =
// max(-x, 0): signed so that the larger magnitude takes code 0; |d| in ad.
__device__ __forceinline__ float q4_scale(float top, float low, float& ad) {
    const bool pos = top >= low;  // the positive extreme takes -8 * d
    const float a = fminf(__bfloat162float(__float2bfloat16_rn((pos ? top : low) * 0.125f)), kQ4MaxScale);
    ad = __half2float(__float2half_rn(a));
    return pos ? -ad : ad;
}

// clamp(floor(x / d + 1/2) + 8, 0, 15) as the last byte of the result (the rest
// is to be masked off), decided exactly.  xs = x with d's sign taken off, inv ~
// 1 / |d|.  k, rounded from a quotient brought down by 2^-10 (far more than
// its error), is the answer or one below it; the border (k + 1/2) * |d| has at
// most 13 significant bits, so comparing xs with it in f32 settles which.  Adding
// 1.5 * 2^23 rounds to an integer and leaves it in the last bits.  NaN, or d = 0:
// code 8.  PLAIN: no NaN, and |d| a normal f16 within 2^-8 of max|x| / 8, so that
// no quotient is below -8.1.
template <bool PLAIN>
__device__ __forceinline__ uint32_t q4_code(float xs, float ad, float inv) {
    constexpr float kRound = 12582912.f;
    const float x = fminf(PLAIN ? xs : fmaxf(xs, -8.f * ad), 7.f * ad);  // exact bounds: codes 0 and 15
    float k = __fadd_rn(__fadd_rn(__fmaf_rn(x, inv, -0.0009765625f), kRound), -kRound);
    if (x >= __fmaf_rn(k, ad, 0.5f * ad)) k += 1.f;
    if (!PLAIN) k = ad > 0.f && xs == xs ? k : 0.f;
    return __float_as_uint(__fadd_rn(k, kRound + 8.f));
}

// One group held as N values by each of 32 / N consecutive lanes (every lane of
// the warp calls this): its codes; returns d.  NaN does not count in the scale.
template <int N>
__device__ __forceinline__ float q4_quant(const float (&x)[N], uint32_t (&code)[N]) {
    float top = 0.f, low = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        top = fmaxf(top, x[i]);
        low = fmaxf(low, -x[i]);
    }
#pragma unroll
    for (int m = 1; m < 32 / N; m <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(kFull, top, m));
        low = fmaxf(low, __shfl_xor_sync(kFull, low, m));
    }
    float ad;
    const float d = q4_scale(top, low, ad);
    const float inv = ad > 0.f ? __fdividef(1.0f, ad) : 0.f;
    const bool neg = top >= low;
    if constexpr (N == 8) {  // rows of a write, which it shortens from 16.2 to 14.9 us (4096 tokens of 8 x 128 f16)
        float odd = 0.f;  // becomes NaN with a NaN or an infinity among the values
#pragma unroll
        for (int i = 0; i < N; ++i) odd = fmaf(x[i], 0.f, odd);
        if (__all_sync(kFull, odd == odd && ad >= 6.103515625e-5f && fmaxf(top, low) <= 8.f * kQ4MaxScale)) {
#pragma unroll
            for (int i = 0; i < N; ++i) code[i] = q4_code<true>(neg ? -x[i] : x[i], ad, inv);
            return d;
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) code[i] = q4_code<false>(neg ? -x[i] : x[i], ad, inv);  // (last bytes)
    return d;
}

// Store a lane's four codes (as q4_code gives them; dims 16i + 2t, +1, +8, +9) of slot `slot`, and
// the group's scale from its first lane, into a tile.
template <int D>
__device__ __forceinline__ void q4_store4(uint8_t* tile, int kvsel, int i, int t, int slot, const uint32_t (&code)[4],
                                          float d) {
    const uint8_t b0 = (uint8_t)((code[0] & 15) | (code[2] << 4)), b1 = (uint8_t)((code[1] & 15) | (code[3] << 4));
    const int e = 16 * i + 2 * t;
    if (kvsel == 0) {
        uint8_t* w = tile + q4_kbyte(slot, e);
        w[0] = b0;
        w[2] = b1;
    } else {
        tile[8 * D + q4_vbyte(slot, e)] = b0;
        tile[8 * D + q4_vbyte(slot, e + 1)] = b1;
    }
    if ((i & 1) == 0 && t == 0) {
        const int off = kvsel ? q4_vscale<D>(slot, i >> 1) : q4_kscale<D>(slot, i >> 1);
        *reinterpret_cast<uint16_t*>(tile + off) = __half_as_ushort(__float2half_rn(d));
    }
}

// A lane's four inputs: values idx, idx+1, idx+8, idx+9.
__device__ __forceinline__ void load4_f32(const void* base, size_t idx, int in_f32, float (&x)[4]) {
    if (in_f32) {
        const float* p = static_cast<const float*>(base) + idx;
        const float2 a = __ldg(reinterpret_cast<const float2*>(p)), b = __ldg(reinterpret_cast<const float2*>(p + 8));
        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    } else {
        const __half* p = static_cast<const __half*>(base) + idx;
        const float2 a = __half22float2(__ldg(reinterpret_cast<const __half2*>(p)));
        const float2 b = __half22float2(__ldg(reinterpret_cast<const __half2*>(p + 8)));
        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    }
}

// --------------------------------------------------------------- write ----
// One CTA per (16 tokens of the call, head): D/8 lanes a row, eight values a lane, a
// group is four lanes.  Bytes belong to one slot, so rows of one block written by
// different warps or CTAs never touch the same byte; but stored one by one
// straight to the pool they cost a 32-byte sector each (V's lie 64 bytes apart).
// Tokens that fill a block (a prefill chunk; `shift` aligns the first block of
// the call) therefore meet in a tile image in shared memory, stored 16 bytes a
// thread.  4096 tokens of 8 x 128 f16 (38 MB, 5.8 us at the copy rate): 23 us byte
// by byte with four values a lane, 20 through the image, 16 with eight values a
// lane, which halves what a group's extremes and scale cost, 15 with the odd values'
// steps left to the warps that hold one.  Instruction issue
// bounds it (the exact codes): 0.76 instructions a cycle and scheduler, DRAM at 13 %.
template <int D>
__global__ void __launch_bounds__(4 * D) kv_write_q4_kernel(uint8_t* __restrict__ pool_layer,
                                                            const int2* __restrict__ cells, int n, int n_kv_heads,
                                                            int shift, const void* __restrict__ k,
                                                            const void* __restrict__ v, int in_f32) {
    constexpr int TILE = q4_tile_bytes(D), L = D / 8;  // lanes of a row
    __shared__ __align__(16) uint8_t image[TILE];
    const int j = threadIdx.x / (2 * L), kvsel = threadIdx.x / L & 1, c = threadIdx.x % L;
    const int h = blockIdx.x % n_kv_heads, tok0 = (int)(blockIdx.x / n_kv_heads) * kBlock - shift, tok = tok0 + j;
    const bool live = tok >= 0 && tok < n;
    const int2 cell = live ? __ldg(cells + tok) : make_int2(-1, -1);
    const int block0 = tok0 >= 0 ? __ldg(cells + tok0).x : -1;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live) load8_f32(kvsel ? v : k, ((size_t)tok * n_kv_heads + h) * D + 8 * c, in_f32, x);
    const bool full = __syncthreads_and(live && cell.y == j && cell.x == block0);
    uint8_t* tile = full ? image : pool_layer + ((size_t)max(cell.x, 0) * n_kv_heads + h) * TILE;
    const int slot = max(cell.y, 0);
    uint32_t code[8];
    const float d = q4_quant<8>(x, code);
    // One code a byte: values 0-3 and 4-7.  Units c and c^1 (dims 16i.. and 16i + 8 ..)
    // share their bytes; the even lane stores dims 0-3 of the pair, the odd one 4-7.
    const uint32_t lo = __byte_perm(__byte_perm(code[0], code[1], 0x0040), __byte_perm(code[2], code[3], 0x0040), 0x5410);
    const uint32_t hi = __byte_perm(__byte_perm(code[4], code[5], 0x0040), __byte_perm(code[6], code[7], 0x0040), 0x5410);
    const bool odd = c & 1;
    const uint32_t got = __shfl_xor_sync(kFull, odd ? lo : hi, 1);
    const uint32_t bytes = odd ? got | (hi << 4) : lo | (got << 4);
    if (live) {
        const int e = 16 * (c >> 1) + (odd ? 4 : 0);
        // dims e .. e + 3: K in two words 16 bytes apart (bytes 0, 2 of each), V in four 64 bytes apart
        uint8_t* at = tile + (kvsel ? 8 * D + q4_vbyte(slot, e) : q4_kbyte(slot, e));
        const int step1 = kvsel ? 64 : 2, step2 = kvsel ? 128 : 16;
        at[0] = (uint8_t)bytes;
        at[step1] = (uint8_t)(bytes >> 8);
        at[step2] = (uint8_t)(bytes >> 16);
        at[step2 + step1] = (uint8_t)(bytes >> 24);
        if ((c & 3) == 0)
            *reinterpret_cast<uint16_t*>(tile + (kvsel ? q4_vscale<D>(slot, c >> 2) : q4_kscale<D>(slot, c >> 2))) =
                __half_as_ushort(__float2half_rn(d));
    }
    if (!full) return;
    __syncthreads();
    uint4* dst = reinterpret_cast<uint4*>(pool_layer + ((size_t)block0 * n_kv_heads + h) * TILE);
    if (threadIdx.x < TILE / 16) dst[threadIdx.x] = reinterpret_cast<const uint4*>(image)[threadIdx.x];
}

// ---------------------------------------------------------------- read ----
// Values 8c..8c+7 of K (kvsel 0) or V of one slot of a (block, head) tile of
// any format.  Q8_0 products are exact in f32; f16 and Q4_0 values are f16s.
template <int D, int FMT>
__device__ __forceinline__ void cell_values8(const uint8_t* pool_layer, size_t tile_no, int kvsel, int slot, int c,
                                             float (&x)[8]) {
    if constexpr (FMT == LT_KV_F16) {
        const uint16_t* src =
            reinterpret_cast<const uint16_t*>(pool_layer) + (tile_no * 2 + kvsel) * (kBlock * D) + chunk_off(c, slot);
        const uint4 r = *reinterpret_cast<const uint4*>(src);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            x[2 * j] = f.x;
            x[2 * j + 1] = f.y;
        }
    } else if constexpr (FMT == LT_KV_Q8_0) {
        const uint8_t* tile = pool_layer + tile_no * q8_tile_bytes(D);
        const float d = __half2float(__ushort_as_half(
            *reinterpret_cast<const uint16_t*>(tile + (kvsel ? 33 : 32) * D + ((c >> 2) * 16 + q8_pos(slot)) * 2)));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = 8 * c + i;
            const int off = kvsel ? 16 * D + e * 16 + q8_pos(slot) : q8_krun<D>(slot, e >> 4) + q8_pos(e & 15);
            x[i] = (float)(int8_t)tile[off] * d;
        }
    } else {
        const uint8_t* tile = pool_layer + tile_no * q4_tile_bytes(D);
        const float d = __half2float(__ushort_as_half(*reinterpret_cast<const uint16_t*>(
            tile + (kvsel ? q4_vscale<D>(slot, c >> 2) : q4_kscale<D>(slot, c >> 2)))));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = 8 * c + i;
            const int b = kvsel ? tile[8 * D + q4_vbyte(slot, e)] : tile[q4_kbyte(slot, e)];
            x[i] = (float)(((c & 1) ? b >> 4 : b & 15) - 8) * d;
        }
    }
}

__device__ __forceinline__ void store8_as(void* out, size_t idx, int out_f32, const float (&x)[8]) {
    if (out_f32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + idx);
        p[0] = make_float4(x[0], x[1], x[2], x[3]);
        p[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = f32_to_f16_ref(x[2 * j]) | ((uint32_t)f32_to_f16_ref(x[2 * j + 1]) << 16);
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + idx) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// cells (lt_kv_read) or a block-table row (lt_kv_rows) name the cells.
template <int D, int FMT>
__global__ void __launch_bounds__(256) kv_read_kernel(const uint8_t* __restrict__ pool_layer,
                                                      const int2* __restrict__ cells, const int32_t* __restrict__ trow,
                                                      int n, int n_kv_heads, void* __restrict__ k_out,
                                                      void* __restrict__ v_out, int out_f32, int n_blocks, int32_t* err) {
    constexpr int CH = D / 8;
    const long long gid = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (gid >= (long long)n * n_kv_heads * 2 * CH) return;
    const int c = (int)(gid % CH);
    long long r = gid / CH;
    const int kvsel = (int)(r & 1);
    r >>= 1;
    const int h = (int)(r % n_kv_heads);
    const int i = (int)(r / n_kv_heads);
    const int2 cell = cells ? cells[i] : make_int2(checked_block(trow[i / kBlock], n_blocks, err), i % kBlock);
    float x[8];
    cell_values8<D, FMT>(pool_layer, (size_t)cell.x * n_kv_heads + h, kvsel, cell.y, c, x);
    store8_as(kvsel ? v_out : k_out, ((size_t)i * n_kv_heads + h) * D + 8 * c, out_f32, x);
}

template <int FMT>
cudaError_t launch_read_fmt(const uint8_t* pool, const int2* cells, const int32_t* trow, int n, int n_kv_heads,
                            int head_dim, void* k_out, void* v_out, int out_f32, int n_blocks, int32_t* err,
                            cudaStream_t s) {
    const long long threads = (long long)n * n_kv_heads * 2 * (head_dim / 8);
    const long long blocks = (threads + 255) / 256;
    if (blocks > 0x7FFFFFFFll) return cudaErrorInvalidValue;
    if (head_dim == 64)
        kv_read_kernel<64, FMT><<<(unsigned)blocks, 256, 0, s>>>(pool, cells, trow, n, n_kv_heads, k_out, v_out,
                                                                 out_f32, n_blocks, err);
    else
        kv_read_kernel<128, FMT><<<(unsigned)blocks, 256, 0, s>>>(pool, cells, trow, n, n_kv_heads, k_out, v_out,
                                                                  out_f32, n_blocks, err);
    return cudaGetLastError();
}

// ----------------------------------------------------------- attention ----
// Stream-K decode attention over 4-bit tiles.  Descriptors, flags and merges
// are those of the f16/Q8_0 kernel (lt_kv_kernels.cu): the call's (token, KV
// head, block) tiles are cut into one contiguous range per resident worker
// warp, and cut (token, head)s are merged over epoch flags.  Each (token, head)
// weighs p.piece_cost tiles more than it has: that many tiles' time go into its
// q rows and its output, and ranges of equal weight then end together (ragged
// batches of short sequences).
//
// One producer warp per CTA feeds the workers: kQ4Lanes of its lanes cut
// a worker's range into pieces and keep its ring of 18*D-byte bulk copies
// full, all workers at once.  The workers only compute.
//
// Per tile the mathematics is turned over: S^T = K Q^T and O^T += V^T P^T, so
// that the 4-bit tile is the A operand of mma.sync m16n8k16 (16 slots x 16
// dims, or 16 dims x 16 slots), one 32-bit word of codes per lane and step, and
// the query heads are the 8 columns of B:
//   K: the codes become code - 8 in f16 (one logic and one f16 operation a
//      pair); each group's partial scores are scaled by the slots' scales in f32.
//      (A masked code read as the subnormal f16 code * 2^-24 would save the f16
//      operation, but the MMA aligns its products by their exponent fields:
//      the scores then lose ~10 bits, 2.5e-6 of an output against 4e-7.  Codes in
//      bytes, read as e4m3 and converted, save a seventh of the instructions, but
//      the conversion shares the logic operations' half-rate pipe: 64 us against
//      57 for 64 sequences of 512 to 4096.)
//   V: the codes become (code - 8) * d in f16, exactly (one operation more).
// q and P are split into an f16 value and its f16 residual (~22 bits).  With a
// group of at most 4 heads (PACK) the 8 columns hold both (columns 0-3 the
// values, 4-7 the residuals), so one MMA carries them; larger groups take two.
// P^T in B-operand form is the transpose of the scores' fragment: movmatrix.
//
// What bounds it: instruction issue.  An mma.sync m16n8k16 keeps its scheduler
// from issuing anything else for 8 cycles on this chip, so a tile (D = 128)
// costs 16 x 8 scheduler cycles of MMA (32 x 8 for larger groups) beside ~290
// other instructions, ~180 of them the half-rate unpacking, where its 2304 bytes
// take ~400 scheduler cycles (4 schedulers x 148 SMs) from HBM.  64 sequences of 512
// to 4096, 32 / 8 heads: 52 us a call (26 at the copy rate; 0.54 instructions issued
// a cycle, DRAM 39 %); 16 of 32768, 64 / 8 heads, f16 q: 158 to 167 us (92).
//
// Q16 (f16 q): q has no residual, so PACK's columns 4-7 repeat the values and
// the scores come out in both halves without an exchange; larger groups take
// half the score MMAs.
//
// A worker takes two tiles a step: their score chains (MMA, scale, max, 2^x,
// transpose, MMA) are independent and fill one another's latencies.
constexpr int kQ4Workers = 4;   // worker warps of a CTA
constexpr int kQ4Step = 2;      // tiles a step
constexpr int kQ4Stages = 4;    // steps' worth of tiles in a worker's ring (a power of two)
constexpr int kQ4Pieces = 8;    // piece descriptors in its ring (> stages ahead + 2; a power of two)
constexpr int kQ4Threads = (kQ4Workers + 1) * 32;
constexpr int kQ4Lanes = 4;  // producer lanes of a worker: two stages' tiles

// D = A * B (f16 operands, f32 accumulators from zero).
__device__ __forceinline__ void mma16816_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// D += A * B.
__device__ __forceinline__ void mma16816_add(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ __half2 as_h2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }

// The low (high) nibbles of bytes 0 and 2 of w, minus 8, as two f16s: 1024 +
// code (64 + code) is the f16 whose last bits are the nibble.  The exponent
// patterns come in registers (`magic`), so that one three-input logic
// operation does mask and exponent (it takes one immediate only).
struct Q4Magic {
    uint32_t low, high;
};
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
    return r;
}
__device__ __forceinline__ __half2 q4_low(uint32_t w, const Q4Magic& m) {
    return __hsub2(as_h2(and_or(w, 0x000f000fu, m.low)), __floats2half2_rn(1032.f, 1032.f));
}
__device__ __forceinline__ __half2 q4_high(uint32_t w, const Q4Magic& m) {
    return __hsub2(as_h2(and_or(w, 0x00f000f0u, m.high)), __floats2half2_rn(72.f, 72.f));
}

// A piece: tiles [b0, b1) (counted from block skip) of (token, head).
// kind: 0 whole (token, head) -> output; 1 it started before this worker's
// range -> partial slot; 2 it starts here and runs past the range -> merged here.
struct Q4Piece {
    int tok, h, pos, b0, b1, kind, last_block, skip;
    int lo, qpos;
    int first;  // first tile of the (token, head), in the partition's units
    int last;   // last piece of the range
};

// What a worker and its producer lanes share.
constexpr int kQ4QBufs = 4;  // q buffers at most
struct Q4Ring {
    unsigned long long full[kQ4Stages];   // a stage's tiles have arrived (one tile at a piece's odd end)
    unsigned long long q_full[kQ4QBufs];  // a piece's q rows have arrived (they come ahead of its tiles)
    uint32_t consumed, q_taken;  // by the worker: stages done, pieces whose q rows it has read
    uint32_t issued, q_issued;   // by the producer: stages, q rows
    uint32_t none, stop, stopped;  // range without tiles; the worker gave up; the producer has seen it
    Q4Piece pieces[kQ4Pieces];
};

__device__ __forceinline__ uint32_t ld_acquire_cta(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory");
    return v;
}
__device__ __forceinline__ void st_release_cta(uint32_t* p, uint32_t v) {
    asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(smem_u32(p)), "r"(v) : "memory");
}

__host__ __device__ inline int q4_qbuf_bytes(int group, int head_dim, int q_f32) {
    return (group * head_dim * (q_f32 ? 4 : 2) + 127) & ~127;
}
// q buffers of a worker: 4 KiB worth, at most kQ4QBufs.
__host__ __device__ inline int q4_qbufs(int group, int head_dim, int q_f32) {
    const int n = 4096 / q4_qbuf_bytes(group, head_dim, q_f32);
    return n < 1 ? 1 : n > kQ4QBufs ? kQ4QBufs : n;
}
__host__ __device__ inline int q4_worker_smem(int group, int head_dim, int q_f32) {
    return kQ4Stages * kQ4Step * q4_tile_bytes(head_dim) +
           q4_qbufs(group, head_dim, q_f32) * q4_qbuf_bytes(group, head_dim, q_f32);
}
__host__ __device__ inline int q4_smem(int group, int head_dim, int q_f32) {
    return kQ4Workers * (q4_worker_smem(group, head_dim, q_f32) + (int)sizeof(Q4Ring));
}

// Turn a 4 x 4 array over within each quad: lane t gives r[s], s = 0..3, and
// gets the r[t] of lanes 0..3.
__device__ __forceinline__ void quad_transpose(uint32_t (&r)[4], int t) {
    const bool odd = t & 1, top = t & 2;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint32_t got = __shfl_xor_sync(kFull, odd ? r[i] : r[i + 1], 1);
        if (odd) r[i] = got; else r[i + 1] = got;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t got = __shfl_xor_sync(kFull, top ? r[i] : r[i + 2], 2);
        if (top) r[i] = got; else r[i + 2] = got;
    }
}

// Values of one part of a 4-bit tile: part = (K 0 | V 1) * D/64 + run ch, the
// dims 64 ch ... of all 16 slots.  put(kvsel, slot, c, x) gets the f16 dims
// 8c .. 8c+7 of a slot.  The words are read and dequantised as the attention
// kernel's A fragments; V's are turned over by movmatrix, so that every register
// is two neighbouring dims of a slot, and quads then gather eight of them.
constexpr int q4_parts(int D) { return 2 * (D / 64); }

template <int D, class Put>
__device__ __forceinline__ void q4_part_values(const uint8_t* tile, int part, int lane, Put put) {
    constexpr int G32 = D / 32, R = D / 64;
    const int g = lane >> 2, t = lane & 3, kvsel = part / R, ch = part % R;
    const Q4Magic magic{0x64006400u, 0x54005400u};
    const uint4 wv = __ldg(reinterpret_cast<const uint4*>(tile + kvsel * 8 * D + ch * 512 + lane * 16));
    const uint32_t ws[4] = {wv.x, wv.y, wv.z, wv.w};
    uint32_t r[2][2][4];  // [slots g, g + 8][dims .., + 8][16-dim step]
    if (kvsel == 0) {
        const __half* ks = reinterpret_cast<const __half*>(tile + 16 * D + g * (4 * G32)) + 2 * ch;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const __half2 d0 = __half2half2(ks[s >> 1]), d1 = __half2half2(ks[G32 + (s >> 1)]);  // slots g, g + 8
            const uint32_t w = ws[s], w8 = w >> 8;
            r[0][0][s] = h2_bits(__hmul2(q4_low(w, magic), d0));
            r[0][1][s] = h2_bits(__hmul2(q4_high(w, magic), d0));
            r[1][0][s] = h2_bits(__hmul2(q4_low(w8, magic), d1));
            r[1][1][s] = h2_bits(__hmul2(q4_high(w8, magic), d1));
        }
    } else {
        const uint4 vd = __ldg(reinterpret_cast<const uint4*>(tile + 17 * D + (t * G32 + 2 * ch) * 8));
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const __half2 dA = as_h2(s < 2 ? vd.x : vd.z), dB = as_h2(s < 2 ? vd.y : vd.w);
            const uint32_t w = ws[s], w8 = w >> 8;
            r[0][0][s] = movmatrix_trans(h2_bits(__hmul2(q4_low(w, magic), dA)));
            r[0][1][s] = movmatrix_trans(h2_bits(__hmul2(q4_high(w, magic), dA)));
            r[1][0][s] = movmatrix_trans(h2_bits(__hmul2(q4_low(w8, magic), dB)));
            r[1][1][s] = movmatrix_trans(h2_bits(__hmul2(q4_high(w8, magic), dB)));
        }
    }
#pragma unroll
    for (int sl = 0; sl < 2; ++sl)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            quad_transpose(r[sl][hf], t);
            put(kvsel, g + 8 * sl, 2 * (4 * ch + t) + hf,
                make_uint4(r[sl][hf][0], r[sl][hf][1], r[sl][hf][2], r[sl][hf][3]));
        }
}

// lt_kv_read of 4-bit cells, one CTA per (16 cells of the call, head) as in the
// write: cells that fill a block are read as a tile, a part a warp; others a
// cell a warp at a time, eight values a lane.
template <int D>
__global__ void __launch_bounds__(q4_parts(D) * 32) kv_read_q4_kernel(const uint8_t* __restrict__ pool_layer,
                                                                      const int2* __restrict__ cells, int n,
                                                                      int n_kv_heads, int shift,
                                                                      void* __restrict__ k_out,
                                                                      void* __restrict__ v_out, int out_f32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.x % n_kv_heads, i0 = (int)(blockIdx.x / n_kv_heads) * kBlock - shift;
    // lane l looks at cell i0 + l % 16: every warp finds the same answer
    const int mine = i0 + (lane & 15);
    const bool live = mine >= 0 && mine < n;
    const int2 cell = live ? __ldg(cells + mine) : make_int2(-1, -1);
    const int block0 = __shfl_sync(kFull, cell.x, 0);
    if (__all_sync(kFull, live && cell.y == (lane & 15) && cell.x == block0)) {
        const uint8_t* tile = pool_layer + ((size_t)block0 * n_kv_heads + h) * q4_tile_bytes(D);
        q4_part_values<D>(tile, warp, lane, [&](int kvsel, int slot, int c, uint4 x) {
            void* out = kvsel ? v_out : k_out;
            const size_t at = ((size_t)(i0 + slot) * n_kv_heads + h) * D + 8 * c;
            if (!out_f32) {
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) = x;
                return;
            }
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            float f[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 y = __half22float2(as_h2(w[j]));
                f[2 * j] = y.x;
                f[2 * j + 1] = y.y;
            }
            store8_as(out, at, 1, f);
        });
        return;
    }
    constexpr int CH = D / 8, W = q4_parts(D);
    for (int j = warp; j < kBlock; j += W) {
        const int blk = __shfl_sync(kFull, cell.x, j), slot = __shfl_sync(kFull, cell.y, j);
        if (blk < 0 || lane >= 2 * CH) continue;
        const int kvsel = lane / CH, c = lane % CH;
        float x[8];
        cell_values8<D, LT_KV_Q4_0>(pool_layer, (size_t)blk * n_kv_heads + h, kvsel, slot, c, x);
        store8_as(kvsel ? v_out : k_out, ((size_t)(i0 + j) * n_kv_heads + h) * D + 8 * c, out_f32, x);
    }
}

// -------------------------------------------------------------- expand ----
// 4-bit tiles -> f16 tiles (lt_kv_layout.cuh) for the shared-prefix pass, whose
// tensor-core operands they are.  One warp per (block, head, part).  Reads
// 18*D bytes a tile and writes 64*D.
struct ExpandParams {
    const uint8_t* pool;
    const int32_t* tables;
    uint16_t* out;
    int32_t* err;
    int max_blocks, n_kv_heads, n_blocks, n_groups, total;  // total: blocks of all groups
    ExpandGroup groups[kExpandGroups];
    int first[kExpandGroups];  // blocks before each group
};

template <int D>
__global__ void __launch_bounds__(256) expand_q4_kernel(const __grid_constant__ ExpandParams p) {
    const int lane = threadIdx.x & 31;
    const int item = (int)((blockIdx.x * 256u + threadIdx.x) >> 5);
    constexpr int P = q4_parts(D);
    if (item >= p.total * p.n_kv_heads * P) return;
    const int part = item % P, h = item / P % p.n_kv_heads, b = item / P / p.n_kv_heads;
    int lo = 0, hi = p.n_groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.first[mid] <= b) lo = mid; else hi = mid - 1;
    }
    const ExpandGroup gr = p.groups[lo];
    const int i = b - p.first[lo];
    const int src = checked_block(__ldg(p.tables + (size_t)gr.root * p.max_blocks + gr.first + i), p.n_blocks, p.err);
    const uint8_t* tile = p.pool + ((size_t)src * p.n_kv_heads + h) * q4_tile_bytes(D);
    uint16_t* out = p.out + ((size_t)(gr.base + i) * p.n_kv_heads + h) * (2 * kBlock * D);
    q4_part_values<D>(tile, part, lane, [&](int kvsel, int slot, int c, uint4 x) {
        *reinterpret_cast<uint4*>(out + kvsel * kBlock * D + chunk_off(c, slot)) = x;
    });
}

// The values of a (token, head)'s result that one lane holds once the columns
// are joined: dims 16m + g + 8*row(v), head col(v).  PACK: lanes t and t^2
// hold the same heads, so each keeps one of the two rows.
template <bool PACK>
struct Own {
    static constexpr int N = PACK ? 2 : 4;
    static __device__ __forceinline__ int row(int v, int t) { return PACK ? t >> 1 : v >> 1; }
    static __device__ __forceinline__ int col(int v) { return v & 1; }
    static __device__ __forceinline__ int head(int v, int t) { return (PACK ? 2 * (t & 1) : 2 * t) + (v & 1); }
};

// Fold partials `first`, first + stride, ... <= last into (M, L, acc).  L and
// M of columns 0 and 1; log2 units.  Loads of a batch of U partials overlap.
template <int D, bool PACK>
__device__ __forceinline__ void q4_merge_slots(const float* po, const float* pml, int G, int g, int t, int first,
                                               int last, int stride, float (&M)[2], float (&L)[2],
                                               float (&acc)[D / 16][Own<PACK>::N]) {
    using O = Own<PACK>;
    constexpr int U = PACK ? 4 : 2;
    const int h0 = O::head(0, t);
    const int lastv = first + ((last - first) / stride) * stride;
    for (int w = first; w <= lastv; w += U * stride) {
        float pm[U][2], pl[U][2], x[U][D / 16][O::N];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t ww = (size_t)min(w + u * stride, lastv);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int h = min(h0 + c, G - 1);
                pm[u][c] = __ldcg(pml + (ww * G + h) * 2);
                pl[u][c] = __ldcg(pml + (ww * G + h) * 2 + 1);
            }
#pragma unroll
            for (int v = 0; v < O::N; ++v) {
                const float* src = po + (ww * G + min(h0 + O::col(v), G - 1)) * D + g + 8 * O::row(v, t);
#pragma unroll
                for (int m = 0; m < D / 16; ++m) x[u][m][v] = __ldcg(src + 16 * m);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (w + u * stride > lastv) break;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float Mn = fmaxf(M[c], pm[u][c]);
                const float a = M[c] == Mn ? 1.f : ex2(M[c] - Mn), b = pm[u][c] == Mn ? 1.f : ex2(pm[u][c] - Mn);
                M[c] = Mn;
                L[c] = L[c] * a + pl[u][c] * b;
#pragma unroll
                for (int v = 0; v < O::N; ++v)
                    if (O::col(v) == c)
#pragma unroll
                        for (int m = 0; m < D / 16; ++m) acc[m][v] = acc[m][v] * a + x[u][m][v] * b;
            }
        }
    }
}

// Fold the prefix pass's partials (lt_kv_kernels.cu) of the blocks before
// `skip` into (M, L, acc); the same log2 units.
template <int D, bool PACK>
__device__ __forceinline__ void q4_fold_prefix(const AttnParams& p, int tok, int h, int g, int t, float (&M)[2],
                                               float (&L)[2], float (&acc)[D / 16][Own<PACK>::N]) {
    using O = Own<PACK>;
    const size_t r0 = ((size_t)tok * p.n_kv_heads + h) * p.group;
#pragma unroll 1
    for (int sp = 0; sp < p.pre_splits; ++sp) {
        const size_t rs = r0 + (size_t)sp * p.pre_split_rows;
        float a[2], b[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const size_t r = rs + min(O::head(c, t), p.group - 1);
            const float mp = __ldcg(p.pre_ml + r * 2), lp = __ldcg(p.pre_ml + r * 2 + 1);
            const float Mn = fmaxf(M[c], mp);
            a[c] = M[c] == Mn ? 1.f : ex2(M[c] - Mn);
            b[c] = mp == Mn ? 1.f : ex2(mp - Mn);
            M[c] = Mn;
            L[c] = L[c] * a[c] + lp * b[c];
        }
#pragma unroll
        for (int v = 0; v < O::N; ++v) {
            const float* src = p.pre_o + (rs + min(O::head(v, t), p.group - 1)) * D + g + 8 * O::row(v, t);
#pragma unroll
            for (int m = 0; m < D / 16; ++m) acc[m][v] = acc[m][v] * a[O::col(v)] + __ldcg(src + 16 * m) * b[O::col(v)];
        }
    }
}

// Store the heads' rows at `dst` ([group][D] f32 or f16), each times inv of its column.
template <int D, bool PACK>
__device__ __forceinline__ void q4_store_rows(void* dst, bool f16, int G, int g, int t, const float (&inv)[2],
                                              const float (&acc)[D / 16][Own<PACK>::N]) {
    using O = Own<PACK>;
    if (f16) {
#pragma unroll
        for (int v = 0; v < O::N; ++v) {
            const int h = O::head(v, t);
            if (h >= G) continue;
            __half* at = static_cast<__half*>(dst) + h * D + g + 8 * O::row(v, t);
#pragma unroll
            for (int m = 0; m < D / 16; ++m) at[16 * m] = __float2half_rn(acc[m][v] * inv[O::col(v)]);
        }
    } else {
#pragma unroll
        for (int v = 0; v < O::N; ++v) {
            const int h = O::head(v, t);
            if (h >= G) continue;
            float* at = static_cast<float*>(dst) + h * D + g + 8 * O::row(v, t);
#pragma unroll
            for (int m = 0; m < D / 16; ++m) at[16 * m] = acc[m][v] * inv[O::col(v)];
        }
    }
}

// The producer warp: kQ4Lanes lanes feed each worker.
template <int D, bool SH>
__device__ __forceinline__ void q4_produce(const AttnParamsOf<SH>& p, uint8_t* stages0, Q4Ring* rings, int lane) {
    constexpr int TILE = q4_tile_bytes(D), S = kQ4Stages, NT = kQ4Step;
    const int G = p.group, Hkv = p.n_kv_heads, C = p.piece_cost;
    const int WSM = q4_worker_smem(G, D, p.q_f32), QBUF = q4_qbuf_bytes(G, D, p.q_f32), nqb = q4_qbufs(G, D, p.q_f32);
    const uint32_t qbytes = (uint32_t)(G * D * (p.q_f32 ? 4 : 2));
    constexpr int LN = kQ4Lanes;
    const int c = min(lane / LN, kQ4Workers - 1), u = lane % LN;
    const int gw = blockIdx.x * kQ4Workers + c;
    Q4Ring* ring = rings + c;
    const uint32_t stages = smem_u32(stages0) + c * WSM, qbufs = stages + S * NT * TILE, bar0 = smem_u32(ring->full);
    const TokenDesc* toks = p.toks ? p.toks : p.inl;
    const uint8_t* pool = reinterpret_cast<const uint8_t*>(p.pool_layer);
    const uint32_t T = (uint32_t)p.tiles_per_head * Hkv, NW = (uint32_t)p.n_warps, quo = T / NW, rem = T % NW;
    bool live = lane / LN < kQ4Workers && gw < p.n_warps;

    // The generator's place: (token, head, offset); offsets below C are the (token, head)'s cost.
    int gi = 0, gh = 0, go = 0, gt = 0, t1 = 0;
    if (live) {
        // Range [T * gw / n, T * (gw + 1) / n) of T < 2^31, in 32 bits: with
        // T = quo * n + rem, floor(T * w / n) = quo * w + floor(rem * w / n).
        gt = (int)(quo * gw + rem * gw / NW);
        t1 = (int)(quo * (gw + 1) + rem * (gw + 1) / NW);
        int lo = 0, hi = p.n_tok - 1;  // last token whose first tile is <= gt
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (toks[mid].prefix * Hkv <= gt) lo = mid; else hi = mid - 1;
        }
        gi = lo;
        const uint32_t nv = (uint32_t)(toks[gi].pos / kBlock + 1 - toks[gi].skip + C), off = (uint32_t)(gt - toks[gi].prefix * Hkv);
        gh = (int)(off / nv);
        go = (int)(off % nv);
    }
    int qslot = nqb - 1;  // q buffer of the piece being issued
    int pi = -1, it = 0, len = 0, head = 0, tok = 0, b_last = -1;  // the piece being issued
    const int32_t* trow = p.tables;
    int id = 0;  // block of tile it + u
    uint32_t issued = 0;
    bool first = true;
    uint32_t idle = 0;  // passes without progress, and when the first of them was
    uint64_t t_idle = 0;
    auto load_id = [&]() {
        if (it + u < len)
            id = it + u == len - 1 && b_last >= 0 ? b_last
                                                  : checked_block(__ldg(trow + it + u), p.n_blocks, p.err, p.check_ids != 0);
    };
    for (;;) {
        bool moved = false;
        // One reading for a worker's lanes, which must decide alike.
        const uint32_t done = __shfl_sync(kFull, ld_acquire_cta(&ring->consumed), lane & ~(LN - 1));
        const uint32_t taken = __shfl_sync(kFull, ld_acquire_cta(&ring->q_taken), lane & ~(LN - 1));
        const uint32_t stop = __shfl_sync(kFull, ld_acquire_cta(&ring->stop), lane & ~(LN - 1));
        if (live) {
            if (stop) {
                if (u == 0) st_release_cta(&ring->stopped, 1);
                live = false;
            } else if (it < len) {
                // lane u issues tile it + u, the u % NT-th of stage issued + u / NT
                const int room = S - (int)(issued - done);
                int n = min(min(LN / NT, room), (len - it + NT - 1) / NT);
                if (it == 0 && pi - (int)taken >= nqb) n = 0;  // no q buffer free
                if (n > 0) {
                    if (it == 0 && u == 0) {
                        const uint32_t qbar = smem_u32(ring->q_full) + 8u * qslot;
                        mbar_arrive_expect_tx(qbar, qbytes);
                        bulk_g2s(qbufs + qslot * QBUF,
                                 static_cast<const uint8_t*>(p.q) + ((size_t)tok * Hkv + head) * qbytes, qbytes, qbar);
                        st_release_cta(&ring->q_issued, (uint32_t)pi + 1);
                    }
                    if (u < n * NT && it + u < len) {
                        const uint32_t st = (issued + u / NT) % S, bar = bar0 + 8u * st;
                        if (u % NT == 0) mbar_arrive_expect_tx(bar, TILE * min(NT, len - it - u));
                        bulk_g2s(stages + (st * NT + u % NT) * TILE, pool + ((size_t)id * Hkv + head) * TILE, TILE, bar);
                    }
                    issued += n;
                    it = min(it + n * NT, len);
                    if (u == 0) st_release_cta(&ring->issued, issued);
                    load_id();
                    moved = true;
                }
            } else {
                // ---- next piece ----
                const TokenDesc td = toks[min(gi, p.n_tok - 1)];
                const int nb = td.pos / kBlock + 1 - td.skip, nv = nb + C;
                if (go < C) {
                    gt += C - go;
                    go = C;
                }
                if (gt >= t1) {  // the range ends here
                    live = false;
                    if (first && u == 0) {  // ... and has no tile: wake the worker
                        st_release_cta(&ring->none, 1);
                        mbar_arrive(smem_u32(ring->q_full));
                    }
                } else {
                    first = false;
                    ++pi;
                    qslot = qslot + 1 == nqb ? 0 : qslot + 1;
                    len = min(nv - go, t1 - gt);
                    it = 0;
                    head = gh;
                    tok = gi;
                    const int b0 = go - C;
                    b_last = b0 + len == nb ? td.last_block : -1;
                    trow = p.tables + (size_t)td.seq * p.max_blocks + td.skip + b0;
                    load_id();
                    if (u == 0) {
                        Q4Piece r;
                        r.tok = gi;
                        r.h = gh;
                        r.pos = td.pos;
                        r.b0 = b0;
                        r.b1 = b0 + len;
                        r.kind = b0 > 0 ? 1 : b0 + len < nb ? 2 : 0;
                        r.last_block = b_last;
                        r.skip = td.skip;
                        r.first = td.prefix * Hkv + gh * nv + C;
                        r.lo = r.qpos = 0;
                        if constexpr (SH) {
                            const ShapeDesc sd = p.shapes ? p.shapes[gi] : p.inl_shapes[gi];
                            r.lo = sd.lo;
                            r.qpos = sd.qpos;
                        }
                        // the next piece, if any, starts after the next (token, head)'s cost
                        r.last = gt + len + (go + len == nv ? C : 0) >= t1;
                        ring->pieces[pi % kQ4Pieces] = r;
                        // the token's last block entry, written once per token (head 0)
                        if (gh == 0 && b_last >= 0) p.tables[(size_t)td.seq * p.max_blocks + td.skip + b0 + len - 1] = b_last;
                    }
                    gt += len;
                    go += len;
                    if (go == nv) {
                        go = 0;
                        if (++gh == Hkv) {
                            gh = 0;
                            ++gi;
                        }
                    }
                    moved = true;
                }
            }
        }
        if (!__any_sync(kFull, live)) break;
        if (__any_sync(kFull, moved)) {
            idle = 0;
        } else {
            if (idle == 0) t_idle = global_ns();
            __nanosleep(20);
            // (the workers' own waits are shorter)
            if ((++idle & 255u) == 0 && __any_sync(kFull, global_ns() - t_idle > 2 * kWaitLimitNs)) {
                if (lane == 0) atomicOr(p.err, kErrTimeout);
                break;
            }
        }
    }
}

template <int D, bool PACK, bool SH, bool Q16>
__global__ void __launch_bounds__(kQ4Threads, 2) attn_q4_kernel(const __grid_constant__ AttnParamsOf<SH> p) {
    constexpr int TILE = q4_tile_bytes(D);
    constexpr int KS = D / 16;   // 16-dim steps of K, and 16-dim row tiles of V
    constexpr int G32 = D / 32;  // scale groups
    constexpr int S = kQ4Stages, NT = kQ4Step;
    using O = Own<PACK>;
    extern __shared__ __align__(1024) uint8_t smem[];

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int Hkv = p.n_kv_heads, G = p.group;
    const int WSM = q4_worker_smem(G, D, p.q_f32);
    Q4Ring* rings = reinterpret_cast<Q4Ring*>(smem + (size_t)kQ4Workers * WSM);
    if (warp < kQ4Workers) {
        Q4Ring* r = rings + warp;
        if (lane < S) mbar_init(smem_u32(r->full) + 8u * lane, 1);
        else if (lane < S + kQ4QBufs) mbar_init(smem_u32(r->q_full) + 8u * (lane - S), 1);
        if (lane == 31) r->consumed = r->q_taken = r->issued = r->q_issued = r->none = r->stop = r->stopped = 0;
        fence_mbar_init();
    }
    __syncthreads();
    if (warp == kQ4Workers) {
        q4_produce<D, SH>(p, smem, rings, lane);
        return;
    }
    const int gw = blockIdx.x * kQ4Workers + warp;
    if (gw >= p.n_warps) return;

    Q4Ring* ring = rings + warp;
    uint8_t* stages = smem + (size_t)warp * WSM;
    uint8_t* qbufs = stages + S * NT * TILE;
    const int QBUF = q4_qbuf_bytes(G, D, p.q_f32), nqb = q4_qbufs(G, D, p.q_f32);
    const uint32_t bar0 = smem_u32(ring->full);
    const uint32_t T = (uint32_t)p.tiles_per_head * Hkv;
    const int g = lane >> 2, t = lane & 3;
    int ci = 0, ct = 0;  // the piece in hand, and its tiles consumed
    uint32_t consumed = 0;  // stages
    int qslot = 0, qphase = 0;  // q buffer of the next piece
    int c_len = 0, c_end = 0, c_lo = 0, c_q = 0;  // its length; its end, first position and own position from its start
    // an opaque zero keeps the exponent patterns in registers (see Q4Magic)
    const uint32_t zero = (uint32_t)p.n_warps >> 31;
    const Q4Magic magic{0x64006400u + zero, 0x54005400u + zero};

    // B fragments: values (PACK: residuals in columns 4-7), residuals
    uint32_t qh[KS][2], ql[PACK || Q16 ? 1 : KS][2];
    float cmul[2] = {0.f, 0.f};                // from the MMA's units to q.k (SH) or log2 units
    float slope[2] = {0.f, 0.f};
    float o[KS][4];
    // Weights are 2^(score - mb): mb trails the running maximum by 7, and moves
    // only when a score passes it by 15, so they stay within (0, 2^15] (an f16
    // and its residual keep 22 bits of all but the smallest) and o is rescaled rarely.
    float mb[2], l_run[2];
    bool ok = true;
    int items_out = 0;
    int lead_to = 0;  // last worker of the group of partials this one combines, 0: none

    // Join lanes and columns of the running piece: M, L of columns 0 and 1, acc.
    auto join = [&](float (&M)[2], float (&L)[2], float (&acc)[KS][O::N]) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float l = l_run[c];
            l += __shfl_xor_sync(kFull, l, 4);
            l += __shfl_xor_sync(kFull, l, 8);
            l += __shfl_xor_sync(kFull, l, 16);
            L[c] = l;
            M[c] = mb[c];
        }
#pragma unroll
        for (int m = 0; m < KS; ++m) {
            if constexpr (PACK) {
                float x[4];
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    // lanes t < 2 hold minus the values' part, t >= 2 the residuals'
                    const float y = __shfl_xor_sync(kFull, o[m][v], 2);
                    x[v] = t < 2 ? y - o[m][v] : o[m][v] - y;
                }
                acc[m][0] = t < 2 ? x[0] : x[2];
                acc[m][1] = t < 2 ? x[1] : x[3];
            } else {
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[m][v] = o[m][v];
            }
        }
    };

    // ---- q rows of a piece -> B fragments ----
    auto load_q = [&](const uint8_t* qbuf) {
        const int qg = PACK ? g & 3 : g;
        const int at = min(qg, G - 1) * D + 2 * t;
        float2 x[2 * KS];  // q values 16 ks + 8 hf + 2t, + 1 at 2 ks + hf
        if constexpr (!Q16) {
#pragma unroll
            for (int i = 0; i < 2 * KS; ++i) x[i] = *reinterpret_cast<const float2*>(qbuf + (at + 8 * i) * 4);
        } else {
#pragma unroll
            for (int i = 0; i < 2 * KS; ++i)
                x[i] = __half22float2(*reinterpret_cast<const __half2*>(qbuf + (at + 8 * i) * 2));
        }
        // Rows past the group repeat its last one; nothing stores their results.
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) mx = fmaxf(mx, fmaxf(fabsf(x[i].x), fabsf(x[i].y)));
        mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 2));
        float f, finv;
        q_row_scale(mx, f, finv);
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) {
            const float y0 = x[i].x * f, y1 = x[i].y * f;
            const __half2 hi = __floats2half2_rn(y0, y1);
            qh[i >> 1][i & 1] = h2_bits(hi);
            if constexpr (!Q16) {
                const float2 back = __half22float2(hi);
                const uint32_t lo = h2_bits(__floats2half2_rn(y0 - back.x, y1 - back.y));
                if constexpr (!PACK) ql[i >> 1][i & 1] = lo;
                else if (g >= 4) qh[i >> 1][i & 1] = lo;
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            cmul[c] = __shfl_sync(kFull, finv, 8 * t + 4 * c);
            if constexpr (SH) {
                const int hh = O::head(c, t);
                slope[c] = p.shape.slopes && hh < G
                               ? __ldg(p.shape.slopes + ring->pieces[ci % kQ4Pieces].h * G + hh) * kLog2e
                               : 0.f;
            } else {
                cmul[c] *= p.scale_log2;
            }
        }
    };

    // Fused append: quantise this token's new K and V row of head h into its
    // pool cell and into the staged tile.
    auto append = [&](uint8_t* tile) {
        constexpr int L = D / 4;  // lanes of one row
        const Q4Piece dc = ring->pieces[ci % kQ4Pieces];
        const int slot = dc.pos % kBlock;
        uint8_t* cell_tile = reinterpret_cast<uint8_t*>(p.pool_layer_w) + ((size_t)dc.last_block * Hkv + dc.h) * TILE;
#pragma unroll 1
        for (int r = 0; r < 2 * L / 32; ++r) {
            const int kvsel = (r * 32 + lane) / L, i = (lane % L) >> 2;
            float x[4];
            load4_f32(kvsel ? p.v_new : p.k_new, (size_t)dc.tok * Hkv * D + (size_t)dc.h * D + 16 * i + 2 * t, p.kv_f32,
                      x);
            uint32_t code[4];
            const float d = q4_quant<4>(x, code);
            q4_store4<D>(tile, kvsel, i, t, slot, code, d);
            q4_store4<D>(cell_tile, kvsel, i, t, slot, code, d);
        }
        __syncwarp();
    };

    // ---- the next nt <= NT staged tiles, blocks ct .. of the piece ----
    // A step short of a tile takes its first tile again with every score -inf
    // (weights 0, finite values): one copy of the code serves both.
    auto step = [&](int nt) {
        const uint8_t* tiles[NT];
        tiles[0] = stages + (consumed % S) * (NT * TILE);
#pragma unroll
        for (int u = 1; u < NT; ++u) tiles[u] = u < nt ? tiles[0] + u * TILE : tiles[0];
        // S^T = K Q^T
        float sc[NT][4];  // (slot g | g+8) x (column 2t | 2t+1)
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            const uint8_t* tile = tiles[u];
            uint32_t kd[G32];  // scales of slot g (first half of the run) and g+8
            const uint8_t* ks_p = tile + 16 * D + g * (4 * G32);
            if constexpr (D == 128) {
                const uint4 r = *reinterpret_cast<const uint4*>(ks_p);
                kd[0] = r.x, kd[1] = r.y, kd[2] = r.z, kd[3] = r.w;
            } else {
                const uint2 r = *reinterpret_cast<const uint2*>(ks_p);
                kd[0] = r.x, kd[1] = r.y;
            }
#pragma unroll
            for (int ch = 0; ch < D / 64; ++ch) {
                const uint4 wv = *reinterpret_cast<const uint4*>(tile + ch * 512 + lane * 16);
                const uint32_t w[4] = {wv.x, wv.y, wv.z, wv.w};
                const float2 dg = __half22float2(as_h2(kd[ch]));              // slot g, groups 2ch, 2ch+1
                const float2 dg8 = __half22float2(as_h2(kd[G32 / 2 + ch]));  // slot g+8
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                    float tt[4];
#pragma unroll
                    for (int q2 = 0; q2 < 2; ++q2) {
                        const int ks = 4 * ch + 2 * cc + q2;
                        const uint32_t w0 = w[2 * cc + q2], w8 = w0 >> 8;
                        const uint32_t a[4] = {h2_bits(q4_low(w0, magic)), h2_bits(q4_low(w8, magic)), h2_bits(q4_high(w0, magic)),
                                               h2_bits(q4_high(w8, magic))};
                        if (q2 == 0) mma16816_zero(tt, a, qh[ks][0], qh[ks][1]);
                        else mma16816_add(tt, a, qh[ks][0], qh[ks][1]);
                        if constexpr (!PACK && !Q16) mma16816_add(tt, a, ql[ks][0], ql[ks][1]);
                    }
                    const float d0 = cc ? dg.y : dg.x, d1 = cc ? dg8.y : dg8.x;
                    const bool first = ch == 0 && cc == 0;
                    sc[u][0] = first ? d0 * tt[0] : sc[u][0] + d0 * tt[0];
                    sc[u][1] = first ? d0 * tt[1] : sc[u][1] + d0 * tt[1];
                    sc[u][2] = first ? d1 * tt[2] : sc[u][2] + d1 * tt[2];
                    sc[u][3] = first ? d1 * tt[3] : sc[u][3] + d1 * tt[3];
                }
            }
        }
        const int j0 = ct * kBlock;  // first position of the step in the piece
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            if constexpr (PACK && !Q16) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[u][e] += __shfl_xor_sync(kFull, sc[u][e], 2);
            }
            if constexpr (SH) {
                const int ju = j0 + u * kBlock, lo = c_lo - ju;
                const TileShape s0{p.shape, slope[0], c_q - ju, lo}, s1{p.shape, slope[1], c_q - ju, lo};
                sc[u][0] = s0.score(sc[u][0] * cmul[0], g);
                sc[u][1] = s1.score(sc[u][1] * cmul[1], g);
                sc[u][2] = s0.score(sc[u][2] * cmul[0], g + 8);
                sc[u][3] = s1.score(sc[u][3] * cmul[1], g + 8);
                if (g < lo) sc[u][0] = sc[u][1] = -INFINITY;
                if (g + 8 < lo) sc[u][2] = sc[u][3] = -INFINITY;
            } else {
                sc[u][0] *= cmul[0];
                sc[u][1] *= cmul[1];
                sc[u][2] *= cmul[0];
                sc[u][3] *= cmul[1];
            }
        }
        const int filled = min(c_end, c_len * kBlock) - j0;  // positions from the step's first to the piece's end
        if (filled < NT * kBlock) {
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                if (g + u * kBlock >= filled) sc[u][0] = sc[u][1] = -INFINITY;
                if (g + 8 + u * kBlock >= filled) sc[u][2] = sc[u][3] = -INFINITY;
            }
        }

        // softmax
        float mx0 = fmaxf(sc[0][0], sc[0][2]), mx1 = fmaxf(sc[0][1], sc[0][3]);
#pragma unroll
        for (int u = 1; u < NT; ++u) {
            mx0 = fmaxf(mx0, fmaxf(sc[u][0], sc[u][2]));
            mx1 = fmaxf(mx1, fmaxf(sc[u][1], sc[u][3]));
        }
        if (__any_sync(kFull, mx0 > mb[0] + 15.f || mx1 > mb[1] + 15.f)) {
#pragma unroll
            for (int m = 4; m < 32; m <<= 1) {
                mx0 = fmaxf(mx0, __shfl_xor_sync(kFull, mx0, m));
                mx1 = fmaxf(mx1, __shfl_xor_sync(kFull, mx1, m));
            }
            const float n0 = fmaxf(mb[0], mx0 - 7.f), n1 = fmaxf(mb[1], mx1 - 7.f);
            const float a0 = n0 == mb[0] ? 1.f : ex2(mb[0] - n0), a1 = n1 == mb[1] ? 1.f : ex2(mb[1] - n1);
            mb[0] = n0;
            mb[1] = n1;
            l_run[0] *= a0;
            l_run[1] *= a1;
#pragma unroll
            for (int m = 0; m < KS; ++m) {
                o[m][0] *= a0;
                o[m][1] *= a1;
                o[m][2] *= a0;
                o[m][3] *= a1;
            }
        }
        // Nothing seen yet (an empty interval): weights ex2(-inf) = 0.
        const float r0 = SH && mb[0] == -INFINITY ? 0.f : mb[0], r1 = SH && mb[1] == -INFINITY ? 0.f : mb[1];
        // P^T as B fragments: value = the leading 11 bits (an f16), residual = the rest.
        constexpr uint32_t kLead = 0xffffe000u;
        uint32_t ph[NT][2];
        [[maybe_unused]] uint32_t pl[PACK ? 1 : NT][2];
        [[maybe_unused]] const float own = t < 2 ? 0.f : 1.f;
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            const float p0 = ex2(sc[u][0] - r0), p1 = ex2(sc[u][1] - r1), p2 = ex2(sc[u][2] - r0),
                        p3 = ex2(sc[u][3] - r1);
            l_run[0] += p0 + p2;
            l_run[1] += p1 + p3;
            auto lead = [&](float v) { return __uint_as_float(__float_as_uint(v) & kLead); };
            if constexpr (PACK) {
                // lanes t < 2: minus the value; t >= 2: the residual (join() puts the sign right)
                ph[u][0] = movmatrix_trans(h2_bits(__floats2half2_rn(fmaf(p0, own, -lead(p0)), fmaf(p1, own, -lead(p1)))));
                ph[u][1] = movmatrix_trans(h2_bits(__floats2half2_rn(fmaf(p2, own, -lead(p2)), fmaf(p3, own, -lead(p3)))));
            } else {
                const float v0 = lead(p0), v1 = lead(p1), v2 = lead(p2), v3 = lead(p3);
                ph[u][0] = movmatrix_trans(h2_bits(__floats2half2_rn(v0, v1)));
                ph[u][1] = movmatrix_trans(h2_bits(__floats2half2_rn(v2, v3)));
                pl[u][0] = movmatrix_trans(h2_bits(__floats2half2_rn(p0 - v0, p1 - v1)));
                pl[u][1] = movmatrix_trans(h2_bits(__floats2half2_rn(p2 - v2, p3 - v3)));
            }
        }

        // O^T += V^T P^T.  The MMA's own accumulation rounds towards zero, which over
        // the ~100 tiles of a range would shrink O by 100 * 2^-25; so the step's
        // products are summed from zero there and added in f32, to nearest.
#pragma unroll
        for (int ch = 0; ch < D / 64; ++ch) {
            uint4 wv[NT], vd[NT];
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                wv[u] = *reinterpret_cast<const uint4*>(tiles[u] + 8 * D + ch * 512 + lane * 16);
                vd[u] = *reinterpret_cast<const uint4*>(tiles[u] + 17 * D + (t * G32 + 2 * ch) * 8);
            }
#pragma unroll
            for (int mm = 0; mm < 4; ++mm) {
                const int m = 4 * ch + mm;
                float tt[4];
#pragma unroll
                for (int u = 0; u < NT; ++u) {
                    const uint32_t w[4] = {wv[u].x, wv[u].y, wv[u].z, wv[u].w};
                    const __half2 dA = as_h2(mm < 2 ? vd[u].x : vd[u].z), dB = as_h2(mm < 2 ? vd[u].y : vd[u].w);
                    const uint32_t w0 = w[mm], w8 = w0 >> 8;
                    const uint32_t a[4] = {h2_bits(__hmul2(q4_low(w0, magic), dA)), h2_bits(__hmul2(q4_high(w0, magic), dA)),
                                           h2_bits(__hmul2(q4_low(w8, magic), dB)), h2_bits(__hmul2(q4_high(w8, magic), dB))};
                    if (u == 0) mma16816_zero(tt, a, ph[u][0], ph[u][1]);
                    else mma16816_add(tt, a, ph[u][0], ph[u][1]);
                    if constexpr (!PACK) mma16816_add(tt, a, pl[u][0], pl[u][1]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) o[m][e] += tt[e];
            }
        }
    };

    // The worker that holds tile x: the last w with floor(T * w / n) <= x, from a
    // rounded quotient (a 64-bit division costs ten times the correction).
    auto warp_of = [&](int x) {
        const uint32_t NW = (uint32_t)p.n_warps, quo = T / NW, rem = T % NW;
        auto start = [&](int w) { return (int)(quo * (uint32_t)w + rem * (uint32_t)w / NW); };
        int w = min(p.n_warps - 1, (int)__fdividef((float)x * (float)p.n_warps, (float)T));
        while (w > 0 && start(w) > x) --w;
        while (w + 1 < p.n_warps && start(w + 1) <= x) ++w;
        return w;
    };
    for (;;) {
        if (ct == c_len) {  // the next piece: its descriptor came before its q rows
            if (!mbar_wait_bounded(smem_u32(ring->q_full) + 8u * qslot, (uint32_t)qphase)) {
                ok = false;
                break;
            }
            if (ld_acquire_cta(&ring->none)) return;
            const Q4Piece& c = ring->pieces[ci % kQ4Pieces];
            const int base = (c.skip + c.b0) * kBlock;
            c_len = c.b1 - c.b0;
            c_end = c.pos + 1 - base;
            c_lo = c.lo - base;
            c_q = c.qpos - base;
            ct = 0;
            load_q(qbufs + qslot * QBUF);
            if (++qslot == nqb) {
                qslot = 0;
                qphase ^= 1;
            }
            __syncwarp();
            if (lane == 0) st_release_cta(&ring->q_taken, (uint32_t)ci + 1);
#pragma unroll
            for (int m = 0; m < KS; ++m) o[m][0] = o[m][1] = o[m][2] = o[m][3] = 0.f;
            mb[0] = mb[1] = -INFINITY;
            l_run[0] = l_run[1] = 0.f;
        }
        const int nt = min(c_len - ct, NT);
        if (!mbar_wait_bounded(bar0 + 8u * (consumed % S), consumed / S & 1)) {
            ok = false;
            break;
        }
        const bool fill = !SH && p.k_new && ct + nt == c_len && ring->pieces[ci % kQ4Pieces].last_block >= 0;
        if (fill) append(stages + ((consumed % S) * NT + nt - 1) * TILE);
        step(nt);
        ++consumed;
        ct += nt;
        if (fill) fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) st_release_cta(&ring->consumed, consumed);
        if (ct < c_len) continue;

        // ---- piece done ----
        // what: 0 store the output, 1 the warp's partial, 2 merge the following
        // warps' partials and store the output, 3 lead: combine the partials of
        // this warp and its next neighbours into a group partial.
        const Q4Piece dc = ring->pieces[ci % kQ4Pieces];
        const bool last_piece = dc.last != 0;
        if (dc.kind == 1 && p.part2_o) {  // the range's first piece
            // Helpers of a cut (token, head) are the workers after the one with
            // its first tile; with more than kMergeGroup of them, every
            // kMergeGroup-th leads, so that the merging one reads one partial a group.
            const int ws = warp_of(dc.first), we = warp_of(dc.first + dc.pos / kBlock - dc.skip);
            if (we - ws > kMergeGroup && (gw - ws - 1) % kMergeGroup == 0) lead_to = min(gw + kMergeGroup - 1, we);
        }
        int what = dc.kind;
        if (last_piece && what == 2) {
            // this warp's own partial is stored: its flag may go up before the merge's wait
            __syncwarp();
            if (lane == 0) st_release_gpu(p.flags + gw, p.epoch);
            if (lead_to) what = 3;
        }
#pragma unroll 1
        for (;;) {
            float M[2], L[2], acc[KS][O::N], inv[2] = {1.f, 1.f};
            if (what != 3) {
                join(M, L, acc);
            } else {
                M[0] = M[1] = -INFINITY;
                L[0] = L[1] = 0.f;
#pragma unroll
                for (int m = 0; m < KS; ++m)
#pragma unroll
                    for (int v = 0; v < O::N; ++v) acc[m][v] = 0.f;
            }
            bool rd = true;
            if (what >= 2) {
                int from = gw, to = lead_to, stride = 1;
                bool groups = false;
                if (what == 2) {
                    from = gw + 1;
                    to = warp_of(dc.first + dc.pos / kBlock - dc.skip);
                    groups = p.part2_o && to - gw > kMergeGroup;
                    stride = groups ? kMergeGroup : 1;
                }
                // (a leader's own flag is up: `from` may be itself)
                rd = wait_flags(groups ? p.flags2 : p.flags, p.epoch, from, to, stride, lane);
                __syncwarp();
                if (rd)
                    q4_merge_slots<D, PACK>(groups ? p.part2_o : p.part_o, groups ? p.part2_ml : p.part_ml, G, g, t,
                                            from, to, stride, M, L, acc);
                else if (lane == 0)
                    atomicOr(p.err, kErrTimeout);
            }
            if (what & 1) {  // 1, 3: a partial of this warp
                float* ml = (what == 1 ? p.part_ml : p.part2_ml) + (size_t)gw * G * 2;
                q4_store_rows<D, PACK>((what == 1 ? p.part_o : p.part2_o) + (size_t)gw * G * D, false, G, g, t, inv, acc);
                if (g == 0 && (!PACK || t < 2)) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int h = O::head(c, t);
                        if (h < G) {
                            ml[h * 2] = M[c];
                            ml[h * 2 + 1] = L[c];
                        }
                    }
                }
            } else {
                ++items_out;
                if (!SH && p.pre_splits > 0 && dc.skip > 0) q4_fold_prefix<D, PACK>(p, dc.tok, dc.h, g, t, M, L, acc);
                const size_t hl = (size_t)Hkv * G;
                const size_t row = p.n_peers == 0 ? dc.tok * hl + (size_t)dc.h * G
                                                  : dc.tok * (size_t)p.n_peers * hl + p.peer_rank * hl + (size_t)dc.h * G;
                uint8_t* out = static_cast<uint8_t*>(p.n_peers == 0 ? p.out : p.gather_out);
                inv[0] = L[0] == 0.f ? 0.f : 1.f / L[0];  // 0: an interval without positions
                inv[1] = L[1] == 0.f ? 0.f : 1.f / L[1];
                if (rd) q4_store_rows<D, PACK>(out + row * D * (p.out_f32 ? 4 : 2), !p.out_f32, G, g, t, inv, acc);
            }
            if (!last_piece) break;
            // Publish: every partial of this warp is visible before its flag.
            __syncwarp();
            if (what == 3) {
                if (lane == 0) st_release_gpu(p.flags2 + gw, p.epoch);  // either way: no second wait
                if (dc.kind != 2) break;
                what = 2;
                continue;
            }
            if (what == 2) break;
            if (lane == 0) st_release_gpu(p.flags + gw, p.epoch);
            if (!lead_to) break;
            what = 3;
        }
        if (last_piece) break;
        ++ci;
    }
    if (!ok) {
        // Stop the producer lanes (bounded), drain the copies in flight
        // (bounded), report; the flag goes up all the same, so that no other
        // worker waits its limit out.
        if (lane == 0) {
            atomicOr(p.err, kErrTimeout);
            st_release_cta(&ring->stop, 1);
            const uint64_t t_stop = global_ns();
            while (!ld_acquire_cta(&ring->stopped) && global_ns() - t_stop < kWaitLimitNs / 4) __nanosleep(100);
            const uint32_t issued = ld_acquire_cta(&ring->issued), q_issued = ld_acquire_cta(&ring->q_issued);
            for (uint32_t j = consumed; j < issued; ++j) mbar_wait_bounded(bar0 + 8u * (j % S), j / S & 1);
            for (uint32_t j = ld_acquire_cta(&ring->q_taken); j < q_issued; ++j)
                mbar_wait_bounded(smem_u32(ring->q_full) + 8u * (j % nqb), j / nqb & 1);
            st_release_gpu(p.flags + gw, p.epoch);
        }
        __syncwarp();
    }
    peer_done(p, lane, items_out);
}

// ------------------------------------------------------------- launches ----
template <int D, bool PACK, bool SH, bool Q16>
cudaError_t ensure_q4_attr(int dev) {
    static bool set[64] = {};
    if (set[dev]) return cudaSuccess;
    const cudaError_t e =
        cudaFuncSetAttribute(attn_q4_kernel<D, PACK, SH, Q16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             q4_smem(PACK ? 4 : kMaxGroup, D, 1));
    if (e == cudaSuccess) set[dev] = true;
    return e;
}

template <int D, bool PACK, bool SH, bool Q16>
int q4_warps_for(int dev, int group, int q_f32) {
    static int cache[64][kMaxGroup + 1][2] = {};
    int& c = cache[dev][group][q_f32 ? 1 : 0];
    if (c == 0) {
        int per_sm = 0, sms = 0;
        if (ensure_q4_attr<D, PACK, SH, Q16>(dev) != cudaSuccess) return 0;
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, attn_q4_kernel<D, PACK, SH, Q16>, kQ4Threads,
                                                          q4_smem(group, D, q_f32)) != cudaSuccess)
            return 0;
        c = (per_sm < 1 ? 1 : per_sm) * sms * kQ4Workers;
    }
    return c;
}

// Cooperative: merging warps wait for other CTAs' flags, so the whole grid
// (sized to the resident capacity) is co-resident.
template <int D, bool PACK, bool SH, bool Q16>
cudaError_t launch_q4(const AttnParamsOf<SH>& p, cudaStream_t s) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if ((e = ensure_q4_attr<D, PACK, SH, Q16>(dev)) != cudaSuccess) return e;
    const dim3 grid((p.n_warps + kQ4Workers - 1) / kQ4Workers), block(kQ4Threads);
    void* args[] = {const_cast<AttnParamsOf<SH>*>(&p)};
    return cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(&attn_q4_kernel<D, PACK, SH, Q16>), grid, block,
                                       args, q4_smem(p.group, D, p.q_f32), s);
}

// f(D, PACK, Q16 as integral constants) of a call: the one place that picks a variant.
template <class F>
auto q4_variant(int head_dim, int group, bool q16, F f) {
    using std::false_type;
    using std::true_type;
    using D64 = std::integral_constant<int, 64>;
    using D128 = std::integral_constant<int, 128>;
    if (group <= 4) {
        if (q16) return head_dim == 64 ? f(D64{}, true_type{}, true_type{}) : f(D128{}, true_type{}, true_type{});
        return head_dim == 64 ? f(D64{}, true_type{}, false_type{}) : f(D128{}, true_type{}, false_type{});
    }
    if (q16) return head_dim == 64 ? f(D64{}, false_type{}, true_type{}) : f(D128{}, false_type{}, true_type{});
    return head_dim == 64 ? f(D64{}, false_type{}, false_type{}) : f(D128{}, false_type{}, false_type{});
}

template <bool SH>
cudaError_t launch_q4_any(const AttnParamsOf<SH>& p, int head_dim, cudaStream_t s) {
    return q4_variant(head_dim, p.group, !p.q_f32, [&](auto d, auto pack, auto q16) {
        return launch_q4<decltype(d)::value, decltype(pack)::value, SH, decltype(q16)::value>(p, s);
    });
}

}  // namespace

int attend_q4_warps(int device, int group, int head_dim, int q_f32, bool shaped) {
    return q4_variant(head_dim, group, !q_f32, [&](auto d, auto pack, auto q16) {
        constexpr int D = decltype(d)::value;
        constexpr bool PACK = decltype(pack)::value, Q16 = decltype(q16)::value;
        return shaped ? q4_warps_for<D, PACK, true, Q16>(device, group, q_f32)
                      : q4_warps_for<D, PACK, false, Q16>(device, group, q_f32);
    });
}

cudaError_t launch_attend_q4(const AttnParams& p, int head_dim, cudaStream_t s) {
    return launch_q4_any<false>(p, head_dim, s);
}

cudaError_t launch_attend_q4_shaped(const AttnShapedParams& p, int head_dim, cudaStream_t s) {
    return launch_q4_any<true>(p, head_dim, s);
}

cudaError_t launch_expand_q4(const uint8_t* pool_layer, const int32_t* tables, int max_blocks, const ExpandGroup* groups,
                             int n_groups, int n_kv_heads, int head_dim, uint16_t* out, int n_blocks, int32_t* err,
                             cudaStream_t s) {
    for (int g0 = 0; g0 < n_groups; g0 += kExpandGroups) {
        ExpandParams p{};
        p.pool = pool_layer;
        p.tables = tables;
        p.out = out;
        p.err = err;
        p.max_blocks = max_blocks;
        p.n_kv_heads = n_kv_heads;
        p.n_blocks = n_blocks;
        p.n_groups = std::min(kExpandGroups, n_groups - g0);
        for (int i = 0; i < p.n_groups; ++i) {
            p.groups[i] = groups[g0 + i];
            p.first[i] = p.total;
            p.total += groups[g0 + i].count;
        }
        const unsigned blocks = (unsigned)(((long long)p.total * n_kv_heads * q4_parts(head_dim) + 7) / 8);
        if (head_dim == 64) expand_q4_kernel<64><<<blocks, 256, 0, s>>>(p);
        else expand_q4_kernel<128><<<blocks, 256, 0, s>>>(p);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

cudaError_t launch_write_q4(uint8_t* pool_layer, const int2* cells, int n, int n_kv_heads, int head_dim, int shift,
                            const void* k, const void* v, int in_f32, cudaStream_t s) {
    const long long blocks = ((long long)n + shift + kBlock - 1) / kBlock * n_kv_heads;
    if (blocks > 0x7FFFFFFFll) return cudaErrorInvalidValue;
    if (head_dim == 64)
        kv_write_q4_kernel<64><<<(unsigned)blocks, 256, 0, s>>>(pool_layer, cells, n, n_kv_heads, shift, k, v, in_f32);
    else
        kv_write_q4_kernel<128><<<(unsigned)blocks, 512, 0, s>>>(pool_layer, cells, n, n_kv_heads, shift, k, v, in_f32);
    return cudaGetLastError();
}

cudaError_t launch_rows_q4(const uint8_t* pool_layer, const int32_t* table_row, int n, int n_kv_heads, int head_dim,
                           uint16_t* k_out, uint16_t* v_out, int n_blocks, int32_t* err, cudaStream_t s) {
    return launch_read_fmt<LT_KV_Q4_0>(pool_layer, nullptr, table_row, n, n_kv_heads, head_dim, k_out, v_out, 0,
                                       n_blocks, err, s);
}

cudaError_t launch_read(const uint16_t* pool_layer, const int2* cells, int n, int n_kv_heads, int head_dim,
                        int first_slot, void* k_out, void* v_out, int out_f32, int fmt, cudaStream_t s) {
    if (n == 0) return cudaSuccess;
    const uint8_t* pool = reinterpret_cast<const uint8_t*>(pool_layer);
    if (fmt == LT_KV_Q4_0) {
        const long long blocks = ((long long)n + first_slot + kBlock - 1) / kBlock * n_kv_heads;
        if (blocks > 0x7FFFFFFFll) return cudaErrorInvalidValue;
        if (head_dim == 64)
            kv_read_q4_kernel<64><<<(unsigned)blocks, q4_parts(64) * 32, 0, s>>>(pool, cells, n, n_kv_heads, first_slot,
                                                                               k_out, v_out, out_f32);
        else
            kv_read_q4_kernel<128><<<(unsigned)blocks, q4_parts(128) * 32, 0, s>>>(pool, cells, n, n_kv_heads, first_slot,
                                                                                 k_out, v_out, out_f32);
        return cudaGetLastError();
    }
    if (fmt == LT_KV_Q8_0)
        return launch_read_fmt<LT_KV_Q8_0>(pool, cells, nullptr, n, n_kv_heads, head_dim, k_out, v_out, out_f32, 0,
                                           nullptr, s);
    return launch_read_fmt<LT_KV_F16>(pool, cells, nullptr, n, n_kv_heads, head_dim, k_out, v_out, out_f32, 0, nullptr,
                                      s);
}

}  // namespace ltkv

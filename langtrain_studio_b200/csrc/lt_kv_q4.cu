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

#include "lt_kv_device.cuh"
#include "lt_kv_internal.h"
#include "lt_kv_layout.cuh"

namespace ltkv {
namespace {

constexpr float kQ4MaxScale = 2720.0f;  // 8 significant bits, and 24 * d is still an f16

// ------------------------------------------------------------ quantise ----
// One 32-value group held as 4 values by each of 8 consecutive lanes (every
// lane of the warp calls this).  Returns d; code[i] = clamp(floor(x / d + 1/2)
// + 8, 0, 15), decided exactly: the borders (k + 1/2) * |d| have at most 13
// significant bits, so comparing x with them in f32 settles what the rounded
// quotient leaves open.  NaN: not counted in d, code 8 (value 0).
__device__ __forceinline__ float q4_quant4(const float (&x)[4], uint32_t (&code)[4]) {
    float top = 0.f, low = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        top = fmaxf(top, x[i]);
        low = fmaxf(low, -x[i]);
    }
#pragma unroll
    for (int m = 1; m < 8; m <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(kFull, top, m));
        low = fmaxf(low, __shfl_xor_sync(kFull, low, m));
    }
    const bool pos = top >= low;  // the positive extreme takes -8 * d
    const float a = fminf(__bfloat162float(__float2bfloat16_rn((pos ? top : low) * 0.125f)), kQ4MaxScale);
    const float ad = __half2float(__float2half_rn(a));
    const float inv = ad > 0.f ? 1.0f / ad : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float xs = pos ? -x[i] : x[i];
        float k = floorf(fmaf(xs, inv, 0.5f));
        k = fminf(fmaxf(k, -9.f), 8.f);  // NaN -> -9, put right below
        if (xs < (k - 0.5f) * ad) k -= 1.f;
        else if (xs >= (k + 0.5f) * ad) k += 1.f;
        k = fminf(fmaxf(k, -8.f), 7.f);
        if (!(ad > 0.f) || xs != xs) k = 0.f;
        code[i] = (uint32_t)((int)k + 8);
    }
    return pos ? -ad : ad;
}

// Store a lane's four codes (dims 16i + 2t, +1, +8, +9) of slot `slot`, and
// the group's scale from its first lane, into a tile.
template <int D>
__device__ __forceinline__ void q4_store4(uint8_t* tile, int kvsel, int i, int t, int slot, const uint32_t (&code)[4],
                                          float d) {
    const uint8_t b0 = (uint8_t)(code[0] | (code[2] << 4)), b1 = (uint8_t)(code[1] | (code[3] << 4));
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
// D/4 lanes per (token, head, K|V) row, four values a lane; 8 lanes share a
// 32-value group.  Bytes belong to one slot, so rows of one block written by
// different warps never touch the same byte.  Lanes past the end only take
// part in the shuffles.
template <int D>
__global__ void __launch_bounds__(256) kv_write_q4_kernel(uint8_t* __restrict__ pool_layer,
                                                          const int2* __restrict__ cells, int n, int n_kv_heads,
                                                          const void* __restrict__ k, const void* __restrict__ v,
                                                          int in_f32) {
    constexpr int L = D / 4;
    const long long gid = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const bool live = gid < (long long)n * n_kv_heads * 2 * L;
    const int lane = (int)(gid % L);
    long long r = gid / L;
    const int kvsel = (int)(r & 1);
    r >>= 1;
    const int h = (int)(r % n_kv_heads);
    const int tok = (int)(r / n_kv_heads);
    const int i = lane >> 2, t = lane & 3;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (live) load4_f32(kvsel ? v : k, ((size_t)tok * n_kv_heads + h) * D + 16 * i + 2 * t, in_f32, x);
    uint32_t code[4];
    const float d = q4_quant4(x, code);
    if (!live) return;
    const int2 cell = cells[tok];
    q4_store4<D>(pool_layer + ((size_t)cell.x * n_kv_heads + h) * q4_tile_bytes(D), kvsel, i, t, cell.y, code, d);
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
// Stream-K decode attention over 4-bit tiles.  Partition, descriptors, flags
// and merges are those of the f16/Q8_0 kernel (lt_kv_kernels.cu): the call's
// (token, KV head, block) tiles are cut into one contiguous range per
// resident warp, each warp streams its 18*D-byte tiles through its own ring of
// bulk copies, and cut (token, head)s are merged over epoch flags.
//
// Per tile the mathematics is turned over: S^T = K Q^T and O^T += V^T P^T, so
// that the 4-bit tile is the A operand of mma.sync m16n8k16 (16 slots x 16
// dims, or 16 dims x 16 slots), one 32-bit word of codes per lane and step, and
// the query heads are the 8 columns of B:
//   K: a code under a 4-bit mask is, read as f16, the subnormal code * 2^-24
//      (or 2^-20 from the high nibble, whose dims meet q / 16): exact, for one
//      logic operation per pair.  sum (code - 8) q = sum code q - 8 sum q, the
//      second term being the accumulator's start value, formed once per q row;
//      each group's partial scores are scaled by the slots' scales in f32.
//   V: the codes become (code - 8) * d in f16, exactly (two f16 operations).
// q and P are split into an f16 value and its f16 residual (~22 bits).  With a
// group of at most 4 heads (PACK) the 8 columns hold both (columns 0-3 the
// values, 4-7 the residuals), so one MMA carries them; larger groups take two.
// P^T in B-operand form is the transpose of the scores' fragment: movmatrix.
constexpr int kQ4Warps = 4;
constexpr int kQ4Stages = 6;

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// D = A * B + C with separate C (the start value of a group's partial scores).
__device__ __forceinline__ void mma16816_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0,
                                              float c1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%11,%10,%11};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}

__device__ __forceinline__ __half2 as_h2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }

// A piece: tiles [b0, b1) (counted from block skip) of (token, head).
// kind: 0 whole (token, head) -> output; 1 it started before this warp's range
// -> partial slot; 2 it starts here and runs past the range -> merged here.
struct Q4Piece {
    int tok, h, seq, pos, b0, b1, kind, last_block, skip;
    int lo, qpos;
    long long ps;
};

__host__ __device__ inline int q4_qbuf_bytes(int group, int head_dim, int q_f32) {
    return (group * head_dim * (q_f32 ? 4 : 2) + 127) & ~127;
}
__host__ __device__ inline int q4_warp_smem(int group, int head_dim, int q_f32) {
    return kQ4Stages * q4_tile_bytes(head_dim) + q4_qbuf_bytes(group, head_dim, q_f32);
}
__host__ __device__ inline int q4_smem(int group, int head_dim, int q_f32) {
    return kQ4Warps * (q4_warp_smem(group, head_dim, q_f32) + kQ4Stages * 8);
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
    constexpr int U = 2;
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

// Store a partial (slot w) or the output rows of (tok, h).
template <int D, bool PACK>
__device__ __forceinline__ void q4_store_partial(float* po, float* pml, int G, int g, int t, size_t w,
                                                 const float (&M)[2], const float (&L)[2],
                                                 const float (&acc)[D / 16][Own<PACK>::N]) {
    using O = Own<PACK>;
#pragma unroll
    for (int v = 0; v < O::N; ++v) {
        const int h = O::head(v, t);
        if (h < G) {
            float* dst = po + (w * G + h) * D + g + 8 * O::row(v, t);
#pragma unroll
            for (int m = 0; m < D / 16; ++m) dst[16 * m] = acc[m][v];
        }
    }
    if (g == 0 && (!PACK || t < 2)) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int h = O::head(c, t);
            if (h < G) {
                pml[(w * G + h) * 2] = M[c];
                pml[(w * G + h) * 2 + 1] = L[c];
            }
        }
    }
}

template <int D, bool PACK>
__device__ __forceinline__ void q4_store_out(const AttnParams& p, int tok, int h, int g, int t, const float (&L)[2],
                                             const float (&acc)[D / 16][Own<PACK>::N]) {
    using O = Own<PACK>;
    const int hl = p.n_kv_heads * p.group;
    const size_t row0 = p.n_peers == 0 ? (size_t)tok * hl + (size_t)h * p.group
                                       : (size_t)tok * p.n_peers * hl + (size_t)p.peer_rank * hl + (size_t)h * p.group;
    void* out = p.n_peers == 0 ? p.out : p.gather_out;
#pragma unroll
    for (int v = 0; v < O::N; ++v) {
        const int hh = O::head(v, t);
        if (hh >= p.group) continue;
        const float l = L[O::col(v)];
        const float inv = l == 0.f ? 0.f : 1.f / l;  // 0: an interval without positions
        const size_t at = (row0 + hh) * D + g + 8 * O::row(v, t);
#pragma unroll
        for (int m = 0; m < D / 16; ++m) {
            if (p.out_f32) static_cast<float*>(out)[at + 16 * m] = acc[m][v] * inv;
            else static_cast<__half*>(out)[at + 16 * m] = __float2half_rn(acc[m][v] * inv);
        }
    }
}

template <int D, bool PACK, bool SH>
__global__ void __launch_bounds__(kQ4Warps * 32, 3) attn_q4_kernel(const __grid_constant__ AttnParamsOf<SH> p) {
    constexpr int TILE = q4_tile_bytes(D);
    constexpr int KS = D / 16;   // 16-dim steps of K, and 16-dim row tiles of V
    constexpr int G32 = D / 32;  // scale groups
    constexpr int S = kQ4Stages;
    using O = Own<PACK>;
    extern __shared__ __align__(1024) uint8_t smem[];

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int gw = blockIdx.x * kQ4Warps + warp;
    const int Hkv = p.n_kv_heads, G = p.group;
    uint8_t* stages = smem + (size_t)warp * q4_warp_smem(G, D, p.q_f32);
    uint8_t* qbuf = stages + S * TILE;
    const uint32_t bar0 = smem_u32(smem + (size_t)kQ4Warps * q4_warp_smem(G, D, p.q_f32)) + 8u * S * warp;
    if (lane < S) mbar_init(bar0 + 8u * lane, 1);
    fence_mbar_init();
    __syncwarp();
    if (gw >= p.n_warps) return;

    const TokenDesc* toks = p.toks ? p.toks : p.inl;
    const uint8_t* pool = reinterpret_cast<const uint8_t*>(p.pool_layer);
    const long long T = (long long)p.tiles_per_head * Hkv;
    const long long t0 = T * gw / p.n_warps, t1 = T * (gw + 1) / p.n_warps;
    const int g = lane >> 2, t = lane & 3;
    const int qelem = p.q_f32 ? 4 : 2;
    const uint32_t qbytes = (uint32_t)(G * D * qelem);

    // ---- piece generator over [t0, t1) ----
    int gi, gh, gb;
    long long gt = t0;
    {
        int lo = 0, hi = p.n_tok - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if ((long long)toks[mid].prefix * Hkv <= t0) lo = mid; else hi = mid - 1;
        }
        gi = lo;
        const TokenDesc td = toks[gi];
        const int nb = td.pos / kBlock + 1 - td.skip;
        const long long off = t0 - (long long)td.prefix * Hkv;
        gh = (int)(off / nb);
        gb = (int)(off % nb);
    }
    auto gen_piece = [&](Q4Piece& r) {
        const TokenDesc td = toks[gi];
        const int nb = td.pos / kBlock + 1 - td.skip;
        const int len = (int)min((long long)(nb - gb), t1 - gt);
        r.tok = gi;
        r.skip = td.skip;
        r.h = gh;
        r.seq = td.seq;
        r.pos = td.pos;
        r.b0 = gb;
        r.b1 = gb + len;
        r.ps = (long long)td.prefix * Hkv + (long long)gh * nb;
        r.kind = r.ps < t0 ? 1 : (r.ps + nb > t1 ? 2 : 0);
        r.last_block = r.b1 == nb ? td.last_block : -1;
        if constexpr (SH) {
            const ShapeDesc sd = p.shapes ? p.shapes[gi] : p.inl_shapes[gi];
            r.lo = sd.lo;
            r.qpos = sd.qpos;
        }
        gt += len;
        gb += len;
        if (gb == nb) {
            gb = 0;
            if (++gh == Hkv) {
                gh = 0;
                ++gi;
            }
        }
    };
    // block ids [b, min(b + 32, b1)) of a piece, lane j holding b + j
    auto load_window = [&](const Q4Piece& r, int b) {
        const int bb = b + lane;
        if (bb >= r.b1) return 0;
        if (bb == r.b1 - 1 && r.last_block >= 0) return r.last_block;
        return checked_block(__ldg(p.tables + (size_t)r.seq * p.max_blocks + r.skip + bb), p.n_blocks, p.err,
                             p.check_ids != 0);
    };

    // ---- issuer ----
    Q4Piece di{}, dn{};
    gen_piece(di);
    const long long f_ps = di.ps;
    const int f_nb = di.pos / kBlock + 1 - di.skip, f_kind = di.kind;
    bool dn_valid = gt < t1;
    if (dn_valid) gen_piece(dn);
    int ii = 0, it = 0, wb = 0;
    int win = load_window(di, di.b0), win_n = 0;
    auto prefetch_window = [&]() {
        if (wb + 32 < di.b1 - di.b0) win_n = load_window(di, di.b0 + wb + 32);
        else if (dn_valid) win_n = load_window(dn, dn.b0);
    };
    prefetch_window();
    auto table_write = [&](const Q4Piece& r) {
        if (r.h == 0 && r.last_block >= 0 && lane == 0)
            p.tables[(size_t)r.seq * p.max_blocks + r.skip + r.b1 - 1] = r.last_block;
    };
    table_write(di);
    int issued = 0, consumed = 0, istage = 0, cstage = 0, cphase = 0;
    auto issue_one = [&]() {
        if (it - wb >= 32) {
            win = win_n;
            wb += 32;
            prefetch_window();
        }
        const int b = __shfl_sync(kFull, win, it - wb);
        if (lane == 0) {
            const uint32_t bar = bar0 + 8u * istage;
            mbar_arrive_expect_tx(bar, TILE + (it == 0 ? qbytes : 0u));
            bulk_g2s(smem_u32(stages + (size_t)istage * TILE), pool + ((size_t)b * Hkv + di.h) * TILE, TILE, bar);
            if (it == 0)
                bulk_g2s(smem_u32(qbuf),
                         static_cast<const uint8_t*>(p.q) + ((size_t)di.tok * Hkv + di.h) * G * D * qelem, qbytes, bar);
        }
        ++it;
        ++issued;
        istage = istage + 1 == S ? 0 : istage + 1;
    };
    auto issuer_advance = [&]() {
        ++ii;
        di = dn;
        dn_valid = gt < t1;
        if (dn_valid) gen_piece(dn);
        it = 0;
        wb = 0;
        win = win_n;
        prefetch_window();
        table_write(di);
    };

    // ---- consumer ----
    int ci = 0, ct = 0;
    Q4Piece dc = di;
    // The issuer runs at most one piece ahead, and only once the consumer has
    // taken its own piece's q rows out of the single q buffer (ct > 0).
    auto try_issue = [&]() {
        while (issued - consumed < S) {
            if (it < di.b1 - di.b0) {
                issue_one();
                continue;
            }
            if (ii != ci || ct == 0 || !dn_valid) break;
            issuer_advance();
        }
    };
    try_issue();

    uint32_t qh[KS][2], ql[PACK ? 1 : KS][2];  // B fragments: values (PACK: residuals in columns 4-7), residuals
    float corr[G32][2];                        // -8 * 2^-24 * (sum of q over the group), columns 2t, 2t + 1
    float cmul[2] = {0.f, 0.f};                // from the MMA's units to q.k (SH) or log2 units
    float slope[2] = {0.f, 0.f};
    float o[KS][4];
#pragma unroll
    for (int m = 0; m < KS; ++m) o[m][0] = o[m][1] = o[m][2] = o[m][3] = 0.f;
    // Weights are 2^(score - mb): mb trails the running maximum by 7, and moves
    // only when a score passes it by 15, so they stay within (0, 2^15] (an f16
    // and its residual keep 22 bits of all but the smallest) and o is rescaled rarely.
    float mb[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
    bool ok = true;
    int items_out = 0;

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

    for (;;) {
        if (!mbar_wait_bounded(bar0 + 8u * cstage, (uint32_t)cphase)) {
            ok = false;
            break;
        }
        uint8_t* tile = stages + (size_t)cstage * TILE;
        if (ct == 0) {
            // ---- q rows of this piece -> B fragments ----
            const int qg = PACK ? g & 3 : g;
            float x[KS][4];
            float mx = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    float2 f = make_float2(0.f, 0.f);
                    if (qg < G) {
                        const int e = qg * D + ks * 16 + hf * 8 + 2 * t;
                        if (p.q_f32) f = *reinterpret_cast<const float2*>(qbuf + e * 4);
                        else f = __half22float2(*reinterpret_cast<const __half2*>(qbuf + e * 2));
                    }
                    x[ks][2 * hf] = f.x;
                    x[ks][2 * hf + 1] = f.y;
                    mx = fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
            }
            // Scale each row by a power of two that brings its largest value
            // near 2^12: value, residual and q / 16 are then normal f16s.
            mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 2));
            const int ex = (int)(__float_as_uint(mx) >> 23);  // 255: Inf, which no scale helps
            const int fe = ex == 255 ? 127 : min(253, max(1, 266 - ex));
            const float f = __uint_as_float((uint32_t)fe << 23), finv = __uint_as_float((uint32_t)(254 - fe) << 23);
            const bool resid = PACK && g >= 4;
            float csum[G32];
#pragma unroll
            for (int c = 0; c < G32; ++c) csum[c] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const float s = hf ? f * 0.0625f : f;  // high nibbles weigh 16 times as much
                    const float y0 = x[ks][2 * hf] * s, y1 = x[ks][2 * hf + 1] * s;
                    __half2 hi = __floats2half2_rn(y0, y1);
                    float2 back = __half22float2(hi);
                    const __half2 lo = __floats2half2_rn(y0 - back.x, y1 - back.y);
                    const float2 lback = __half22float2(lo);
                    if constexpr (PACK) {
                        if (resid) {
                            hi = lo;
                            back = lback;
                        }
                        qh[ks][hf] = h2_bits(hi);
                        csum[ks >> 1] += (back.x + back.y) * (hf ? 16.f : 1.f);
                    } else {
                        qh[ks][hf] = h2_bits(hi);
                        ql[ks][hf] = h2_bits(lo);
                        csum[ks >> 1] += ((back.x + back.y) + (lback.x + lback.y)) * (hf ? 16.f : 1.f);
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < G32; ++c) {
                float v = csum[c];
                v += __shfl_xor_sync(kFull, v, 1);
                v += __shfl_xor_sync(kFull, v, 2);
                corr[c][0] = __shfl_sync(kFull, v, 8 * t) * -4.76837158203125e-7f;  // -8 * 2^-24
                corr[c][1] = __shfl_sync(kFull, v, 8 * t + 4) * -4.76837158203125e-7f;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                cmul[c] = __shfl_sync(kFull, finv, 8 * t + 4 * c) * 16777216.f;  // 2^24
                if constexpr (SH) {
                    const int hh = O::head(c, t);
                    slope[c] = p.shape.slopes && hh < G ? __ldg(p.shape.slopes + dc.h * G + hh) * kLog2e : 0.f;
                } else {
                    cmul[c] *= p.scale_log2;
                }
            }
        }
        const int b = dc.b0 + ct;  // from block dc.skip
        const int valid = min(kBlock, dc.pos + 1 - (dc.skip + b) * kBlock);
        bool touched = false;
        if (!SH && p.k_new && dc.last_block >= 0 && b == dc.b1 - 1) {
            // Fused append: quantise this token's new K and V row of head h
            // into its pool cell and into the staged tile.
            constexpr int L = D / 4;  // lanes of one row
            const int slot = dc.pos % kBlock;
            uint8_t* cell_tile = reinterpret_cast<uint8_t*>(p.pool_layer_w) + ((size_t)dc.last_block * Hkv + dc.h) * TILE;
#pragma unroll
            for (int r = 0; r < 2 * L / 32; ++r) {
                const int kvsel = (r * 32 + lane) / L, i = (lane % L) >> 2;
                float x[4];
                load4_f32(kvsel ? p.v_new : p.k_new, (size_t)dc.tok * Hkv * D + (size_t)dc.h * D + 16 * i + 2 * t,
                          p.kv_f32, x);
                uint32_t code[4];
                const float d = q4_quant4(x, code);
                q4_store4<D>(tile, kvsel, i, t, slot, code, d);
                q4_store4<D>(cell_tile, kvsel, i, t, slot, code, d);
            }
            touched = true;
            __syncwarp();
        }

        // ---- S^T = K Q^T ----
        float sc[4] = {0.f, 0.f, 0.f, 0.f};  // (slot g | g+8) x (column 2t | 2t+1)
        {
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
                    const int c = 2 * ch + cc;
                    float tt[4];
#pragma unroll
                    for (int q2 = 0; q2 < 2; ++q2) {
                        const int ks = 2 * c + q2;
                        const uint32_t w0 = w[2 * cc + q2], w8 = w0 >> 8;
                        const uint32_t a[4] = {w0 & 0x000f000fu, w8 & 0x000f000fu, w0 & 0x00f000f0u, w8 & 0x00f000f0u};
                        if (q2 == 0) mma16816_from(tt, a, qh[ks][0], qh[ks][1], corr[c][0], corr[c][1]);
                        else mma16816(tt, a, qh[ks][0], qh[ks][1]);
                        if constexpr (!PACK) mma16816(tt, a, ql[ks][0], ql[ks][1]);
                    }
                    const float d0 = cc ? dg.y : dg.x, d1 = cc ? dg8.y : dg8.x;
                    sc[0] += d0 * tt[0];
                    sc[1] += d0 * tt[1];
                    sc[2] += d1 * tt[2];
                    sc[3] += d1 * tt[3];
                }
            }
        }
        if constexpr (PACK) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[e] += __shfl_xor_sync(kFull, sc[e], 2);
        }
        if constexpr (SH) {
            const int j0 = (dc.skip + b) * kBlock, lo = dc.lo - j0;
            const TileShape s0{p.shape, slope[0], dc.qpos - j0, lo}, s1{p.shape, slope[1], dc.qpos - j0, lo};
            sc[0] = s0.score(sc[0] * cmul[0], g);
            sc[1] = s1.score(sc[1] * cmul[1], g);
            sc[2] = s0.score(sc[2] * cmul[0], g + 8);
            sc[3] = s1.score(sc[3] * cmul[1], g + 8);
            if (g < lo) sc[0] = sc[1] = -INFINITY;
            if (g + 8 < lo) sc[2] = sc[3] = -INFINITY;
        } else {
            sc[0] *= cmul[0];
            sc[1] *= cmul[1];
            sc[2] *= cmul[0];
            sc[3] *= cmul[1];
        }
        if (valid < kBlock) {
            if (g >= valid) sc[0] = sc[1] = -INFINITY;
            if (g + 8 >= valid) sc[2] = sc[3] = -INFINITY;
        }

        // ---- softmax ----
        float mx0 = fmaxf(sc[0], sc[2]), mx1 = fmaxf(sc[1], sc[3]);
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
        const float p0 = ex2(sc[0] - r0), p1 = ex2(sc[1] - r1), p2 = ex2(sc[2] - r0), p3 = ex2(sc[3] - r1);
        l_run[0] += p0 + p2;
        l_run[1] += p1 + p3;
        // P^T as B fragments: value = the leading 11 bits (an f16), residual = the rest.
        constexpr uint32_t kLead = 0xffffe000u;
        uint32_t ph[2], pl[2];
        if constexpr (PACK) {
            // lanes t < 2: minus the value; t >= 2: the residual (join() puts the sign right)
            const float own = t < 2 ? 0.f : 1.f;
            auto part = [&](float v) { return fmaf(v, own, -__uint_as_float(__float_as_uint(v) & kLead)); };
            ph[0] = movmatrix_trans(h2_bits(__floats2half2_rn(part(p0), part(p1))));
            ph[1] = movmatrix_trans(h2_bits(__floats2half2_rn(part(p2), part(p3))));
        } else {
            const float v0 = __uint_as_float(__float_as_uint(p0) & kLead), v1 = __uint_as_float(__float_as_uint(p1) & kLead);
            const float v2 = __uint_as_float(__float_as_uint(p2) & kLead), v3 = __uint_as_float(__float_as_uint(p3) & kLead);
            ph[0] = movmatrix_trans(h2_bits(__floats2half2_rn(v0, v1)));
            ph[1] = movmatrix_trans(h2_bits(__floats2half2_rn(v2, v3)));
            pl[0] = movmatrix_trans(h2_bits(__floats2half2_rn(p0 - v0, p1 - v1)));
            pl[1] = movmatrix_trans(h2_bits(__floats2half2_rn(p2 - v2, p3 - v3)));
        }

        // ---- O^T += V^T P^T ----
        const __half2 k1032 = __floats2half2_rn(1032.f, 1032.f), k72 = __floats2half2_rn(72.f, 72.f);
#pragma unroll
        for (int ch = 0; ch < D / 64; ++ch) {
            const uint4 wv = *reinterpret_cast<const uint4*>(tile + 8 * D + ch * 512 + lane * 16);
            const uint32_t w[4] = {wv.x, wv.y, wv.z, wv.w};
            const uint4 vd = *reinterpret_cast<const uint4*>(tile + 17 * D + (t * G32 + 2 * ch) * 8);
#pragma unroll
            for (int mm = 0; mm < 4; ++mm) {
                const int m = 4 * ch + mm;
                const __half2 dA = as_h2(mm < 2 ? vd.x : vd.z), dB = as_h2(mm < 2 ? vd.y : vd.w);
                const uint32_t w0 = w[mm], w8 = w0 >> 8;
                // 1024 + code and 64 + code are f16s whose last bits are the nibble
                const uint32_t a[4] = {
                    h2_bits(__hmul2(__hsub2(as_h2((w0 & 0x000f000fu) | 0x64006400u), k1032), dA)),
                    h2_bits(__hmul2(__hsub2(as_h2((w0 & 0x00f000f0u) | 0x54005400u), k72), dA)),
                    h2_bits(__hmul2(__hsub2(as_h2((w8 & 0x000f000fu) | 0x64006400u), k1032), dB)),
                    h2_bits(__hmul2(__hsub2(as_h2((w8 & 0x00f000f0u) | 0x54005400u), k72), dB))};
                mma16816(o[m], a, ph[0], ph[1]);
                if constexpr (!PACK) mma16816(o[m], a, pl[0], pl[1]);
            }
        }
        ++consumed;
        if (++cstage == S) {
            cstage = 0;
            cphase ^= 1;
        }
        ++ct;
        if (touched) fence_proxy_async_smem();
        __syncwarp();

        if (ct == dc.b1 - dc.b0) {
            if (dc.kind == 2) break;  // merged after the loop
            float M[2], L[2], acc[KS][O::N];
            join(M, L, acc);
            if (dc.kind == 0) {
                ++items_out;
                q4_store_out<D, PACK>(p, dc.tok, dc.h, g, t, L, acc);
            } else {
                q4_store_partial<D, PACK>(p.part_o, p.part_ml, G, g, t, (size_t)gw, M, L, acc);
            }
#pragma unroll
            for (int m = 0; m < KS; ++m) o[m][0] = o[m][1] = o[m][2] = o[m][3] = 0.f;
            mb[0] = mb[1] = -INFINITY;
            l_run[0] = l_run[1] = 0.f;
            if (ii == ci) {
                if (!dn_valid) break;
                issuer_advance();
            }
            ++ci;
            dc = di;
            ct = 0;
        }
        try_issue();
    }
    if (!ok) {
        for (int jj = consumed + 1; jj < issued; ++jj) mbar_wait_bounded(bar0 + 8u * (jj % S), (jj / S) & 1);
        if (lane == 0) atomicOr(p.err, kErrTimeout);
    }
    __syncwarp();
    if (lane == 0) st_release_gpu(p.flags + gw, p.epoch);
    const long long NW = p.n_warps;

    // ---- two-level merge: lead a group of helpers of a long cut (token, head) ----
    if (ok && f_kind == 1 && p.part2_o) {
        const int ws = (int)(((f_ps + 1) * NW - 1) / T), we = (int)(((f_ps + f_nb) * NW - 1) / T);
        if (we - ws > kMergeGroup && (gw - ws - 1) % kMergeGroup == 0) {
            const int last = min(gw + kMergeGroup - 1, we);
            const bool rd = wait_flags(p.flags, p.epoch, gw + 1, last, 1, lane);
            __syncwarp();
            if (rd) {
                float M[2] = {-INFINITY, -INFINITY}, L[2] = {0.f, 0.f}, acc[KS][O::N];
#pragma unroll
                for (int m = 0; m < KS; ++m)
#pragma unroll
                    for (int v = 0; v < O::N; ++v) acc[m][v] = 0.f;
                q4_merge_slots<D, PACK>(p.part_o, p.part_ml, G, g, t, gw, last, 1, M, L, acc);
                q4_store_partial<D, PACK>(p.part2_o, p.part2_ml, G, g, t, (size_t)gw, M, L, acc);
            }
            if (!rd && lane == 0) atomicOr(p.err, kErrTimeout);
            __syncwarp();
            if (lane == 0) st_release_gpu(p.flags2 + gw, p.epoch);
        }
    }
    if (!ok || dc.kind != 2 || ct != dc.b1 - dc.b0) {
        peer_done(p, lane, items_out);
        return;
    }

    // ---- merge the cut (token, head) this range ends with ----
    const int nb = dc.pos / kBlock + 1 - dc.skip;
    const int w_last = (int)(((dc.ps + nb) * NW - 1) / T);
    const bool grouped = p.part2_o && w_last - gw > kMergeGroup;
    const int stride = grouped ? kMergeGroup : 1;
    const bool ready = wait_flags(grouped ? p.flags2 : p.flags, p.epoch, gw + 1, w_last, stride, lane);
    __syncwarp();
    if (!ready) {
        if (lane == 0) atomicOr(p.err, kErrTimeout);
        peer_done(p, lane, items_out + 1);
        return;
    }
    {
        float M[2], L[2], acc[KS][O::N];
        join(M, L, acc);
        q4_merge_slots<D, PACK>(grouped ? p.part2_o : p.part_o, grouped ? p.part2_ml : p.part_ml, G, g, t, gw + 1,
                                w_last, stride, M, L, acc);
        q4_store_out<D, PACK>(p, dc.tok, dc.h, g, t, L, acc);
    }
    peer_done(p, lane, items_out + 1);
}

// ------------------------------------------------------------- launches ----
template <int D, bool PACK, bool SH>
cudaError_t ensure_q4_attr(int dev) {
    static bool set[64] = {};
    if (set[dev]) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(attn_q4_kernel<D, PACK, SH>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               q4_smem(PACK ? 4 : kMaxGroup, D, 1));
    if (e == cudaSuccess) set[dev] = true;
    return e;
}

template <int D, bool PACK, bool SH>
int q4_warps_for(int dev, int group, int q_f32) {
    static int cache[64][kMaxGroup + 1][2] = {};
    int& c = cache[dev][group][q_f32 ? 1 : 0];
    if (c == 0) {
        int per_sm = 0, sms = 0;
        if (ensure_q4_attr<D, PACK, SH>(dev) != cudaSuccess) return 0;
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, attn_q4_kernel<D, PACK, SH>, kQ4Warps * 32,
                                                          q4_smem(group, D, q_f32)) != cudaSuccess)
            return 0;
        c = (per_sm < 1 ? 1 : per_sm) * sms * kQ4Warps;
    }
    return c;
}

// Cooperative: merging warps wait for other CTAs' flags, so the whole grid
// (sized to the resident capacity) is co-resident.
template <int D, bool PACK, bool SH>
cudaError_t launch_q4(const AttnParamsOf<SH>& p, cudaStream_t s) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if ((e = ensure_q4_attr<D, PACK, SH>(dev)) != cudaSuccess) return e;
    const dim3 grid((p.n_warps + kQ4Warps - 1) / kQ4Warps), block(kQ4Warps * 32);
    void* args[] = {const_cast<AttnParamsOf<SH>*>(&p)};
    return cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(&attn_q4_kernel<D, PACK, SH>), grid, block, args,
                                       q4_smem(p.group, D, p.q_f32), s);
}

template <bool SH>
cudaError_t launch_q4_any(const AttnParamsOf<SH>& p, int head_dim, cudaStream_t s) {
    if (p.group <= 4) return head_dim == 64 ? launch_q4<64, true, SH>(p, s) : launch_q4<128, true, SH>(p, s);
    return head_dim == 64 ? launch_q4<64, false, SH>(p, s) : launch_q4<128, false, SH>(p, s);
}

}  // namespace

int attend_q4_warps(int device, int group, int head_dim, int q_f32, bool shaped) {
    if (shaped) {
        if (group <= 4)
            return head_dim == 64 ? q4_warps_for<64, true, true>(device, group, q_f32)
                                  : q4_warps_for<128, true, true>(device, group, q_f32);
        return head_dim == 64 ? q4_warps_for<64, false, true>(device, group, q_f32)
                              : q4_warps_for<128, false, true>(device, group, q_f32);
    }
    if (group <= 4)
        return head_dim == 64 ? q4_warps_for<64, true, false>(device, group, q_f32)
                              : q4_warps_for<128, true, false>(device, group, q_f32);
    return head_dim == 64 ? q4_warps_for<64, false, false>(device, group, q_f32)
                          : q4_warps_for<128, false, false>(device, group, q_f32);
}

cudaError_t launch_attend_q4(const AttnParams& p, int head_dim, cudaStream_t s) {
    return launch_q4_any<false>(p, head_dim, s);
}

cudaError_t launch_attend_q4_shaped(const AttnShapedParams& p, int head_dim, cudaStream_t s) {
    return launch_q4_any<true>(p, head_dim, s);
}

cudaError_t launch_write_q4(uint8_t* pool_layer, const int2* cells, int n, int n_kv_heads, int head_dim, const void* k,
                            const void* v, int in_f32, cudaStream_t s) {
    const long long blocks = ((long long)n * n_kv_heads * 2 * (head_dim / 4) + 255) / 256;
    if (blocks > 0x7FFFFFFFll) return cudaErrorInvalidValue;
    if (head_dim == 64)
        kv_write_q4_kernel<64><<<(unsigned)blocks, 256, 0, s>>>(pool_layer, cells, n, n_kv_heads, k, v, in_f32);
    else
        kv_write_q4_kernel<128><<<(unsigned)blocks, 256, 0, s>>>(pool_layer, cells, n, n_kv_heads, k, v, in_f32);
    return cudaGetLastError();
}

cudaError_t launch_rows_q4(const uint8_t* pool_layer, const int32_t* table_row, int n, int n_kv_heads, int head_dim,
                           uint16_t* k_out, uint16_t* v_out, int n_blocks, int32_t* err, cudaStream_t s) {
    return launch_read_fmt<LT_KV_Q4_0>(pool_layer, nullptr, table_row, n, n_kv_heads, head_dim, k_out, v_out, 0,
                                       n_blocks, err, s);
}

cudaError_t launch_read(const uint16_t* pool_layer, const int2* cells, int n, int n_kv_heads, int head_dim, void* k_out,
                        void* v_out, int out_f32, int fmt, cudaStream_t s) {
    if (n == 0) return cudaSuccess;
    const uint8_t* pool = reinterpret_cast<const uint8_t*>(pool_layer);
    if (fmt == LT_KV_Q4_0)
        return launch_read_fmt<LT_KV_Q4_0>(pool, cells, nullptr, n, n_kv_heads, head_dim, k_out, v_out, out_f32, 0,
                                           nullptr, s);
    if (fmt == LT_KV_Q8_0)
        return launch_read_fmt<LT_KV_Q8_0>(pool, cells, nullptr, n, n_kv_heads, head_dim, k_out, v_out, out_f32, 0,
                                           nullptr, s);
    return launch_read_fmt<LT_KV_F16>(pool, cells, nullptr, n, n_kv_heads, head_dim, k_out, v_out, out_f32, 0, nullptr,
                                      s);
}

}  // namespace ltkv

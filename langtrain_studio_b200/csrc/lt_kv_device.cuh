// Device helpers shared by the cache's kernels: mbarriers and bulk copies,
// bounded flag waits, the f16 tensor-core step, input conversion and the
// stream-K launch's flag protocol.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "lt_kv_internal.h"
#include "lt_kv_layout.cuh"

namespace ltkv {

constexpr uint64_t kWaitLimitNs = 2000000000ull;  // bounded mbarrier wait: 2 s
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ uint64_t global_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void fence_mbar_init() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

__device__ __forceinline__ void fence_proxy_async_smem() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void mbar_arrive_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// Wait for `parity` of an mbarrier, giving up after kWaitLimitNs.
__device__ __forceinline__ bool mbar_wait_bounded(uint32_t bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 15u) == 0 && global_ns() - t0 > kWaitLimitNs) return false;
    }
}

// Non-multicast 1-D bulk copy global -> this CTA's shared memory.
__device__ __forceinline__ void bulk_g2s(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
        "l"(src), "r"(bytes), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void st_release_gpu(uint32_t* p, uint32_t v) {
    asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}

__device__ __forceinline__ uint32_t ld_acquire_gpu(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

// System scope (another GPU over NVLink reads or writes the word).
__device__ __forceinline__ void fence_acq_rel_sys() { asm volatile("fence.acq_rel.sys;" ::: "memory"); }

__device__ __forceinline__ void st_relaxed_sys(uint32_t* p, uint32_t v) {
    asm volatile("st.relaxed.sys.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}

__device__ __forceinline__ uint32_t ld_acquire_sys(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.acquire.sys.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

__device__ __forceinline__ uint32_t atom_add_acq_rel_gpu(uint32_t* p, uint32_t v) {
    uint32_t old;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
    return old;
}


// Wait until *flag == epoch, giving up after limit_ns.
__device__ __forceinline__ int wait_flag_bounded(const uint32_t* flag, uint32_t epoch,
                                                 uint64_t limit_ns = kWaitLimitNs) {
    if (ld_acquire_gpu(flag) == epoch) return 1;
    const uint64_t t0 = global_ns();
    for (;;) {
        __nanosleep(64);
        if (ld_acquire_gpu(flag) == epoch) return 1;
        if (global_ns() - t0 > limit_ns) return 0;
    }
}

// A block id read from a block table.  Builds with LT_BOUNDS_CHECK test it
// against the pool (n_blocks > 0), and so does every build when `check` is
// set (tables the caller owns): a bad id raises kErrBounds and block 0
// stands in for it, so the access stays inside the pool and only the
// output is wrong (and reported).  Otherwise the host bookkeeping that
// wrote the table is trusted.
__device__ __forceinline__ int checked_block(int b, int n_blocks, int32_t* err, bool check = false) {
#ifdef LT_BOUNDS_CHECK
    check = true;
#endif
    if (check && n_blocks > 0 && (unsigned)b >= (unsigned)n_blocks) {
        atomicOr(err, kErrBounds);
        return 0;
    }
    return b;
}

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
                 : "r"(addr));
}

__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
                 : "r"(addr));
}

// D(16x8 f32) += A(16x16 f16, row) * B(16x8 f16, col)
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 2^x on the SFU (hardware instruction; relative error ~2^-22).
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// Load 8 consecutive input values (f32 or f16) and return them as 8 f16.
__device__ __forceinline__ uint4 load8_as_f16(const void* base, size_t idx, int in_f32) {
    uint4 r;
    if (in_f32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + idx);
        const float4 a = __ldg(p), b = __ldg(p + 1);
        r.x = f32_to_f16_ref(a.x) | (uint32_t(f32_to_f16_ref(a.y)) << 16);
        r.y = f32_to_f16_ref(a.z) | (uint32_t(f32_to_f16_ref(a.w)) << 16);
        r.z = f32_to_f16_ref(b.x) | (uint32_t(f32_to_f16_ref(b.y)) << 16);
        r.w = f32_to_f16_ref(b.z) | (uint32_t(f32_to_f16_ref(b.w)) << 16);
    } else {
        r = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + idx));
    }
    return r;
}

// Load 8 consecutive input values (f32, or f16 widened exactly).
__device__ __forceinline__ void load8_f32(const void* base, size_t idx, int in_f32, float (&x)[8]) {
    if (in_f32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + idx);
        const float4 a = __ldg(p), b = __ldg(p + 1);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 r = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + idx));
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            x[2 * j] = f.x;
            x[2 * j + 1] = f.y;
        }
    }
}

// A power of two that brings a row of q whose largest magnitude is mx near 2^12, and
// its inverse: value and residual of the row are then normal f16s.
__device__ __forceinline__ void q_row_scale(float mx, float& mul, float& inv) {
    const int ex = (int)(__float_as_uint(mx) >> 23);  // 255: Inf, which no scale helps
    const int fe = ex == 255 ? 127 : min(253, max(1, 266 - ex));
    mul = __uint_as_float((uint32_t)fe << 23);
    inv = __uint_as_float((uint32_t)(254 - fe) << 23);
}

// Peer gather: a warp is done and stored the output rows of `items`
// (token, head) items into this rank's gather half (local memory).  Only
// such warps take part: after the warp barrier, lane 0 adds the items to
// this launch's count with an acq_rel RMW on this GPU, so the warp that
// completes the count (n_tok * n_kv_heads items) has every row ordered
// before it, in this GPU's memory.  It publishes this launch's epoch into
// every rank's flag for this rank: one system-scope fence, then relaxed
// system-scope stores (fence + store is a release; a release store per rank
// would pay the fence once per rank).  A rank that acquires the flag then
// reads the rows from here over NVLink.
__device__ __forceinline__ void peer_done(const AttnParams& p, int lane, int items) {
    if (p.n_peers == 0 || items == 0) return;
    __syncwarp();
    const uint32_t total = (uint32_t)p.n_tok * (uint32_t)p.n_kv_heads;
    if (lane == 0 && atom_add_acq_rel_gpu(p.done_count, (uint32_t)items) + (uint32_t)items == total) {
        *p.done_count = 0u;  // ready for the next launch (which starts after this one ends)
        fence_acq_rel_sys();
        for (int r = 0; r < p.n_peers; ++r) st_relaxed_sys(p.peer_flag[r], p.peer_epoch);
    }
}

// Wait (bounded) until flags[w] == epoch for w = first, first + stride, ...
// <= last; lane j polls every 32nd of them, so the round trips overlap.
// Warp-uniform result.
__device__ __forceinline__ bool wait_flags(const uint32_t* flags, uint32_t epoch, int first, int last, int stride,
                                           int lane) {
    int ready = 1;
    for (int w0 = first; w0 <= last && ready; w0 += 32 * stride) {
        int ok = 1;
        const int w = w0 + lane * stride;
        if (w <= last) ok = wait_flag_bounded(flags + w, epoch);
        ready = __all_sync(kFull, ok);
    }
    return ready != 0;
}

// Score terms of one tile of a shaped call for one query row (lt_kv_score).
struct TileShape {
    ShapeTerms c;
    float slope;  // log2 units per position
    int q_off;    // the token's position minus the tile's first
    int lo;       // slots before this one are masked (<= 0: none)
    // q.k of a slot -> score in log2 units.  tanh is the library's: near 0 it
    // keeps the relative accuracy that 1 - 2 / (1 + e^2x) loses.
    __device__ __forceinline__ float score(float s, int slot) const {
        const float v = c.capped ? c.cap_log2 * tanhf(s * c.scale_cap) : s * c.scale_log2;
        return v - slope * (float)abs(q_off - slot);
    }
};

}  // namespace ltkv

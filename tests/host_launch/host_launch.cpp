// The host side of the library (lt_kv.cpp) without a GPU: the CUDA runtime and
// the kernels' launchers are replaced by stand-ins over host memory, so that
// what a launch is given can be looked at as the launch is made.  Copies and
// launches take effect when they are issued, which is the order of one stream.
// `host_launch <scenario>` exits 0 if the scenario holds.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <string>
#include <vector>

#include "lt_kv.h"
#include "lt_kv_internal.h"

// ------------------------------------------------------- the CUDA runtime
namespace {
bool g_capturing = false;
}
extern "C" {
cudaError_t CUDARTAPI cudaMalloc(void** p, size_t n) { return (*p = std::calloc(1, n ? n : 1)) ? cudaSuccess : cudaErrorMemoryAllocation; }
cudaError_t CUDARTAPI cudaFree(void* p) { return std::free(p), cudaSuccess; }
cudaError_t CUDARTAPI cudaHostAlloc(void** p, size_t n, unsigned) { return cudaMalloc(p, n); }
cudaError_t CUDARTAPI cudaFreeHost(void* p) { return cudaFree(p); }
cudaError_t CUDARTAPI cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind) { return std::memcpy(d, s, n), cudaSuccess; }
cudaError_t CUDARTAPI cudaMemcpyAsync(void* d, const void* s, size_t n, cudaMemcpyKind, cudaStream_t) { return std::memcpy(d, s, n), cudaSuccess; }
cudaError_t CUDARTAPI cudaMemset(void* d, int v, size_t n) { return std::memset(d, v, n), cudaSuccess; }
cudaError_t CUDARTAPI cudaMemsetAsync(void* d, int v, size_t n, cudaStream_t) { return std::memset(d, v, n), cudaSuccess; }
cudaError_t CUDARTAPI cudaGetDevice(int* d) { return *d = 0, cudaSuccess; }
cudaError_t CUDARTAPI cudaSetDevice(int) { return cudaSuccess; }
cudaError_t CUDARTAPI cudaDeviceSynchronize() { return cudaSuccess; }
cudaError_t CUDARTAPI cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t CUDARTAPI cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { return *v = 148, cudaSuccess; }
cudaError_t CUDARTAPI cudaEventCreate(cudaEvent_t* e) { return *e = reinterpret_cast<cudaEvent_t>(std::malloc(1)), cudaSuccess; }
cudaError_t CUDARTAPI cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) { return cudaEventCreate(e); }
cudaError_t CUDARTAPI cudaEventDestroy(cudaEvent_t e) { return std::free(e), cudaSuccess; }
cudaError_t CUDARTAPI cudaEventRecord(cudaEvent_t, cudaStream_t) { return cudaSuccess; }
cudaError_t CUDARTAPI cudaEventSynchronize(cudaEvent_t) { return cudaSuccess; }
cudaError_t CUDARTAPI cudaEventElapsedTime(float* ms, cudaEvent_t, cudaEvent_t) { return *ms = 0.f, cudaSuccess; }
const char* CUDARTAPI cudaGetErrorString(cudaError_t) { return "an error"; }
cudaError_t CUDARTAPI cudaIpcCloseMemHandle(void*) { return cudaErrorNotSupported; }
cudaError_t CUDARTAPI cudaIpcGetMemHandle(cudaIpcMemHandle_t*, void*) { return cudaErrorNotSupported; }
cudaError_t CUDARTAPI cudaIpcOpenMemHandle(void**, cudaIpcMemHandle_t, unsigned) { return cudaErrorNotSupported; }
cudaError_t CUDARTAPI cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* s) {
    return *s = g_capturing ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone, cudaSuccess;
}
}

// ------------------------------------------------------------ the launches
namespace {
std::function<void(const ltkv::AttnParams&, const ltkv::AttnShapedParams*)> on_attend;
std::function<void(const ltkv::PrefixParams&, int)> on_prefix;
int n_attend = 0, n_prefix = 0, n_plan = 0, n_write = 0, n_rows = 0;
}  // namespace
namespace ltkv {
int attend_warps(int, int, int, int, int, bool) { return 1184; }
int attend_launches(const AttnParams&) { return 1; }
bool bounds_checked_build() { return false; }
cudaError_t launch_attend(const AttnParams& p, int, cudaStream_t) {
    ++n_attend;
    if (on_attend) on_attend(p, nullptr);
    return cudaSuccess;
}
cudaError_t launch_attend_shaped(const AttnShapedParams& p, int, cudaStream_t) {
    ++n_attend;
    if (on_attend) on_attend(p, &p);
    return cudaSuccess;
}
cudaError_t launch_prefix(const PrefixParams& p, int n_items, int, bool, bool, cudaStream_t) {
    ++n_prefix;
    if (on_prefix) on_prefix(p, n_items);
    return cudaSuccess;
}
cudaError_t launch_expand_q4(const uint8_t*, const int32_t*, int, const ExpandGroup*, int, int, int, uint16_t*, int,
                             int32_t*, cudaStream_t) {
    return cudaSuccess;
}
cudaError_t launch_write(uint16_t*, const int2*, int, int, int, int, const void*, const void*, int, int, cudaStream_t) {
    ++n_write;
    return cudaSuccess;
}
cudaError_t launch_read(const uint16_t*, const int2*, int, int, int, int, void*, void*, int, int, cudaStream_t) {
    ++n_rows;
    return cudaSuccess;
}
cudaError_t launch_rows(const uint16_t*, const int32_t*, int, int, int, uint16_t*, uint16_t*, int, int, int32_t*,
                        cudaStream_t) {
    ++n_rows;
    return cudaSuccess;
}
cudaError_t launch_apply_plan(uint16_t*, size_t, size_t, int, const int2*, int, int32_t* tables, const int2* tw, int n_tw,
                              int, long long, int32_t*, cudaStream_t) {
    ++n_plan;
    for (int i = 0; i < n_tw; ++i) tables[tw[i].x] = tw[i].y;
    return cudaSuccess;
}
cudaError_t launch_gather_wait_copy(const uint32_t*, int, uint32_t, void* const*, void*, uint32_t, size_t, int32_t*,
                                    cudaStream_t) {
    return cudaErrorNotSupported;
}
cudaError_t launch_wait_selftest(uint64_t, int32_t*, cudaStream_t) { return cudaErrorNotSupported; }
}  // namespace ltkv

// ---------------------------------------------------------- the scenarios
namespace {

#define NEED(cond, ...)                                                     \
    do {                                                                    \
        if (!(cond)) {                                                      \
            std::printf("%s:%d: %s\n  ", __FILE__, __LINE__, #cond);        \
            std::printf(__VA_ARGS__);                                       \
            std::printf("\n");                                              \
            std::exit(1);                                                   \
        }                                                                   \
    } while (0)

struct Cache {
    lt_kv* kv = nullptr;
    std::vector<uint32_t> seq, pos;  // tokens of the next call
    alignas(16) char dummy[64] = {};

    Cache(uint32_t fmt, uint32_t hkv, uint32_t group, uint32_t tokens, uint32_t seqs, uint32_t batch) {
        lt_kv_config c{};
        c.n_layers = 1, c.n_kv_heads = hkv, c.head_dim = 64, c.n_heads = hkv * group, c.n_tokens = tokens;
        c.max_seqs = seqs, c.max_batch = batch, c.kv_format = fmt;
        NEED(lt_kv_create(&c, &kv) == LT_OK, "create");
    }
    ~Cache() { lt_kv_destroy(kv); }
    void fill(uint32_t s, uint32_t n) {
        for (uint32_t p = lt_kv_len(kv, s); p < n; ++p) {
            int32_t b, sl;
            uint32_t done;
            NEED(lt_kv_append(kv, &s, &p, 1, &b, &sl, &done, nullptr) == LT_OK, "%s", lt_kv_last_error(kv));
        }
    }
    void tokens(uint32_t s, uint32_t p0, uint32_t p1) {
        for (uint32_t p = p0; p < p1; ++p) seq.push_back(s), pos.push_back(p);
    }
    lt_status attend(const lt_kv_score* score = nullptr) {
        const uint32_t n = (uint32_t)seq.size();
        return score ? lt_kv_attend_shaped(kv, 0, dummy, LT_F32, seq.data(), pos.data(), n, score, dummy, LT_F32, 1.f, nullptr)
                     : lt_kv_attend(kv, 0, dummy, LT_F32, seq.data(), pos.data(), n, dummy, LT_F32, 1.f, nullptr);
    }
};

// Shaped calls past the inline descriptors stage their tokens and their
// intervals apart.  The tokens' staging is the same call after call, the
// intervals' is not: a call must not put its intervals where its tokens lie.
void staging(uint32_t fmt) {
    Cache c(fmt, 1, 1, 16 * 64, 4, 1024);
    for (uint32_t s = 0; s < 4; ++s) c.fill(s, 160), c.tokens(s, 16, 160);
    const size_t n = c.seq.size();
    NEED(n > (size_t)ltkv::kInlineTokens, "%zu tokens", n);
    std::vector<uint32_t> first(n);
    on_attend = [&](const ltkv::AttnParams& p, const ltkv::AttnShapedParams* sp) {
        NEED(sp && p.toks && sp->shapes && p.n_tok == (int32_t)n, "a shaped launch of %zu tokens", n);
        for (size_t i = 0; i < n; ++i) {
            NEED(p.toks[i].seq == (int32_t)c.seq[i] && p.toks[i].pos == (int32_t)c.pos[i] && p.toks[i].skip == 0,
                 "token %zu of launch %d: (%d, %d) for (%u, %u)", i, n_attend, p.toks[i].seq, p.toks[i].pos, c.seq[i],
                 c.pos[i]);
            NEED(sp->shapes[i].lo == (int32_t)first[i], "interval %zu of launch %d", i, n_attend);
        }
    };
    lt_kv_score score{};
    score.first_host = first.data();
    for (int call = 0; call < 40; ++call) {
        for (size_t i = 0; i < n; ++i) first[i] = (uint32_t)((call + i) % 16);
        NEED(c.attend(&score) == LT_OK, "%s", lt_kv_last_error(c.kv));
    }
    NEED(n_attend == 40, "%d launches", n_attend);
}

// A call that is refused in a capture leaves everything as it was, one of no
// tokens too: a plan put into a graph would reach the tables only as it replays.
void capture(uint32_t fmt, bool shaped) {
    Cache c(fmt, 2, 2, 16 * 16, 2, 64);
    c.fill(0, 20);
    lt_kv_score score{};
    g_capturing = true;
    NEED(c.attend(shaped ? &score : nullptr) == LT_E_ARG && n_plan == 0, "no tokens: %d plans", n_plan);
    c.tokens(0, 19, 20);
    NEED(c.attend(shaped ? &score : nullptr) == LT_E_ARG && n_plan == 0, "one token: %d plans", n_plan);
    g_capturing = false;
    NEED(c.attend(shaped ? &score : nullptr) == LT_OK && n_attend == 1, "%s", lt_kv_last_error(c.kv));
}

// Device pointers that the kernels' 16-byte accesses cannot take, or that are
// none, are refused before anything is queued; with no tokens none is looked at.
void pointers(uint32_t fmt) {
    Cache c(fmt, 2, 2, 16 * 16, 2, 64);
    c.fill(0, 20);
    alignas(16) static char buf[64];
    void *ok = buf, *odd = buf + 2;
    const int32_t block = 0, slot = 3;
    const uint32_t seq = 0, pos = 19;
    int32_t last[2];
    NEED(lt_kv_seq_blocks(c.kv, 0, last, 2) == 2, "blocks");
    auto refused = [&](lt_status rc, const char* what) {
        NEED(rc == LT_E_ARG && n_plan == 0 && n_attend == 0 && n_write == 0 && n_rows == 0, "%s: status %d", what, rc);
    };
    for (void* bad : {odd, (void*)nullptr})
        for (int which = 0; which < 2; ++which) {
            void *a = which ? ok : bad, *b = which ? bad : ok;
            refused(lt_kv_write(c.kv, 0, &block, &slot, 1, a, b, LT_F16, nullptr), "write");
            refused(lt_kv_rows(c.kv, 0, 0, 20, a, b, nullptr), "rows");
            refused(lt_kv_read(c.kv, 0, &block, &slot, 1, a, b, LT_F16, nullptr), "read");
            refused(lt_kv_attend(c.kv, 0, a, LT_F32, &seq, &pos, 1, b, LT_F32, 1.f, nullptr), "attend");
            const int32_t own = 3;
            refused(lt_kv_write_attend(c.kv, 0, &last[1], &own, a, b, LT_F32, ok, LT_F32, &seq, &pos, 1, ok, LT_F32, 1.f,
                                       nullptr), "write_attend");
        }
    NEED(lt_kv_write(c.kv, 0, nullptr, nullptr, 0, nullptr, nullptr, LT_F16, nullptr) == LT_OK, "no tokens");
    NEED(lt_kv_read(c.kv, 0, nullptr, nullptr, 0, nullptr, nullptr, LT_F16, nullptr) == LT_OK, "no tokens");
    NEED(lt_kv_rows(c.kv, 0, 0, 0, nullptr, nullptr, nullptr) == LT_OK, "no rows");
    NEED(lt_kv_attend(c.kv, 0, nullptr, LT_F32, nullptr, nullptr, 0, nullptr, LT_F32, 1.f, nullptr) == LT_OK, "no tokens");
    NEED(lt_kv_write(c.kv, 0, &block, &slot, 1, ok, ok, LT_F16, nullptr) == LT_OK && n_write == 1, "write");
}

}  // namespace

int main(int argc, char** argv) {
    const std::string what = argc > 1 ? argv[1] : "";
    if (what == "staging-f16") staging(LT_KV_F16);
    else if (what == "staging-q8_0") staging(LT_KV_Q8_0);
    else if (what == "capture-q4_0") capture(LT_KV_Q4_0, false);
    else if (what == "capture-shaped") capture(LT_KV_F16, true);
    else if (what == "pointers-f16") pointers(LT_KV_F16);
    else if (what == "pointers-q8_0") pointers(LT_KV_Q8_0);
    else if (what == "pointers-q4_0") pointers(LT_KV_Q4_0);
    else return std::printf("no scenario '%s'\n", what.c_str()), 2;
    std::printf("ok\n");
    return 0;
}

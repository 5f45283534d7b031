// Internal interface between the host bookkeeping (lt_kv.cpp) and the sm_100a
// kernels (lt_kv_kernels.cu).  Not part of the C ABI.
#pragma once
#include <cuda_runtime.h>
#include <nvtx3/nvToolsExt.h>
#include <stdint.h>
#include <string.h>

#include "lt_kv.h"

namespace ltkv {

// Whether an lt_dtype argument names LT_F32 or LT_F16.  A C caller may pass
// any 32-bit value; reading an out-of-range value through the C++ enum type
// is undefined, so the argument's bytes are read instead.
static_assert(sizeof(lt_dtype) == sizeof(int32_t), "lt_dtype is passed as a 32-bit int");
inline bool dtype_valid(const lt_dtype& d) {
    int32_t v;
    memcpy(&v, &d, sizeof v);
    return v == (int32_t)LT_F32 || v == (int32_t)LT_F16;
}

constexpr float kLog2e = 1.4426950408889634f;  // scores are in log2 units
constexpr int kBlock = 16;           // tokens per block (kv.rs:13)
constexpr int kMaxGroup = 8;         // q heads per KV head the attention kernel handles

// Bits of the device error word (lt_kv_check turns them into statuses).
constexpr int32_t kErrTimeout = 1;   // a bounded wait gave up -> LT_E_TIMEOUT
constexpr int32_t kErrBounds = 2;    // a table entry named no block of the pool -> LT_E_BOUNDS
                                     // (tested by LT_BOUNDS_CHECK builds, and by every build
                                     // for tables the caller owns)

// Per-token input of one attention launch: the token's sequence, its
// position (it attends over blocks [0, pos/16]), the physical id of its last
// block, the tile prefix P = sum of (pos_j/16 + 1 - skip_j) over tokens
// j < i, and skip: its first `skip` blocks are a shared prefix whose
// attention the prefix pass already computed (partial in pre_o / pre_ml).
struct TokenDesc {
    int32_t seq, pos, last_block, prefix, skip;
};

constexpr int kInlineTokens = 512;  // tokens passed inside the kernel parameters
constexpr int kMaxPeers = 8;        // ranks of a head-sharded peer gather
constexpr int kMergeGroup = 8;      // partials a group leader combines (two-level merge)

struct AttnParams {
    const uint16_t* pool_layer;  // pool + layer offset
    uint16_t* pool_layer_w;      // same, for the fused append
    int32_t* tables;             // [max_seqs][max_blocks]; each token's last entry is (re)written
    int32_t max_blocks;
    int32_t n_blocks;            // blocks in the pool, for LT_BOUNDS_CHECK builds (0: not checked)
    int32_t check_ids;           // test every block id read from `tables` against n_blocks in every
                                 // build (caller-owned tables, lt_paged_attend_noalloc)
    const TokenDesc* toks;       // n_tok entries in global memory, or null: use inl
    int32_t n_tok;
    int32_t tiles_per_head;      // prefix of n_tok (total blocks over the tokens)
    int32_t piece_cost;          // LT_KV_Q4_0: tiles a (token, head) weighs in the partition beside its
                                 // blocks; TokenDesc.prefix and tiles_per_head count them
    int32_t n_warps;             // stream-K ranges; tile total = tiles_per_head * n_kv_heads
    int32_t n_kv_heads;
    int32_t group;
    const void* q;               // [n][n_heads*D]
    int32_t q_f32;
    void* out;                   // [n][n_heads*D]
    int32_t out_f32;
    float scale_log2;            // scale * log2(e)
    float* part_o;               // [n_warps][group][D]: partial of warp w's first piece
    float* part_ml;              // [n_warps][group][2]
    uint32_t* flags;             // [n_warps]: warp w stores `epoch` once its range is done
    // Two-level merge of (token, head)s cut into more than kMergeGroup + 1
    // pieces: the helper warps' partials are first combined in groups of
    // kMergeGroup by each group's first warp (into slot w of part2_*, flag
    // flags2[w]); the merging warp then reads one partial per group.  Null:
    // one level (the merging warp reads every helper's partial).
    float* part2_o;
    float* part2_ml;
    uint32_t* flags2;
    uint32_t epoch;              // distinct per launch on a flags array
    int32_t* err;                // device error flag
    const void* k_new;           // fused append: new K/V rows [n][n_kv_heads*D], or null
    const void* v_new;
    int32_t kv_f32;
    const float* pre_o;          // [pre_splits][rows][D]: shared-prefix partial O (tokens with skip > 0),
    const float* pre_ml;         // [pre_splits][rows][2]: its (m, l); row = (token*n_kv_heads + h)*group + g
    int32_t pre_splits;          // partials per row (the prefix blocks split over that many CTAs)
    int64_t pre_split_rows;      // rows between split slabs
    int32_t fmt;                 // lt_kv_format of the pool's tiles; LT_KV_Q8_0 has no prefix partials
    // Head-sharded gather over NVLink (lt_kv_attend_gather).  With n_peers > 0
    // every output row goes, instead of to `out`, to this rank's gather half
    // gather_out at row tok*(n_peers*n_heads) + peer_rank*n_heads + head, and
    // the (token, head) that completes the count publishes peer_epoch into
    // every rank's flag for this rank (peer_flag[r]); the ranks then read
    // each other's rows (launch_gather_wait_copy).
    int32_t n_peers;
    int32_t peer_rank;
    uint32_t peer_epoch;
    uint32_t* done_count;        // this rank's count of stored (token, head)s (zero between launches)
    void* gather_out;
    uint32_t* peer_flag[kMaxPeers];
    TokenDesc inl[kInlineTokens];
};

// Score terms of a shaped call (lt_kv_score), the same for all its tokens.
// q.k becomes, in log2 units, cap_log2 * tanh(q.k * scale_cap) with a cap,
// else q.k * scale_log2; then slope * |distance| is taken off.
struct ShapeTerms {
    int32_t capped;
    float scale_cap;      // scale / cap
    float cap_log2;       // cap * log2(e)
    float scale_log2;     // scale * log2(e)
    const float* slopes;  // [n_heads], natural units, or null
};

// Per-token part of a shaped call beside its TokenDesc, whose pos is the last
// position attended and whose skip counts the blocks before position lo.
// An empty interval is described by one block with lo past pos.
struct ShapeDesc {
    int32_t lo;    // first position attended
    int32_t qpos;  // the token's own position (distances count from it)
};

struct AttnShapedParams : AttnParams {
    ShapeTerms shape;
    const ShapeDesc* shapes;  // n_tok entries in global memory, or null: use inl_shapes
    ShapeDesc inl_shapes[kInlineTokens];
};

template <bool SH>
struct AttnParamsSel {
    using type = AttnParams;
};
template <>
struct AttnParamsSel<true> {
    using type = AttnShapedParams;
};
template <bool SH>
using AttnParamsOf = typename AttnParamsSel<SH>::type;

// Shared-prefix (cascade) pass: one CTA per item attends up to
// prefix_tokens_per_cta(group) tokens of one prefix group (128 query rows on
// the tensor cores) to the group's first n_blocks blocks for one KV head,
// each K/V tile staged once for all of them, and writes (m, l, O) partials
// that the stream-K launch folds into the tokens' outputs.
struct PrefixItem {
    int32_t root_seq;  // a member whose table row holds the shared blocks (LT_KV_Q4_0: where block 0 would
                       // lie in the workspace)
    int32_t blk0;      // this item's part of the shared blocks: [blk0, blk1)
    int32_t blk1;
    int32_t full;      // blocks before this one count for every token of the item
    int32_t split;     // which partial slab it writes
    int32_t head;      // KV head
    int32_t tok_off;   // first of the item's tokens in the token list
    int32_t n_tok;     // tokens of this item
};
constexpr int kPreMaxSplits = 4;
struct PrefixParams {
    const uint16_t* pool_layer;
    const int32_t* tables;
    int32_t max_blocks;
    int32_t n_blocks;  // blocks in the pool, for LT_BOUNDS_CHECK builds (0: not checked)
    const PrefixItem* items;
    const int32_t* tok_list;  // token indices of the call (into q, pre_o, pre_ml)
    const int32_t* tok_lim;   // parallel to tok_list: the token attends positions [0, tok_lim) here
    int32_t n_kv_heads, group;
    const void* q;
    int32_t q_f32;
    int32_t scale_q;     // q4: rows of q go to the tensor core times a power of two
    float scale_log2;
    float* pre_o;
    float* pre_ml;
    int64_t split_rows;  // rows between split slabs of pre_o / pre_ml
    void* out;           // not null: every token's positions are all attended here, by one split; rows of
                         // [token][n_heads][head_dim] go to out instead of pre_o, pre_ml
    int32_t out_f32;
    // Shaped scores (launch_prefix's `shaped`; with out alone): parallel to tok_list
    const int32_t* tok_lo;    // first position attended
    const int32_t* tok_qpos;  // the token's own position
    ShapeTerms shape;
    int32_t* err;
};
// Tokens one prefix CTA covers: 128 query rows / group.
inline int prefix_tokens_per_cta(int group) { return 128 / group; }
// q4: the tiles are an expanded 4-bit cache's; only those have shaped scores.
cudaError_t launch_prefix(const PrefixParams& p, int n_items, int head_dim, bool q4, bool shaped, cudaStream_t s);

// Warps of one attention launch on `device` (all resident at once), or 0.
// fmt: lt_kv_format of the pool; shaped: the launch is launch_attend_shaped.
int attend_warps(int device, int group, int head_dim, int q_f32, int fmt, bool shaped = false);
cudaError_t launch_attend(const AttnParams& p, int head_dim, cudaStream_t s);
cudaError_t launch_attend_shaped(const AttnShapedParams& p, int head_dim, cudaStream_t s);
// The same for LT_KV_Q4_0 pools, on the current device (called by the above).
int attend_q4_warps(int device, int group, int head_dim, int q_f32, bool shaped);
cudaError_t launch_attend_q4(const AttnParams& p, int head_dim, cudaStream_t s);
cudaError_t launch_attend_q4_shaped(const AttnShapedParams& p, int head_dim, cudaStream_t s);
constexpr int kQ4PieceCost = 4;  // AttnParams.piece_cost
// Kernel launches made by launch_attend(p).
int attend_launches(const AttnParams& p);

// Head-sharded output assembly: gathered [nranks][n][row bytes] ->
// out [n][nranks][row bytes] (row = one token's local heads).
cudaError_t launch_gather_permute(const void* gathered, void* out, int nranks, uint32_t n, size_t row_bytes,
                                  cudaStream_t s);

// first_slot: slot of cells[0], which the host knows (LT_KV_Q4_0 aligns blocks by it).
cudaError_t launch_write(uint16_t* pool_layer, const int2* cells, int n, int n_kv_heads, int head_dim, int first_slot,
                         const void* k, const void* v, int in_f32, int fmt, cudaStream_t s);
// shift: slot of the call's first cell (0..15): blocks are tried from token -shift on.
cudaError_t launch_write_q4(uint8_t* pool_layer, const int2* cells, int n, int n_kv_heads, int head_dim, int shift,
                            const void* k, const void* v, int in_f32, cudaStream_t s);

// Blocks [first, first + count) of sequence root's table, expanded to f16 tiles
// as blocks base, base + 1, ... of a workspace.
struct ExpandGroup {
    int32_t root, base, count, first;
};
constexpr int kExpandGroups = 128;  // groups of one launch (kernel parameters)
cudaError_t launch_expand_q4(const uint8_t* pool_layer, const int32_t* tables, int max_blocks, const ExpandGroup* groups,
                             int n_groups, int n_kv_heads, int head_dim, uint16_t* out, int n_blocks, int32_t* err,
                             cudaStream_t s);

// Values of n cells of a pool of any format -> k_out, v_out [n][n_kv_heads*head_dim], f32 or f16.
cudaError_t launch_read(const uint16_t* pool_layer, const int2* cells, int n, int n_kv_heads, int head_dim,
                        int first_slot, void* k_out, void* v_out, int out_f32, int fmt, cudaStream_t s);

// Block copies (copy-on-write and compaction moves) and table scatter.
// copies: (src, dst) pairs; tw: (flat table index, value) pairs.  n_blocks
// and n_entries (pool blocks, table entries) bound the indices in
// LT_BOUNDS_CHECK builds, which report a bad one through err.
cudaError_t launch_apply_plan(uint16_t* pool, size_t layer_stride_elems, size_t block_elems, int n_layers,
                              const int2* copies, int n_copies, int32_t* tables, const int2* tw, int n_tw,
                              int n_blocks, long long n_entries, int32_t* err, cudaStream_t s);

cudaError_t launch_rows(const uint16_t* pool_layer, const int32_t* table_row, int n, int n_kv_heads,
                        int head_dim, uint16_t* k_out, uint16_t* v_out, int fmt, int n_blocks, int32_t* err,
                        cudaStream_t s);
cudaError_t launch_rows_q4(const uint8_t* pool_layer, const int32_t* table_row, int n, int n_kv_heads, int head_dim,
                           uint16_t* k_out, uint16_t* v_out, int n_blocks, int32_t* err, cudaStream_t s);

// One warp waits, through the kernels' bounded flag wait with a limit of
// limit_ns, for a device word that nothing sets, then raises kErrTimeout in
// err: the failure path of every bounded wait, made to run out on purpose.
cudaError_t launch_wait_selftest(uint64_t limit_ns, int32_t* err, cudaStream_t s);
// Whether this build checks table entries on the device (LT_BOUNDS_CHECK).
bool bounds_checked_build();

// Peer gather, receiving side: wait (bounded, system-scope acquire) until
// every rank's flag in `flags` has reached `epoch`, then assemble `out`
// [n][nranks][slice_bytes]: slice r of every token comes from rank r's
// gather half srcs[r] (the same layout; over NVLink for the other ranks).
// A wait that gives up raises kErrTimeout and copies nothing.
cudaError_t launch_gather_wait_copy(const uint32_t* flags, int nranks, uint32_t epoch, void* const* srcs, void* out,
                                    uint32_t n, size_t slice_bytes, int32_t* err, cudaStream_t s);

}  // namespace ltkv

// Accessors of the opaque handle for the other translation units.
struct lt_kv;
struct lt_kv_config;
namespace ltkv {
size_t local_out_row_bytes(const lt_kv* kv, int dtype);  // n_heads*head_dim*elem of this handle
int handle_device(const lt_kv* kv);
const lt_kv_config* handle_config(const lt_kv* kv);
void count_launch(lt_kv* kv);
// Host bookkeeping reads for the scheduler driver: entry idx of seq's block
// list, and a block's refcount.
int32_t seq_block_at(const lt_kv* kv, uint32_t seq, uint32_t idx);
uint32_t block_refs(const lt_kv* kv, int32_t block);
}  // namespace ltkv

namespace ltkv {
// NVTX range over one C ABI call, named after it, so a timeline from a
// profiler shows the host bookkeeping and launches of each call.  With no
// profiler attached the push/pop cost one test of a null pointer each.
struct NvtxRange {
    explicit NvtxRange(const char* name) { nvtxRangePushA(name); }
    ~NvtxRange() { nvtxRangePop(); }
    NvtxRange(const NvtxRange&) = delete;
    NvtxRange& operator=(const NvtxRange&) = delete;
};
}  // namespace ltkv

// Launcher interface of the attention operators and of the attention branch's
// gradients, between the C-ABI layer (t2h_api.hip) and t2h_attn.hip,
// t2h_attn_bwd.hip and t2h_qk_bwd.hip. Arguments arrive validated.
#pragma once

#include "t2h_internal.h"

namespace t2h {

// Attention and its backward pass (t2h_attention, t2h_attention_backward).
// Strides in elements. A side's segments: from its offsets, or nbatch equal shares.
struct AttnSide {
    const int64_t* offsets;  // [nbatch + 1] or nullptr
    int32_t rows;
    int32_t share;           // rows / nbatch
};
struct AttnArgs {
    const void* q;           // [q_rows, heads, head_dim]
    const void* k;           // [k_rows, kv_heads, head_dim]
    const void* v;
    void* out;               // [q_rows, heads, head_dim]
    float* lse;              // [heads, q_rows] or nullptr
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;
    int64_t q_rows, k_rows;
    int32_t heads;
    int32_t group;           // query heads per key/value head
    int32_t head_dim;
    int32_t dtype;
    float scale;
    AttnSide qs, ks;
    const int64_t* k_lens;   // [nbatch] keys of a segment that count, or nullptr
    int32_t nbatch;
    int32_t nsplit;          // parts of a segment's keys, joined afterwards
    float* part;             // workspace: [nsplit, q_rows, heads, head_dim] parts' outputs
    float* part_lse;         // workspace: [nsplit, heads, q_rows], log2
    int32_t q_tiles;         // set by the launcher: numbers of query tiles
    int32_t nblocks;         // set by the launcher
};

struct AttnBwdArgs {
    AttnArgs f;              // the forward's operands, output and log-sum-exp
    const void* dout;        // [q_rows, heads, head_dim]
    void* dq;
    void* dk;
    void* dv;
    int64_t do_row, do_head, dq_row, dq_head, dk_row, dk_head, dv_row, dv_head;
    int32_t kv_heads;
    // set by attn_bwd_plan: forms, parts, and the workspace's pieces
    int32_t kv_split, q_split;
    bool kv_small, q_small, fine, q_first;
    float* delta;            // [heads, q_rows]
    float* lse2;             // [heads, q_rows] log2, less the rounding shift of P
    float* g_most;           // [heads, prep_q_tiles] f16: largest squared row length of dout in each tile
    float* v_most;           // [kv_heads, prep_k_tiles]   ... of v
    float* part_kv;          // [2, kv_split, k_rows, kv_heads, head_dim] dk's and dv's parts
    float* part_q;           // [q_split, q_rows, heads, head_dim]
    int32_t prep_q_tiles, prep_k_tiles, prep_blocks;
    int32_t k_tiles, kv_blocks, q_blocks;   // set by the launcher
};

// Backward pass of the q/k epilogue (t2h_qk_rmsnorm_rope_backward).
struct QkBwdTensor {
    const void* x;           // the forward's input rows (read for the norm)
    const void* dy;          // gradient of its output
    void* dx;                // gradient of its input; may alias dy
    const float* bias;
    const float* gamma;      // nullptr = no RMS
    float* dgamma;           // [heads, head_dim] or nullptr
    float* dbias;
};
struct QkBwdArgs {
    QkBwdTensor t[2];
    int32_t tensors;
    int64_t rows;
    int64_t x_stride, dy_stride, dx_stride;
    int32_t heads;
    int32_t head_dim;
    int32_t dtype;
    float rms_scale;
    int32_t use_rope;
    int32_t pos_dim;
    int32_t freq_dim;
    const float* phases;
    int64_t phase_rows;
    const int32_t* coords;
    int32_t coord_cols;
    int32_t grid_res;
    float* part;             // workspace: [tensors, blocks, 2, heads * head_dim]
    int64_t blocks;          // set by the launcher: partial rows per tensor
};

// t2h_attn.hip
int attn_splits(const AttnArgs& a);                         // parts that suit the sizes (1: none)
int64_t attn_split_bytes(const AttnArgs& a, int nsplit);    // workspace of that many parts
hipError_t launch_attn(AttnArgs a, hipStream_t s);
// t2h_attn_bwd.hip
int64_t attn_bwd_plan(AttnBwdArgs& a, void* workspace);     // places the workspace's pieces, returns its bytes
hipError_t launch_attn_bwd(const AttnBwdArgs& a, hipStream_t s);
// t2h_qk_bwd.hip
int64_t qk_bwd_bytes(int64_t rows, int32_t heads, int32_t head_dim, int32_t tensors);   // workspace of the sums
hipError_t launch_qk_bwd(QkBwdArgs a, const RopeSlots& tab, hipStream_t s);

}  // namespace t2h

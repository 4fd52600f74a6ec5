// Arguments of the attention kernels, shared by the device code and the host side that fills them.
#pragma once

namespace kmc {

typedef long long i64;

constexpr int ATT_MAX_SLOTS = 128;          // partial results of a row
// A dimension of a grid holds fewer than 2^32 threads, so this many workgroups of 256; larger grids are several launches, each a multiple of the 8 XCDs.
constexpr int ATT_MAX_BLOCKS = (1 << 24) - 8;

// Keys and values of one segment; strides in elements.
struct AttentionKeys {
    const void *k, *v;
    i64 k_ls, k_ns, k_gs, v_ls, v_ns, v_gs;
    const int *lengths;                     // per batch entry, or null: all n take part
    const unsigned char *mask;              // per batch entry and key, or null
    i64 mask_ls, mask_ns;
    int n;
    int causal;                             // the queries are the last m of `lengths` tokens
};

// A list of workgroups: (batch entry, head of keys, range of keys, tile of rows), the tile of rows fastest.
struct AttentionJob {
    int first_segment, last_segment;
    int entries, rows, row_tiles, splits;
    int slot;                               // of its first partial result
    int partial, own_keys;
    int workgroups, grid;                   // grid: workgroups rounded up to a multiple of the 8 XCDs
};

struct AttentionArgs {
    const void *q;
    i64 q_ls, q_ms, q_hs;
    void *out;
    i64 out_ls, out_ms, out_hs;
    float *lse;                             // [l, m, g r], or null
    AttentionKeys keys[2];
    AttentionJob job[2];
    int first_block;                        // of this launch
    int m, g, r, k, o;
    float scale_log2;                       // |scale| log2(e), above 0
    float query_factor;                     // 1; -1 for a negative scale; 0 for a scale of 0
    float *partial_out;                     // [slots, rows_total, partial_width]
    float *partial_shift, *partial_lse;     // [slots, rows_total]: a score that was subtracted (-inf: no keys), and the lse beside it to base 2
    int slots, partial_width;
    i64 rows_total;                         // l m g r
};

struct AttentionGradArgs {
    const void *q, *out, *grad_out;
    i64 q_ls, q_ms, q_hs, out_ls, out_ms, out_hs, grad_out_ls, grad_out_ms, grad_out_hs;
    const float *lse;                       // [l, m, g r]
    AttentionKeys keys;
    void *grad_q, *grad_k, *grad_v;         // contiguous [l, m, g r, k], [key_entries, n, g, k], [key_entries, n, g, o]
    int first_block;                        // of this launch
    int l, m, g, r, k, o;
    int key_entries;                        // l, or 1: one source for all entries
    float scale, scale_log2, query_factor;
    float *stats;                           // [2, l, g r, m]: lse to base 2 (+inf without keys) and delta, for weights times a power of two, from the first kernel for the second; behind them +inf and 0
    // For rows of large scores, or null: [l, g r, m], what is subtracted from a row's scores in front of the scale, and [l, g, q_row_tiles], whether a tile of 128 rows
    // has such rows (their lse is the one beside the shift).
    float *row_shift;
    int *row_flags;
    int q_row_tiles, q_splits, q_workgroups, q_grid;
    int key_tiles, k_splits, k_workgroups, k_grid;
    float *partial_q, *partial_k, *partial_v;   // [splits, rows, width rounded up to 4], where the work is cut
    int partial_k_width, partial_o_width;
};

// Sums of partial results, times a factor, in the operands' type: up to three results in one launch.
struct AttentionSum {
    const float *partial;
    void *out;
    i64 rows;
    int splits, width, partial_width;
    float factor;
};

struct AttentionSumArgs {
    AttentionSum part[3];
    i64 first[4];                           // elements in front of each part, of all
};

}  // namespace kmc

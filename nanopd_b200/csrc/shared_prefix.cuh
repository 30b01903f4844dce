// What the three launches of the shared-prefix attention hand to one another (see shared_prefix.cu).
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace {

// Rows between the records of two CTAs of the prefix pass: an item holds up to two query tiles of 128 rows.  The row r of
// item i in the piece of CTA w is record row R_i + w * kPrefixRows + r, with R_i the (query, head) rows of the items before
// i.  Items and CTAs follow the same line of units, so no two pieces share a row and the whole takes
// num_seqs * num_q_heads + CTAs * kPrefixRows rows.
constexpr int kPrefixRows = 256;

struct PrefixPlanHead {
    int total_units;      // key tiles over all (group, query tiles, kv head) items
    int units_per_worker;
    int pad[2];
};
struct PrefixGroup {
    int begin, seqs;      // sequences of the group
    int tokens;           // shared tokens that the prefix pass covers, a multiple of 16
    int key_tiles;        // K/V tiles of them
    int table_seq;        // the group's first sequence that is not empty: its table row names the shared pages
};
struct PrefixSeed {
    int group, pair, head, tile;      // where a CTA's run of units begins
};
struct PrefixSeqPlan {
    int first_tile;       // 16-token tiles of the sequence that the prefix pass covers
    int unit0;            // first unit of this sequence's item for kv head 0
    int key_tiles;        // units of one item (0: nothing is shared)
    int item_first_seq;   // first sequence of the item
    int item_seqs;        // sequences of the item
    int pad[3];
};

}  // namespace

namespace npd {

// The prefix pass (prefix_pass.cu): its arguments as the C ABI names them.
struct PrefixPass {
    const void *q, *k_cache, *v_cache;
    const int32_t *block_tables;
    float scale;
    int64_t num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, num_blocks, cache_block_stride,
        bt_row_stride;
    int dtype;
    int32_t *status;
    const void *groups, *seeds, *plan_head;
    float *prefix_o, *prefix_lse;
    int ctas;
    void *stream;
};
int launch_prefix_pass(const PrefixPass &a);

// A shared-prefix call (scored_attention.cu): answered without sharing, by the small form of the decode kernel, where that
// form takes the batch; *taken says whether it did.
struct SharedCall {
    void *out;
    const void *q, *k_cache, *v_cache;
    const int32_t *block_tables, *seq_lens, *group_offsets, *shared_lens;
    float scale;
    int64_t num_seqs, num_groups, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, num_blocks,
        cache_block_stride, bt_row_stride;
    int dtype;
    void *workspace;
    size_t workspace_bytes;
    int32_t *status;
    int flags;
    void *stream;
};
int decode_unshared_if_small(const SharedCall &a, bool *taken);

}  // namespace npd

// Paged decode attention with shaped scores: capped by a tanh, biased by the distance to the key, seen through a sliding
// window.  For the query of sequence s (at position n - 1, n = seq_lens[s]) and key j, with n - window <= j < n:
//   x_j = scale * q . k_j;   x_j = cap * tanh(x_j / cap);   x_j -= slope[h] * (n - 1 - j);   out = softmax(x) . V
// The kernel is the streaming one of decode_kernel.cuh in its mode kScored: HBM-bound, every visible K/V byte read once.
// A tile of 16 keys costs a thread four scores, so the tanh (capped_scores.cuh) disappears behind the tile's loads.  A window moves the first tile of each sequence: the split into equal work, the small-batch form and the
// merge then count its tiles only, and neither the pages before it nor their table entries are read.
#include "decode_kernel.cuh"

extern "C" int npd_paged_scored_attention(void *out, const void *q, const void *k_cache, const void *v_cache,
                                          const int32_t *block_tables, const int32_t *seq_lens, float scale,
                                          float score_cap, const float *distance_slopes, int64_t window,
                                          int64_t num_seqs, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                          int64_t block_size, int64_t max_blocks_per_seq, int64_t num_blocks,
                                          int64_t cache_block_stride, int64_t bt_row_stride, int dtype, void *workspace,
                                          size_t workspace_bytes, int32_t *status, int flags, void *stream) {
    DecodeCall c{out, q, k_cache, v_cache, block_tables, seq_lens, scale, num_seqs, num_q_heads, num_kv_heads, head_dim,
                 block_size, max_blocks_per_seq, num_blocks, cache_block_stride, bt_row_stride, dtype, workspace,
                 workspace_bytes, flags, stream};
    NPD_REQUIRE((flags & ~0xffff00) == 0, NPD_ERR_INVALID_ARG, "scored attention: only NPD_FLAG_MAX_CTAS is a flag here");
    const int rs = npd::check_score_shape("scored attention", scale, score_cap, distance_slopes, window);
    if (rs != NPD_OK) return rs;
    c.status = status;
    c.score_cap = score_cap;
    c.slopes = distance_slopes;
    c.window = window;
    const int rc = check_decode_call(c);
    return rc != NPD_OK || num_seqs == 0 ? rc : run_decode<kScored>(c);
}

int npd::decode_unshared_if_small(const npd::SharedCall &a, bool *taken) {
    DecodeCall c{a.out, a.q, a.k_cache, a.v_cache, a.block_tables, a.seq_lens, a.scale, a.num_seqs, a.num_q_heads, a.num_kv_heads,
                 a.head_dim, a.block_size, a.max_blocks_per_seq, a.num_blocks, a.cache_block_stride, a.bt_row_stride, a.dtype,
                 a.workspace, a.workspace_bytes, a.flags, a.stream};
    c.status = a.status;
    c.group_offsets = a.group_offsets;
    c.shared_lens = a.shared_lens;
    c.num_groups = a.num_groups;
    *taken = takes_cluster_form(c);
    return *taken ? run_decode<kScored>(c) : NPD_OK;
}

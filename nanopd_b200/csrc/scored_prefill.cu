// Prompt attention with shaped scores: capped by a tanh, biased by the distance to the key, seen through a sliding window
// (the formula is in scored_attention.cu; here a query at position i sees the keys i - window < j <= i).  The kernel is the
// tcgen05 one of prefill_kernel.cuh in its modes kShaped and kCapped.  A window moves the first key tile of each pair of query tiles, so
// that the work grows with the window and not with the context.
#include "prefill_kernel.cuh"

extern "C" int npd_paged_scored_prefill_attention(
    void *out, const void *q, const void *k_cache, const void *v_cache, const int32_t *block_tables,
    const int32_t *chunk_q_offset_host, const int32_t *chunk_tokens_host, const int32_t *chunk_start_host, int64_t num_chunks,
    float scale, float score_cap, const float *distance_slopes, int64_t window, int64_t num_q_heads, int64_t num_kv_heads,
    int64_t head_dim, int64_t block_size, int64_t max_blocks_per_seq, int64_t num_blocks, int64_t cache_block_stride,
    int64_t bt_row_stride, int dtype, void *workspace, size_t workspace_bytes, int32_t *status, int flags, void *stream) {
    NPD_REQUIRE((flags & ~0xffff00) == 0, NPD_ERR_INVALID_ARG, "scored prefill attention: only NPD_FLAG_MAX_CTAS is a flag here");
    const int rs = npd::check_score_shape("scored prefill attention", scale, score_cap, distance_slopes, window);
    if (rs != NPD_OK) return rs;
    PrefillCall c{out, q, k_cache, v_cache, block_tables, chunk_q_offset_host, chunk_tokens_host, chunk_start_host, num_chunks,
                  scale, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, num_blocks, cache_block_stride,
                  bt_row_stride, dtype, workspace, workspace_bytes, flags, stream};
    c.status = status;
    c.score_cap = score_cap;
    c.slopes = distance_slopes;
    c.window = window;
    try {
        return score_cap > 0.f ? run_prefill<kCapped>(c) : run_prefill<kShaped>(c);
    } catch (const std::exception &e) {          // the list of work items is host memory
        return npd::fail(NPD_ERR_CUDA, "scored prefill attention: %s", e.what());
    }
}

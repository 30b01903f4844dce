// Entry point of chunked-prefill attention; the kernel and its design notes are in prefill_kernel.cuh.
#include "prefill_kernel.cuh"

extern "C" size_t npd_prefill_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int) { return 256; }

extern "C" int npd_paged_prefill_attention(void *out, const void *q, const void *k_cache, const void *v_cache,
                                           const int32_t *block_tables, const int32_t *chunk_q_offset_host,
                                           const int32_t *chunk_tokens_host, const int32_t *chunk_start_host,
                                           int64_t num_chunks, float scale, int64_t num_q_heads, int64_t num_kv_heads,
                                           int64_t head_dim, int64_t block_size, int64_t max_blocks_per_seq,
                                           int64_t num_blocks, int64_t cache_block_stride, int64_t bt_row_stride,
                                           int dtype, void *workspace, size_t workspace_bytes, int flags,
                                           void *stream) {
    try {
        return run_prefill<kCausal>({out, q, k_cache, v_cache, block_tables, chunk_q_offset_host, chunk_tokens_host, chunk_start_host,
                                     num_chunks, scale, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq,
                                     num_blocks, cache_block_stride, bt_row_stride, dtype, workspace, workspace_bytes, flags, stream});
    } catch (const std::exception &e) {          // the list of work items is host memory
        return npd::fail(NPD_ERR_CUDA, "prefill attention: %s", e.what());
    }
}

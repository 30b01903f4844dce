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
    NPD_REQUIRE(dtype == NPD_DTYPE_F16 || dtype == NPD_DTYPE_BF16, NPD_ERR_UNSUPPORTED,
                "prefill attention supports float16 and bfloat16 only (dtype code %d)", dtype);
    NPD_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, NPD_ERR_UNSUPPORTED,
                "prefill attention: head_dim %lld not in {64,128,256}", (long long)head_dim);
    NPD_REQUIRE(block_size == 4 || block_size == 8 || block_size == 16 || block_size == 32, NPD_ERR_UNSUPPORTED,
                "prefill attention: block_size %lld not in {4,8,16,32}", (long long)block_size);
    NPD_REQUIRE(num_chunks >= 0 && num_q_heads > 0 && num_kv_heads > 0 && max_blocks_per_seq > 0 && num_blocks > 0,
                NPD_ERR_INVALID_ARG, "prefill attention: non-positive dimension");
    NPD_REQUIRE(num_q_heads % num_kv_heads == 0, NPD_ERR_INVALID_ARG,
                "prefill attention: num_q_heads is not a multiple of num_kv_heads");
    const int group = static_cast<int>(num_q_heads / num_kv_heads);
    NPD_REQUIRE(group <= 128, NPD_ERR_UNSUPPORTED, "prefill attention: more than 128 q heads per kv head");
    if (num_chunks == 0) return NPD_OK;
    NPD_REQUIRE(out && q && k_cache && v_cache && block_tables && chunk_q_offset_host && chunk_tokens_host &&
                    chunk_start_host,
                NPD_ERR_INVALID_ARG, "prefill attention: NULL pointer");
    NPD_REQUIRE(workspace != nullptr && workspace_bytes >= 256, NPD_ERR_WORKSPACE,
                "prefill attention: workspace of at least 256 bytes needed (status word)");
    NPD_REQUIRE(npd::aligned16(q) && (reinterpret_cast<uintptr_t>(out) & 31u) == 0, NPD_ERR_INVALID_ARG,
                "prefill attention: q must be 16-byte and out 32-byte aligned");
    NPD_REQUIRE(num_blocks < INT32_MAX && max_blocks_per_seq * block_size < INT32_MAX, NPD_ERR_INVALID_ARG,
                "prefill attention: dimension exceeds int32");

    int64_t total_tokens = 0;
    for (int64_t i = 0; i < num_chunks; ++i) {
        NPD_REQUIRE(chunk_tokens_host[i] >= 0 && chunk_start_host[i] >= 0 && chunk_q_offset_host[i] >= 0,
                    NPD_ERR_INVALID_ARG, "prefill attention: negative chunk field");
        NPD_REQUIRE((int64_t)chunk_start_host[i] + chunk_tokens_host[i] <= max_blocks_per_seq * block_size,
                    NPD_ERR_INVALID_ARG, "prefill attention: chunk %lld reaches beyond its block table", (long long)i);
        const int64_t end = (int64_t)chunk_q_offset_host[i] + chunk_tokens_host[i];
        if (end > total_tokens) total_tokens = end;
    }
    if (total_tokens == 0) return NPD_OK;

    const int tq = kRows / group;
    CUtensorMap tq_map, tk, tv;
    {
        const uint64_t dims[3] = {(uint64_t)head_dim, (uint64_t)num_q_heads, (uint64_t)total_tokens};
        const uint64_t strides[2] = {(uint64_t)head_dim * 2u, (uint64_t)num_q_heads * head_dim * 2u};
        const uint32_t box[3] = {64u, (uint32_t)group, (uint32_t)tq};
        const int rc = npd::encode_tiled_3d(&tq_map, q, dtype, dims, strides, box);
        if (rc != NPD_OK) return rc;
    }
    const int box_rows = block_size < 16 ? static_cast<int>(block_size) : 16;
    int rc = npd::encode_cache_tensor_map(&tk, k_cache, dtype, head_dim, num_kv_heads * block_size, num_blocks,
                                          cache_block_stride, box_rows);
    if (rc != NPD_OK) return rc;
    rc = npd::encode_cache_tensor_map(&tv, v_cache, dtype, head_dim, num_kv_heads * block_size, num_blocks,
                                      cache_block_stride, box_rows);
    if (rc != NPD_OK) return rc;

    const size_t halves = static_cast<size_t>(head_dim / 64);
    const int query_tiles = head_dim == 256 ? 1 : 2, tile_keys = head_dim == 256 ? 64 : kKeys;
    const size_t smem = 1024 + query_tiles * halves * kQHalfBytes + (size_t)(kStagesK + kStagesV) * halves * tile_keys * 128 +
                        sizeof(SmemCtrl) + 64;
    const bool f16 = dtype == NPD_DTYPE_F16;
    using Kernel = void (*)(PrefillParams, CUtensorMap, CUtensorMap, CUtensorMap);
    Kernel kern = nullptr;
#define NPD_PICK_B(D_, B_) (f16 ? paged_prefill_kernel<__half, D_, B_> : paged_prefill_kernel<__nv_bfloat16, D_, B_>)
#define NPD_PICK(D_) kern = box_rows == 4 ? NPD_PICK_B(D_, 4) : (box_rows == 8 ? NPD_PICK_B(D_, 8) : NPD_PICK_B(D_, 16))
    if (head_dim == 64) NPD_PICK(64);
    else if (head_dim == 128) NPD_PICK(128);
    else NPD_PICK(256);
#undef NPD_PICK
#undef NPD_PICK_B
    NPD_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));

    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int dev = 0;
    NPD_CUDA_TRY(cudaGetDevice(&dev));
    const long long sms = npd::sm_count(dev);
    for (int64_t c0 = 0; c0 < num_chunks; c0 += kMaxChunks) {
        const int nc = static_cast<int>(num_chunks - c0 < kMaxChunks ? num_chunks - c0 : kMaxChunks);
        PrefillParams p;
        p.out = out;
        p.block_tables = block_tables + c0 * bt_row_stride;
        p.status = static_cast<int32_t *>(workspace);
        p.scale_log2 = scale * 1.4426950408889634f;
        p.num_chunks = nc;
        p.num_q_heads = static_cast<int>(num_q_heads);
        p.num_kv_heads = static_cast<int>(num_kv_heads);
        p.group = group;
        p.tq = tq;
        p.block_size = static_cast<int>(block_size);
        p.box_rows = box_rows;
        p.query_tiles = query_tiles;
        p.half_steps_per_tile = tile_keys / kHalfKeys;
        p.max_blocks_per_seq = static_cast<int>(max_blocks_per_seq);
        p.num_blocks = static_cast<int>(num_blocks);
        p.bt_row_stride = bt_row_stride;
#ifdef NPD_PREFILL_TRACE
        p.trace = workspace_bytes >= 256 + 11 * 4096 * sizeof(long long)
                      ? reinterpret_cast<long long *>(static_cast<uint8_t *>(workspace) + 256) : nullptr;
#endif
        // Pairs of query tiles of the launch, heaviest (most key tiles) first; the kernel hands them out in
        // this order through an atomic counter.
        struct Entry { int weight; uint32_t code; };
        std::vector<Entry> entries;
        for (int i = 0; i < nc; ++i) {
            p.chunk_q_offset[i] = chunk_q_offset_host[c0 + i];
            p.chunk_tokens[i] = chunk_tokens_host[c0 + i];
            p.chunk_start[i] = chunk_start_host[c0 + i];
            const int pairs = (p.chunk_tokens[i] + query_tiles * tq - 1) / (query_tiles * tq);
            NPD_REQUIRE(pairs <= 0xffff, NPD_ERR_INVALID_ARG, "prefill attention: chunk %d is too long", i);
            for (int pr = 0; pr < pairs; ++pr) {
                const int last_tok = std::min(p.chunk_tokens[i], (pr + 1) * query_tiles * tq);
                entries.push_back({(p.chunk_start[i] + last_tok + kKeys - 1) / kKeys,
                                   (static_cast<uint32_t>(i) << 16) | static_cast<uint32_t>(pr)});
            }
        }
        std::stable_sort(entries.begin(), entries.end(), [](const Entry &a, const Entry &b) { return a.weight > b.weight; });
        cudaStream_t launch_stream = st;
        for (size_t e0 = 0; e0 < entries.size(); e0 += kMaxPairs) {
            const int ne = static_cast<int>(std::min<size_t>(kMaxPairs, entries.size() - e0));
            for (int e = 0; e < ne; ++e) p.pair_order[e] = entries[e0 + e].code;
            p.num_pairs = ne;
            p.work_counter = reinterpret_cast<int *>(static_cast<uint8_t *>(workspace) + 64);   // zero: see the kernel's end
            const long long items = (long long)ne * num_kv_heads;
            long long grid = items < sms ? items : sms;           // persistent: one CTA per SM
            const int cta_cap = (flags >> 8) & 0xffff;
            if (cta_cap > 0 && cta_cap < grid) grid = cta_cap;
            kern<<<static_cast<unsigned>(grid), kThreads, smem, launch_stream>>>(p, tq_map, tk, tv);
            NPD_CUDA_TRY(cudaGetLastError());
        }
    }
    return NPD_OK;
}

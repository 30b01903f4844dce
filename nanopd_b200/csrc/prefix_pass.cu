// The prefix pass of the shared-prefix attention: the queries of a group of sequences over the pages they share, on the
// tensor cores.  The kernel is the one of prompt attention (prefill_kernel.cuh) in its mode kPrefix: the rows of a query
// tile are the sequences of the group times the q heads of a kv head, every key is visible to every row.
#include "prefill_kernel.cuh"

int npd::launch_prefix_pass(const PrefixPass &a) {
    PrefillCall c{nullptr, a.q, a.k_cache, a.v_cache, a.block_tables, nullptr, nullptr, nullptr, 0, a.scale, a.num_q_heads,
                  a.num_kv_heads, a.head_dim, a.block_size, a.max_blocks_per_seq, a.num_blocks, a.cache_block_stride,
                  a.bt_row_stride, a.dtype, nullptr, 0, 0, a.stream};
    PrefillLaunch l;
    const int rc = prepare_launch<kPrefix>(c, a.num_seqs, l);
    if (rc != NPD_OK) return rc;
    PrefillParams p;
    fill_geometry(c, l, p);
    p.out = nullptr;
    p.block_tables = a.block_tables;
    p.status = a.status;
    p.num_chunks = 0;
    p.num_pairs = 0;
    p.work_counter = nullptr;
    p.groups = static_cast<const PrefixGroup *>(a.groups);
    p.seeds = static_cast<const PrefixSeed *>(a.seeds);
    p.plan = static_cast<const PrefixPlanHead *>(a.plan_head);
    p.prefix_o = a.prefix_o;
    p.prefix_lse = a.prefix_lse;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(a.ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = l.smem;
    cfg.stream = static_cast<cudaStream_t>(a.stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // set up while the plan kernel runs
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    NPD_CUDA_TRY(cudaLaunchKernelEx(&cfg, l.kernel, p, l.q, l.k, l.v));
    return NPD_OK;
}

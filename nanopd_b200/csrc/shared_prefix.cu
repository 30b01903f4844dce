// Decode attention for a batch whose sequences share the first pages of their tables (a system prompt, a document): the
// shared keys are read and multiplied once per group of sequences instead of once per sequence.
//
// softmax over [prefix | own pages] is joined from its parts: with (m, l, O) the running maximum, sum and weighted rows of
// one part, the whole is  sum_i 2^(lse_i - M) O_i / l_i  over  sum_i 2^(lse_i - M),  lse_i = m_i + log2 l_i, M = max lse_i.
// Three launches on one stream, everything decided on the device (lengths may change between replays of a graph):
//   plan    one CTA: per group the tokens that all its sequences share and none ends in, in 16-token tiles; the line of
//           (group, query tiles, kv head, key tile) units cut into equal runs, one per SM; per sequence where its rows are
//   prefix  prefix_pass.cu: the rows of a group (sequences x heads of a kv head, 256 at a time, 128 at head size 256) over the
//           shared pages on the tensor cores, a piece per cut, normalised fp32 rows and their log2 sums
//   tail    the streaming decode kernel over each sequence's own pages, which joins the pieces where it writes the row
// Bytes: prefix pages once per 256 (128) rows of a kv head + own pages; flops of the prefix 4 * Hq * D * tokens * sequences.
#include "decode_kernel.cuh"

namespace {

constexpr int kMaxGroups = 4096;
constexpr int kPlanThreads = 1024;

struct PlanParams {
    const int32_t *group_offsets, *shared_lens, *seq_lens;
    int32_t *status;
    PrefixPlanHead *head;
    PrefixGroup *groups;
    PrefixSeed *seeds;
    PrefixSeqPlan *seqs;
    long long cap;              // tokens a table row can name
    int num_groups, num_seqs, num_kv_heads;
    int item_seqs;              // sequences of one item of the prefix pass
    int tile_keys;              // keys of one unit
    int workers;
};

// Exclusive prefix over v[0..n) in place, v[n] = the total; the whole CTA.  Ends with a barrier.
__device__ void exclusive_prefix(int *v, int n) {
    __shared__ int warp_sums[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
    const int chunk = (n + threads - 1) / threads;
    const int lo = min(tid * chunk, n), hi = min(lo + chunk, n);
    int sum = 0;
    for (int i = lo; i < hi; ++i) sum += v[i];
    int incl = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += u;
    }
    int run = incl - sum;
    if (n > 32 * chunk) {                        // more than the first warp has some
        if (lane == 31) warp_sums[warp] = incl;
        __syncthreads();
        for (int w = 0; w < warp; ++w) run += warp_sums[w];
    }
    for (int i = lo; i < hi; ++i) {
        const int x = v[i];
        v[i] = run;
        run += x;
    }
    if (hi == n && lo < n) v[n] = run;
    __syncthreads();
}

__global__ void __launch_bounds__(kPlanThreads) shared_prefix_plan_kernel(const PlanParams p) {
    extern __shared__ int plan_smem[];
    int *offs = plan_smem;                       // [num_groups + 1] group_offsets
    int *unit = offs + p.num_groups + 1;         // [num_groups + 1] units in front of each group
    int *least = unit + p.num_groups + 1;        // [num_groups] shortest sequence that is not empty
    int *first = least + p.num_groups;           // [num_groups] first sequence that is not empty: an empty one's table row may
                                                 // name anything (an idle slot's is parked on a page that nobody reads)
    __shared__ int bad;
    const int tid = threadIdx.x;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int my_len = tid < p.num_seqs ? p.seq_lens[tid] : 0;      // under way together with the offsets
    if (tid == 0) bad = 0;
    for (int g = tid; g <= p.num_groups; g += blockDim.x) {
        offs[g] = p.group_offsets[g];
        if (g < p.num_groups) least[g] = first[g] = INT32_MAX;
    }
    __syncthreads();                             // `bad` and the offsets are set
    // Groups must be consecutive ranges of the batch.  Anything else shares nothing (every row is still right: the tail
    // then covers whole sequences) and is flagged.
    for (int g = tid; g < p.num_groups; g += blockDim.x)
        if (offs[g] < 0 || offs[g + 1] < offs[g] || offs[g + 1] > p.num_seqs) bad = 1;
    __syncthreads();
    const bool none = bad != 0;
    if (none && tid == 0) atomicOr(p.status, NPD_STATUS_BAD_POSITION);
    // the last group that begins at or before sequence s, or -1
    auto group_of = [&](int s) {
        if (none || s < offs[0] || s >= offs[p.num_groups]) return -1;
        int lo = 0, hi = p.num_groups - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (offs[mid] <= s) lo = mid; else hi = mid - 1;
        }
        return lo;
    };
    for (int s = tid; s < p.num_seqs; s += blockDim.x) {
        const int n = s == tid ? my_len : p.seq_lens[s];
        const int g = group_of(s);
        if (g >= 0 && n > 0) {
            atomicMin(least + g, n);
            atomicMin(first + g, s);
        }
    }
    __syncthreads();
    for (int g = tid; g < p.num_groups; g += blockDim.x) {
        PrefixGroup out{0, 0, 0, 0, 0};
        if (!none) {
            out.begin = offs[g];
            out.seqs = offs[g + 1] - offs[g];
            const int shared = p.shared_lens[g];
            if (shared < 0) atomicOr(p.status, NPD_STATUS_BAD_POSITION);
            // at least one token stays with each sequence, so that the tail kernel visits (and writes) every row
            if (out.seqs > 1 && least[g] != INT32_MAX) {
                const long long most = min((long long)least[g], p.cap) - 1;
                out.tokens = static_cast<int>(min((long long)max(shared, 0), most)) / kTile * kTile;
                out.table_seq = first[g];
            }
            out.key_tiles = (out.tokens + p.tile_keys - 1) / p.tile_keys;
        }
        p.groups[g] = out;
        unit[g] = out.key_tiles * ((out.seqs + p.item_seqs - 1) / p.item_seqs) * p.num_kv_heads;
    }
    __syncthreads();
    exclusive_prefix(unit, p.num_groups);
    const int total = unit[p.num_groups], units_per_worker = max(1, (total + p.workers - 1) / p.workers);
    if (tid == 0) *p.head = PrefixPlanHead{total, units_per_worker, {0, 0}};
    for (int s = tid; s < p.num_seqs; s += blockDim.x) {
        PrefixSeqPlan sp{0, 0, 0, 0, 0, {0, 0, 0}};
        const int lo = group_of(s);
        if (lo >= 0) {
            const PrefixGroup g = p.groups[lo];
            const int item = (s - g.begin) / p.item_seqs;
            sp.first_tile = g.tokens / kTile;
            sp.key_tiles = g.key_tiles;
            sp.unit0 = unit[lo] + item * p.num_kv_heads * g.key_tiles;
            sp.item_first_seq = g.begin + item * p.item_seqs;
            sp.item_seqs = min(p.item_seqs, g.seqs - item * p.item_seqs);
        }
        p.seqs[s] = sp;
    }
    for (int w = tid; w < p.workers; w += blockDim.x) {
        PrefixSeed seed{0, 0, 0, 0};
        const long long u = (long long)w * units_per_worker;
        if (u < total) {
            int lo = 0, hi = p.num_groups - 1;   // the last group whose units begin at or before u
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (unit[mid] <= u) lo = mid; else hi = mid - 1;
            }
            const PrefixGroup g = p.groups[lo];
            const int r = static_cast<int>(u) - unit[lo], item = r / g.key_tiles;
            seed = PrefixSeed{lo, item / p.num_kv_heads, item % p.num_kv_heads, r - item * g.key_tiles};
        }
        p.seeds[w] = seed;
    }
}

struct SharedLayout {
    size_t head, groups, seeds, seqs, lse, rows_o, total;
};

SharedLayout shared_layout(size_t decode_bytes, int64_t num_seqs, int64_t num_groups, int64_t num_q_heads, int64_t head_dim,
                           int workers) {
    SharedLayout l;
    const size_t rows = (size_t)num_seqs * num_q_heads + (size_t)workers * kPrefixRows;
    l.head = align_up(decode_bytes, 256);
    l.groups = l.head + 256;
    l.seeds = align_up(l.groups + (size_t)num_groups * sizeof(PrefixGroup), 256);
    l.seqs = align_up(l.seeds + (size_t)workers * sizeof(PrefixSeed), 256);
    l.lse = align_up(l.seqs + (size_t)num_seqs * sizeof(PrefixSeqPlan), 256);
    l.rows_o = align_up(l.lse + rows * sizeof(float), 256);
    l.total = l.rows_o + rows * head_dim * sizeof(float);
    return l;
}

size_t tail_bytes(int64_t num_seqs, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int device) {
    LaunchShape ls = launch_shape(static_cast<int>(head_dim), 16, 0, 1 << 20, device);
    if (ls.nwarps < NPD_DECODE_MAX_WARPS) ls.nwarps = NPD_DECODE_MAX_WARPS;
    return plan_workspace(num_seqs, num_q_heads, num_kv_heads, head_dim, ls).total;
}

}  // namespace

extern "C" size_t npd_shared_prefix_workspace_bytes(int64_t num_seqs, int64_t num_groups, int64_t num_q_heads, int64_t num_kv_heads,
                                                    int64_t head_dim, int device) {
    if (num_seqs < 0 || num_groups < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
    return shared_layout(tail_bytes(num_seqs, num_q_heads, num_kv_heads, head_dim, device), num_seqs, num_groups, num_q_heads,
                         head_dim, npd::sm_count(device)).total;
}

extern "C" int npd_paged_shared_prefix_attention(void *out, const void *q, const void *k_cache, const void *v_cache,
                                                 const int32_t *block_tables, const int32_t *seq_lens,
                                                 const int32_t *group_offsets, const int32_t *shared_lens, float scale,
                                                 int64_t num_seqs, int64_t num_groups, int64_t num_q_heads,
                                                 int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                                 int64_t max_blocks_per_seq, int64_t num_blocks, int64_t cache_block_stride,
                                                 int64_t bt_row_stride, int dtype, void *workspace, size_t workspace_bytes,
                                                 int32_t *status, int flags, void *stream) {
    NPD_REQUIRE((flags & ~0xffff00) == 0, NPD_ERR_INVALID_ARG, "shared-prefix attention: only NPD_FLAG_MAX_CTAS is a flag here");
    const int rs = npd::check_score_shape("shared-prefix attention", scale, 0.f, nullptr, 0);
    if (rs != NPD_OK) return rs;
    NPD_REQUIRE(num_groups >= 1 && num_groups <= kMaxGroups, NPD_ERR_INVALID_ARG, "shared-prefix attention: between 1 and %d groups", kMaxGroups);
    DecodeCall c{out, q, k_cache, v_cache, block_tables, seq_lens, scale, num_seqs, num_q_heads, num_kv_heads, head_dim,
                 block_size, max_blocks_per_seq, num_blocks, cache_block_stride, bt_row_stride, dtype, workspace,
                 workspace_bytes, flags, stream};
    int rc = check_decode_call(c);
    if (rc != NPD_OK) return rc;
    if (num_seqs == 0) return NPD_OK;
    NPD_REQUIRE(group_offsets && shared_lens, NPD_ERR_INVALID_ARG, "shared-prefix attention: NULL pointer");
    const int64_t group = num_q_heads / num_kv_heads;
    NPD_REQUIRE(group <= 128, NPD_ERR_UNSUPPORTED, "shared-prefix attention: more than 128 q heads per kv head");
    int dev = 0;
    NPD_CUDA_TRY(cudaGetDevice(&dev));
    const size_t decode_bytes = tail_bytes(num_seqs, num_q_heads, num_kv_heads, head_dim, dev);
    const int sms = npd::sm_count(dev), cap = (flags >> 8) & 0xffff;
    const SharedLayout l = shared_layout(decode_bytes, num_seqs, num_groups, num_q_heads, head_dim, sms);
    NPD_REQUIRE(workspace != nullptr && workspace_bytes >= l.total, NPD_ERR_WORKSPACE,
                "shared-prefix attention: workspace of %zu bytes given, %zu needed", workspace_bytes, l.total);
    const int query_tiles = head_dim == 256 ? 1 : 2, tile_keys = head_dim == 256 ? 64 : 128;
    const int64_t max_tiles = (max_blocks_per_seq * block_size + tile_keys - 1) / tile_keys;
    NPD_REQUIRE(num_seqs * num_kv_heads * max_tiles < INT32_MAX, NPD_ERR_INVALID_ARG,
                "shared-prefix attention: batch times context exceeds int32");
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    if (status == nullptr) status = reinterpret_cast<int32_t *>(ws);
    {
        // A small batch whose sequences fit a cluster of CTAs each is answered by that one launch: reading the shared pages
        // again (they are in L2) costs less than three launches.  Measured at 2 to 74 sequences behind 512 to 16000 shared
        // tokens, 100 of their own, 12/2, 32/8 and 16/16 heads and 16/2 of 256: one launch / sharing 7 / 22 us for 16
        // sequences (12/2) behind 512 tokens, 8.8 / 24 behind 992, 18 / 25 for 18 sequences (32/8) behind 2000, 35 / 62 for
        // 37 (16/2 of 256) behind 2000; the one point of 89 where sharing won was 2 sequences (32/8) behind 16000, 36 / 32.
        const npd::SharedCall sc{out, q, k_cache, v_cache, block_tables, seq_lens, group_offsets, shared_lens, scale, num_seqs, num_groups,
                                 num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, num_blocks, cache_block_stride,
                                 bt_row_stride, dtype, workspace, decode_bytes, status, flags, stream};
        bool taken = false;
        rc = npd::decode_unshared_if_small(sc, &taken);
        if (taken || rc != NPD_OK) return rc;
    }
    PlanParams pp;
    pp.group_offsets = group_offsets;
    pp.shared_lens = shared_lens;
    pp.seq_lens = seq_lens;
    pp.status = status;
    pp.head = reinterpret_cast<PrefixPlanHead *>(ws + l.head);
    pp.groups = reinterpret_cast<PrefixGroup *>(ws + l.groups);
    pp.seeds = reinterpret_cast<PrefixSeed *>(ws + l.seeds);
    pp.seqs = reinterpret_cast<PrefixSeqPlan *>(ws + l.seqs);
    pp.cap = max_blocks_per_seq * block_size;
    pp.num_groups = static_cast<int>(num_groups);
    pp.num_seqs = static_cast<int>(num_seqs);
    pp.num_kv_heads = static_cast<int>(num_kv_heads);
    pp.item_seqs = query_tiles * (128 / static_cast<int>(group));
    pp.tile_keys = tile_keys;
    pp.workers = cap > 0 && cap < sms ? cap : sms;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    constexpr size_t plan_most = (size_t)(4 * kMaxGroups + 2) * sizeof(int);
    static std::atomic<unsigned long long> plan_done{0};
    if (npd::first_on_device(plan_done, dev)) {
        NPD_CUDA_TRY(cudaFuncSetAttribute(shared_prefix_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)plan_most));
        npd::set_up_on_device(plan_done, dev);
    }
    // a barrier of 1024 threads costs more than what a batch of a few hundred sequences gives them to do
    const int plan_threads = num_seqs <= 512 && num_groups <= 512 ? 256 : kPlanThreads;
    shared_prefix_plan_kernel<<<1, plan_threads, (size_t)(4 * num_groups + 2) * sizeof(int), st>>>(pp);
    NPD_CUDA_TRY(cudaGetLastError());
    npd::PrefixPass pass{q, k_cache, v_cache, block_tables, scale, num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
                         max_blocks_per_seq, num_blocks, cache_block_stride, bt_row_stride, dtype, status, pp.groups, pp.seeds,
                         pp.head, reinterpret_cast<float *>(ws + l.rows_o), reinterpret_cast<float *>(ws + l.lse), pp.workers, stream};
    rc = npd::launch_prefix_pass(pass);
    if (rc != NPD_OK) return rc;
    c.workspace_bytes = decode_bytes;
    c.status = status;
    c.seq_plan = pp.seqs;
    c.plan_head = pp.head;
    c.prefix_o = pass.prefix_o;
    c.prefix_lse = pass.prefix_lse;
    return run_decode<kTail>(c);
}

// Entry points of paged decode attention; the kernel and its design notes are in decode_kernel.cuh.
#include "decode_kernel.cuh"

extern "C" size_t npd_decode_workspace_bytes(int64_t num_seqs, int64_t num_q_heads, int64_t num_kv_heads,
                                             int64_t head_dim, int device) {
    if (num_seqs < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
    // Sized for the largest grid/warp shape the launcher may pick, so tuning knobs never outgrow it.
    LaunchShape ls = launch_shape(static_cast<int>(head_dim), 16, 0, 1 << 20, device);
    if (ls.nwarps < NPD_DECODE_MAX_WARPS) ls.nwarps = NPD_DECODE_MAX_WARPS;
    return plan_workspace(num_seqs, num_q_heads, num_kv_heads, head_dim, ls).total;
}

extern "C" int npd_paged_decode_attention(void *out, const void *q, const void *k_cache, const void *v_cache,
                                          const int32_t *block_tables, const int32_t *seq_lens, float scale,
                                          int64_t num_seqs, int64_t num_q_heads, int64_t num_kv_heads,
                                          int64_t head_dim, int64_t block_size, int64_t max_blocks_per_seq,
                                          int64_t num_blocks, int64_t cache_block_stride, int64_t bt_row_stride,
                                          int dtype, void *workspace, size_t workspace_bytes, int flags,
                                          void *stream) {
    DecodeCall c{out, q, k_cache, v_cache, block_tables, seq_lens, scale, num_seqs, num_q_heads, num_kv_heads, head_dim,
                 block_size, max_blocks_per_seq, num_blocks, cache_block_stride, bt_row_stride, dtype, workspace,
                 workspace_bytes, flags, stream};
    const int rc = check_decode_call(c);
    return rc != NPD_OK || num_seqs == 0 ? rc : run_decode<kPlain>(c);
}

// ---------------------------------------------------------------------------
// Decode attention for callers that must not allocate device memory
// ---------------------------------------------------------------------------
// Some hosts of this library cannot hand it a workspace: a decode worker that gave all free
// HBM to the KV block pool and the weights at start-up, a step loop with a "no allocation
// after initialisation" rule, or a foreign-language runtime binding the C ABI without a device
// allocator of its own (and cudaMalloc / cudaFree would stall every stream of the device
// anyway).  For them the scratch below is part of the library image: every GPU that loads the
// library holds these 32 MiB until the process exits.  It is large enough for every supported
// shape on a B200 (148 SMs x 12 workers x 2 partial records of at most 8320 B, plus the ticket region and header).
#define NPD_STATIC_SCRATCH_BYTES (32u << 20)
static __device__ __align__(256) unsigned char g_decode_static_scratch[NPD_STATIC_SCRATCH_BYTES];

namespace {

// In host code `g_decode_static_scratch` is only a stand-in for the device array; the device
// address has to be asked for, once per device, with that device current.
int static_scratch_address(void **ptr_out) {
    static std::atomic<void *> resolved[64];
    int dev = -1;
    NPD_CUDA_TRY(cudaGetDevice(&dev));
    NPD_REQUIRE(dev >= 0 && dev < 64, NPD_ERR_UNSUPPORTED, "static scratch: device index %d out of range", dev);
    void *ptr = resolved[dev].load(std::memory_order_acquire);
    if (ptr == nullptr) {
        NPD_CUDA_TRY(cudaGetSymbolAddress(&ptr, g_decode_static_scratch));
        NPD_REQUIRE(ptr != nullptr, NPD_ERR_CUDA, "static scratch: cudaGetSymbolAddress returned NULL");
        resolved[dev].store(ptr, std::memory_order_release);
    }
    *ptr_out = ptr;
    return NPD_OK;
}

}  // namespace

extern "C" size_t npd_decode_static_scratch_bytes(void) { return NPD_STATIC_SCRATCH_BYTES; }

extern "C" int npd_paged_decode_attention_static(void *out, const void *q, const void *k_cache,
                                                 const void *v_cache, const int32_t *block_tables,
                                                 const int32_t *seq_lens, float scale, int64_t num_seqs,
                                                 int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                                 int64_t block_size, int64_t max_blocks_per_seq,
                                                 int64_t num_blocks, int64_t cache_block_stride,
                                                 int64_t bt_row_stride, int dtype, int32_t *status_out,
                                                 int flags, void *stream) {
    int dev = 0;
    NPD_CUDA_TRY(cudaGetDevice(&dev));
    const size_t need = npd_decode_workspace_bytes(num_seqs, num_q_heads, num_kv_heads, head_dim, dev);
    NPD_REQUIRE(need != 0, NPD_ERR_INVALID_ARG, "decode attention (static scratch): non-positive dimension");
    NPD_REQUIRE(need <= NPD_STATIC_SCRATCH_BYTES, NPD_ERR_WORKSPACE,
                "decode attention (static scratch): this shape needs %zu bytes of scratch, the built-in array "
                "holds %u; use npd_paged_decode_attention with a caller-owned workspace",
                need, (unsigned)NPD_STATIC_SCRATCH_BYTES);
    void *scratch = nullptr;
    const int rc_addr = static_scratch_address(&scratch);   // first call on a device: resolves the symbol
    if (rc_addr != NPD_OK) return rc_addr;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // The array keeps whatever the previous call left.  The status word must start at zero, and so must the
    // arrival tickets: the kernel leaves them at zero itself, except when an earlier launch gave up on a bounded
    // wait — and this caller has no pointer to clean up with.  The partial records are written before they are read.
    // Only the tickets one launch can touch are cleared: one per (sequence of a sub-batch, virtual kv head).
    const LaunchShape ls = launch_shape(static_cast<int>(head_dim), static_cast<int>(block_size), (flags >> 8) & 0xffff,
                                        (long long)num_seqs * num_kv_heads, dev);
    const WorkspacePlan wp = plan_workspace(num_seqs, num_q_heads, num_kv_heads, head_dim, ls);
    const int64_t vheads = num_kv_heads * wp.kv_rep;
    int64_t batch_cap = vheads > 0 ? kTicketCapacity / vheads : 0;
    if (batch_cap > kMaxSeqsPerLaunch) batch_cap = kMaxSeqsPerLaunch;
    const int64_t tickets = (num_seqs < batch_cap ? num_seqs : batch_cap) * vheads;
    NPD_CUDA_TRY(cudaMemsetAsync(scratch, 0, kStatusBytes + (size_t)tickets * sizeof(int32_t), st));
    const int rc = npd_paged_decode_attention(out, q, k_cache, v_cache, block_tables, seq_lens, scale, num_seqs,
                                              num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq,
                                              num_blocks, cache_block_stride, bt_row_stride, dtype, scratch,
                                              NPD_STATIC_SCRATCH_BYTES, flags, st);
    if (rc != NPD_OK) return rc;
    if (status_out != nullptr)
        NPD_CUDA_TRY(cudaMemcpyAsync(status_out, scratch, sizeof(int32_t), cudaMemcpyDeviceToDevice, st));
    return NPD_OK;
}

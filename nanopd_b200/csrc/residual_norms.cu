// What stands between two blocks of a decoder layer, in one pass over the rows:
//   y = x                                  the block's output
//   y = y * rsqrt(mean(y^2) + eps) * (post_weight + offset)     if there is a norm behind the block
//   y = gate * y                           if there is a gate: one value per channel, or one per token and channel
//   r = residual + residual_scale * y      -> residual_out
//   h = r * rsqrt(mean(r^2) + eps) * (weight + offset)          -> out, the next block's input
// All of it in 32 bits from the loads to the two stores, each rounded once; the second norm reads the unrounded sum.
//
// HBM-bound: x, residual and a per-token gate are read once, two rows are written.  The two means are warp shuffles and,
// across the warps of a row, one exchange through shared memory each.  8191 rows of 4096 bf16 values with both norms: 46.8 us,
// 5.7 TB/s.  What it took from a plain kernel's 67 us: rows fetched ahead into shared memory (51), packed fp32 pairs and
// pointers that are stepped instead of computed (47; the first form spent 44 instructions for 32 values, as many cycles as
// the bytes need); fewer registers for more CTAs cost more in spills than they gave (52-57).
#include "npd_common.cuh"

namespace {

struct NormParams {
    void *residual_out, *out;
    const void *x, *residual, *weight, *post_weight, *gate;
    float residual_scale, eps, offset, inv_hidden;
    long long num_rows;
    int vecs;                  // 8-element vectors per row
    int warps_per_row;         // one row: 32 * warps_per_row threads
    long long x_stride, residual_stride, gate_stride, residual_out_stride, out_stride;   // in elements; gate 0 = per channel
};

// Eight values of T as they are stored, and as four pairs of floats (the arithmetic is in packed pairs: half the
// instructions, and instructions are what a row of 16-bit values costs beside its bytes).
template <typename T> struct Vec8;
template <> struct Vec8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const void *p) {
        a = reinterpret_cast<const float4 *>(p)[0];
        b = reinterpret_cast<const float4 *>(p)[1];
    }
    __device__ __forceinline__ void unpack(float2 (&f)[4]) const {
        f[0] = make_float2(a.x, a.y), f[1] = make_float2(a.z, a.w), f[2] = make_float2(b.x, b.y), f[3] = make_float2(b.z, b.w);
    }
    __device__ __forceinline__ void pack(const float2 (&f)[4]) {
        a = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
        b = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
    }
    __device__ __forceinline__ void store(void *p) const {
        reinterpret_cast<float4 *>(p)[0] = a;
        reinterpret_cast<float4 *>(p)[1] = b;
    }
};
struct Vec8Half {
    uint4 v;
    __device__ __forceinline__ void load(const void *p) { v = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void store(void *p) const { *reinterpret_cast<uint4 *>(p) = v; }
};
template <> struct Vec8<__half> : Vec8Half {
    __device__ __forceinline__ void unpack(float2 (&f)[4]) const {
        const __half2 *h = reinterpret_cast<const __half2 *>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __half22float2(h[i]);
    }
    __device__ __forceinline__ void pack(const float2 (&f)[4]) {
        __half2 *h = reinterpret_cast<__half2 *>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __float22half2_rn(f[i]);
    }
};
template <> struct Vec8<__nv_bfloat16> : Vec8Half {
    __device__ __forceinline__ void unpack(float2 (&f)[4]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
    __device__ __forceinline__ void pack(const float2 (&f)[4]) {
        __nv_bfloat162 *h = reinterpret_cast<__nv_bfloat162 *>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __float22bfloat162_rn(f[i]);
    }
};

constexpr int kMaxThreads = 512;
// Threads of a row: one vector each up to 256, then two (more rows in flight on an SM beat more threads to a row), then as
// many as 512 threads need.
constexpr int kOneVecThreads = 256;

// Sum over the warps of one row; every thread of the CTA takes part.  `buf`: one float per warp of the CTA.
__device__ __forceinline__ float row_sum(float v, int warps_per_row, float *buf) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if (warps_per_row == 1) return v;
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) buf[warp] = v;
    __syncthreads();
    if (warps_per_row >= 4) {            // the CTA holds this row alone; what is behind its warps is zero
        const float4 *b4 = reinterpret_cast<const float4 *>(buf);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < kMaxThreads / 128; ++i) {
            if (i * 4 >= warps_per_row) break;
            const float4 q = b4[i];
            s += (q.x + q.y) + (q.z + q.w);
        }
        return s;
    }
    float s = 0.f;
    const int first = warp / warps_per_row * warps_per_row;
    for (int i = 0; i < warps_per_row; ++i) s += buf[first + i];      // the same order in every thread
    return s;
}
__device__ __forceinline__ float sum_of_squares(float ss, const float2 (&f)[4]) {
    float2 a = __fmul2_rn(f[0], f[0]), b = __fmul2_rn(f[1], f[1]);
    a = __ffma2_rn(f[2], f[2], a);
    b = __ffma2_rn(f[3], f[3], b);
    a = __fadd2_rn(a, b);
    return ss + (a.x + a.y);
}

__device__ __forceinline__ void copy16_async(uint32_t smem, const void *global) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(global) : "memory");
}

// A CTA takes every gridDim-th set of rows.  kStaged: a thread copies its pieces of the next rows (x, residual, a per-token
// gate) into a ring in shared memory with asynchronous copies, kStages rows ahead, and reads them back itself, so the ring
// needs no barrier; registers would have to hold what is under way otherwise.  Rows too long for that are read where they
// are.  The sum r is held in fp32 between its mean and the outputs; the weights stay in registers up to kHeld vectors a
// thread.
constexpr int kHeld = 2;
constexpr int kStages = 3;

template <typename T, int kVecs, bool kStaged>
__global__ void __maxnreg__(kVecs <= kHeld ? 96 : 128) residual_norms_kernel(const NormParams p) {
    extern __shared__ __align__(16) uint8_t ring[];
    // two buffers per sum: a fast warp may be a row ahead of a slow one that still reads
    __shared__ __align__(16) float sums[2][2][kMaxThreads / 32];
    constexpr bool kHold = kVecs <= kHeld;
    constexpr int kPiece = 8 * sizeof(T);
    const int row_threads = p.warps_per_row * 32, rows_per_cta = blockDim.x / row_threads;
    const int sub = rows_per_cta == 1 ? 0 : threadIdx.x / row_threads, t = threadIdx.x - sub * row_threads;
    const bool post = p.post_weight != nullptr, gated = p.gate != nullptr, gate_per_row = gated && p.gate_stride != 0;
    const long long step = (long long)gridDim.x * rows_per_cta;
    const int vec_bytes = row_threads * kPiece;                      // from one vector of a thread to its next
    const int off = t * kPiece;
    if (threadIdx.x < 4 * kMaxThreads / 32) (&sums[0][0][0])[threadIdx.x] = 0.f;
    __syncthreads();

    bool in[kVecs];                                                  // vectors of this thread that lie in the row
#pragma unroll
    for (int i = 0; i < kVecs; ++i) in[i] = t + i * row_threads < p.vecs;

    // ring: [stage][x, residual, gate][thread piece]; a thread's pieces are a CTA's width apart, consecutive lanes side by side
    const uint32_t slab = blockDim.x * kVecs * kPiece;               // bytes of one operand of one stage
    const uint32_t stage_bytes = slab * (gate_per_row ? 3 : 2);
    const uint32_t my_slot = threadIdx.x * kPiece, piece_step = blockDim.x * kPiece;
    const uint32_t ring_addr = npd::smem_u32(ring);

    // this thread's place in the row that is fetched next, and in the outputs' row
    long long fetch_row = (long long)blockIdx.x * rows_per_cta + sub, row = fetch_row;
    const uint8_t *fx = static_cast<const uint8_t *>(p.x) + fetch_row * p.x_stride * (long long)sizeof(T) + off;
    const uint8_t *fr = static_cast<const uint8_t *>(p.residual) + fetch_row * p.residual_stride * (long long)sizeof(T) + off;
    const uint8_t *fg = static_cast<const uint8_t *>(p.gate) + (gate_per_row ? fetch_row * p.gate_stride * (long long)sizeof(T) : 0) + off;
    uint8_t *out_r = static_cast<uint8_t *>(p.residual_out) + row * p.residual_out_stride * (long long)sizeof(T) + off;
    uint8_t *out_h = static_cast<uint8_t *>(p.out) + row * p.out_stride * (long long)sizeof(T) + off;
    const long long step_x = step * p.x_stride * (long long)sizeof(T), step_r = step * p.residual_stride * (long long)sizeof(T);
    const long long step_g = gate_per_row ? step * p.gate_stride * (long long)sizeof(T) : 0;
    const long long step_or = step * p.residual_out_stride * (long long)sizeof(T), step_oh = step * p.out_stride * (long long)sizeof(T);
    auto fetch = [&](uint32_t at) {
        if (fetch_row < p.num_rows) {
            const uint32_t dst = ring_addr + at + my_slot;
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                if (!in[i]) continue;
#pragma unroll
                for (int b = 0; b < kPiece; b += 16) {
                    copy16_async(dst + i * piece_step + b, fx + i * vec_bytes + b);
                    copy16_async(dst + slab + i * piece_step + b, fr + i * vec_bytes + b);
                    if (gate_per_row) copy16_async(dst + 2 * slab + i * piece_step + b, fg + i * vec_bytes + b);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");         // a group per row, rows past the end included
        fetch_row += step;
        fx += step_x;
        fr += step_r;
        fg += step_g;
    };
    if (kStaged) {
#pragma unroll
        for (int k = 0; k < kStages; ++k) fetch(k * stage_bytes);
    }
    Vec8<T> wv[kHold ? kVecs : 1], pv[kHold ? kVecs : 1], gv[kHold ? kVecs : 1];
    if (kHold) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            if (!in[i]) continue;
            wv[i].load(static_cast<const uint8_t *>(p.weight) + off + i * vec_bytes);
            if (post) pv[i].load(static_cast<const uint8_t *>(p.post_weight) + off + i * vec_bytes);
            if (gated && !gate_per_row) gv[i].load(static_cast<const uint8_t *>(p.gate) + off + i * vec_bytes);
        }
    }
    const float2 offset2 = make_float2(p.offset, p.offset);
    uint32_t stage = 0;                                              // byte offset of the ring stage
    int turn = 0;
    // all rows of a set take part in its barriers: the set goes on while its first row is there
    for (long long row0 = (long long)blockIdx.x * rows_per_cta; row0 < p.num_rows; row0 += step, turn ^= 1) {
        const bool live = rows_per_cta == 1 || row < p.num_rows;
        if (kStaged) asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");      // this thread's pieces have landed
        const uint8_t *slot = ring + stage + my_slot;
        // plain loads where nothing is staged: the outputs may be the same rows
        auto x_at = [&](int i) {
            Vec8<T> a;
            a.load(kStaged ? slot + i * piece_step : fx + i * vec_bytes);
            return a;
        };
        float ss = 0.f, inv = p.residual_scale;
        if (post) {
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                if (!live || !in[i]) continue;
                float2 y[4];
                x_at(i).unpack(y);
                ss = sum_of_squares(ss, y);
            }
            inv *= rsqrtf(row_sum(ss, p.warps_per_row, sums[turn][0]) * p.inv_hidden + p.eps);
        }
        const float2 inv2 = make_float2(inv, inv);
        float2 r[kVecs][4];
        ss = 0.f;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            if (!live || !in[i]) continue;
            float2 y[4], w[4];
            x_at(i).unpack(y);
            Vec8<T> a;
            a.load(kStaged ? slot + slab + i * piece_step : fr + i * vec_bytes);
            a.unpack(r[i]);
            if (post) {
                if (kHold) a = pv[i];
                else a.load(static_cast<const uint8_t *>(p.post_weight) + off + i * vec_bytes);
                a.unpack(w);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = __fmul2_rn(y[e], __fadd2_rn(w[e], offset2));
            }
            if (gated) {
                if (gate_per_row) a.load(kStaged ? slot + 2 * slab + i * piece_step : fg + i * vec_bytes);
                else if (kHold) a = gv[i];
                else a.load(static_cast<const uint8_t *>(p.gate) + off + i * vec_bytes);
                a.unpack(w);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = __fmul2_rn(y[e], w[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) r[i][e] = __ffma2_rn(y[e], inv2, r[i][e]);
            ss = sum_of_squares(ss, r[i]);
            a.pack(r[i]);
            a.store(out_r + i * vec_bytes);
        }
        if (kStaged) {                                               // the slot is read: the row that comes kStages sets later
            fetch(stage);
            stage = stage + stage_bytes == kStages * stage_bytes ? 0 : stage + stage_bytes;
        } else {
            fx += step_x;
            fr += step_r;
            fg += step_g;
        }
        const float inv_r = rsqrtf(row_sum(ss, p.warps_per_row, sums[turn][1]) * p.inv_hidden + p.eps);
        const float2 inv_r2 = make_float2(inv_r, inv_r);
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            if (!live || !in[i]) continue;
            float2 w[4];
            Vec8<T> a;
            if (kHold) a = wv[i];
            else a.load(static_cast<const uint8_t *>(p.weight) + off + i * vec_bytes);
            a.unpack(w);
#pragma unroll
            for (int e = 0; e < 4; ++e) r[i][e] = __fmul2_rn(__fmul2_rn(r[i][e], inv_r2), __fadd2_rn(w[e], offset2));
            a.pack(r[i]);
            a.store(out_h + i * vec_bytes);
        }
        row += step;
        out_r += step_or;
        out_h += step_oh;
    }
    if (kStaged) asm volatile("cp.async.wait_group 0;" ::: "memory");
}

constexpr int kMaxRing = 96 * 1024;       // two CTAs to an SM at least

template <typename T, int kVecs, bool kStaged>
int launch_kernel(const NormParams &p, int rows_per_cta, size_t smem, int device, cudaStream_t stream) {
    auto kern = residual_norms_kernel<T, kVecs, kStaged>;
    const int threads = rows_per_cta * p.warps_per_row * 32;
    static std::atomic<unsigned long long> done{0};
    if (npd::first_on_device(done, device)) {
        NPD_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxRing));
        NPD_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
        npd::set_up_on_device(done, device);
    }
    // resident CTAs: by the register limit of the kernel's declaration and by the ring (the rest follows from these two)
    const int by_registers = 65536 / ((kVecs <= kHeld ? 96 : 128) * threads), by_ring = static_cast<int>((size_t)npd::kMaxDynamicSmem / (smem + 1280));
    const int per_sm = by_registers < by_ring ? by_registers : by_ring;
    const long long sets = (p.num_rows + rows_per_cta - 1) / rows_per_cta;
    const long long most = (long long)npd::sm_count(device) * (per_sm > 0 ? per_sm : 1);
    kern<<<static_cast<unsigned>(sets < most ? sets : most), threads, smem, stream>>>(p);
    NPD_CUDA_TRY(cudaGetLastError());
    return NPD_OK;
}

template <typename T, int kVecs>
int launch_vecs(const NormParams &p, int rows_per_cta, int device, cudaStream_t stream) {
    const int operands = p.gate != nullptr && p.gate_stride != 0 ? 3 : 2;
    const size_t ring = (size_t)kStages * operands * rows_per_cta * p.warps_per_row * 32 * kVecs * 8 * sizeof(T);
    if (ring <= kMaxRing) return launch_kernel<T, kVecs, true>(p, rows_per_cta, ring, device, stream);
    return launch_kernel<T, kVecs, false>(p, rows_per_cta, 0, device, stream);
}

template <typename T>
int launch(NormParams &p, cudaStream_t stream) {
    int vecs_per_thread = 1;
    while (vecs_per_thread < 8 && (p.vecs + vecs_per_thread - 1) / vecs_per_thread > (vecs_per_thread < 2 ? kOneVecThreads : kMaxThreads)) vecs_per_thread *= 2;
    p.warps_per_row = ((p.vecs + vecs_per_thread - 1) / vecs_per_thread + 31) / 32;
    const int rows_per_cta = p.warps_per_row >= 4 ? 1 : 4 / p.warps_per_row;
    int dev = 0;
    NPD_CUDA_TRY(cudaGetDevice(&dev));
    if (vecs_per_thread == 1) return launch_vecs<T, 1>(p, rows_per_cta, dev, stream);
    if (vecs_per_thread == 2) return launch_vecs<T, 2>(p, rows_per_cta, dev, stream);
    if (vecs_per_thread == 4) return launch_vecs<T, 4>(p, rows_per_cta, dev, stream);
    return launch_vecs<T, 8>(p, rows_per_cta, dev, stream);
}

}  // namespace

extern "C" int npd_residual_norms(void *residual_out, void *out, const void *x, const void *residual, const void *weight,
                                  const void *post_weight, const void *gate, float residual_scale, float eps,
                                  float weight_offset, int64_t num_rows, int64_t hidden, int64_t x_row_stride,
                                  int64_t residual_row_stride, int64_t gate_row_stride, int64_t residual_out_row_stride,
                                  int64_t out_row_stride, int dtype, void *stream) {
    NPD_REQUIRE(dtype == NPD_DTYPE_F16 || dtype == NPD_DTYPE_BF16 || dtype == NPD_DTYPE_F32, NPD_ERR_UNSUPPORTED,
                "npd_residual_norms: unsupported dtype code %d", dtype);
    NPD_REQUIRE(num_rows >= 0 && hidden > 0, NPD_ERR_INVALID_ARG, "npd_residual_norms: non-positive dimension");
    NPD_REQUIRE(hidden % 8 == 0 && hidden <= NPD_NORMS_MAX_HIDDEN, NPD_ERR_UNSUPPORTED,
                "npd_residual_norms: hidden size %lld is not a multiple of 8 up to %d", (long long)hidden, NPD_NORMS_MAX_HIDDEN);
    NPD_REQUIRE(num_rows <= INT32_MAX, NPD_ERR_INVALID_ARG, "npd_residual_norms: more than 2^31 - 1 rows in one call");
    if (num_rows == 0) return NPD_OK;
    NPD_REQUIRE(residual_out && out && x && residual && weight, NPD_ERR_INVALID_ARG, "npd_residual_norms: NULL pointer");
    NPD_REQUIRE(npd::aligned16(residual_out) && npd::aligned16(out) && npd::aligned16(x) && npd::aligned16(residual) &&
                    npd::aligned16(weight) && npd::aligned16(post_weight) && npd::aligned16(gate),
                NPD_ERR_INVALID_ARG, "npd_residual_norms: pointers must be 16-byte aligned");
    const int64_t unit = dtype == NPD_DTYPE_F32 ? 4 : 8;
    for (const int64_t stride : {x_row_stride, residual_row_stride, residual_out_row_stride, out_row_stride})
        NPD_REQUIRE(stride % unit == 0 && stride >= hidden, NPD_ERR_INVALID_ARG,
                    "npd_residual_norms: row strides must be multiples of 16 bytes and at least a row");
    NPD_REQUIRE(gate == nullptr || gate_row_stride == 0 || (gate_row_stride % unit == 0 && gate_row_stride >= hidden),
                NPD_ERR_INVALID_ARG, "npd_residual_norms: the gate's row stride must be 0 or a multiple of 16 bytes of at least a row");
    NormParams p{residual_out, out, x, residual, weight, post_weight, gate, residual_scale, eps, weight_offset,
                 1.f / static_cast<float>(hidden), num_rows, static_cast<int>(hidden / 8), 1, x_row_stride, residual_row_stride,
                 gate ? gate_row_stride : 0, residual_out_row_stride, out_row_stride};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == NPD_DTYPE_F32) return launch<float>(p, st);
    return dtype == NPD_DTYPE_BF16 ? launch<__nv_bfloat16>(p, st) : launch<__half>(p, st);
}

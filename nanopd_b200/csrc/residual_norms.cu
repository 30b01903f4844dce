// What stands between two blocks of a decoder layer, in one pass over the rows:
//   y = x                                  the block's output
//   y = y * rsqrt(mean(y^2) + eps) * (post_weight + offset)     if there is a norm behind the block
//   y = gate * y                           if there is a gate: one value per channel, or one per token and channel
//   r = residual + residual_scale * y      -> residual_out
//   h = r * rsqrt(mean(r^2) + eps) * (weight + offset)          -> out, the next block's input
// All of it in 32 bits from the loads to the two stores, each rounded once; the second norm reads the unrounded sum.
//
// HBM-bound: x, residual and a per-token gate are read once, two rows are written; a row lives in registers between its
// loads and its stores.  A row belongs to kWarps warps, eight elements to a thread and vector, kVecs vectors to a thread;
// the two means are warp shuffles and, across warps, one exchange through shared memory each.
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

template <typename T> struct Vec8;
template <> struct Vec8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const void *p) {
        a = reinterpret_cast<const float4 *>(p)[0];
        b = reinterpret_cast<const float4 *>(p)[1];
    }
    __device__ __forceinline__ void unpack(float (&f)[8]) const {
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    }
    __device__ __forceinline__ void pack(const float (&f)[8]) {
        a = make_float4(f[0], f[1], f[2], f[3]);
        b = make_float4(f[4], f[5], f[6], f[7]);
    }
    __device__ __forceinline__ void store(void *p) const {
        reinterpret_cast<float4 *>(p)[0] = a;
        reinterpret_cast<float4 *>(p)[1] = b;
    }
};
template <typename T, typename T2>
struct Vec8Half {
    uint4 v;
    __device__ __forceinline__ void load(const void *p) { v = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void store(void *p) const { *reinterpret_cast<uint4 *>(p) = v; }
};
template <> struct Vec8<__half> : Vec8Half<__half, __half2> {
    __device__ __forceinline__ void unpack(float (&f)[8]) const {
        const __half2 *h = reinterpret_cast<const __half2 *>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = __half22float2(h[i]);
            f[2 * i] = t.x, f[2 * i + 1] = t.y;
        }
    }
    __device__ __forceinline__ void pack(const float (&f)[8]) {
        __half2 *h = reinterpret_cast<__half2 *>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    }
};
template <> struct Vec8<__nv_bfloat16> : Vec8Half<__nv_bfloat16, __nv_bfloat162> {
    __device__ __forceinline__ void unpack(float (&f)[8]) const {
        const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = __bfloat1622float2(h[i]);
            f[2 * i] = t.x, f[2 * i + 1] = t.y;
        }
    }
    __device__ __forceinline__ void pack(const float (&f)[8]) {
        __nv_bfloat162 *h = reinterpret_cast<__nv_bfloat162 *>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    }
};

constexpr int kMaxThreads = 512;

// Sum over the warps of one row; every thread of the CTA takes part.  `buf`: one float per warp of the CTA.
__device__ __forceinline__ float row_sum(float v, int warps_per_row, float *buf) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if (warps_per_row == 1) return v;
    const int warp = threadIdx.x >> 5, first = warp / warps_per_row * warps_per_row;
    if ((threadIdx.x & 31) == 0) buf[warp] = v;
    __syncthreads();
    float s = 0.f;
    for (int i = 0; i < warps_per_row; ++i) s += buf[first + i];      // the same order in every thread
    return s;
}

// A CTA takes every gridDim-th set of rows; the loads of its next set are issued before it works on this one, and the
// weights stay in registers (16 bits each).
template <typename T, int kVecs>
__global__ void __launch_bounds__(kMaxThreads) residual_norms_kernel(const NormParams p) {
    // two buffers per sum: a fast warp may be a row ahead of a slow one that still reads
    __shared__ float sums[2][2][kMaxThreads / 32];
    const int row_threads = p.warps_per_row * 32, rows_per_cta = blockDim.x / row_threads;
    const int sub = threadIdx.x / row_threads, t = threadIdx.x - sub * row_threads;
    const bool post = p.post_weight != nullptr, gated = p.gate != nullptr, gate_per_row = gated && p.gate_stride != 0;

    Vec8<T> wv[kVecs], pv[kVecs], gv[kVecs], xv[kVecs], rv[kVecs];
    auto load_rows = [&](long long row) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int v = t + i * row_threads;
            if (row >= p.num_rows || v >= p.vecs) continue;
            // plain loads: the outputs may be the same rows
            xv[i].load(static_cast<const T *>(p.x) + row * p.x_stride + v * 8);
            rv[i].load(static_cast<const T *>(p.residual) + row * p.residual_stride + v * 8);
            if (gate_per_row) gv[i].load(static_cast<const T *>(p.gate) + row * p.gate_stride + v * 8);
        }
    };
    long long row = (long long)blockIdx.x * rows_per_cta + sub;
    load_rows(row);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int v = t + i * row_threads;
        if (v >= p.vecs) continue;
        wv[i].load(static_cast<const T *>(p.weight) + v * 8);
        if (post) pv[i].load(static_cast<const T *>(p.post_weight) + v * 8);
        if (gated && !gate_per_row) gv[i].load(static_cast<const T *>(p.gate) + v * 8);
    }
    int turn = 0;
    for (long long row0 = (long long)blockIdx.x * rows_per_cta; row0 < p.num_rows; row0 += (long long)gridDim.x * rows_per_cta) {
        const long long row = row0 + sub;
        float y[kVecs][8], r[kVecs][8];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            if (row >= p.num_rows || t + i * row_threads >= p.vecs) continue;
            xv[i].unpack(y[i]);
            rv[i].unpack(r[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += y[i][e] * y[i][e];
            if (gated) {
                float g[8];
                gv[i].unpack(g);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[i][e] *= g[e];
            }
        }
        load_rows(row + (long long)gridDim.x * rows_per_cta);
        float inv = p.residual_scale;
        if (post) inv *= rsqrtf(row_sum(ss, p.warps_per_row, sums[turn][0]) * p.inv_hidden + p.eps);
        ss = 0.f;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int v = t + i * row_threads;
            if (row >= p.num_rows || v >= p.vecs) continue;
            if (post) {
                float w[8];
                pv[i].unpack(w);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[i][e] *= w[e] + p.offset;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                r[i][e] += y[i][e] * inv;
                ss += r[i][e] * r[i][e];
            }
            Vec8<T> o;
            o.pack(r[i]);
            o.store(static_cast<T *>(p.residual_out) + row * p.residual_out_stride + v * 8);
        }
        const float inv_r = rsqrtf(row_sum(ss, p.warps_per_row, sums[turn][1]) * p.inv_hidden + p.eps);
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int v = t + i * row_threads;
            if (row >= p.num_rows || v >= p.vecs) continue;
            float w[8];
            wv[i].unpack(w);
#pragma unroll
            for (int e = 0; e < 8; ++e) r[i][e] *= inv_r * (w[e] + p.offset);
            Vec8<T> o;
            o.pack(r[i]);
            o.store(static_cast<T *>(p.out) + row * p.out_stride + v * 8);
        }
        turn ^= 1;
    }
}

template <typename T, int kVecs>
int launch_vecs(const NormParams &p, int rows_per_cta, int device, cudaStream_t stream) {
    const int threads = rows_per_cta * p.warps_per_row * 32;
    int per_sm = 1;
    NPD_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, residual_norms_kernel<T, kVecs>, threads, 0));
    const long long sets = (p.num_rows + rows_per_cta - 1) / rows_per_cta;
    const long long most = (long long)npd::sm_count(device) * (per_sm > 0 ? per_sm : 1);
    residual_norms_kernel<T, kVecs><<<static_cast<unsigned>(sets < most ? sets : most), threads, 0, stream>>>(p);
    NPD_CUDA_TRY(cudaGetLastError());
    return NPD_OK;
}

template <typename T>
int launch(NormParams &p, cudaStream_t stream) {
    int vecs_per_thread = 1;
    while (vecs_per_thread < 8 && (p.vecs + vecs_per_thread - 1) / vecs_per_thread > (vecs_per_thread < 2 ? 256 : kMaxThreads)) vecs_per_thread *= 2;
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

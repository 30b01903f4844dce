// One entry point for hosts to which every argument of a foreign call costs time: the operator's arguments come as an array
// of 8-byte slots, in the order of its own entry point, with the device in front.
#include "npd_common.cuh"

namespace {

// Makes `device` current for the call, and the caller's device again behind it.
struct DeviceScope {
    int before = -1;
    bool switched = false;
    int enter(int device) {
        NPD_CUDA_TRY(cudaGetDevice(&before));
        if (before != device) {
            NPD_CUDA_TRY(cudaSetDevice(device));
            switched = true;
        }
        return NPD_OK;
    }
    ~DeviceScope() {
        if (switched) (void)cudaSetDevice(before);
    }
};

template <typename T> T *ptr(const npd_slot &s) { return reinterpret_cast<T *>(static_cast<uintptr_t>(s.u)); }

}  // namespace

extern "C" int npd_call_packed(int op, const npd_slot *a) {
    NPD_REQUIRE(a != nullptr, NPD_ERR_INVALID_ARG, "npd_call_packed: NULL pointer");
    DeviceScope scope;
    const int rc = scope.enter(static_cast<int>(a[0].i));
    if (rc != NPD_OK) return rc;
    ++a;
    auto f = [&](int k) { return static_cast<float>(a[k].f); };
    auto n = [&](int k) { return a[k].i; };
    switch (op) {
        case NPD_OP_RESIDUAL_NORMS:
            return npd_residual_norms(ptr<void>(a[0]), ptr<void>(a[1]), ptr<const void>(a[2]), ptr<const void>(a[3]), ptr<const void>(a[4]),
                                      ptr<const void>(a[5]), ptr<const void>(a[6]), f(7), f(8), f(9), n(10), n(11), n(12), n(13), n(14), n(15),
                                      n(16), static_cast<int>(n(17)), ptr<void>(a[18]));
        case NPD_OP_SCORED_ATTENTION:
            return npd_paged_scored_attention(ptr<void>(a[0]), ptr<const void>(a[1]), ptr<const void>(a[2]), ptr<const void>(a[3]),
                                              ptr<const int32_t>(a[4]), ptr<const int32_t>(a[5]), f(6), f(7), ptr<const float>(a[8]), n(9), n(10),
                                              n(11), n(12), n(13), n(14), n(15), n(16), n(17), n(18), static_cast<int>(n(19)), ptr<void>(a[20]),
                                              static_cast<size_t>(n(21)), ptr<int32_t>(a[22]), static_cast<int>(n(23)), ptr<void>(a[24]));
        case NPD_OP_SCORED_PREFILL_ATTENTION:
            return npd_paged_scored_prefill_attention(ptr<void>(a[0]), ptr<const void>(a[1]), ptr<const void>(a[2]), ptr<const void>(a[3]),
                                                      ptr<const int32_t>(a[4]), ptr<const int32_t>(a[5]), ptr<const int32_t>(a[6]),
                                                      ptr<const int32_t>(a[7]), n(8), f(9), f(10), ptr<const float>(a[11]), n(12), n(13), n(14),
                                                      n(15), n(16), n(17), n(18), n(19), n(20), static_cast<int>(n(21)), ptr<void>(a[22]),
                                                      static_cast<size_t>(n(23)), ptr<int32_t>(a[24]), static_cast<int>(n(25)), ptr<void>(a[26]));
        case NPD_OP_SHARED_PREFIX_ATTENTION:
            return npd_paged_shared_prefix_attention(ptr<void>(a[0]), ptr<const void>(a[1]), ptr<const void>(a[2]), ptr<const void>(a[3]),
                                                     ptr<const int32_t>(a[4]), ptr<const int32_t>(a[5]), ptr<const int32_t>(a[6]),
                                                     ptr<const int32_t>(a[7]), f(8), n(9), n(10), n(11), n(12), n(13), n(14), n(15), n(16), n(17),
                                                     n(18), static_cast<int>(n(19)), ptr<void>(a[20]), static_cast<size_t>(n(21)),
                                                     ptr<int32_t>(a[22]), static_cast<int>(n(23)), ptr<void>(a[24]));
        default:
            return npd::fail(NPD_ERR_INVALID_ARG, "npd_call_packed: unknown operator %d", op);
    }
}

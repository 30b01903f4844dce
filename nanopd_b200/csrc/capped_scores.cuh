// Scores capped by a tanh, cap * tanh(scale * x / cap) of a raw score x = q . k, in the log2 domain.
//
// capped_near and capped_far keep the score's own relative accuracy (2e-7 and the two roundings of fp32 products), however large the cap is
// beside the score:
//   |z| < 0.6   tanh(z) = z (1 + w R(w)), z = scale x / cap, w = z^2; R of degree 3 fitted by Remez exchange for the least
//               relative error of the whole, 8.4e-8; exact as z goes to 0
//   elsewhere   tanh(z) = 1 - 2 / (1 + e^2z) with z > 0, the sign put back behind it: at z = 0.6 and beyond the difference has
//               lost no digits yet.  Near z = 0 this form has an absolute error of 2^-23 cap, which for a cap of 1e6 is a tenth;
//               where speed asks for one form it serves small caps alone (capped_low)
#pragma once
#include "npd_common.cuh"

namespace {

constexpr float kLowCap = 128.f;
struct ScoreCap {
    float in;         // 2 log2(e) * scale / cap; 0 = scores are not capped (or the scale is 0)
    float log2;       // cap * log2(e)
    float per;        // scale / cap
    float edge;       // |x| where z = 0.6; +inf where no finite x reaches it
    bool low;         // the cap is small enough for capped_low
};
inline ScoreCap make_score_cap(float scale, float cap) {
    if (cap <= 0.f || scale <= 0.f) return {0.f, 0.f, 0.f, INFINITY, true};
    // a quotient below fp32's normal numbers: any such number serves, w is 0 for every finite score
    const double per = (double)scale / cap < 1.2e-38 ? 1.2e-38 : (double)scale / cap;
    return {static_cast<float>(2.0 * 1.4426950408889634 * per), cap * 1.4426950408889634f, static_cast<float>(per),
            static_cast<float>(0.6 / per), cap <= kLowCap};
}

// A pair of raw scores with |x| < edge.
__device__ __forceinline__ float2 capped_near(float2 x, float scale_log2, const ScoreCap &cap) {
    constexpr float kR[4] = {-0.3333259750883f, 0.1331311667739f, -0.05221180760144f, 0.01561263411914f};
    const float2 z = __fmul2_rn(x, make_float2(cap.per, cap.per)), w = __fmul2_rn(z, z);
    float2 r = make_float2(kR[3], kR[3]);
#pragma unroll
    for (int k = 2; k >= 0; --k) r = __ffma2_rn(r, w, make_float2(kR[k], kR[k]));
    const float2 y = __fmul2_rn(x, make_float2(scale_log2, scale_log2));
    return __ffma2_rn(__fmul2_rn(y, w), r, y);
}
// Any raw score with |x| >= edge, infinite ones included; NaN stays NaN.
__device__ __forceinline__ float capped_far(float x, const ScoreCap &cap) {
    return copysignf(cap.log2 - __fdividef(2.f * cap.log2, 1.f + npd::fast_exp2(fabsf(x) * cap.in)), x);
}
// Any raw score under a cap of up to kLowCap: the exponential's form near z = 0 too.  Its absolute error there, 2^-23 cap or
// 1.6e-5, is what the score's own sums are off by.
__device__ __forceinline__ float capped_low(float x, const ScoreCap &cap) {
    return cap.log2 - __fdividef(2.f * cap.log2, 1.f + npd::fast_exp2(x * cap.in));
}
// A pair of any raw scores under any cap.
__device__ __forceinline__ float2 capped_any(float2 x, float scale_log2, const ScoreCap &cap) {
    const float2 y = capped_near(x, scale_log2, cap);
    return make_float2(fabsf(x.x) < cap.edge ? y.x : capped_far(x.x, cap), fabsf(x.y) < cap.edge ? y.y : capped_far(x.y, cap));
}

}  // namespace

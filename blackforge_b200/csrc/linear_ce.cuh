// Device helpers shared by the two routes of the linear cross entropy (linear_ce.cu, linear_ce_tc.cu).
#pragma once

#include <cstdint>

namespace bfb {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Class index of a label held in a float32 (as token ids are everywhere): -1 for a row that does not count (negative,
// at or above `vocab`, not finite).
__device__ __forceinline__ int64_t ceLabel(float label, int64_t vocab) {
    if (!(fabsf(label) < 2147483648.0f)) return -1;   // NaN and infinities too
    const int64_t id = static_cast<int64_t>(lroundf(label));
    return id >= 0 && id < vocab ? id : -1;
}

// A label that is neither a class nor one of the negative marks: a mistake in the data, counted for the caller.
__device__ __forceinline__ bool ceLabelIsBad(float label, int64_t vocab) {
    if (!(fabsf(label) < 2147483648.0f)) return true;
    return static_cast<int64_t>(lroundf(label)) >= vocab;
}

__device__ __forceinline__ float ceScale(const float* dGradScale, float gradScale) {
    return dGradScale != nullptr ? gradScale * *dGradScale : gradScale;
}
__device__ __forceinline__ float ceRowGrad(const float* gradLoss, int64_t row, const float* dGradScale, float gradScale) {
    float g = ceScale(dGradScale, gradScale);
    if (gradLoss != nullptr) g *= gradLoss[row];
    return g;
}

// exp(z - top) summed into (top, sum) for a batch of values. While nothing but -inf has been seen the reference point is
// 0, so that exp(-inf - -inf) never arises; a NaN reaches the sum and stays there. The difference is taken before the
// factor log2(e): masks of the lowest finite value would overflow the other way round.
template <int kN>
__device__ __forceinline__ void ceAccumulate(const float (&v)[kN], float& top, float& sum) {
    float most = v[0];
#pragma unroll
    for (int j = 1; j < kN; ++j) most = fmaxf(most, v[j]);
    const float next = fmaxf(top, most);
    const float at = next == -INFINITY ? 0.0f : next;
    sum *= top == -INFINITY ? 1.0f : exp2f((top - at) * kLog2e);
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < kN; ++j) s += exp2f((v[j] - at) * kLog2e);
    sum += s;
    top = next;
}

}  // namespace bfb

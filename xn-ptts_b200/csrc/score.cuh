// Score arithmetic shared by the kernels of attention with score rules.
#pragma once

#include "common.cuh"

namespace ptts {

constexpr float kScoreLog2e = 1.4426950408889634f;
constexpr float kScoreLow = -3.0e38f;  // below every score: a running maximum's start

__device__ __forceinline__ float score_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// u * log2(e) of a score s = q . k / 8 at a distance (either sign), in f32 with the library's
// tanh: small scores under a large cap keep their digits.
__device__ __forceinline__ float score_exact(float s, float cap, float slope, int distance) {
    if (cap > 0.f) s = cap * tanhf(s / cap);
    return (s - slope * (float)abs(distance)) * kScoreLog2e;
}

}  // namespace ptts

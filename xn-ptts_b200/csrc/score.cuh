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

// The same in the exp2 domain, for scores out of the matrix products. Exact: x = s log2(e), by tanhf.
__device__ __forceinline__ float cap_exact(float x, float cap) {
    const float c = cap * kScoreLog2e;
    return c * tanhf(x / c);
}
// Fast: x = 2 s log2(e) / cap, and tanh(y) = 1 - 2 / (1 + e^2y) by one exp2 and one reciprocal. Near
// y = 0 the difference cancels: an absolute error of about cap x 2^-20, which moves a weight by at
// most 2^-13 for cap <= kScoreFastCap, below bf16's own 2^-9.
__device__ __forceinline__ float cap_fast(float x, float cap) {
    const float c = cap * kScoreLog2e;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + score_exp2(x)));
    return fmaf(-2.f * c, r, c);
}

// Takes the bf16s that are not finite out of a pair; whether there was one.
__device__ __forceinline__ bool drop_not_finite(uint32_t& u) {
    const bool lo = (u & 0x7f80u) == 0x7f80u, hi = (u & 0x7f800000u) == 0x7f800000u;
    u = lo ? u & 0xffff0000u : u;
    u = hi ? u & 0x0000ffffu : u;
    return lo || hi;
}

}  // namespace ptts

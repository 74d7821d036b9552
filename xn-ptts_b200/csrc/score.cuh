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

// tanh in f32: y p(y^2), the best fit of degree 5, on |y| <= 1/2 (largest error 2.1e-9 with its constants
// in f32, a seventh of f32's half step there), else tanhf. Each lane by its own y: a vote of the warp
// would let a key that a row does not see choose the form, and with it the last bits, of one that it sees.
__device__ __forceinline__ float f32_tanh(float y) {
    if (fabsf(y) > 0.5f) return tanhf(y);
    const float z = y * y;
    return y * fmaf(fmaf(fmaf(fmaf(fmaf(-0.00646002789f, z, 0.0211690968f), z, -0.0538669695f), z, 0.133326121f), z,
                         -0.333333112f), z, 0.999999998f);
}

// u * log2(e) of a score s = q . k / 8 at a distance (either sign), in f32: small scores under a large cap
// keep their digits. `inv_cap` = 1 / cap.
__device__ __forceinline__ float score_exact(float s, float cap, float inv_cap, float slope, int distance) {
    if (cap > 0.f) s = cap * f32_tanh(s * inv_cap);
    return (s - slope * (float)abs(distance)) * kScoreLog2e;
}

// The same in the exp2 domain, for scores out of the matrix products. Exact: x = s log2(e), by tanhf.
__device__ __forceinline__ float cap_exact(float x, float cap) {
    const float c = cap * kScoreLog2e;
    return c * tanhf(x / c);
}
// Fast: y = s / cap, for N scores of a thread. tanh(y) = y p(y^2) with the polynomial of degree 3
// that fits it best (least largest error, 3.6e-6) on |y| <= 3/4, fitted to numpy's tanh by reweighted
// least squares; where some score is past that, tanh(y) = 1 - 2 / (1 + e^2y) by one exp2
// and one reciprocal, whose difference cancels near 0 (an absolute error near 2^-20). Either moves a
// weight by less than 2^-10 for cap <= kScoreFastCap, a quarter of bf16's own half step of 2^-8.
// On the packed FMAs the polynomial costs 5 pipe cycles a score, the other form 2 of the 3 operations
// at exp2's rate (8 cycles each) that would then bound a capped softmax.
// No row's bits depend on a key that it does not see. Either each thread chooses its form, whose scores are
// one key's, or one row's with those that it does not see set to 0 by the caller; or (VOTE) the warp does,
// the polynomial only where all its rows see all its keys (`all_seen`).
// LESS: less three quarters of the cap, for weights without a maximum. They then lie within 2^-81 and 2^12
// (kScoreBoundedCap), so that values up to 2^94 of a million keys, and down to 2^-45, stay among f32's normal
// numbers beside scores at either end of the cap.
template <int N, bool VOTE, bool LESS>
__device__ __forceinline__ void cap_fast(float* y, float cap, bool all_seen = true) {
    const float c = cap * kScoreLog2e;
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 v = make_float2(y[i], y[i + 1]), z = __fmul2_rn(v, v);
        asm("max.f32 %0, %0, %1, %2;" : "+f"(most) : "f"(z.x), "f"(z.y));
    }
    bool small = most <= 0.5625f;  // a NaN score passes, and stays NaN
    if (VOTE) small = all_seen && __all_sync(0xffffffffu, small);
    if (small) {
        const float2 k0 = make_float2(0.999955601f * c, 0.999955601f * c), k1 = make_float2(-0.332227634f * c, -0.332227634f * c),
                     k2 = make_float2(0.125770911f * c, 0.125770911f * c), k3 = make_float2(-0.0337782684f * c, -0.0337782684f * c),
                     less = make_float2(-0.75f * c, -0.75f * c);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 v = make_float2(y[i], y[i + 1]), z = __fmul2_rn(v, v);
            const float2 p = __ffma2_rn(__ffma2_rn(__ffma2_rn(k3, z, k2), z, k1), z, k0);
            const float2 t = LESS ? __ffma2_rn(v, p, less) : __fmul2_rn(v, p);
            y[i] = t.x;
            y[i + 1] = t.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float r;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + score_exp2(2.f * kScoreLog2e * y[i])));
            y[i] = fmaf(-2.f * c, r, LESS ? 0.25f * c : c);
        }
    }
}

// Takes the bf16s that are not finite out of a pair; whether there was one.
__device__ __forceinline__ bool drop_not_finite(uint32_t& u) {
    const bool lo = (u & 0x7f80u) == 0x7f80u, hi = (u & 0x7f800000u) == 0x7f800000u;
    u = lo ? u & 0xffff0000u : u;
    u = hi ? u & 0x0000ffffu : u;
    return lo || hi;
}

// 16-byte chunks c0 .. c0 + N - 1 of key `key` in a V tile: zeros if the key is gone, else without what is
// not finite (x 0 is NaN then), which `bad` records. Swizzled 16-byte chunks; visible to the products
// afterwards.
template <int N>
__device__ __forceinline__ void clean_v(unsigned char* tile, int key, int c0, bool gone, int* bad) {
    uint4* v = reinterpret_cast<uint4*>(tile + key * 128);
    const uint32_t zero = 0;
    uint32_t probe = 0;
    uint4 w[N];
#pragma unroll
    for (int c = 0; c < N; ++c) {
        w[c] = v[(c0 + c) ^ (key & 7)];
        const uint32_t* u = &w[c].x;
#pragma unroll
        for (int j = 0; j < 4; ++j) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(probe) : "r"(u[j]), "r"(zero));
    }
    const bool drop = (probe & 0x7fff7fffu) != 0;  // NaN in either half
    if (gone || drop) {
        if (!gone) {  // recorded first: whoever reads the cleaned row finds the record
            *bad = 1;
            __threadfence_block();
        }
#pragma unroll
        for (int c = 0; c < N; ++c) {
            uint32_t* u = &w[c].x;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (gone) u[j] = 0u;
                else drop_not_finite(u[j]);
            }
            v[(c0 + c) ^ (key & 7)] = w[c];
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// The greatest bias (in log2 units) of a row at `pos` over its visible positions from .. to: the nearest
// one's, or the farthest one's where the slope is negative. 0 for a row that sees nothing.
__device__ __forceinline__ float most_bias(float slope, int pos, int from, int to) {
    if (from > to) return 0.f;
    const int near = max(max(from - pos, pos - to), 0), far = max(abs(pos - from), abs(pos - to));
    return -slope * (float)(slope < 0.f ? far : near);
}

}  // namespace ptts

// Attention with score rules on CUDA cores, f32 arithmetic: one warp per (row, head), 8 lanes per
// key, 4 keys per step, an online softmax in the exp2 domain per lane group, merged at the end.
// Keys a row does not see are not read, so whatever they hold stays out of its result.
#include "common.cuh"
#include "score.cuh"
#include "score.h"

namespace ptts {
namespace {

template <typename T>
__global__ void __launch_bounds__(256) score_core_kernel(ScoreCoreArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    const long long w = blockIdx.x * 8LL + (threadIdx.x >> 5);
    if (w >= (long long)a.n_rows * a.heads) return;
    const int lane = threadIdx.x & 31, g = lane >> 3, j = lane & 7;
    const int row = (int)(w / a.heads), h = (int)(w % a.heads);
    const int sid = a.rows.stream[row], pos = a.rows.pos[row];
    const int lo = a.rows.lo[row], hi = sid < 0 ? -1 : a.rows.hi[row];
    const unsigned long long lineage = a.rows.lineage ? a.rows.lineage[row] : 0;
    const int base = a.rows.lineage ? a.rows.base[row] : 0x7fffffff;
    const float slope = a.rule.slopes ? a.rule.slopes[h] : 0.f;
    const float inv_cap = a.rule.cap > 0.f ? 1.f / a.rule.cap : 0.f;
    float q[8], m = kScoreLow, l = 0.f, acc[8];
    const long long at = ((long long)row * a.heads + h) * kHeadDim + 8 * j;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        q[i] = a.q[at + i] * 0.125f;
        acc[i] = 0.f;
    }
    const T* kb = static_cast<const T*>(a.k_cache) + kv_offset(sid < 0 ? 0 : sid, 0, h, a.num_streams, a.capacity);
    const T* vb = static_cast<const T*>(a.v_cache) + kv_offset(sid < 0 ? 0 : sid, 0, h, a.num_streams, a.capacity);
    for (int s0 = lo; s0 <= hi; s0 += 4) {
        const int slot = s0 + g;
        const bool node = slot >= base;
        const bool seen = slot <= hi && (!node || (lineage >> (slot - base) & 1));
        float d = 0.f;
        if (seen) {
            const T* k = kb + (long long)slot * kRowWidth + 8 * j;
#pragma unroll
            for (int i = 0; i < 8; ++i) d = fmaf(q[i], to_f32(k[i]), d);
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        const int kp = seen && node ? a.rows.pos[a.rows.row0[row] + slot - base] : slot;
        d = score_exact(d, a.rule.cap, inv_cap, slope, pos - kp);
        if (seen) {
            const float mn = fmaxf(m, d);
            const float corr = score_exp2(m - mn), e = score_exp2(d - mn);
            l = fmaf(l, corr, e);
            const T* v = vb + (long long)slot * kRowWidth + 8 * j;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = fmaf(e, to_f32(v[i]), acc[i] * corr);
            m = mn;
        }
    }
#pragma unroll
    for (int o = 8; o <= 16; o <<= 1) {
        const float mo = __shfl_xor_sync(0xffffffffu, m, o), lo2 = __shfl_xor_sync(0xffffffffu, l, o);
        const float mn = fmaxf(m, mo);
        const float fa = score_exp2(m - mn), fb = score_exp2(mo - mn);
        l = l * fa + lo2 * fb;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = acc[i] * fa + __shfl_xor_sync(0xffffffffu, acc[i], o) * fb;
        m = mn;
    }
    if (g != 0) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;  // nothing visible: zeros (a NaN sum stays NaN)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float o = acc[i] * inv;
        if (a.out_bf16) static_cast<__nv_bfloat16*>(a.out)[at + i] = __float2bfloat16_rn(o);
        else static_cast<float*>(a.out)[at + i] = o;
    }
}

}  // namespace

void launch_score_core(const ScoreCoreArgs& a, bool cache_bf16, cudaStream_t s) {
    const long long blocks = ((long long)a.n_rows * a.heads + 7) / 8;
    if (cache_bf16) launch_k(score_core_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(256), 0, s, a);
    else launch_k(score_core_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, s, a);
}

}  // namespace ptts

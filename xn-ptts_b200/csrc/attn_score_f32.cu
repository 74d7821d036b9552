// Attention with score rules for prompts and drafted trees on f32 caches: f32 arithmetic on the CUDA
// cores, one CTA per (tile of up to 32 rows of one sequence, head, share of its keys).
//
// Bound by the FMAs (two of 64 per row and key; 128 lanes) as long as shared memory keeps up: each
// thread holds a 4 x 4 block of S (rows x keys) and of O (rows x dims), so 16-byte reads of q, k, p and
// v feed 8 FMAs each, 12 cycles of shared memory under 16 of FMAs. Rows of 68 floats keep the 16-byte
// reads of 16 keys (or 16 dim groups) free of bank conflicts. Two to six CTAs share an SM.
//
// Few rows over a long cache would leave most SMs idle: then the tile's keys are cut into `splits` equal
// shares (whole 64-key tiles), which leave (max, sum, acc) records that a second kernel joins.
//
// Measured (one B200, 8 heads): 5 streams of 65-301 rows on up to 130 keys, cap, bias and documents, 47 us
// a call, 37 of them this kernel (a warp a row, a key a lane: 242 a call).
//
// A tile of keys that some row does not see whole takes values that are not finite out of V (0 x NaN is
// NaN); rows that see such a value get it back at the end, from the cache.
#include "common.cuh"
#include "score.cuh"
#include "score.h"

namespace ptts {
namespace {

constexpr int TR = kScoreF32Rows, TK = 64, kLd = 68, kThreads32 = 128;
static_assert(TR == 32, "8 row groups of 4");
struct Smem32 {
    float q[TR][kLd], p[TR][kLd], k[TK][kLd], v[TK][kLd];
};

__global__ void __launch_bounds__(kThreads32) score_f32_kernel(ScoreF32Args a) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Smem32& sm = *reinterpret_cast<Smem32*>(smem_raw);
    __shared__ int s_lo, s_hi, s_lo_most, s_hi_least, s_bad;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    if (tid == 0) s_lo = 0x7fffffff, s_hi = -1, s_lo_most = 0, s_hi_least = 0x7fffffff, s_bad = 0;
    __syncthreads();
    grid_dep_wait();
    grid_dep_launch();
    const int head = blockIdx.y, split = blockIdx.z;
    const int2 tile = a.tiles[blockIdx.x];
    const int row0 = tile.x, nrows = tile.y, sid = a.rows.stream[row0];
    const float slope = a.rule.slopes ? a.rule.slopes[head] : 0.f, inv_cap = a.rule.cap > 0.f ? 1.f / a.rule.cap : 0.f;
    // This thread's rows 4 ty .. + 3, and the slots that the tile's rows see: any and all.
    int lo[4], hi[4], pos[4];
    unsigned long long line[4];
    int base = 0x7fffffff, node0 = 0;
    if (a.rows.lineage) base = a.rows.base[row0], node0 = a.rows.row0[row0];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 4 * ty + i, row = row0 + min(r, nrows - 1);
        lo[i] = a.rows.lo[row];
        hi[i] = r < nrows ? a.rows.hi[row] : -1;
        pos[i] = a.rows.pos[row];
        line[i] = a.rows.lineage ? a.rows.lineage[row] : 0;
        if (tx == 0 && r < nrows) {
            if (lo[i] <= hi[i]) {
                atomicMin(&s_lo, lo[i]);
                atomicMax(&s_hi, hi[i]);
            }
            atomicMax(&s_lo_most, lo[i]);
            atomicMin(&s_hi_least, min(hi[i], base - 1));
        }
    }
    for (int i = tid; i < TR * 16; i += kThreads32) {
        const int r = i >> 4, c = i & 15;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < nrows) x = *reinterpret_cast<const float4*>(a.q + (long long)(row0 + r) * a.heads * kHeadDim + head * kHeadDim + 4 * c);
        *reinterpret_cast<float4*>(&sm.q[r][4 * c]) = make_float4(x.x * 0.125f, x.y * 0.125f, x.z * 0.125f, x.w * 0.125f);
    }
    __syncthreads();
    // This CTA's share: key tiles t0 .. t1 - 1 from the first slot any row sees.
    const int first = s_lo, end = sid < 0 ? 0 : s_hi + 1, n = end <= 0 ? 0 : (end - first + TK - 1) / TK;
    const int t0 = (int)((long long)n * split / a.splits), t1 = (int)((long long)n * (split + 1) / a.splits);
    const long long kv0 = kv_offset(max(sid, 0), 0, head, a.num_streams, a.capacity);
    const float* kc = static_cast<const float*>(a.k_cache) + kv0;
    const float* vc = static_cast<const float*>(a.v_cache) + kv0;
    float o[4][4] = {}, m[4], l[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = kScoreLow;
    for (int t = t0; t < t1; ++t) {
        const int s0 = first + t * TK;
        const bool whole = s0 >= s_lo_most && s0 + TK - 1 <= s_hi_least;
        __syncthreads();  // the tile before is read
        for (int i = tid; i < TK * 16; i += kThreads32) {
            const int j = i >> 4, c = i & 15;
            float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
            if (s0 + j < end) {
                k = *reinterpret_cast<const float4*>(kc + (long long)(s0 + j) * kRowWidth + 4 * c);
                v = *reinterpret_cast<const float4*>(vc + (long long)(s0 + j) * kRowWidth + 4 * c);
            }
            if (!whole && !(isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w))) {
                v = make_float4(isfinite(v.x) ? v.x : 0.f, isfinite(v.y) ? v.y : 0.f, isfinite(v.z) ? v.z : 0.f,
                                isfinite(v.w) ? v.w : 0.f);
                s_bad = 1;
            }
            *reinterpret_cast<float4*>(&sm.k[j][4 * c]) = k;
            *reinterpret_cast<float4*>(&sm.v[j][4 * c]) = v;
        }
        __syncthreads();
        // S: rows 4 ty + i, keys tx + 16 j.
        float s[4][4] = {};
#pragma unroll 4
        for (int d = 0; d < kHeadDim; d += 4) {
            float4 q[4], k[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const float4*>(&sm.q[4 * ty + i][d]);
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const float4*>(&sm.k[tx + 16 * j][d]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    s[i][j] = fmaf(q[i].w, k[j].w, fmaf(q[i].z, k[j].z, fmaf(q[i].y, k[j].y, fmaf(q[i].x, k[j].x, s[i][j]))));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int slot = s0 + tx + 16 * j, node = slot - base;
                const bool seen = whole || (slot >= lo[i] && slot <= hi[i] && (node < 0 || (line[i] >> (node & 63) & 1)));
                const int at = seen && node >= 0 && slope != 0.f ? a.rows.pos[node0 + node] : slot;
                s[i][j] = score_exact(s[i][j], a.rule.cap, inv_cap, slope, pos[i] - at);
                if (!seen) s[i][j] = -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            const float mn = fmaxf(m[i], top), f = score_exp2(m[i] - mn);
            m[i] = mn;
            l[i] *= f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float e = score_exp2(s[i][j] - mn);
                l[i] += e;
                o[i][j] *= f;
                sm.p[4 * ty + i][tx + 16 * j] = e;
            }
        }
        __syncwarp();  // a row group's p is written and read by its own 16 threads
        // O: rows 4 ty + i, dims 4 tx + j.
#pragma unroll 4
        for (int k = 0; k < TK; k += 4) {
            float4 p[4], v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4*>(&sm.p[4 * ty + i][k]);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float4*>(&sm.v[k + j][4 * tx]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float pp[4] = {p[i].x, p[i].y, p[i].z, p[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    o[i][0] = fmaf(pp[j], v[j].x, o[i][0]);
                    o[i][1] = fmaf(pp[j], v[j].y, o[i][1]);
                    o[i][2] = fmaf(pp[j], v[j].z, o[i][2]);
                    o[i][3] = fmaf(pp[j], v[j].w, o[i][3]);
                }
            }
        }
    }
    __syncthreads();
    const bool bad = s_bad != 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
        const int r = 4 * ty + i;
        if (r >= nrows) continue;
        if (bad) {  // values taken out of V, for the rows that see them
            for (int slot = max(lo[i], first + t0 * TK); slot <= min(hi[i], first + t1 * TK - 1); ++slot) {
                if (slot >= base && !(line[i] >> (slot - base) & 1)) continue;
                for (int j = 0; j < 4; ++j) {
                    const float x = vc[(long long)slot * kRowWidth + 4 * tx + j];
                    if (!isfinite(x)) o[i][j] += x;
                }
            }
        }
        if (a.splits > 1) {
            float* rec = a.part + (((long long)(row0 + r) * a.heads + head) * a.splits + split) * kPartStride;
            *reinterpret_cast<float4*>(rec + 4 * tx) = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
            if (tx == 0) *reinterpret_cast<float2*>(rec + 64) = make_float2(m[i], l[i]);
            continue;
        }
        const float f = l[i] == 0.f ? 0.f : 1.f / l[i];  // a row that sees nothing: zeros
        const long long at = ((long long)(row0 + r) * a.heads + head) * kHeadDim + 4 * tx;
        if (a.out_bf16)
            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) =
                make_uint2(pack_bf16x2(o[i][0] * f, o[i][1] * f), pack_bf16x2(o[i][2] * f, o[i][3] * f));
        else
            *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(o[i][0] * f, o[i][1] * f, o[i][2] * f, o[i][3] * f);
    }
}

// Joins a row's and head's splits: one warp each, lane = 2 dims.
__global__ void __launch_bounds__(256) score_f32_merge_kernel(ScoreF32Args a) {
    grid_dep_wait();
    grid_dep_launch();
    const long long w = blockIdx.x * 8LL + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (w >= (long long)a.n_rows * a.heads) return;
    const float* rec = a.part + w * a.splits * kPartStride;
    float mx = kScoreLow, den = 0.f, x0 = 0.f, x1 = 0.f;
    for (int s = 0; s < a.splits; ++s) mx = fmaxf(mx, rec[s * kPartStride + 64]);
    for (int s = 0; s < a.splits; ++s, rec += kPartStride) {
        const float2 ml = *reinterpret_cast<const float2*>(rec + 64), v = *reinterpret_cast<const float2*>(rec + 2 * lane);
        const float f = score_exp2(ml.x - mx);
        den = fmaf(f, ml.y, den);
        x0 = fmaf(f, v.x, x0);
        x1 = fmaf(f, v.y, x1);
    }
    const float f = den == 0.f ? 0.f : 1.f / den;
    if (a.out_bf16) reinterpret_cast<uint32_t*>(a.out)[w * 32 + lane] = pack_bf16x2(x0 * f, x1 * f);
    else reinterpret_cast<float2*>(a.out)[w * 32 + lane] = make_float2(x0 * f, x1 * f);
}

}  // namespace

int score_f32_splits(int tiles, int heads, int most_keys, int sms) {
    // Four CTAs an SM (their shared memory and registers fit), each with two key tiles or more.
    const long long ctas = (long long)tiles * heads, want = (4LL * sms + ctas - 1) / ctas, most = most_keys / (2 * TK);
    return (int)(want < most ? (want > 1 ? want : 1) : (most > 1 ? most : 1));
}

void launch_score_f32(const ScoreF32Args& a, cudaStream_t s) {
    set_max_dynamic_smem(reinterpret_cast<const void*>(score_f32_kernel), sizeof(Smem32));
    launch_k(score_f32_kernel, dim3(a.n_tiles, a.heads, a.splits), dim3(kThreads32), sizeof(Smem32), s, a);
    if (a.splits > 1)
        launch_k(score_f32_merge_kernel, dim3((unsigned)(((long long)a.n_rows * a.heads + 7) / 8)), dim3(256), 0, s, a);
}

}  // namespace ptts

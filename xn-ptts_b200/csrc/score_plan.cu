// The plan of attention with score rules, in one launch: each row's position, visible slots and
// (in a tree call) lineage, its RoPE and its cache rows; and, in CTA 0, the key partition of the
// split kernels. The ordinary attention op plans and appends in two launches.
//
// RoPE and append as in rope_append.cu (rope.rs:81-95, complete_kv at transformer.rs:84-91): one
// warp per row, whose lanes compute the 32 pairs' sines and cosines once for all heads.
//
// Bound by memory for prompts (per row (H + 2 KVH) x 64 inputs read, H x 64 x 2 cache elements and
// the q planes written) and by launch latency for single tokens. Measured (one B200): 54,073 rows of
// 8 heads, 388 MB, 88 us, 67 % of a copy's rate; fetching a row's q, k and v ahead of the rotation 102,
// registers bounded for 5 or 6 CTAs an SM 97, for 8 126.
#include "common.cuh"
#include "score.h"

namespace ptts {
namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanWarps = kPlanThreads / 32;

// The last sequence whose rows begin at or before row r.
__device__ __forceinline__ int seq_of(const ScorePlanArgs& a, const int32_t* offsets, int r) {
    if (a.n_seq == a.n_rows) return r;  // single tokens
    int lo = 0, hi = a.n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (offsets[mid] <= r) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// The same by a warp for one row: 31 probes a step.
__device__ __forceinline__ int seq_of_warp(const ScorePlanArgs& a, const int32_t* offsets, int r, int lane) {
    if (a.n_seq == a.n_rows) return r;
    int lo = 0, hi = a.n_seq - 1;  // offsets[lo] <= r, offsets[hi + 1] > r
    while (lo < hi) {
        const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
        const int below = __popc(__ballot_sync(0xffffffffu, at <= hi && offsets[min(at, hi)] <= r));
        lo += below * step;
        hi = min(hi, lo + step - 1);
    }
    return lo;
}

// Whether a sequence of `rows` rows fits behind the device's length `base`. The host has checked its own
// lengths; the device's can be others (a caller's graph that advances, a caller that writes them).
__device__ __forceinline__ bool fits(const ScorePlanArgs& a, int base, int rows) {
    return base >= 0 && base <= a.capacity - rows;
}

// Row r's visible slots, from the caller's spans clamped to the filled slots; an empty span is
// 0..-1 whatever the caller wrote.
__device__ __forceinline__ void row_span(const ScorePlanArgs& a, int r, int base, int row0, int rows, int& lo, int& hi) {
    const int end = base + rows - 1;
    lo = a.first ? max(a.first[r], 0) : 0;
    hi = a.parents ? end : (a.last ? min(a.last[r], end) : base + r - row0);
    if (lo > hi) lo = 0, hi = -1;
}

// CTA 0: the units' key counts, end to end. Every unit has at least one key, so that a CTA visits
// it and writes its rows even where they see nothing; a sequence that does not fit has that one, in slot 0.
__device__ __forceinline__ void plan_units(const ScorePlanArgs& a, const int32_t* list) {
    __shared__ int warp_tot[kPlanWarps];
    __shared__ int carry;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool spans = a.first || a.last, blocks = a.blocks_at >= 0;
    const int32_t *streams = list, *offsets = list + a.n_seq, *units = list + a.blocks_at;
    auto unit = [&](int u) { return blocks ? make_int2(units[2 * u], units[2 * u + 1]) : make_int2(u, 1); };
    if (tid == 0) {
        carry = 0;
        a.prefix[0] = 0;
    }
    // A block's union of spans: a warp per block, two rows a lane.
    if (blocks && spans) {
        for (int u = warp; u < a.n_units; u += kPlanWarps) {
            const int2 b = unit(u);
            const int sq = seq_of(a, offsets, b.x), row0 = offsets[sq];
            const int base = a.lengths[streams[sq]], rows = offsets[sq + 1] - row0;
            int lo = 0x7fffffff, hi = -1;
            for (int i = lane; i < b.y; i += 32) {
                int x = 0, y = -1;
                if (fits(a, base, rows)) row_span(a, b.x + i, base, row0, rows, x, y);
                if (x <= y) lo = min(lo, x), hi = max(hi, y);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            }
            if (lane == 0) {
                a.unit_lo[u] = hi < 0 ? 0 : lo;
                a.prefix[u + 1] = hi < 0 ? 1 : hi - lo + 1;
            }
        }
    }
    __syncthreads();
    for (int at = 0; at < a.n_units; at += kPlanThreads) {
        const int u = at + tid;
        int v = 0;
        if (u < a.n_units) {
            if (blocks && spans) {
                v = a.prefix[u + 1];
            } else {
                const int2 b = unit(u);
                const int sq = seq_of(a, offsets, b.x), row0 = offsets[sq];
                const int base = a.lengths[streams[sq]], rows = offsets[sq + 1] - row0;
                int lo = 0, hi = -1;
                if (fits(a, base, rows)) row_span(a, b.x + b.y - 1, base, row0, rows, lo, hi);  // without spans the last row sees the most
                a.unit_lo[u] = lo;
                v = max(hi - lo + 1, 1);
            }
            if (blocks) v = v * score_key_cost(unit(u).y) + kScoreBlockCost;
        }
        int x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += t;
        }
        if (lane == 31) warp_tot[warp] = x;
        __syncthreads();
        int before = carry;
        for (int w = 0; w < warp; ++w) before += warp_tot[w];
        if (u < a.n_units) a.prefix[u + 1] = before + x;
        __syncthreads();
        if (tid == kPlanThreads - 1) carry = before + x;
        __syncthreads();
    }
    const long long total = carry;
    const int G = blocks ? score_ctas(total, a.grid) : ctas_in_use(total, a.grid);
    for (int u = tid; u < a.n_units; u += kPlanThreads) {
        const long long pb = a.prefix[u], pe = a.prefix[u + 1];
        for (int c = cta_of(pb, total, G); c <= cta_of(pe - 1, total, G); ++c)
            if (cta_start(c, total, G) >= pb) a.cta_first[c] = u;
    }
}

// 16 bytes of an input row as floats: 8 bf16 or 4 f32.
__device__ __forceinline__ void load_in(const __nv_bfloat16* p, float* x) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    x[0] = bf16lo(u.x), x[1] = bf16hi(u.x), x[2] = bf16lo(u.y), x[3] = bf16hi(u.y);
    x[4] = bf16lo(u.z), x[5] = bf16hi(u.z), x[6] = bf16lo(u.w), x[7] = bf16hi(u.w);
}
__device__ __forceinline__ void load_in(const float* p, float* x) {
    const float4 u = *reinterpret_cast<const float4*>(p);
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
}
template <int E>
__device__ __forceinline__ void store_out(float* p, const float* x) {
#pragma unroll
    for (int i = 0; i < E; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
}
template <int E>
__device__ __forceinline__ void store_out(__nv_bfloat16* p, const float* x) {
    uint32_t w[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    if constexpr (E == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}

template <typename Tin, typename T>
__device__ __forceinline__ void plan(const ScorePlanArgs& a, const int32_t* list) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int block = blockIdx.x;
    if (a.n_units > 0) {
        if (block == 0) {
            plan_units(a, list);
            return;
        }
        block -= 1;
    }
    const int32_t* offsets = list + a.n_seq;
    // A warp per row.
    const int r = block * kPlanWarps + warp;
    if (r >= a.n_rows) return;
    const int sq = seq_of_warp(a, offsets, r, lane), row0 = offsets[sq];
    const int rows = offsets[sq + 1] - row0, sid = list[sq];
    const bool known = sid >= 0 && sid < a.num_streams;
    const int length = known ? a.lengths[sid] : 0;
    bool good = known && fits(a, length, rows);  // the whole sequence: its rows see each other's slots
    const int base = good ? length : 0;          // a refused row's numbers mean nothing, and stay small
    const int node = r - row0, slot = base + node;
    if (!good && lane == 0) set_error(a.err, known ? DEV_ERR_CAPACITY : DEV_ERR_BOUNDS);
    int pos = slot, lo = 0, hi = -1;
    if (good) row_span(a, r, base, row0, rows, lo, hi);
    unsigned long long seen = 0;
    if (a.parents) {
        // Lane i holds the parents of nodes i and 32 + i. One bad parent refuses the whole tree: every
        // row's warp sees it.
        const int p0 = lane < rows ? a.parents[row0 + lane] : -1;
        const int p1 = lane + 32 < rows ? a.parents[row0 + lane + 32] : -1;
        if (__any_sync(0xffffffffu, p0 < -1 || p0 >= lane || p1 < -1 || p1 >= lane + 32)) {
            if (lane == 0) set_error(a.err, DEV_ERR_BOUNDS);
            good = false;
            lo = 0, hi = -1;
        }
        // The path to the root: parents fall, so it ends; the node and its ancestors, a bit each.
        int depth = 0;
        for (int i = node; good && i >= 0;) {
            seen |= 1ull << i;
            const int up = __shfl_sync(0xffffffffu, i < 32 ? p0 : p1, i & 31);
            depth += up >= 0;
            i = up;
        }
        pos = base + depth;
        // Of these, the ones at positions from `lo` on: positions fall by one from node to parent,
        // so drop the lowest bits (the roots' end) of those before it.
        for (int drop = lo - base; drop > 0 && seen; --drop) seen &= seen - 1;
        if (hi < 0) seen = 0;
    }
    if (lane == 0) {
        a.rows.stream[r] = good ? sid : -1;
        a.rows.pos[r] = good ? pos : 0;
        a.rows.lo[r] = lo;
        a.rows.hi[r] = hi;
        if (a.parents) {
            a.rows.base[r] = base;
            a.rows.row0[r] = row0;
            a.rows.lineage[r] = seen;
        }
    }
    // RoPE and append, 16 bytes of input a lane: E dims of one of the HS heads a warp takes at a time.
    // Lane i turns pair i; a lane's own pairs' factors come from there.
    constexpr int E = 16 / (int)sizeof(Tin), HS = 32 * E / kHeadDim;
    float cs[E / 2], sn[E / 2];
    if (a.rotate) {
        // The f32 angle's sine and cosine in f64, rounded once (attend's are sincosf's: a key in one of
        // ten thousand ends up a bf16 step apart). Beside the row's memory traffic it does not show.
        double sd, cd;
        sincos((double)((float)pos * a.inv_freq[lane]), &sd, &cd);
        const float s = (float)sd, c = (float)cd;
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            const int pair = lane % (kHeadDim / E) * (E / 2) + i;
            cs[i] = __shfl_sync(0xffffffffu, c, pair);
            sn[i] = __shfl_sync(0xffffffffu, s, pair);
        }
    }
    auto rotate = [&](float* x) {
        if (!a.rotate) return;
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            const float x0 = x[2 * i], x1 = x[2 * i + 1];
            x[2 * i] = __fsub_rn(__fmul_rn(x0, cs[i]), __fmul_rn(x1, sn[i]));
            x[2 * i + 1] = __fadd_rn(__fmul_rn(x0, sn[i]), __fmul_rn(x1, cs[i]));
        }
    };
    const int mine = lane / (kHeadDim / E), dim = lane % (kHeadDim / E) * E;  // of a step's heads; first dim
    const Tin* q = static_cast<const Tin*>(a.q) + (long long)r * a.heads * kHeadDim + dim;
#pragma unroll 1  // (by two: 1 to 2 us more a call, the code has to be fetched)
    for (int h = mine; h < a.heads; h += HS) {
        const long long at = ((long long)r * a.heads + h) * kHeadDim + dim;
        float x[E];
        load_in(q + h * kHeadDim, x);
        rotate(x);
        if (a.q_hi) {
            float lo[E];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                x[i] *= a.q_scale;
                lo[i] = x[i] - __bfloat162float(__float2bfloat16_rn(x[i]));
            }
            store_out<E>(a.q_hi + at, x);
            store_out<E>(a.q_lo + at, lo);
        } else {
            store_out<E>(a.q_out + at, x);
        }
    }
    if (!good) return;
    const int group = a.heads / a.kv_heads;
    const Tin* k = static_cast<const Tin*>(a.k) + (long long)r * a.kv_heads * kHeadDim + dim;
    const Tin* v = static_cast<const Tin*>(a.v) + (long long)r * a.kv_heads * kHeadDim + dim;
    T* kc = static_cast<T*>(a.k_cache) + dim;
    T* vc = static_cast<T*>(a.v_cache) + dim;
#pragma unroll 1  // (by two: 1 to 2 us more a call, the code has to be fetched)
    for (int h = mine; h < a.kv_heads; h += HS) {
        float x[E], y[E];
        load_in(k + h * kHeadDim, x);
        load_in(v + h * kHeadDim, y);
        rotate(x);
        for (int rep = 0; rep < group; ++rep) {
            const long long to = kv_offset(sid, slot, h * group + rep, a.num_streams, a.capacity);
            store_out<E>(kc + to, x);
            store_out<E>(vc + to, y);
        }
    }
}

template <typename Tin, typename T>
__global__ void __launch_bounds__(kPlanThreads) score_plan_kernel(ScorePlanArgs a) {
    grid_dep_wait();
    grid_dep_launch();
    plan<Tin, T>(a, a.list);
}

template <typename Tin, typename T>
__global__ void __launch_bounds__(kPlanThreads) score_plan_inline_kernel(ScorePlanArgs a, const __grid_constant__ ScoreInline l) {
    grid_dep_wait();
    grid_dep_launch();
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < a.list_ints; i += kPlanThreads) a.list[i] = l.list[i];
    plan<Tin, T>(a, l.list);
}

template <typename Tin, typename T>
void launch_typed(const ScorePlanArgs& a, const ScoreInline* list, cudaStream_t s) {
    const dim3 grid((a.n_rows + kPlanWarps - 1) / kPlanWarps + (a.n_units > 0 ? 1 : 0)), block(kPlanThreads);
    if (list) launch_k(score_plan_inline_kernel<Tin, T>, grid, block, 0, s, a, *list);
    else launch_k(score_plan_kernel<Tin, T>, grid, block, 0, s, a);
}

}  // namespace

void launch_score_plan(const ScorePlanArgs& a, const ScoreInline* list, bool in_bf16, bool cache_bf16, cudaStream_t s) {
    if (in_bf16 && cache_bf16) launch_typed<__nv_bfloat16, __nv_bfloat16>(a, list, s);
    else if (in_bf16) launch_typed<__nv_bfloat16, float>(a, list, s);
    else if (cache_bf16) launch_typed<float, __nv_bfloat16>(a, list, s);
    else launch_typed<float, float>(a, list, s);
}

}  // namespace ptts

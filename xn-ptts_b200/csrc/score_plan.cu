// The plan of attention with score rules, in one launch: each row's position, visible slots and
// (in a tree call) lineage, its RoPE and its cache rows; and, in CTA 0, the key partition of the
// split kernels. The ordinary attention op plans and appends in two launches.
//
// RoPE and append as in rope_append.cu (rope.rs:81-95, complete_kv at transformer.rs:84-91): one
// CTA per row, one warp per head, a lane per pair, so the angle's sine and cosine are computed
// once per warp rather than once per head.
//
// Bound by memory for prompts (per row (H + 2 KVH) x 64 inputs read, H x 64 x 2 cache elements and
// the q planes written) and by launch latency for single tokens.
#include "common.cuh"
#include "score.h"

namespace ptts {
namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanWarps = kPlanThreads / 32;

// The last sequence whose rows begin at or before row r.
__device__ __forceinline__ int seq_of(const ScorePlanArgs& a, int r) {
    if (a.n_seq == a.n_rows) return r;  // single tokens
    const int32_t* offsets = a.row_offsets;
    int lo = 0, hi = a.n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (offsets[mid] <= r) lo = mid;
        else hi = mid - 1;
    }
    return lo;
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
// it and writes its rows even where they see nothing.
__device__ void plan_units(const ScorePlanArgs& a) {
    __shared__ int warp_tot[kPlanWarps];
    __shared__ int carry;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool spans = a.first || a.last;
    if (tid == 0) {
        carry = 0;
        a.prefix[0] = 0;
    }
    // A block's union of spans: a warp per block, two rows a lane.
    if (a.blocks && spans) {
        for (int u = warp; u < a.n_units; u += kPlanWarps) {
            const int2 b = a.blocks[u];
            const int sq = seq_of(a, b.x), row0 = a.row_offsets[sq];
            const int base = a.lengths[a.seq_stream[sq]], rows = a.row_offsets[sq + 1] - row0;
            int lo = 0x7fffffff, hi = -1;
            for (int i = lane; i < b.y; i += 32) {
                int x, y;
                row_span(a, b.x + i, base, row0, rows, x, y);
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
            if (a.blocks && spans) {
                v = a.prefix[u + 1];
            } else {
                const int2 b = a.blocks ? a.blocks[u] : make_int2(u, 1);
                const int sq = seq_of(a, b.x), row0 = a.row_offsets[sq];
                const int base = a.lengths[a.seq_stream[sq]], rows = a.row_offsets[sq + 1] - row0;
                int lo, hi;
                row_span(a, b.x + b.y - 1, base, row0, rows, lo, hi);  // without spans the last row sees the most
                a.unit_lo[u] = lo;
                v = max(hi - lo + 1, 1);
            }
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
    const int G = ctas_in_use(total, a.grid);
    for (int u = tid; u < a.n_units; u += kPlanThreads) {
        const long long pb = a.prefix[u], pe = a.prefix[u + 1];
        for (int c = cta_of(pb, total, G); c <= cta_of(pe - 1, total, G); ++c)
            if (cta_start(c, total, G) >= pb) a.cta_first[c] = u;
    }
}

template <typename Tin>
__device__ __forceinline__ float2 load_pair(const void* p, long long pair);
template <>
__device__ __forceinline__ float2 load_pair<float>(const void* p, long long pair) {
    return static_cast<const float2*>(p)[pair];
}
template <>
__device__ __forceinline__ float2 load_pair<__nv_bfloat16>(const void* p, long long pair) {
    const uint32_t u = static_cast<const uint32_t*>(p)[pair];
    return make_float2(bf16lo(u), bf16hi(u));
}
__device__ __forceinline__ void store_pair(float* p, float2 v) { *reinterpret_cast<float2*>(p) = v; }
__device__ __forceinline__ void store_pair(__nv_bfloat16* p, float2 v) {
    *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(v.x, v.y);
}

template <typename Tin, typename T>
__global__ void __launch_bounds__(kPlanThreads) score_plan_kernel(ScorePlanArgs a) {
    __shared__ int s_parent[kTreeNodes];
    __shared__ int s_pos;
    grid_dep_wait();
    grid_dep_launch();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int r = blockIdx.x;
    if (a.n_units > 0) {
        if (r == 0) {
            plan_units(a);
            return;
        }
        r -= 1;
    }
    const int sq = seq_of(a, r), row0 = a.row_offsets[sq];
    const int rows = a.row_offsets[sq + 1] - row0, sid = a.seq_stream[sq];
    const bool known = sid >= 0 && sid < a.num_streams;
    const int base = known ? a.lengths[sid] : 0;
    const int node = r - row0, slot = base + node;
    bool good = known && base >= 0 && slot < a.capacity;
    if (!good && tid == 0) set_error(a.err, known ? DEV_ERR_CAPACITY : DEV_ERR_BOUNDS);
    int pos = slot;
    if (a.parents) {  // one bad parent refuses the whole tree: every node's CTA sees it
        const int p = tid < rows ? a.parents[row0 + tid] : -1;
        if (tid < kTreeNodes) s_parent[tid] = p;
        if (__syncthreads_or(tid < rows && (p < -1 || p >= tid))) {
            if (tid == 0) set_error(a.err, DEV_ERR_BOUNDS);
            good = false;
        }
        if (good && tid == 0) {
            int depth = 0;
            for (int i = s_parent[node]; i >= 0; i = s_parent[i]) ++depth;
            s_pos = base + depth;
        }
        __syncthreads();
        if (good) pos = s_pos;
    }
    if (tid == 0) {
        int lo = 0, hi = -1;
        if (good) row_span(a, r, base, row0, rows, lo, hi);
        a.rows.stream[r] = good ? sid : -1;
        a.rows.pos[r] = pos;
        a.rows.lo[r] = lo;
        a.rows.hi[r] = hi;
        if (a.parents) {
            // Itself and its ancestors, those at positions from `lo` on (a path's positions
            // fall by one from node to parent).
            unsigned long long seen = 0;
            if (good && hi >= 0)
                for (int i = node, at = pos; i >= 0 && at >= lo; i = s_parent[i], --at) seen |= 1ull << i;
            a.rows.base[r] = base;
            a.rows.row0[r] = row0;
            a.rows.lineage[r] = seen;
        }
    }
    // RoPE and append: lane = pair, warps over the heads of q, k and v.
    float sn = 0.f, cs = 1.f;
    if (a.rotate) sincosf((float)pos * a.inv_freq[lane], &sn, &cs);
    const int group = a.heads / a.kv_heads;
    for (int h = warp; h < a.heads + 2 * a.kv_heads; h += kPlanWarps) {
        const int part = h < a.heads ? 0 : (h < a.heads + a.kv_heads ? 1 : 2);  // q, k, v
        const int hh = part == 0 ? h : h - a.heads - (part - 1) * a.kv_heads;
        const long long at = ((long long)r * (part == 0 ? a.heads : a.kv_heads) + hh) * (kHeadDim / 2) + lane;
        float2 x = load_pair<Tin>(part == 0 ? a.q : (part == 1 ? a.k : a.v), at);
        if (part < 2 && a.rotate) {
            const float y0 = __fsub_rn(__fmul_rn(x.x, cs), __fmul_rn(x.y, sn));
            const float y1 = __fadd_rn(__fmul_rn(x.x, sn), __fmul_rn(x.y, cs));
            x = make_float2(y0, y1);
        }
        if (part == 0) {
            if (a.q_hi) {
                const float y0 = x.x * a.q_scale, y1 = x.y * a.q_scale;
                const uint32_t hi = pack_bf16x2(y0, y1);
                reinterpret_cast<uint32_t*>(a.q_hi)[at] = hi;
                reinterpret_cast<uint32_t*>(a.q_lo)[at] = pack_bf16x2(y0 - bf16lo(hi), y1 - bf16hi(hi));
            } else {
                store_pair(a.q_out + 2 * at, x);
            }
        } else if (good) {
            T* cache = static_cast<T*>(part == 1 ? a.k_cache : a.v_cache);
            for (int rep = 0; rep < group; ++rep)
                store_pair(cache + kv_offset(sid, slot, hh * group + rep, a.num_streams, a.capacity) + 2 * lane, x);
        }
    }
}

}  // namespace

void launch_score_plan(const ScorePlanArgs& a, bool in_bf16, bool cache_bf16, cudaStream_t s) {
    const dim3 grid(a.n_rows + (a.n_units > 0 ? 1 : 0)), block(kPlanThreads);
    if (in_bf16 && cache_bf16) launch_k(score_plan_kernel<__nv_bfloat16, __nv_bfloat16>, grid, block, 0, s, a);
    else if (in_bf16) launch_k(score_plan_kernel<__nv_bfloat16, float>, grid, block, 0, s, a);
    else if (cache_bf16) launch_k(score_plan_kernel<float, __nv_bfloat16>, grid, block, 0, s, a);
    else launch_k(score_plan_kernel<float, float>, grid, block, 0, s, a);
}

}  // namespace ptts

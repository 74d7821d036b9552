// Attention with score rules for a few rows per stream over its whole cache (drafted trees, short
// prompts on long caches), bf16 caches: blocks of up to 64 rows of one sequence, split over the keys,
// on tcgen05 with the keys as the tall side.
//
// Bound by HBM: a block's keys and values are read once for all its rows. Per key and head 256 bytes
// arrive, about 11 cycles of an SM's share of HBM. With rows as an MMA's M side, half or more of its
// 128 rows would be empty, and mma.sync (2048 flops a cycle and SM) needs those 11 cycles for 64 rows
// alone; so keys are M and rows are N, which a call pays for in steps of 16:
//   S^T = K Q^T     128 keys x N rows, q as a bf16 hi/lo pair: 2 x 2 N cycles
//   O^T += V^T P^T  (64 dims and a row of ones) x N rows over 128 keys: 4 N cycles; the ones give the
//                   rows' sums of P beside their products, in lane 64
// At N = 64 that is 4 cycles a key, and the softmax 4 (64 exp2 at 16 a cycle), side by side.
//
// Work split as in attn_decode.cu: the blocks' keys lie end to end, each at its cost (score.h: ranges of
// equal keys end 64 to 106 us after their start, of equal cost 73 to 92), and every CTA takes an equal range,
// for two heads (f32 outputs: one), each head a pipeline of its own:
//   warps 0-3, 4-7  a thread per key (TMEM lane) of the head's 128-key item, its scores against all rows
//                   in registers: rules, mask, exp2 against the rows' maxima in shared memory, P^T as
//                   bf16 into shared memory (key by key, rows adjacent: the MMA's B operand). No sums and
//                   no maxima cross threads, unless a score passes its row's maximum by 2^8: then the
//                   128 threads take the item's maxima (an integer reduction per row) and rescale O.
//                   Caps up to kScoreBoundedCap need no maxima at all (see attn_score_prompt.cu).
//   warps 8, 9      one lane each issues a head's MMAs; the next item's S starts when this one's scores
//                   are in registers.
//   warp 10         one lane copies the heads' Q tiles and K and V items by TMA, two slots each.
// Measured (one B200, 8 heads, bf16): 128 streams of 64-2048 cached rows with trees of 8-64 nodes, cap 30,
// 107 us a call, about 85 of them this kernel (an item 1.2 us at 16 rows, 2.1 at 64, 1.46 at HBM's rate; a
// block's start and end 4-6 that nothing overlaps); 4 full trees over 20000-33000 rows, 77 us a call. Rows
// as M on mma.sync took 213 and 125 where this form then took 129 and 87.
// A block inside one CTA's range is written at once; the pieces of a cut block leave (max, sum, acc)
// records that a second kernel joins, one warp per row and head: 64 rows x 8 heads are too many for
// the warp that finishes last.
//
// f32 outputs hold P as a bf16 hi/lo pair in two tiles; bf16 outputs round P once to bf16, as the output
// itself is rounded. An item that some row does not see whole has a bit per row in each key's thread, and
// takes values that are not finite out of the V tile (0 x NaN is NaN); rows that see such a value get it
// back at the piece's end, from the cache.
#include <type_traits>

#include "common.cuh"
#include "fa_tc.cuh"
#include "score.cuh"
#include "score.h"

namespace ptts {
namespace {

constexpr int KT = 128;                 // keys per item
constexpr int NR = kTreeNodes;          // rows per block at most
constexpr int kTile = KT * 128;         // a K, V, P or ones tile: 128 keys x 64 bf16
constexpr int kQTile = NR * 128;        // a plane of a head's q
constexpr int kSlots = 2;
// 8 softmax warps, 2 MMA issuers, a producer, a spare. The softmax holds 64 scores a thread: its two
// warpgroups take most of the launch's 384 x 168 registers.
constexpr int kThreadsR = 12 * 32, kRegsR = 168, kRegsSoft = 232, kRegsRest = 40;
static_assert(256 * kRegsSoft + 128 * kRegsRest <= kThreadsR * kRegsR, "the split fits the launch");
constexpr float kRaiseR = 8.f;

// Shared memory of a CTA of HC heads with PT P tiles a head (1024-aligned tiles).
template <int HC, int PT>
struct Smem {
    static constexpr int kQ = 0;                                  // head: hi, lo
    static constexpr int kK = kQ + HC * 2 * kQTile;               // head, slot
    static constexpr int kV = kK + HC * kSlots * kTile;
    static constexpr int kP = kV + HC * kSlots * kTile;           // head, tile
    static constexpr int kOnes = kP + HC * PT * kTile;            // past every V slot (an MMA's offset is positive)
    static constexpr int kRows = kOnes + kTile;
    static constexpr int kBytes = 1024 + kRows + HC * 4096;
};
// A head's rows of the block at hand.
struct HeadRows {
    float m[NR], shift[NR], scale[NR], pos[NR], sum[NR];  // pos: less the first row's
    int lo[NR], hi[NR], top[NR], has[NR];  // has: the row has a maximum (or sees nothing)
    unsigned long long lineage[NR];
    int bad;
};
static_assert(sizeof(HeadRows) <= 4096 - 512, "rows and barriers of a head");
// Barriers of a head. Single buffers for S, P, O and Q: item i completes phase i of sfull, sfree, pfull
// and odone, piece k phase k of qready and qfree; every waiter asks for every phase in turn.
struct HeadBars {
    uint64_t kfull[kSlots], kempty[kSlots], vfull[kSlots], vempty[kSlots], qready, qfree, sfull, sfree, pfull, odone;
};
static_assert(sizeof(HeadBars) <= 512, "rows and barriers of a head");

constexpr uint32_t kIdescBase = (1u << 4) | (1u << 7) | (1u << 10) | (8u << 24);  // f32 += bf16 x bf16, M = 128

// Whether `v` held in any of a head's 128 softmax threads (named barrier 1 + head): they all come here.
__device__ __forceinline__ bool head_any(int hl, bool v) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, %2, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"((uint32_t)v), "r"(1 + hl)
        : "memory");
    return any != 0;
}
// Floats in an order that integers share (NaN below everything).
__device__ __forceinline__ int ordered(float x) {
    const int i = __float_as_int(fmaxf(x, kScoreLow));
    return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }

// The CTA's pieces in order, the same walk for every role: block u, its keys s0 .. s1 - 1 of it.
struct Walk {
    const ScoreRowsArgs& a;
    long long start, end;
    int u;
    int s0, s1, lo, row0, nrows;
    bool whole, begins;
    __device__ Walk(const ScoreRowsArgs& a_, int c, long long total, int G)
        : a(a_), start(cta_start(c, total, G)), end(cta_start(c + 1, total, G)), u(a_.cta_first[c] - 1) {}
    __device__ bool next() {
        while (++u < a.n_units) {
            const long long pb = a.prefix[u], pe = a.prefix[u + 1];
            if (pb >= end) return false;
            row0 = a.blocks[u].x;
            nrows = a.blocks[u].y;
            const unsigned cost = score_key_cost(nrows), keys = (unsigned)(pe - pb - kScoreBlockCost) / cost;
            s0 = start > pb ? (int)min(keys, (unsigned)(start - pb) / cost) : 0;
            s1 = (int)min(keys, (unsigned)(end - pb) / cost);
            if (s0 >= s1) continue;  // its keys are other CTAs'
            begins = s0 == 0;
            whole = begins && s1 == (int)keys;
            lo = a.unit_lo[u];
            return true;
        }
        return false;
    }
    __device__ int items() const { return (s1 - s0 + KT - 1) / KT; }
};

// The values of the piece's keys that are not finite, from the cache, for one dim of the rows that see them
// (rows r0 .. r0 + 15).
__device__ __forceinline__ void add_not_finite(const ScoreRowsArgs& a, const HeadRows& R, const Walk& w, int base_slot,
                                               int head, int dim, int r0, float* o) {
    const int sid = max(a.rows.stream[w.row0], 0);
    const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.v_cache) + kv_offset(sid, w.lo, head, a.num_streams, a.capacity) + dim;
#pragma unroll 1
    for (int j = w.s0; j < w.s1; ++j) {
        const float x = __bfloat162float(v[(long long)j * kRowWidth]);
        if (isfinite(x)) continue;
        const int slot = w.lo + j, node = slot - base_slot;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = r0 + i;
            if (r < w.nrows && slot >= R.lo[r] && slot <= R.hi[r] && (node < 0 || (R.lineage[r] >> node & 1))) o[i] += x;
        }
    }
}

template <int HC, int CAP, bool BOUNDED, bool P2>
__global__ void __launch_bounds__(kThreadsR, 1) score_rows_kernel(ScoreRowsArgs a, const __grid_constant__ CUtensorMap tm_k,
                                                                 const __grid_constant__ CUtensorMap tm_v,
                                                                 const __grid_constant__ CUtensorMap tm_qh,
                                                                 const __grid_constant__ CUtensorMap tm_ql) {
    using L = Smem<HC, P2 ? 2 : 1>;
    constexpr uint32_t kCols = HC * 128;  // per head: S in 64 columns, O in 64
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* sm = smem_raw + (base - raw);
    __shared__ uint32_t s_tmem;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    auto rows_of = [&](int hl) { return reinterpret_cast<HeadRows*>(sm + L::kRows + hl * 4096); };
    auto bars_of = [&](int hl) { return reinterpret_cast<HeadBars*>(sm + L::kRows + hl * 4096 + 4096 - 512); };
    if (tid < HC) {
        HeadBars* b = bars_of(tid);
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&b->kfull[i], 1);
            mbar_init(&b->kempty[i], 1);
            mbar_init(&b->vfull[i], 1);
            mbar_init(&b->vempty[i], 1);
        }
        mbar_init(&b->qready, 1);
        mbar_init(&b->qfree, 1);
        mbar_init(&b->sfull, 1);
        mbar_init(&b->sfree, 4);
        mbar_init(&b->pfull, 4);
        mbar_init(&b->odone, 1);
        rows_of(tid)->bad = 0;
        fence_mbar_init();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // The ones: dim 0 of every key is 1, the others 0 (swizzled: chunk 0 of key k is at chunk k % 8).
    for (int i = tid; i < kTile / 16; i += kThreadsR) {
        const int key = i >> 3, chunk = (i & 7) ^ (key & 7);
        reinterpret_cast<uint4*>(sm + L::kOnes)[i] = make_uint4(chunk == 0 ? 0x3f80u : 0u, 0u, 0u, 0u);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    fa_before();
    __syncthreads();
    fa_after();
    const uint32_t tmem = s_tmem;
    grid_dep_wait();
    grid_dep_launch();
    const long long total = a.prefix[a.n_units];
    const int G = score_ctas(total, gridDim.x), c = blockIdx.x;
    const int head0 = blockIdx.y * HC;
    const bool idle = c >= G;

    if (warp < 4 * HC) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoft));
        // ---- softmax: thread = key ----------------------------------------------------------------
        const int hl = warp >> 2, key = tid & 127, head = head0 + hl;
        HeadRows* R = rows_of(hl);
        HeadBars* b = bars_of(hl);
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 128 * hl;
        const bool biased = a.rule.slopes != nullptr;
        const float slope = biased ? a.rule.slopes[head] * kScoreLog2e : 0.f;
        unsigned char* pt = sm + L::kP + hl * (P2 ? 2 : 1) * kTile + key * 128;
        bool ok = true;
        int i = 0;  // items of this CTA so far
        Walk w(a, idle ? 0 : c, total, G);
        // A wait that gives up clears `ok`; the head's other warps learn of it at their next barrier,
        // and all leave there.
        while (!idle && w.next()) {
            // The block's rows.
            const int base_slot = a.rows.lineage ? a.rows.base[w.row0] : 0x7fffffff;
            // Positions for the bias count from the block's first row: the block's rows are near it, so the
            // distances of near keys are exact in f32 wherever the block is (positions past 2^24 are not).
            const int origin = a.rows.pos[w.row0];
            if (key < NR) {
                const bool there = key < w.nrows;
                const int row = w.row0 + (there ? key : 0);
                const int lo = there ? a.rows.lo[row] : 0, hi = there ? a.rows.hi[row] : -1, pos = a.rows.pos[row];
                R->lo[key] = lo;
                R->hi[key] = hi;
                R->pos[key] = (float)(pos - origin);
                R->lineage[key] = there && a.rows.lineage ? a.rows.lineage[row] : 0;
                // BOUNDED: exp2 against the row's greatest bias (a node sees positions lo .. its own), and
                // three quarters of the cap, which cap_fast takes off. Else the
                // row's first scores set m.
                R->m[key] = BOUNDED && biased ? most_bias(slope, pos, lo, a.rows.lineage ? min(hi, pos) : hi) : 0.f;
                R->has[key] = lo > hi;
            }
            bool fresh = !BOUNDED;  // some row has no maximum yet
            if (head_any(hl, !ok)) break;
            // Rows lane and 32 + lane: what they see, and the slots that every row sees.
            int full_lo = 0, full_hi = 0x7fffffff, row_lo[2], row_hi[2];
            unsigned long long row_line[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int r = 32 * x + lane;
                row_lo[x] = R->lo[r], row_hi[x] = R->hi[r], row_line[x] = R->lineage[r];
                if (r < w.nrows) full_lo = max(full_lo, row_lo[x]), full_hi = min(full_hi, min(row_hi[x], base_slot - 1));
            }
            full_lo = __reduce_max_sync(0xffffffffu, full_lo);
            full_hi = __reduce_min_sync(0xffffffffu, full_hi);
            const int n = w.items(), groups = (w.nrows + 15) / 16;
            for (int it = 0; it < n; ++it, ++i) {
                const int slot0 = w.lo + w.s0 + it * KT, slot = slot0 + key;
                const int count = min(KT, w.s1 - w.s0 - it * KT);  // keys of this item in this CTA's range
                const bool whole = count == KT && slot0 >= full_lo && slot0 + KT - 1 <= full_hi;
                // Rows that see this thread's key, a bit each: every lane has its two rows' 32 keys of the
                // warp, and 32 ballots turn rows of keys into keys of rows.
                uint32_t seen[2] = {~0u, ~0u};
                if (!whole) {
                    const int mine = slot0 + 32 * (warp & 3), last = w.lo + w.s1 - 1;  // the warp's first key; the range's last
                    const int past_base = mine - base_slot;                           // the first key's node, if not negative
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        if (32 * y >= w.nrows) {
                            seen[y] = 0;
                            continue;
                        }
                        const int from = row_lo[y] - mine, to = min(row_hi[y], last) - mine;
                        uint32_t keys = (from <= 0 ? ~0u : from > 31 ? 0u : ~0u << from) & (to >= 31 ? ~0u : to < 0 ? 0u : ~0u >> (31 - to));
                        if (past_base > -32) {  // cached keys, then nodes in the row's lineage
                            const unsigned long long line = past_base >= 0 ? (past_base < NR ? row_line[y] >> past_base : 0ull)
                                                                           : row_line[y] << -past_base | ((1ull << -past_base) - 1);
                            keys &= (uint32_t)line;
                        }
#pragma unroll 8
                        for (int k = 0; k < 32; ++k) {
                            const uint32_t rows = __ballot_sync(0xffffffffu, keys >> k & 1);
                            if (lane == k) seen[y] = rows;
                        }
                    }
                }
                float at = (float)(slot - origin);  // the key's position
                if (biased && slot >= base_slot) at = R->pos[min(slot - base_slot, NR - 1)];
                ok = ok && __all_sync(0xffffffffu, mbar_wait(&b->sfull, i & 1));
                float s[NR];
                float past = -INFINITY;  // how far the scores pass their rows' maxima
                if (ok) {
                    fa_after();
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        if (g < groups) ld16(lanes + 16 * g, s + 16 * g);
                    fa_wait_ld();
                    fa_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&b->sfree);
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        if (g >= groups) continue;
                        float* x = s + 16 * g;
                        if (CAP == kCapFast) cap_fast<16, false, BOUNDED>(x, a.rule.cap);  // (a vote of the warp: tree_batch 113 us, 107 so)
                        if (CAP == kCapExact) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) x[j] = cap_exact(x[j], a.rule.cap);
                        }
                        if (biased) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) x[j] = fmaf(-slope, fabsf(R->pos[16 * g + j] - at), x[j]);
                        }
                        if (!whole) {
                            const uint32_t bits = seen[g >> 1] >> (16 * (g & 1));
#pragma unroll
                            for (int j = 0; j < 16; ++j) x[j] = bits >> j & 1 ? x[j] : -INFINITY;
                        }
                        // From here on the scores are past their rows' maxima (or BOUNDED's references, m = 0 without a bias).
                        if (!BOUNDED || biased) {
#pragma unroll
                            for (int j = 0; j < 16; j += 4) {
                                const float4 m = *reinterpret_cast<const float4*>(&R->m[16 * g + j]);
                                x[j] -= m.x, x[j + 1] -= m.y, x[j + 2] -= m.z, x[j + 3] -= m.w;
                            }
                        }
                        if (!BOUNDED) {
#pragma unroll
                            for (int j = 0; j < 16; j += 2) past = fa_max3(past, x[j], x[j + 1]);
                        }
                    }
                }
                if (!BOUNDED && (head_any(hl, !ok || past > kRaiseR) || fresh)) {
                    // The item's most past each row's maximum: 32 rows over a warp's keys by halving, each lane
                    // left with one row, then over the warps. It becomes the maximum of rows that have none, and raises
                    // rows that it passes by more than kRaiseR.
                    if (key < NR) R->top[key] = ordered(kScoreLow);
                    if (head_any(hl, !ok)) break;
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        if (2 * y >= groups) continue;
                        float v[16];
                        const bool up = lane & 16;
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const bool both = 2 * y + 1 < groups;  // a half group of rows that are not there: lowest
                            const float lo = s[32 * y + j], hi = both ? s[32 * y + 16 + j] : kScoreLow;
                            v[j] = fmaxf(up ? hi : lo, __shfl_xor_sync(0xffffffffu, up ? lo : hi, 16));
                        }
#pragma unroll
                        for (int d = 8; d > 0; d >>= 1) {
                            const bool u = lane & d;
#pragma unroll
                            for (int j = 0; j < d; ++j) {
                                const float lo = v[j], hi = v[j + d];
                                v[j] = fmaxf(u ? hi : lo, __shfl_xor_sync(0xffffffffu, u ? lo : hi, d));
                            }
                        }
                        atomicMax(&R->top[32 * y + lane], ordered(v[0]));
                    }
                    head_any(hl, false);
                    if (key < NR) {
                        const float x = unordered(R->top[key]);
                        const bool first = !R->has[key] && x > kScoreLow, raise = R->has[key] && x > kRaiseR;
                        R->shift[key] = first || raise ? x : 0.f;
                        R->scale[key] = raise ? score_exp2(-x) : 1.f;
                        if (first || raise) R->m[key] += x;
                        if (first) R->has[key] = 1;
                    }
                    if (fresh) fresh = head_any(hl, key < w.nrows && key < NR && !R->has[key & (NR - 1)]);
                    if (it > 0) ok = __all_sync(0xffffffffu, mbar_wait(&b->odone, (i - 1) & 1));
                    if (head_any(hl, !ok)) break;
                    if (it > 0) {  // O of the piece's items before this one
                        fa_after();
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            if (g >= groups) continue;
                            float o[16];
                            uint32_t x[16];
                            ld16(lanes + 64 + 16 * g, o);
                            fa_wait_ld();
#pragma unroll
                            for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(o[j] * R->scale[16 * g + j]);
                            st16(lanes + 64 + 16 * g, x);
                        }
                        wait_st();
                    }
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        if (g >= groups) continue;
#pragma unroll
                        for (int j = 0; j < 16; ++j) s[16 * g + j] -= R->shift[16 * g + j];
                    }
                } else if (i > 0) {  // P V of the item before has read P
                    ok = ok && __all_sync(0xffffffffu, mbar_wait(&b->odone, (i - 1) & 1));
                }
                if (ok) {
                    fa_after();
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        if (g >= groups) continue;
                        uint32_t hi[8], lo[P2 ? 8 : 1];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float e0 = score_exp2(s[16 * g + 2 * j]), e1 = score_exp2(s[16 * g + 2 * j + 1]);
                            hi[j] = pack_bf16x2(e0, e1);
                            if constexpr (P2) lo[j] = pack_bf16x2(e0 - bf16lo(hi[j]), e1 - bf16hi(hi[j]));
                        }
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const int chunk = (2 * g + q) ^ (key & 7);
                            *reinterpret_cast<uint4*>(pt + 16 * chunk) = make_uint4(hi[4 * q], hi[4 * q + 1], hi[4 * q + 2], hi[4 * q + 3]);
                            if constexpr (P2)
                                *reinterpret_cast<uint4*>(pt + kTile + 16 * chunk) = make_uint4(lo[4 * q], lo[4 * q + 1], lo[4 * q + 2], lo[4 * q + 3]);
                        }
                    }
                    if (!whole) {
                        ok = __all_sync(0xffffffffu, mbar_wait(&b->vfull[i % kSlots], (i / kSlots) & 1));
                        if (ok) clean_v<8>(sm + L::kV + (hl * kSlots + i % kSlots) * kTile, key, 0, (seen[0] | seen[1]) == 0, &R->bad);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // P, and V where it was cleaned
                    fa_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&b->pfull);
                }
            }
            // The piece's end: O^T has a dim a lane (threads 0-63), the rows' sums in lane 64.
            ok = ok && __all_sync(0xffffffffu, mbar_wait(&b->odone, (i - 1) & 1));
            if (ok && (warp & 3) == 2) {
                fa_after();
#pragma unroll 1
                for (int g = 0; g < groups; ++g) {
                    float o[16];
                    ld16(lanes + 64 + 16 * g, o);
                    fa_wait_ld();
                    if (lane == 0) {
#pragma unroll
                        for (int j = 0; j < 16; j += 4)
                            *reinterpret_cast<float4*>(&R->sum[16 * g + j]) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                    }
                }
                __syncwarp();
                // As factors of a finished block's rows: zeros for those that see nothing.
                for (int r = lane; w.whole && r < NR; r += 32) R->sum[r] = R->sum[r] == 0.f ? 0.f : 1.f / R->sum[r];
            }
            if (head_any(hl, !ok)) {
                ok = false;
                break;
            }
            if (key < NR) {
                fa_after();
                const bool bad = R->bad != 0;
                const long long at = (long long)w.row0 * a.ld + head * kHeadDim + key;
                // Record 2 c of a piece that began before this CTA's range, 2 c + 1 of one that begins in it.
                float* rec = a.part + ((long long)(2 * c + (w.begins ? 1 : 0)) * a.heads + head) * a.most_rows * kPartStride;
                // Rolled: code that runs once a piece costs more to fetch than to run.
#pragma unroll 1
                for (int g = 0; g < groups; ++g) {
                    float o[16];
                    ld16(lanes + 64 + 16 * g, o);
                    fa_wait_ld();
                    if (bad) add_not_finite(a, *R, w, base_slot, head, key, 16 * g, o);
                    const int rows = w.nrows - 16 * g;  // of these 16
                    if (w.whole) {
                        using Out = typename std::conditional<P2, float, __nv_bfloat16>::type;
                        Out* out = static_cast<Out*>(a.out) + at + (long long)(16 * g) * a.ld;
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            const float4 f = *reinterpret_cast<const float4*>(&R->sum[16 * g + j]);
                            o[j] *= f.x, o[j + 1] *= f.y, o[j + 2] *= f.z, o[j + 3] *= f.w;
                        }
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (j < rows) out[j * a.ld] = from_f32<Out>(o[j]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (j < rows) rec[(16 * g + j) * kPartStride + key] = o[j];
                    }
                }
                fa_before();  // O is read before the next piece's first P V (through pfull)
                if (!w.whole && key < w.nrows)
                    *reinterpret_cast<float2*>(rec + key * kPartStride + NR) =
                        make_float2(BOUNDED || R->has[key] ? R->m[key] : kScoreLow, R->sum[key]);
            }
            head_any(hl, false);  // the rows' arrays are the next block's from here
        }
        if (!ok && lane == 0) set_error(a.err, DEV_ERR_TIMEOUT);
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsRest));
      if ((warp == 8 || warp == 8 + HC - 1) && lane == 0 && !idle) {
        // ---- MMA issuer of a head -------------------------------------------------------------------
        const int hl = warp - 8;
        HeadBars* b = bars_of(hl);
        const uint32_t ts = tmem + 128 * hl, to = ts + 64;
        const uint32_t q = base + L::kQ + hl * 2 * kQTile, k = base + L::kK + hl * kSlots * kTile,
                       v = base + L::kV + hl * kSlots * kTile, p = base + L::kP + hl * (P2 ? 2 : 1) * kTile;
        auto k_full = [&](int i) { return &b->kfull[i % kSlots]; };
        auto issue_s = [&](int i, uint32_t rows, bool last) {
            fa_after();
            const uint64_t dk = desc_k(k + (i % kSlots) * kTile), qh = desc_k(q), ql = desc_k(q + kQTile);
            const uint32_t idesc = kIdescBase | rows / 8 << 17;
#pragma unroll
            for (int d = 0; d < 4; ++d) {  // 64 dims, 16 (32 bytes) a step
                fa_mma_ss(ts, dk + 2 * d, qh + 2 * d, idesc, d ? 1u : 0u);
                fa_mma_ss(ts, dk + 2 * d, ql + 2 * d, idesc, 1u);
            }
            fa_commit(&b->sfull);
            fa_commit(&b->kempty[i % kSlots]);
            if (last) fa_commit(&b->qfree);
        };
        auto issue_pv = [&](int i, uint32_t rows, bool first) {
            fa_after();
            const uint32_t vt = v + (i % kSlots) * kTile;
            // A: dims 0-63 of V, then the ones tile, 128-byte rows of keys (both operands MN-major).
            const uint64_t dv = (uint64_t)((vt >> 4) & 0x3FFFu) | ((uint64_t)((base + L::kOnes - vt) >> 4) << 16) |
                                ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
            const uint64_t dp = desc_mn(p);
            const uint32_t idesc = kIdescBase | rows / 8 << 17 | 1u << 15 | 1u << 16;
#pragma unroll
            for (int d = 0; d < 8; ++d) {  // 128 keys, 16 (2048 bytes) a step
                fa_mma_ss(to, dv + 128 * d, dp + 128 * d, idesc, !first || d ? 1u : 0u);
                if (P2) fa_mma_ss(to, dv + 128 * d, dp + (kTile >> 4) + 128 * d, idesc, 1u);
            }
            fa_commit(&b->odone);
            fa_commit(&b->vempty[i % kSlots]);
        };
        bool ok = true;
        int i = 0, piece = 0;
        uint32_t last_rows = 0;   // of the item before, whose P V is still to come
        bool last_first = false;
        auto pv_before = [&]() {
            ok = ok && mbar_wait(&b->pfull, (i - 1) & 1) && mbar_wait(&b->vfull[(i - 1) % kSlots], ((i - 1) / kSlots) & 1);
            if (ok) issue_pv(i - 1, last_rows, last_first);
        };
        Walk w(a, c, total, G);
        for (; ok && w.next(); ++piece) {
            const int n = w.items();
            const uint32_t rows = (uint32_t)((w.nrows + 15) / 16 * 16);
            for (int it = 0; it < n && ok; ++it, ++i) {
                // S goes first where its keys are there; else P V of the item before, then S.
                const bool there = it == 0 || mbar_test_wait(k_full(i), (i / kSlots) & 1);
                if (!there) pv_before();
                ok = ok && mbar_wait(k_full(i), (i / kSlots) & 1) && mbar_wait(&b->qready, piece & 1) &&
                     (i == 0 || mbar_wait(&b->sfree, (i - 1) & 1));
                if (ok) issue_s(i, rows, it == n - 1);
                if (there && it > 0) pv_before();
                last_rows = rows;
                last_first = it == 0;
            }
            pv_before();  // the piece's last
        }
        if (!ok) set_error(a.err, DEV_ERR_TIMEOUT);
      } else if (warp == 10 && lane == 0 && !idle) {
        // ---- producer -------------------------------------------------------------------------------
        bool ok = true;
        int i = 0, piece = 0, q_out = 0, k_out = 0, v_out = 0;  // copies are issued for all heads up to these
        // Item j's keys or values: its 128 rows of the cache from row `at` on.
        auto copy = [&](bool value, int j, int at) {
            const int slot = j % kSlots;
            for (int hl = 0; hl < HC && ok; ++hl) {
                HeadBars* b = bars_of(hl);
                const int head = head0 + hl;
                if (j >= kSlots && !(ok = mbar_wait(value ? &b->vempty[slot] : &b->kempty[slot], ((j / kSlots) & 1) ^ 1))) break;
                uint64_t* full = value ? &b->vfull[slot] : &b->kfull[slot];
                mbar_arrive_expect_tx(full, kTile);
                fa_tma(base + (value ? L::kV : L::kK) + (hl * kSlots + slot) * kTile, value ? &tm_v : &tm_k,
                       head % kGroupHeads * kHeadDim, head / kGroupHeads * a.num_streams * a.capacity + at, full);
                (value ? v_out : k_out) = j * HC + hl + 1;
            }
        };
        // An item's values come after the next item's keys: their slot is free an item later (P V ends where
        // the next softmax begins, S before it), and keys behind that wait would have one item's time to
        // arrive, not two.
        int before = 0;  // where the item before begins
        Walk w(a, c, total, G);
        for (; ok && w.next(); ++piece) {
            const int sid = max(a.rows.stream[w.row0], 0);  // a refused tree reads slot 0 and sees nothing
            for (int hl = 0; hl < HC && ok; ++hl) {
                HeadBars* b = bars_of(hl);
                if (piece > 0 && !(ok = mbar_wait(&b->qfree, (piece - 1) & 1))) break;
                const uint32_t q = base + L::kQ + hl * 2 * kQTile;
                mbar_arrive_expect_tx(&b->qready, 2 * kQTile);
                fa_tma(q, &tm_qh, (head0 + hl) * kHeadDim, w.row0, &b->qready);
                fa_tma(q + kQTile, &tm_ql, (head0 + hl) * kHeadDim, w.row0, &b->qready);
                q_out = piece * HC + hl + 1;
            }
            const int n = w.items(), first = sid * a.capacity + w.lo + w.s0;
            for (int it = 0; it < n && ok; ++it, ++i) {
                copy(false, i, first + it * KT);
                if (i > 0 && ok) copy(true, i - 1, before);
                before = first + it * KT;
            }
        }
        if (i > 0 && ok) copy(true, i - 1, before);
        if (!ok) set_error(a.err, DEV_ERR_TIMEOUT);
        // The last copies into each buffer land before the shared memory goes (a completed phase returns at
        // once). Copy j of a kind is head j % HC's item (or piece) j / HC.
        for (int j = max(0, q_out - HC); j < q_out; ++j) mbar_wait(&bars_of(j % HC)->qready, (j / HC) & 1);
        for (int j = max(0, k_out - HC * kSlots); j < k_out; ++j)
            mbar_wait(&bars_of(j % HC)->kfull[j / HC % kSlots], (j / HC / kSlots) & 1);
        for (int j = max(0, v_out - HC * kSlots); j < v_out; ++j)
            mbar_wait(&bars_of(j % HC)->vfull[j / HC % kSlots], (j / HC / kSlots) & 1);
      }
    }
    fa_before();
    __syncthreads();
    if (warp == 0) {
        fa_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
    }
}

// Joins the pieces of the blocks that CTAs' ranges cut: one warp per row and head, lane = 2 dims.
// Every warp reads the pieces' maxima and sums lane by lane and then all records at once.
// A grid over the blocks, or where they are more than the CTAs' ranges (BY_CUT) over the ranges' beginnings:
// 128 blocks cut by 37 ranges, 115 us a call over the blocks, 110 over the beginnings.
template <bool P2, bool BY_CUT>
__global__ void __launch_bounds__(256) score_rows_merge_kernel(ScoreRowsArgs a, int grid) {
    grid_dep_wait();
    grid_dep_launch();
    const long long total = a.prefix[a.n_units];
    const int G = score_ctas(total, grid), head = blockIdx.y, lane = threadIdx.x & 31;
    const int cut = BY_CUT ? (int)blockIdx.x + 1 : 0;  // CTA `cut`'s range begins in the block, and is its first such
    if (cut >= G) return;
    const int u = BY_CUT ? a.cta_first[cut] : blockIdx.x;
    const long long pb = a.prefix[u], pe = a.prefix[u + 1];
    const int2 rows = a.blocks[u];
    // The CTAs that hold its first key and its last (see Walk).
    const int c0 = cta_of(pb + score_key_cost(rows.y) - 1, total, G), c1 = cta_of(pe - kScoreBlockCost - 1, total, G);
    if (c0 == c1 || (BY_CUT && cut != c0 + 1)) return;
    const int r = blockIdx.z * 8 + (threadIdx.x >> 5);
    if (r >= rows.y) return;
    auto rec = [&](int c) {
        return a.part + (((long long)(2 * c + (c == c0 ? 1 : 0)) * a.heads + head) * a.most_rows + r) * kPartStride;
    };
    float mx = kScoreLow, den = 0.f, x0 = 0.f, x1 = 0.f;
    for (int cb = c0; cb <= c1; cb += 32) {  // a lane's piece's maximum and sum, then all its records
        const int n = min(32, c1 - cb + 1);
        float2 ml = make_float2(kScoreLow, 0.f);
        if (lane < n) ml = *reinterpret_cast<const float2*>(rec(cb + lane) + 64);
        float top = ml.x;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = fmaxf(top, mx);
        const float before = score_exp2(mx - top), w = lane < n ? score_exp2(ml.x - top) : 0.f;
        mx = top;
        den = fmaf(w, ml.y, den * before);
        x0 *= before, x1 *= before;
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const float f = __shfl_sync(0xffffffffu, w, i);
            const float2 v = *reinterpret_cast<const float2*>(rec(cb + i) + 2 * lane);
            x0 = fmaf(f, v.x, x0);
            x1 = fmaf(f, v.y, x1);
        }
    }
    den = warp_sum(den);
    const float inv = den == 0.f ? 0.f : 1.f / den;
    const long long at = (long long)(rows.x + r) * a.ld + head * kHeadDim + 2 * lane;
    if constexpr (P2) *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at) = make_float2(x0 * inv, x1 * inv);
    else *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.out) + at) = pack_bf16x2(x0 * inv, x1 * inv);
}

template <bool P2>
void merge(const ScoreRowsArgs& a, int grid, cudaStream_t s) {
    if (grid == 1) return;
    const bool by_cut = a.n_units >= grid;
    launch_k(by_cut ? score_rows_merge_kernel<P2, true> : score_rows_merge_kernel<P2, false>,
             dim3(by_cut ? grid - 1 : a.n_units, a.heads, (a.most_rows + 7) / 8), dim3(256), 0, s, a, grid);
}

template <int HC, int CAP, bool BOUNDED, bool P2>
void launch_rules(const ScoreRowsArgs& a, const CUtensorMap* m, int grid, cudaStream_t s) {
    auto kernel = score_rows_kernel<HC, CAP, BOUNDED, P2>;
    constexpr int smem = Smem<HC, P2 ? 2 : 1>::kBytes;
    static_assert(smem <= 227 * 1024, "a CTA per SM");
    set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
    launch_k(kernel, dim3(grid, a.heads / HC), dim3(kThreadsR), smem, s, a, m[0], m[1], m[2], m[3]);
    merge<P2>(a, grid, s);
}

}  // namespace

int score_rows_grid(bool out_bf16, int heads, int sms, long long keys, int blocks) {
    const int slabs = heads / (out_bf16 ? 2 : 1);
    return score_ctas(keys * score_key_cost(kTreeNodes) + (long long)blocks * kScoreBlockCost, sms / slabs > 1 ? sms / slabs : 1);
}

size_t score_rows_part_floats(int heads, int grid, int most_rows) { return (size_t)2 * grid * heads * most_rows * kPartStride; }

bool launch_score_rows(const ScoreRowsArgs& a, int grid, cudaStream_t s) {
    CUtensorMap m[4];
    const long long rows = (long long)(a.heads / kGroupHeads) * a.num_streams * a.capacity;
    if (rows >= (1LL << 31) || !bf16_rows_map(&m[0], a.k_cache, rows, kRowWidth, kHeadDim, KT) ||
        !bf16_rows_map(&m[1], a.v_cache, rows, kRowWidth, kHeadDim, KT) ||
        !bf16_rows_map(&m[2], a.q_hi, a.n_rows, a.ld, kHeadDim, NR) || !bf16_rows_map(&m[3], a.q_lo, a.n_rows, a.ld, kHeadDim, NR))
        return false;
    const int cap = score_cap_mode(a.rule.cap, !a.out_bf16);
    if (!a.out_bf16) {
        if (cap == kCapNone) launch_rules<1, kCapNone, false, true>(a, m, grid, s);
        else launch_rules<1, kCapExact, false, true>(a, m, grid, s);
    } else if (cap == kCapNone) {
        launch_rules<2, kCapNone, false, false>(a, m, grid, s);
    } else if (cap == kCapExact) {
        launch_rules<2, kCapExact, false, false>(a, m, grid, s);
    } else if (a.rule.cap <= kScoreBoundedCap) {
        launch_rules<2, kCapFast, true, false>(a, m, grid, s);
    } else {
        launch_rules<2, kCapFast, false, false>(a, m, grid, s);
    }
    return true;
}

}  // namespace ptts

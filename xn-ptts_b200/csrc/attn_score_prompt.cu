// Attention with score rules for prompts, bf16 caches, on tcgen05: one CTA per (tile of up to 128
// query rows of one sequence, head), two CTAs on an SM.
//
// Bound by the softmax's exponentials: a 128 x 128 tile has 16,384 scores for 2 x 2.1 MFLOP, and an
// SM makes 16 exp2 a cycle (1024 cycles a tile) while the tensor cores need 512 cycles for S (q as
// a bf16 hi/lo pair) and 256 for P V. So the products hide behind the softmax of the other CTA on
// the SM, whose items run half a step apart, and one CTA keeps a plain order per 128-key item:
//   warps 0-3  a thread per query row (TMEM lane): S from TMEM, rules and mask, the row's maximum
//              (raised only when a score passes it by 2^8, the one time O is rescaled, in TMEM), P as
//              bf16 into TMEM, the row's sum in f32; at the end O / l to the output.
//   warp 4     one lane issues S = Q K^T (both planes of q) and O += P V with P from TMEM. The next
//              item's S goes ahead of this item's P V: the softmax waits for S alone.
//   warp 5     one lane copies the Q tile once and each item's K and V by TMA into two-slot rings.
// A row per thread leaves nothing to exchange between threads. The scores are read twice from TMEM
// (for the maximum, then for P): keeping 128 of them in registers would leave no room for two CTAs.
// Where a cap up to kBoundedCap bounds the scores there is no maximum pass: exp2 runs against the
// row's nearest key's bias, which the largest score passes by at most cap x log2(e) < 58 either way.
//
// f32 outputs hold P as a bf16 hi/lo pair over the columns of S (its next item waits for P V);
// bf16 outputs round P once to bf16, as the output itself is rounded.
//
// Items start at the first slot any row of the tile sees and end at the last. An item that some row
// does not see whole masks scores by a 32-bit word per 32 keys (32 keys that no row of a warp sees
// are skipped), and takes values that are not finite, or that no row sees, out of the V tile: 0 x
// NaN is NaN. Rows that do see such a value get it back at the end, from the cache.
#include "common.cuh"
#include "fa_tc.cuh"
#include "score.cuh"
#include "score.h"

namespace ptts {
namespace {

constexpr int QT = 128, KT = 128;
constexpr int kMmaW = 4, kLoadW = 5, kThreadsP = 192;
constexpr int kTile = 128 * 128;  // bytes of a Q plane, a K tile or a V tile: 128 rows x 64 bf16
constexpr int kSlots = 2;
constexpr int kOffK = 2 * kTile, kOffV = kOffK + kSlots * kTile, kOffBars = kOffV + kSlots * kTile;
constexpr int kSmemP = 1024 + kOffBars + 256;
static_assert(2 * (kSmemP + 1024 + 1024) <= 228 * 1024, "two CTAs per SM");
constexpr uint32_t kCols = 256, kColS = 0, kColO = 128, kColP = 192;
constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | ((KT / 8) << 17) | (8u << 24);
constexpr uint32_t kIdescPV = (1u << 4) | (1u << 7) | (1u << 10) | (8u << 17) | (8u << 24) | (1u << 16);
constexpr float kRaiseP = 8.f;
constexpr float kBoundedCap = 40.f;  // 40 log2(e) < 58: weights and sums of 2^58 stay far inside f32 and bf16

// Single buffers for S, P and O: item i completes phase i of sfull, pfull and odone, and each waiter
// asks for every phase (or one that the last wait on another implies), so none is two behind.
struct Bars {
    uint64_t qready, kfull[kSlots], kempty[kSlots], vfull[kSlots], vempty[kSlots], sfull, pfull, odone;
};

__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 scores of a row (keys slot .. slot + 31) with the rules: capped, biased, and -inf where `seen`
// has no bit.
template <int CAP, bool BIAS>
__device__ __forceinline__ void apply_rules(float* s, float cap, float slope, float ahead, uint32_t seen) {
    if (CAP == kCapFast) {
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = cap_fast(s[j], cap);
    }
    if (CAP == kCapExact) {
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = cap_exact(s[j], cap);
    }
    if (BIAS) {  // ahead = position - slot
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = fmaf(-slope, fabsf(ahead - (float)j), s[j]);
    }
    if (seen != 0xffffffffu) {
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = seen >> j & 1 ? s[j] : -INFINITY;
    }
}

// The values of slots lo .. hi that are not finite, from the cache, onto 32 dims of a row.
__device__ __forceinline__ void add_not_finite(const ScorePromptArgs& a, int kv_row, int x, int lo, int hi, float* o) {
    const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.v_cache) + ((long long)kv_row + lo) * kRowWidth + x;
    for (int k = lo; k <= hi; ++k, v += kRowWidth)
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const float y = __bfloat162float(v[j]);
            if (!isfinite(y)) o[j] += y;
        }
}

// BOUNDED: the cap bounds the scores, no maximum is taken.
template <int CAP, bool BOUNDED, bool BIAS, bool P2>
__global__ void __launch_bounds__(kThreadsP, 2) score_prompt_kernel(ScorePromptArgs a, const __grid_constant__ CUtensorMap tm_k,
                                                                   const __grid_constant__ CUtensorMap tm_v,
                                                                   const __grid_constant__ CUtensorMap tm_qh,
                                                                   const __grid_constant__ CUtensorMap tm_ql) {
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* sm = smem_raw + (base - raw);
    Bars* b = reinterpret_cast<Bars*>(sm + kOffBars);
    __shared__ uint32_t s_tmem;
    __shared__ int s_lo[4], s_hi[4], s_lo_most[4], s_hi_least[4], s_bad, s_k_issued, s_v_issued;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        mbar_init(&b->qready, 1);
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&b->kfull[i], 1);
            mbar_init(&b->kempty[i], 1);
            mbar_init(&b->vfull[i], 1);
            mbar_init(&b->vempty[i], 1);
        }
        mbar_init(&b->sfull, 1);
        mbar_init(&b->pfull, 4);
        mbar_init(&b->odone, 1);
        s_bad = s_k_issued = s_v_issued = 0;
        fence_mbar_init();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    grid_dep_wait();
    grid_dep_launch();
    const int head = blockIdx.x % a.heads;
    const int2 tile = a.tiles[blockIdx.x / a.heads];
    const int row0 = tile.x, nrows = tile.y;
    // The row of each softmax thread, and the slots the tile's rows see: any (min lo .. max hi) and
    // all (max lo .. min hi).
    int lo = 0, hi = -1;
    const bool there = tid < nrows;
    if (warp < 4) {
        if (there) lo = a.rows.lo[row0 + tid], hi = a.rows.hi[row0 + tid];
        const bool sees = lo <= hi;
        const int x0 = __reduce_min_sync(0xffffffffu, sees ? lo : 0x7fffffff), x1 = __reduce_max_sync(0xffffffffu, sees ? hi : -1);
        const int y0 = __reduce_max_sync(0xffffffffu, there ? lo : 0), y1 = __reduce_min_sync(0xffffffffu, there ? hi : 0x7fffffff);
        if (lane == 0) s_lo[warp] = x0, s_hi[warp] = x1, s_lo_most[warp] = y0, s_hi_least[warp] = y1;
    }
    fa_before();
    __syncthreads();
    fa_after();
    const uint32_t tmem = s_tmem;
    const int first = min(min(s_lo[0], s_lo[1]), min(s_lo[2], s_lo[3]));
    const int end = max(max(s_hi[0], s_hi[1]), max(s_hi[2], s_hi[3])) + 1;
    const int lo_most = max(max(s_lo_most[0], s_lo_most[1]), max(s_lo_most[2], s_lo_most[3]));
    const int hi_least = min(min(s_hi_least[0], s_hi_least[1]), min(s_hi_least[2], s_hi_least[3]));
    const int sid = a.rows.stream[row0];
    const int n = sid < 0 || end <= 0 ? 0 : (end - first + KT - 1) / KT;
    // The head's rows of this stream in the layer: [group][stream][slot] rows of 8 heads.
    const int kv_row = (int)(((long long)(head / kGroupHeads) * a.num_streams + max(sid, 0)) * a.capacity);
    const int kv_x = (head % kGroupHeads) * kHeadDim;

    if (warp < 4) {
        const uint32_t lanes = tmem + ((uint32_t)(32 * warp) << 16);
        const float slope = BIAS ? a.rule.slopes[head] * kScoreLog2e : 0.f;
        const int pos = BIAS && there ? a.rows.pos[row0 + tid] : 0;
        // BOUNDED: exp2 against the bias of the nearest visible key.
        float m = BOUNDED ? (BIAS ? -slope * (float)max(max(lo - pos, pos - hi), 0) : 0.f) : kScoreLow, l = 0.f;
        bool ok = true;
        for (int i = 0; i < n; ++i) {
            const int k0 = first + i * KT;
            ok = __all_sync(0xffffffffu, mbar_wait(&b->sfull, i & 1));
            if (!ok) break;
            fa_after();
            // This row's visible keys of the item, a bit each.
            uint32_t seen[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int x = lo - k0 - 32 * c, y = hi - k0 - 32 * c;  // bits x .. y
                const uint32_t from = x <= 0 ? 0xffffffffu : (x > 31 ? 0u : 0xffffffffu << x);
                const uint32_t to = y >= 31 ? 0xffffffffu : (y < 0 ? 0u : 0xffffffffu >> (31 - y));
                seen[c] = from & to;
            }
            if (!BOUNDED) {
                float mt = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (!__any_sync(0xffffffffu, seen[c] != 0)) continue;
                    float s[32];
                    fa_ld32(lanes + kColS + 32 * c, s);
                    fa_wait_ld();
                    const bool whole = __all_sync(0xffffffffu, seen[c] == 0xffffffffu);
                    apply_rules<CAP, BIAS>(s, a.rule.cap, slope, (float)(pos - k0 - 32 * c), whole ? 0xffffffffu : seen[c]);
                    float m4[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float* sq = s + 8 * q;
                        m4[q] = fa_max3(fa_max3(fa_max3(sq[0], sq[1], sq[2]), sq[3], sq[4]), sq[5], sq[6]);
                        m4[q] = fmaxf(m4[q], sq[7]);
                    }
                    mt = fmaxf(mt, fmaxf(fa_max3(m4[0], m4[1], m4[2]), m4[3]));
                    if (CAP != kCapNone || BIAS) {  // the second pass takes the scores as they are now
                        uint32_t w[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(s[j]);
                        fa_st32(lanes + kColS + 32 * c, w);
                    }
                }
                if (CAP != kCapNone || BIAS) wait_st();
                const bool raise = mt > m + kRaiseP;
                if (__any_sync(0xffffffffu, raise)) {
                    const float mn = raise ? mt : m, f = score_exp2(m - mn);
                    l *= f;
                    m = mn;
                    if (i > 0) {  // O holds the items before this one once their P V is done
                        ok = __all_sync(0xffffffffu, mbar_wait(&b->odone, (i - 1) & 1));
                        if (!ok) break;
                        fa_after();
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float o[32];
                            uint32_t w[32];
                            fa_ld32(lanes + kColO + 32 * c, o);
                            fa_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(o[j] * f);
                            fa_st32(lanes + kColO + 32 * c, w);
                        }
                        wait_st();
                    }
                }
            }
            if (!P2 && i > 0) {  // P V of the item before has read P (a raise has waited for it already)
                ok = __all_sync(0xffffffffu, mbar_wait(&b->odone, (i - 1) & 1));
                if (!ok) break;
                fa_after();
            }
            // P, 32 keys at a time: bf16 pairs into its own columns, or (P2) hi and lo over the 32
            // columns of S that were read just before.
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            const float2 neg_m = make_float2(-m, -m), minus1 = make_float2(-1.f, -1.f);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t ph[16], pl[P2 ? 16 : 1];
                if (!__any_sync(0xffffffffu, seen[c] != 0)) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        ph[j] = 0u;
                        if constexpr (P2) pl[j] = 0u;
                    }
                } else {
                    float s[32];
                    fa_ld32(lanes + kColS + 32 * c, s);
                    fa_wait_ld();
                    if (BOUNDED || (CAP == kCapNone && !BIAS)) {
                        const bool whole = __all_sync(0xffffffffu, seen[c] == 0xffffffffu);
                        apply_rules<CAP, BIAS>(s, a.rule.cap, slope, (float)(pos - k0 - 32 * c), whole ? 0xffffffffu : seen[c]);
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float2 x = __fadd2_rn(make_float2(s[2 * j], s[2 * j + 1]), neg_m);
                        const float2 e = make_float2(score_exp2(x.x), score_exp2(x.y));
                        sum[j & 1] = __fadd2_rn(sum[j & 1], e);
                        ph[j] = pack_bf16x2(e.x, e.y);
                        if constexpr (P2) {
                            const float2 d = __ffma2_rn(make_float2(bf16lo(ph[j]), bf16hi(ph[j])), minus1, e);
                            pl[j] = pack_bf16x2(d.x, d.y);
                        }
                    }
                }
                if constexpr (P2) {
                    st16(lanes + kColS + 32 * c, ph);
                    st16(lanes + kColS + 32 * c + 16, pl);
                } else {
                    st16(lanes + kColP + 16 * c, ph);
                }
            }
            l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
            wait_st();
            if (k0 < lo_most || k0 + KT - 1 > hi_least) {
                // Some row does not see some key: thread = key, its V row cleaned in shared memory.
                ok = __all_sync(0xffffffffu, mbar_wait(&b->vfull[i % kSlots], (i / kSlots) & 1));
                if (!ok) break;
                uint4* v = reinterpret_cast<uint4*>(sm + kOffV + (i % kSlots) * kTile + tid * 128);
                const bool gone = k0 + tid >= end;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint4 w = gone ? make_uint4(0u, 0u, 0u, 0u) : v[c ^ (tid & 7)];
                    const bool bad = drop_not_finite(w.x) | drop_not_finite(w.y) | drop_not_finite(w.z) | drop_not_finite(w.w);
                    if (gone || bad) v[c ^ (tid & 7)] = w;
                    if (bad) s_bad = 1;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            fa_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b->pfull);
        }
        // O / l to the output (zeros for rows that see nothing).
        if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait(&b->odone, (n - 1) & 1));
        if (!ok && lane == 0) set_error(a.err, DEV_ERR_TIMEOUT);
        asm volatile("bar.sync 1, 128;" ::: "memory");  // s_bad of every softmax warp (all come here)
        const bool bad = *const_cast<volatile int*>(&s_bad) != 0;
        if (ok) {
            fa_after();
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const long long at = (long long)(row0 + tid) * a.ld + head * kHeadDim;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float o[32];
                if (n > 0) {
                    fa_ld32(lanes + kColO + 32 * c, o);
                    fa_wait_ld();
                }
                if (there) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = n > 0 ? o[j] * inv : 0.f;
                    if (bad) add_not_finite(a, kv_row, kv_x + 32 * c, lo, hi, o);
                    if constexpr (P2) {
                        float4* out = reinterpret_cast<float4*>(static_cast<float*>(a.out) + at + 32 * c);
#pragma unroll
                        for (int j = 0; j < 8; ++j) out[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                    } else {
                        uint4* out = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + at + 32 * c);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            out[j] = make_uint4(pack_bf16x2(o[8 * j], o[8 * j + 1]), pack_bf16x2(o[8 * j + 2], o[8 * j + 3]),
                                                pack_bf16x2(o[8 * j + 4], o[8 * j + 5]), pack_bf16x2(o[8 * j + 6], o[8 * j + 7]));
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp == kMmaW && lane == 0) {
        // ---- MMA issuer ------------------------------------------------------------------------
        auto issue_s = [&](int i) {
            fa_after();
            const uint64_t qh = desc_k(base), ql = desc_k(base + kTile), dk = desc_k(base + kOffK + (i % kSlots) * kTile);
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // 64 dims, 16 (32 bytes) a step
                fa_mma_ss(tmem + kColS, qh + 2 * k, dk + 2 * k, kIdescS, k ? 1u : 0u);
                fa_mma_ss(tmem + kColS, ql + 2 * k, dk + 2 * k, kIdescS, 1u);
            }
            fa_commit(&b->sfull);
            fa_commit(&b->kempty[i % kSlots]);
        };
        auto issue_pv = [&](int i) {
            fa_after();
            const uint64_t dv = desc_mn(base + kOffV + (i % kSlots) * kTile);
#pragma unroll
            for (int k = 0; k < 8; ++k) {  // 128 keys, 16 a step: 8 columns of P, 16 rows (2048 bytes) of V
                const uint32_t p = P2 ? tmem + kColS + 32 * (k >> 1) + 8 * (k & 1) : tmem + kColP + 8 * k;
                fa_mma_ts(tmem + kColO, p, dv + 128 * k, kIdescPV, (i || k) ? 1u : 0u);
                if (P2) fa_mma_ts(tmem + kColO, p + 16, dv + 128 * k, kIdescPV, 1u);
            }
            fa_commit(&b->odone);
            fa_commit(&b->vempty[i % kSlots]);
        };
        auto k_there = [&](int i) { return mbar_wait(&b->kfull[i % kSlots], (i / kSlots) & 1); };
        bool ok = n == 0 || (mbar_wait(&b->qready, 0) && k_there(0));
        if (ok && n > 0) issue_s(0);
        for (int i = 0; i < n && ok; ++i) {
            ok = mbar_wait(&b->pfull, i & 1);
            if (!P2 && ok && i + 1 < n && (ok = k_there(i + 1))) issue_s(i + 1);
            if (ok && (ok = mbar_wait(&b->vfull[i % kSlots], (i / kSlots) & 1))) issue_pv(i);
            // P lies over S: the next scores wait for P V.
            if (P2 && ok && i + 1 < n && (ok = k_there(i + 1) && mbar_wait(&b->odone, i & 1))) issue_s(i + 1);
        }
        if (!ok) set_error(a.err, DEV_ERR_TIMEOUT);
    } else if (warp == kLoadW && lane == 0 && n > 0) {
        // ---- Q, K and V producer -----------------------------------------------------------------
        mbar_arrive_expect_tx(&b->qready, 2 * kTile);
        fa_tma(base, &tm_qh, head * kHeadDim, row0, &b->qready);
        fa_tma(base + kTile, &tm_ql, head * kHeadDim, row0, &b->qready);
        bool ok = true;
        for (int i = 0; i < n && ok; ++i) {
            const int slot = i % kSlots, y = kv_row + first + i * KT;
            if (i >= kSlots) ok = mbar_wait(&b->kempty[slot], ((i / kSlots) & 1) ^ 1);
            if (!ok) break;
            mbar_arrive_expect_tx(&b->kfull[slot], kTile);
            fa_tma(base + kOffK + slot * kTile, &tm_k, kv_x, y, &b->kfull[slot]);
            s_k_issued = i + 1;
            if (i >= kSlots) ok = mbar_wait(&b->vempty[slot], ((i / kSlots) & 1) ^ 1);
            if (!ok) break;
            mbar_arrive_expect_tx(&b->vfull[slot], kTile);
            fa_tma(base + kOffV + slot * kTile, &tm_v, kv_x, y, &b->vfull[slot]);
            s_v_issued = i + 1;
        }
        if (!ok) set_error(a.err, DEV_ERR_TIMEOUT);
    }
    fa_before();
    __syncthreads();
    if (tid == 0 && n > 0) {
        // The last copies into each slot land before the shared memory goes (a completed phase returns
        // at once).
        mbar_wait(&b->qready, 0);
        for (int i = max(0, s_k_issued - kSlots); i < s_k_issued; ++i) mbar_wait(&b->kfull[i % kSlots], (i / kSlots) & 1);
        for (int i = max(0, s_v_issued - kSlots); i < s_v_issued; ++i) mbar_wait(&b->vfull[i % kSlots], (i / kSlots) & 1);
    }
    if (warp == 0) {
        fa_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
    }
}

template <int CAP, bool BOUNDED, bool P2>
void launch_bias(const ScorePromptArgs& a, const CUtensorMap* m, cudaStream_t s) {
    auto go = [&](auto kernel) {
        set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), kSmemP);
        launch_k(kernel, dim3((unsigned)(a.n_tiles * a.heads)), dim3(kThreadsP), kSmemP, s, a, m[0], m[1], m[2], m[3]);
    };
    if (a.rule.slopes) go(score_prompt_kernel<CAP, BOUNDED, true, P2>);
    else go(score_prompt_kernel<CAP, BOUNDED, false, P2>);
}

}  // namespace

bool launch_score_prompt(const ScorePromptArgs& a, cudaStream_t s) {
    CUtensorMap m[4];
    const long long rows = (long long)(a.heads / kGroupHeads) * a.num_streams * a.capacity;
    if (rows >= (1LL << 31) || !bf16_rows_map(&m[0], a.k_cache, rows, kRowWidth, kHeadDim, KT) ||
        !bf16_rows_map(&m[1], a.v_cache, rows, kRowWidth, kHeadDim, KT) ||
        !bf16_rows_map(&m[2], a.q_hi, a.n_rows, a.ld, kHeadDim, QT) || !bf16_rows_map(&m[3], a.q_lo, a.n_rows, a.ld, kHeadDim, QT))
        return false;
    const int cap = score_cap_mode(a.rule.cap, !a.out_bf16);
    if (!a.out_bf16) {
        if (cap == kCapNone) launch_bias<kCapNone, false, true>(a, m, s);
        else launch_bias<kCapExact, false, true>(a, m, s);
    } else if (cap == kCapNone) {
        launch_bias<kCapNone, false, false>(a, m, s);
    } else if (cap == kCapExact) {
        launch_bias<kCapExact, false, false>(a, m, s);
    } else if (a.rule.cap <= kBoundedCap) {
        launch_bias<kCapFast, true, false>(a, m, s);
    } else {
        launch_bias<kCapFast, false, false>(a, m, s);
    }
    return true;
}

}  // namespace ptts

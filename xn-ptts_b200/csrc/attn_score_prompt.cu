// Attention with score rules for prompts, bf16 caches, on tcgen05: one CTA per (tile of up to 128
// query rows of one sequence, 1 to 8 heads one after another), two CTAs on an SM.
//
// Bound by the softmax: a 128 x 128 tile has 16,384 scores for 2 x 2.1 MFLOP. An SM makes 16 exp2 a
// cycle (1024 cycles a tile) and issues 4 to 9 instructions a score on 128 lanes (500 to 1200),
// while the tensor cores need 512 cycles for S (q as a bf16 hi/lo pair) and 256 for P V.
//   warps 0-7  two threads per query row (TMEM lane), 64 of the item's 128 keys and 32 dims each: the
//              scores from TMEM into registers, rules and mask, the row's maximum (the halves agree by
//              one barrier that it stays; it is raised, and O rescaled in TMEM, only when a score passes
//              it by 2^8), P as bf16 into TMEM, the row's sum in f32; at a head's end O / l to the output.
//   warp 8     one lane issues S = Q K^T (both planes of q) and O += P V with P from TMEM. The next
//              item's S starts as soon as the softmax holds this one's in registers.
//   warp 9     one lane copies each head's Q tile and each item's K and V (128 keys) by TMA, K and V
//              in two-slot rings, so the next head's data come during this head's last item.
// Measured (one B200, bf16): 96 streams of 200-900 rows in documents, cap 30, 8 heads, 140 us (issue 39 %,
// tensor 20 %); 4 streams of 3900-4096 rows, 16 heads, a distance bias, 300 us (exp2 43 %, issue 48 %,
// tensor 35 %: 430 TFLOP/s of the products that count). A thread a row: 172 and 318; two tiles a CTA
// sharing K and V: 167 and 373.
// Two threads a row and two CTAs an SM make four softmax warps a scheduler, which fill each other's
// waits (with a thread a row, half as many, the issue slots were 35 to 46 % used). Where a cap up to
// kScoreBoundedCap bounds the scores there is no maximum: exp2 runs against the row's greatest bias and
// three quarters of the cap, which a score is from 81 below to 12 above. Items run from the last keys to
// the first: a causal row's nearest keys, whose bias is the least, set the maximum at once.
//
// f32 outputs hold P as a bf16 hi/lo pair over the columns of S (its next item waits for P V);
// bf16 outputs round P once to bf16, as the output itself is rounded.
//
// Items start at the first slot any row of the tile sees and end at the last. An item that some row
// does not see whole masks scores by a 32-bit word per 32 keys (32 keys that no row of a warp sees are
// passed over), and takes values that are not finite,
// or that no row sees, out of the V tile: 0 x NaN is NaN. Rows that do see such a value get it back at
// the end, from the cache.
#include "common.cuh"
#include "fa_tc.cuh"
#include "score.cuh"
#include "score.h"

namespace ptts {
namespace {

constexpr int QT = 128, KT = 128;
constexpr int kSoftW = 8, kMmaW = kSoftW, kLoadW = kSoftW + 1, kThreadsP = (kSoftW + 2) * 32;
constexpr int kTile = 128 * 128;  // bytes of a Q plane, a K tile or a V tile: 128 rows x 64 bf16
constexpr int kSlots = 2;
constexpr int kOffK = 2 * kTile, kOffV = kOffK + kSlots * kTile, kOffBars = kOffV + kSlots * kTile;
constexpr int kOffKx = kOffBars + 1024, kOffQx = kOffKx + 4096;  // the bias operands: 128 rows of 16 bf16 each
constexpr int kSmemP = 1024 + kOffQx + 4096;
constexpr int kStaticP = 4608;  // s_xmax, s_xsum and the small ones
static_assert(2 * (kSmemP + kStaticP + 1024) <= 228 * 1024, "two CTAs per SM");
constexpr uint32_t kCols = 256, kColS = 0, kColO = 128, kColP = 192;
constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | ((KT / 8) << 17) | (8u << 24);
constexpr uint32_t kIdescPV = (1u << 4) | (1u << 7) | (1u << 10) | (8u << 17) | (8u << 24) | (1u << 16);
constexpr float kRaiseP = 8.f;

// Single buffers for S, P and O: item i completes phase i of sfull, sfree, pfull and odone, head hh
// phase hh of qready and qfree, and each waiter asks for every phase (or for one that its last wait on
// another implies), so none is two behind.
struct Bars {
    uint64_t qready, kfull[kSlots], kempty[kSlots], vfull[kSlots], vempty[kSlots], qfree, sfull, sfree, pfull, odone;
};

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

// Named barrier 1 + quarter over the two softmax warps of 32 rows: whether `v` held in any thread.
__device__ __forceinline__ bool pair_any(int quarter, bool v) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, %2, 64, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"((uint32_t)v), "r"(1 + quarter)
        : "memory");
    return any != 0;
}
// K-major, 32-byte swizzle (8-row groups 256 B apart): the bias operands.
__device__ __forceinline__ uint64_t desc_x(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)1u << 16) | ((uint64_t)(256 >> 4) << 32) |
           ((uint64_t)1u << 46) | ((uint64_t)6u << 61);
}
// Row r of a bias operand: three values, then zeros.
__device__ __forceinline__ void put_x(unsigned char* x, int r, uint32_t v01, uint32_t v2) {
    uint4* row = reinterpret_cast<uint4*>(x + 32 * r);
    row[r >> 2 & 1] = make_uint4(v01, v2, 0u, 0u);
    row[(r >> 2 & 1) ^ 1] = make_uint4(0u, 0u, 0u, 0u);
}

// 32 scores of a row: capped, biased (`ahead` = position - first key), -inf where `seen` has no bit.
// Without a cap the products have added slope x (key's place in the item) already, which is the bias up to
// a constant per row as long as no visible key is ahead of the row; `over`: some may be.
template <int CAP, bool BOUNDED, bool BIAS>
__device__ __forceinline__ void rules(float* s, float cap, float slope, int ahead, bool over, uint32_t seen) {
    const bool some = __any_sync(0xffffffffu, seen != 0xffffffffu);  // a key of some row of the warp's is not seen
    // The fast tanh's form by each row, or by the warp (see cap_fast), measured against a vote over all scores,
    // seen or not, of 231 us (documents, cap 30), 232 (and a bias), 298 (cap 50), 406 and 660 (long prompts with
    // a bias, caps 30 and 50): by row 225, 241, 315, 424, 680; by warp 249, 250, 298, 406, 678.
    if (CAP == kCapFast && BOUNDED) {
        if (some) {
#pragma unroll
            for (int j = 0; j < 32; ++j) s[j] = seen >> j & 1 ? s[j] : 0.f;
        }
        cap_fast<32, false, true>(s, cap);
    }
    if (CAP == kCapFast && !BOUNDED) cap_fast<32, true, false>(s, cap, !some);
    if (CAP == kCapExact) {
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = cap_exact(s[j], cap);
    }
    if (BIAS && CAP != kCapNone) {
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = fmaf(-slope, fabsf((float)ahead - (float)j), s[j]);
    }
    if (BIAS && CAP == kCapNone && over) {
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = fmaf(-2.f * slope, fmaxf((float)j - (float)ahead, 0.f), s[j]);
    }
    if (some) {
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = seen >> j & 1 ? s[j] : -INFINITY;
    }
}
__device__ __forceinline__ float most_of(const float* s) {  // four chains of three-input maxima
    float m[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float* x = s + 8 * q;
        m[q] = fmaxf(fa_max3(fa_max3(fa_max3(x[0], x[1], x[2]), x[3], x[4]), x[5], x[6]), x[7]);
    }
    return fmaxf(fa_max3(m[0], m[1], m[2]), m[3]);
}
// Half c (32 dims) of a head's output row.
template <bool P2>
__device__ __forceinline__ void store_half(const ScorePromptArgs& a, int row, int head, int c, const float* o) {
    const long long at = (long long)row * a.ld + head * kHeadDim + 32 * c;
    if constexpr (P2) {
        float4* out = reinterpret_cast<float4*>(static_cast<float*>(a.out) + at);
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
    } else {
        uint4* out = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + at);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            out[j] = make_uint4(pack_bf16x2(o[8 * j], o[8 * j + 1]), pack_bf16x2(o[8 * j + 2], o[8 * j + 3]),
                                pack_bf16x2(o[8 * j + 4], o[8 * j + 5]), pack_bf16x2(o[8 * j + 6], o[8 * j + 7]));
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
    // Without a cap the bias comes out of the products: S += Qx Kx^T with the slope, as three bf16 parts
    // of its 24 bits, against the key's place in the item (exact in bf16), one MMA step of 16.
    constexpr bool kBiasMma = BIAS && CAP == kCapNone;
    __shared__ uint32_t s_tmem;
    __shared__ float s_xmax[2][2][QT], s_xsum[2][2][QT];  // [item or head parity][half][row]
    __shared__ int s_lo[4], s_hi[4], s_lo_most[4], s_hi_least[4], s_bad, s_q_issued, s_k_issued, s_v_issued;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        mbar_init(&b->qready, kBiasMma ? 2 : 1);  // the copies, and the slope
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&b->kfull[i], 1);
            mbar_init(&b->kempty[i], 1);
            mbar_init(&b->vfull[i], 1);
            mbar_init(&b->vempty[i], 1);
        }
        mbar_init(&b->qfree, 1);
        mbar_init(&b->sfull, 1);
        mbar_init(&b->sfree, kSoftW);
        mbar_init(&b->pfull, kSoftW);
        mbar_init(&b->odone, 1);
        s_bad = s_q_issued = s_k_issued = s_v_issued = 0;
        fence_mbar_init();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (kBiasMma && tid < KT) {
        const float j = (float)tid;
        put_x(sm + kOffKx, tid, pack_bf16x2(j, j), pack_bf16x2(j, 0.f));
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    grid_dep_wait();
    grid_dep_launch();
    const int slabs = a.heads / a.heads_per_cta, head0 = blockIdx.x % slabs * a.heads_per_cta;
    const int2 tile = a.tiles[blockIdx.x / slabs];
    const int row0 = tile.x, nrows = tile.y;
    // The row of each softmax thread, and the slots the tile's rows see: any (min lo .. max hi) and
    // all (max lo .. min hi).
    int lo = 0, hi = -1;
    const int r = 32 * (warp & 3) + lane, half = warp >> 2;  // softmax threads: row r, keys 64 half ..
    const bool there = r < nrows;
    if (warp < kSoftW) {
        if (there) lo = a.rows.lo[row0 + r], hi = a.rows.hi[row0 + r];
        const bool sees = lo <= hi;
        const int x0 = __reduce_min_sync(0xffffffffu, sees ? lo : 0x7fffffff), x1 = __reduce_max_sync(0xffffffffu, sees ? hi : -1);
        const int y0 = __reduce_max_sync(0xffffffffu, there ? lo : 0), y1 = __reduce_min_sync(0xffffffffu, there ? hi : 0x7fffffff);
        if (lane == 0 && half == 0) s_lo[warp] = x0, s_hi[warp] = x1, s_lo_most[warp] = y0, s_hi_least[warp] = y1;
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
    // Items: n key tiles for each of the CTA's heads; item i is key tile i % n of head head0 + i / n.
    const int n = sid < 0 || end <= 0 ? 0 : (end - first + KT - 1) / KT, items = n * a.heads_per_cta;
    // A head's rows of this stream in the layer: [group][stream][slot] rows of 8 heads.
    auto kv_row = [&](int head) {
        return (int)(((long long)(head / kGroupHeads) * a.num_streams + max(sid, 0)) * a.capacity);
    };
    auto kv_x = [&](int head) { return (head % kGroupHeads) * kHeadDim; };

    if (warp < kSoftW) {
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const int pos = BIAS && there ? a.rows.pos[row0 + r] : 0;
        const float2 minus1 = make_float2(-1.f, -1.f);
        float m = 0.f, l = 0.f, slope = 0.f;
        bool ok = true;
        if (n == 0 && there) {  // no row sees anything: zeros
            float o[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = 0.f;
            for (int hh = 0; hh < a.heads_per_cta; ++hh) store_half<P2>(a, row0 + r, head0 + hh, half, o);
        }
        // A wait that gives up clears `ok`; the row's other half learns of it at the next barrier they
        // share (per item, or BOUNDED per head), and both leave there.
        for (int i = 0, kt = 0, hh = 0; i < items; ++i) {
            const int head = head0 + hh;
            if (kt == 0) {
                if (BIAS) slope = a.rule.slopes[head] * kScoreLog2e;
                m = BOUNDED ? (BIAS ? most_bias(slope, pos, lo, hi) : 0.f) : kScoreLow;
                l = 0.f;
            }
            const int k0 = first + (n - 1 - kt) * KT, mine = k0 + 64 * half;  // this thread's first key
            ok = ok && __all_sync(0xffffffffu, mbar_wait(&b->sfull, i & 1));
            // The scores are taken 32 at a time, for the maximum and again for P (capped ones go back to
            // TMEM in between): all 64 in registers spill, which cost more than the second read.
            float mt = -INFINITY;
            const bool whole = k0 >= lo_most && k0 + KT - 1 <= hi_least;  // every row sees every key
            uint32_t seen[2] = {~0u, ~0u};  // this row's visible keys, a bit each
            bool alive[2] = {true, true};   // whether some row of the warp sees some of the 32 keys
            if (!whole) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int x = lo - mine - 32 * c, y = hi - mine - 32 * c;  // bits x .. y
                    const uint32_t from = x <= 0 ? 0xffffffffu : (x > 31 ? 0u : 0xffffffffu << x);
                    const uint32_t to = y >= 31 ? 0xffffffffu : (y < 0 ? 0u : 0xffffffffu >> (31 - y));
                    seen[c] = from & to;
                    alive[c] = __any_sync(0xffffffffu, seen[c] != 0);
                }
            }
            const bool over = kBiasMma && __any_sync(0xffffffffu, min(hi, mine + 63) > pos);
            const float bias = kBiasMma ? slope * (float)(k0 - pos) : 0.f;  // the products' bias is slope x (key - k0)
            if (ok) fa_after();
            if (!BOUNDED && ok) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if (alive[c]) {
                        float s[32];
                        const uint32_t at = lanes + kColS + 64 * half + 32 * c;
                        fa_ld32(at, s);
                        fa_wait_ld();
                        rules<CAP, BOUNDED, BIAS>(s, a.rule.cap, slope, pos - mine - 32 * c, over, seen[c]);
                        mt = fmaxf(mt, most_of(s) + bias);
                        if (CAP != kCapNone) {
                            uint32_t w[32];
#pragma unroll
                            for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(s[j]);
                            fa_st32(at, w);
                            wait_st();
                        }
                    }
                }
            }
            bool waited = i == 0;  // for P V of the item before
            // One barrier of the two warps of 32 rows: unless a score of theirs passed m by more than
            // kRaiseP (or a wait gave up), m stays and nothing is exchanged.
            if (!BOUNDED && pair_any(warp & 3, !ok || mt > m + kRaiseP)) {
                s_xmax[i & 1][half][r] = mt;
                if (pair_any(warp & 3, !ok)) break;
                mt = fmaxf(mt, s_xmax[i & 1][half ^ 1][r]);
                const bool raise = mt > m + kRaiseP;
                const float mn = raise ? mt : m, f = score_exp2(m - mn);
                l *= f;
                m = mn;
                if (kt > 0) {  // O holds the head's items before this one once their P V is done
                    ok = __all_sync(0xffffffffu, mbar_wait(&b->odone, (i - 1) & 1));
                    waited = true;
                    if (ok) {
                        fa_after();
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            float o[8];
                            uint32_t w[8];
                            ld8(lanes + kColO + 32 * half + 8 * c, o);
                            fa_wait_ld();
#pragma unroll
                            for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(o[j] * f);
                            fa_st8(lanes + kColO + 32 * half + 8 * c, w);
                        }
                        wait_st();
                    }
                }
            }
            if (!P2 && ok && !waited) {  // P V of the item before has read P
                ok = __all_sync(0xffffffffu, mbar_wait(&b->odone, (i - 1) & 1));
                fa_after();
            }
            if (ok) {
                // P, 32 keys at a time: bf16 pairs into its own columns, or (P2) hi and lo over the 32
                // columns of S they came from.
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                const float2 neg_m = make_float2(bias - m, bias - m);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t ph[16], pl[P2 ? 16 : 1];
                    float s[32];
                    if (alive[c]) {
                        fa_ld32(lanes + kColS + 64 * half + 32 * c, s);
                        fa_wait_ld();
                    }
                    if (!P2 && c == 1) {  // the scores are read: S may take the next item's
                        fa_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&b->sfree);
                    }
                    if (alive[c]) {
                        if (BOUNDED || CAP == kCapNone)
                            rules<CAP, BOUNDED, BIAS>(s, a.rule.cap, slope, pos - mine - 32 * c, over, seen[c]);
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            float2 x = make_float2(s[2 * j], s[2 * j + 1]);
                            if (!BOUNDED || BIAS) x = __fadd2_rn(x, neg_m);
                            const float2 e = make_float2(score_exp2(x.x), score_exp2(x.y));
                            sum[j & 1] = __fadd2_rn(sum[j & 1], e);
                            ph[j] = pack_bf16x2(e.x, e.y);
                            if constexpr (P2) {
                                const float2 d = __ffma2_rn(make_float2(bf16lo(ph[j]), bf16hi(ph[j])), minus1, e);
                                pl[j] = pack_bf16x2(d.x, d.y);
                            }
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            ph[j] = 0u;
                            if constexpr (P2) pl[j] = 0u;
                        }
                    }
                    if constexpr (P2) {
                        st16(lanes + kColS + 64 * half + 32 * c, ph);
                        st16(lanes + kColS + 64 * half + 32 * c + 16, pl);
                    } else {
                        st16(lanes + kColP + 32 * half + 16 * c, ph);
                    }
                }
                l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
                wait_st();
                if (!whole) {
                    // Some row does not see some key: half a key's V row a thread, cleaned in shared memory.
                    ok = __all_sync(0xffffffffu, mbar_wait(&b->vfull[i % kSlots], (i / kSlots) & 1));
                    if (ok) clean_v<4>(sm + kOffV + (i % kSlots) * kTile, tid >> 1, 4 * (tid & 1), k0 + (tid >> 1) >= end, &s_bad);
                }
                fa_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b->pfull);
            }
            if (++kt < n) continue;
            // The head's end: O / l, the sum over both halves, to the output. P V done also means that
            // every warp's s_bad is seen (they wrote it before their arrivals on pfull).
            ok = ok && __all_sync(0xffffffffu, mbar_wait(&b->odone, i & 1));
            s_xsum[hh & 1][half][r] = l;
            if (pair_any(warp & 3, !ok)) {
                ok = false;
                break;
            }
            fa_after();
            l += s_xsum[hh & 1][half ^ 1][r];
            const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing: zeros
            float o[32];
            ld16(lanes + kColO + 32 * half, o);
            ld16(lanes + kColO + 32 * half + 16, o + 16);
            fa_wait_ld();
            fa_before();  // O is read before the next head's first P V (through pfull)
            if (there) {
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] *= inv;
                if (*const_cast<volatile int*>(&s_bad)) add_not_finite(a, kv_row(head), kv_x(head) + 32 * half, lo, hi, o);
                store_half<P2>(a, row0 + r, head, half, o);
            }
            __syncwarp();
            kt = 0;
            ++hh;
        }
        if (!ok && lane == 0) set_error(a.err, DEV_ERR_TIMEOUT);
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
            if (kBiasMma) fa_mma_ss(tmem + kColS, desc_x(base + kOffQx), desc_x(base + kOffKx), kIdescS, 1u);
            fa_commit(&b->sfull);
            fa_commit(&b->kempty[i % kSlots]);
            if (i % n == n - 1) fa_commit(&b->qfree);  // the head's last use of Q
        };
        auto issue_pv = [&](int i) {
            fa_after();
            const uint64_t dv = desc_mn(base + kOffV + (i % kSlots) * kTile);
#pragma unroll
            for (int k = 0; k < 8; ++k) {  // 128 keys, 16 a step: 8 columns of P, 16 rows (2048 bytes) of V
                const uint32_t p = P2 ? tmem + kColS + 32 * (k >> 1) + 8 * (k & 1) : tmem + kColP + 8 * k;
                fa_mma_ts(tmem + kColO, p, dv + 128 * k, kIdescPV, (i % n || k) ? 1u : 0u);
                if (P2) fa_mma_ts(tmem + kColO, p + 16, dv + 128 * k, kIdescPV, 1u);
            }
            fa_commit(&b->odone);
            fa_commit(&b->vempty[i % kSlots]);
        };
        auto there_for_s = [&](int i) {
            return mbar_wait(&b->kfull[i % kSlots], (i / kSlots) & 1) && mbar_wait(&b->qready, (i / n) & 1);
        };
        bool ok = items == 0 || there_for_s(0);
        if (ok && items > 0) issue_s(0);
        for (int i = 0; i < items && ok; ++i) {
            // The next scores as soon as the softmax holds these in registers (P2: P lies over S, so
            // after P V).
            if (!P2 && i + 1 < items && (ok = there_for_s(i + 1) && mbar_wait(&b->sfree, i & 1))) issue_s(i + 1);
            if (ok && (ok = mbar_wait(&b->pfull, i & 1) && mbar_wait(&b->vfull[i % kSlots], (i / kSlots) & 1))) issue_pv(i);
            if (P2 && ok && i + 1 < items && (ok = there_for_s(i + 1) && mbar_wait(&b->odone, i & 1))) issue_s(i + 1);
        }
        if (!ok) set_error(a.err, DEV_ERR_TIMEOUT);
    } else if (warp == kLoadW && lane == 0) {
        // ---- Q, K and V producer -----------------------------------------------------------------
        bool ok = true;
        // An item's values come after the next item's keys: their slot is free an item later (P V ends where
        // the next softmax begins, S before it), and keys behind that wait would have one item's time to
        // arrive, not two.
        int v_x = 0, v_y = 0;  // the item before
        auto copy_v = [&](int i, int x, int y) {
            const int slot = i % kSlots;
            if (i >= kSlots && !(ok = mbar_wait(&b->vempty[slot], ((i / kSlots) & 1) ^ 1))) return;
            mbar_arrive_expect_tx(&b->vfull[slot], kTile);
            fa_tma(base + kOffV + slot * kTile, &tm_v, x, y, &b->vfull[slot]);
            s_v_issued = i + 1;
        };
        for (int i = 0, kt = 0, hh = 0; i < items && ok; ++i) {
            const int slot = i % kSlots, head = head0 + hh, y = kv_row(head) + first + (n - 1 - kt) * KT;
            if (kt == 0) {
                if (hh > 0 && !(ok = mbar_wait(&b->qfree, (hh - 1) & 1))) break;
                mbar_arrive_expect_tx(&b->qready, 2 * kTile);
                fa_tma(base, &tm_qh, head * kHeadDim, row0, &b->qready);
                fa_tma(base + kTile, &tm_ql, head * kHeadDim, row0, &b->qready);
                s_q_issued = hh + 1;
                if (kBiasMma) {  // the head's slope in three parts, for every row
                    const float slope = a.rule.slopes[head] * kScoreLog2e;
                    const float p0 = __bfloat162float(__float2bfloat16_rn(slope)), p1 = __bfloat162float(__float2bfloat16_rn(slope - p0));
                    for (int q = 0; q < QT; ++q) put_x(sm + kOffQx, q, pack_bf16x2(p0, p1), pack_bf16x2(slope - p0 - p1, 0.f));
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_arrive(&b->qready);
                }
            }
            if (i >= kSlots && !(ok = mbar_wait(&b->kempty[slot], ((i / kSlots) & 1) ^ 1))) break;
            mbar_arrive_expect_tx(&b->kfull[slot], kTile);
            fa_tma(base + kOffK + slot * kTile, &tm_k, kv_x(head), y, &b->kfull[slot]);
            s_k_issued = i + 1;
            if (i > 0) copy_v(i - 1, v_x, v_y);
            v_x = kv_x(head), v_y = y;
            if (++kt == n) kt = 0, ++hh;
        }
        if (ok && items > 0) copy_v(items - 1, v_x, v_y);
        if (!ok) set_error(a.err, DEV_ERR_TIMEOUT);
    }
    fa_before();
    __syncthreads();
    if (tid == 0) {
        // The last copies into each slot land before the shared memory goes (a completed phase returns
        // at once).
        if (s_q_issued > 0) mbar_wait(&b->qready, (s_q_issued - 1) & 1);
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
        launch_k(kernel, dim3((unsigned)(a.n_tiles * (a.heads / a.heads_per_cta))), dim3(kThreadsP), kSmemP, s, a, m[0], m[1], m[2], m[3]);
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
    } else if (a.rule.cap <= kScoreBoundedCap) {
        launch_bias<kCapFast, true, false>(a, m, s);
    } else {
        launch_bias<kCapFast, false, false>(a, m, s);
    }
    return true;
}

}  // namespace ptts

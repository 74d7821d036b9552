// Attention with score rules for a few rows per stream over its whole cache (drafted trees, short
// prompts on long caches), bf16 caches: blocks of up to 64 rows of one sequence, split over the keys.
//
// Bound by HBM: a block's keys and values are read once for all its rows, so the time is that of
// the cache bytes as long as the matrix products keep up. Per key and head 256 bytes arrive (about
// 11 cycles of an SM's share of HBM); 64 rows need 64 x 64 x 3 multiply-adds there (q as a bf16
// hi/lo pair, P as one bf16), which mma.sync does within that time, so the rows stay in registers
// as mma fragments and the 128-row tiles of tcgen05, half or three quarters empty here, are left
// to the prompts (attn_score_prompt.cu).
//
// Work split as in attn_decode.cu: the blocks' keys lie end to end and every CTA takes an equal
// range, cut at no tile boundary. One producer lane copies chunks of 32 keys by TMA (one 3-D copy
// each for K and V: 64 dims x 32 keys x the CTA's heads, 128-byte swizzle, so that ldmatrix reads
// are free of bank conflicts) into a ring of 192 KB. The consumer warps each own (a head, 16 or 32
// rows): S = Q K^T in f32 fragments, rules and mask, an online softmax whose maximum is raised only
// when a score passes it by 2^8, then O += P V from the S fragments' registers. A block inside one
// CTA's range is written at once; the pieces of a cut block leave (max, sum, acc) records that a
// second kernel joins, one warp per row and head: 64 rows x 8 heads are too many for the warp that
// finishes last.
//
// Shapes: up to 16 rows, 8 heads a CTA and a warp a head; up to 32 the same with two 16-row tiles
// a warp; up to 64, 4 heads a CTA (half the grid for each half of the heads) and two warps a head.
//
// A chunk that some row does not see whole masks scores by select, and takes values that are not
// finite out of the V fragments, to add them to the rows that do see them (0 x NaN is NaN, and a
// visible key's weight is positive).
#include "common.cuh"
#include "score.cuh"
#include "score.h"

namespace ptts {
namespace {

constexpr int KC = 32;             // keys per chunk
constexpr int kRingBytes = 192 * 1024;
constexpr int kHeadTile = KC * 128;  // one head's K (or V) chunk: 32 keys x 64 bf16
constexpr int kWarps = 8;
// Eight consumer warps and a warpgroup of which one lane produces. Two row tiles a warp need about
// 220 registers; the launch has 168 a thread (12 warps), so the producers give theirs up: 2 x 128 x
// 232 + 128 x 24 of the launch's 384 x 168.
constexpr int kThreadsR = (kWarps + 4) * 32;
constexpr int kRegsLaunch = 168, kRegsConsumer = 232, kRegsProducer = 24;
static_assert(kWarps * 32 * kRegsConsumer + 128 * kRegsProducer <= kThreadsR * kRegsLaunch, "the split fits the launch");
constexpr float kRaise = 8.f;

// MT 16-row tiles a warp, WPH warps a head.
template <int MT_, int WPH_>
struct Shape {
    static constexpr int MT = MT_, WPH = WPH_;
    static constexpr int kRows = 16 * MT * WPH;
    static constexpr int kHeads = kWarps / WPH;  // heads a CTA
    static constexpr int kStageBytes = 2 * kHeads * kHeadTile;
    static constexpr int kStages = kRingBytes / kStageBytes;
    static constexpr int kSmem = 1024 + kRingBytes + kStages * 64 + 2 * kStages * 8;
};

struct RowsHdr {
    int unit, slot, n, flags;  // the chunk's unit, first slot and keys
    int row0, nrows;           // the unit's rows
};
static_assert(sizeof(RowsHdr) <= 64, "a header per stage");
constexpr int kRFirst = 1, kRLast = 2, kRWhole = 4, kREnd = 8;
constexpr int kRBegins = 16;  // the block's keys begin in this CTA's range

__device__ __forceinline__ void ldsm_x4(uint32_t a, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t a, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a));
}
__device__ __forceinline__ void mma_bf16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int y, int z, uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(y), "r"(z), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}
// The slots a row sees, for chunks that some row does not see whole.
struct Sees {
    int lo, hi, base;
    unsigned long long lineage;
    __device__ __forceinline__ bool operator()(int slot) const {
        return slot >= lo && slot <= hi && (slot < base || (lineage >> (slot - base) & 1));
    }
};

__device__ __forceinline__ Sees sees_of(const ScoreRows& rows, long long row) {
    Sees s{rows.lo[row], rows.hi[row], 0x7fffffff, 0};
    if (rows.lineage) s.base = rows.base[row], s.lineage = rows.lineage[row];
    return s;
}

template <class S, int CAP, bool P2>
__global__ void __launch_bounds__(kThreadsR, 1) score_rows_kernel(ScoreRowsArgs a, const __grid_constant__ CUtensorMap tm_k,
                                                                 const __grid_constant__ CUtensorMap tm_v) {
    constexpr int MT = S::MT;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    unsigned char* hdrs = smem + kRingBytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(hdrs + S::kStages * 64);
    uint64_t* empty = full + S::kStages;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kWarps);
        }
        fence_mbar_init();
    }
    __syncthreads();
    grid_dep_wait();
    grid_dep_launch();
    const long long total = a.prefix[a.n_units];
    const int G = ctas_in_use(total, gridDim.x), c = blockIdx.x;
    if (c >= G) return;
    const int head0 = blockIdx.y * S::kHeads;  // this CTA's heads: within one group of 8

    if (warp >= kWarps) {
        // ---- producer ------------------------------------------------------------------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsProducer));
        if (warp != kWarps || lane != 0) return;
        const long long start = cta_start(c, total, G), end = cta_start(c + 1, total, G);
        const uint64_t pol = policy_evict_first();
        const int group = head0 / kGroupHeads;
        int it = 0;
        bool ok = true;
        auto stage_free = [&](int k) {
            if (mbar_wait(&empty[k % S::kStages], ((k / S::kStages) & 1) ^ 1)) return true;
            set_error(a.err, DEV_ERR_TIMEOUT);
            return false;
        };
        for (int u = a.cta_first[c]; u < a.n_units && ok; ++u) {
            const long long pb = a.prefix[u], pe = a.prefix[u + 1];
            if (pb >= end) break;
            const int s0 = (int)((start > pb ? start : pb) - pb), s1 = (int)((end < pe ? end : pe) - pb);
            const int2 rows = a.blocks[u];
            const int sid = max(a.rows.stream[rows.x], 0);  // a refused tree reads slot 0 and sees nothing
            const int lo = a.unit_lo[u];
            const int row = (int)(((long long)group * a.num_streams + sid) * a.capacity);
            const int whole = pb >= start && pe <= end ? kRWhole : 0;
            for (int p = s0; p < s1; p += KC, ++it) {
                if (!(ok = stage_free(it))) break;
                const int st = it % S::kStages;
                RowsHdr* hd = reinterpret_cast<RowsHdr*>(hdrs + st * 64);
                hd->unit = u;
                hd->slot = lo + p;
                hd->n = min(KC, s1 - p);
                hd->flags = (p == s0 ? kRFirst : 0) | (p + KC >= s1 ? kRLast : 0) | whole | (pb < start ? 0 : kRBegins);
                hd->row0 = rows.x;
                hd->nrows = rows.y;
                unsigned char* sb = smem + st * S::kStageBytes;
                mbar_arrive_expect_tx(&full[st], S::kStageBytes);
                tma_3d(sb, &tm_k, row + lo + p, head0 % kGroupHeads, &full[st], pol);
                tma_3d(sb + S::kStageBytes / 2, &tm_v, row + lo + p, head0 % kGroupHeads, &full[st], pol);
            }
        }
        if (ok && stage_free(it)) {
            reinterpret_cast<RowsHdr*>(hdrs + (it % S::kStages) * 64)->flags = kREnd;
            mbar_arrive(&full[it % S::kStages]);
            ++it;
        }
        // Let every copy in flight land before the CTA's shared memory goes.
        for (int k = it > S::kStages ? it - S::kStages : 0; k < it; ++k)
            if (!mbar_wait(&full[k % S::kStages], (k / S::kStages) & 1)) set_error(a.err, DEV_ERR_TIMEOUT);
        return;
    }

    // ---- consumers: warp = (head, 16 MT rows) --------------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsConsumer));
    const int hl = warp / S::WPH, head = head0 + hl, rbase = (warp % S::WPH) * 16 * MT;
    const int g = lane >> 2, t = lane & 3;
    const float slope = a.rule.slopes ? a.rule.slopes[head] * kScoreLog2e : 0.f;
    const bool biased = a.rule.slopes != nullptr;
    uint32_t qh[MT][4][4], ql[MT][4][4];
    float o[MT][8][4], m[MT][2], l[MT][2], posf[MT][2];
    int full_lo = 0, full_hi = -1;
    bool any = false;  // this warp has rows of the block
    // ldmatrix addresses within a head's tile: K takes 8 keys x 32 dims a time (matrix = dims), V
    // 16 keys x 16 dims (matrices: keys, then dims).
    const int k_row = lane & 7, k_chunk = lane >> 3;
    const int v_row = (lane & 7) + (lane & 8), v_chunk = lane >> 4;
    for (int it = 0;; ++it) {
        const int st = it % S::kStages;
        if (!mbar_wait(&full[st], (it / S::kStages) & 1)) {
            set_error(a.err, DEV_ERR_TIMEOUT);
            break;
        }
        const RowsHdr hd = *reinterpret_cast<const RowsHdr*>(hdrs + st * 64);
        if (hd.flags & kREnd) break;
        if (hd.flags & kRFirst) {
            any = rbase < hd.nrows;
            full_lo = 0, full_hi = 0x7fffffff;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int r = rbase + 16 * i + g + 8 * b;
                    const bool there = r < hd.nrows;
                    const long long row = hd.row0 + (there ? r : 0);
                    if (there) {
                        full_lo = max(full_lo, a.rows.lo[row]);
                        full_hi = min(full_hi, a.rows.lineage ? min(a.rows.hi[row], a.rows.base[row] - 1) : a.rows.hi[row]);
                    }
                    posf[i][b] = biased ? (float)a.rows.pos[row] : 0.f;
                    m[i][b] = kScoreLow;
                    l[i][b] = 0.f;
                    // Rows that are not there have q = 0: finite scores that go nowhere.
                    const uint32_t* ph = reinterpret_cast<const uint32_t*>(a.q_hi + row * a.ld + head * kHeadDim) + t;
                    const uint32_t* pl = reinterpret_cast<const uint32_t*>(a.q_lo + row * a.ld + head * kHeadDim) + t;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        qh[i][k][b] = there ? ph[8 * k] : 0u;
                        qh[i][k][b + 2] = there ? ph[8 * k + 4] : 0u;
                        ql[i][k][b] = there ? pl[8 * k] : 0u;
                        ql[i][k][b + 2] = there ? pl[8 * k + 4] : 0u;
                    }
                }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int d = 0; d < 8; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i][d][e] = 0.f;
            full_lo = __reduce_max_sync(0xffffffffu, full_lo);
            full_hi = __reduce_min_sync(0xffffffffu, full_hi);
        }
        const unsigned char* kt = smem + st * S::kStageBytes + hl * kHeadTile;
        const uint32_t ka = smem_u32(kt), va = ka + S::kStageBytes / 2;
        const bool edge = hd.n < KC || hd.slot < full_lo || hd.slot + KC - 1 > full_hi;
        if (any) {
            // S = Q K^T: key 8 n + 2 t (+1) of rows g and g + 8 in s[i][n][0..3].
            float s[MT][4][4];
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[i][n][e] = 0.f;
            // A dims half at a time, its eight accumulators in turn: each mma waits for the one before
            // it on the same accumulator, 8 (or 4) back.
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                uint32_t kb[4][4];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int key = 8 * n + k_row;
                    ldsm_x4(ka + key * 128 + (((4 * hf + k_chunk) ^ (key & 7)) << 4), kb[n]);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int i = 0; i < MT; ++i) mma_bf16(s[i][n], qh[i][2 * hf + k], kb[n][2 * k], kb[n][2 * k + 1]);
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int i = 0; i < MT; ++i) mma_bf16(s[i][n], ql[i][2 * hf + k], kb[n][2 * k], kb[n][2 * k + 1]);
                }
            }
            // Rules.
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if (CAP == kCapFast) cap_fast<16>(&s[i][0][0], a.rule.cap);
                if (CAP == kCapExact) {
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[i][n][e] = cap_exact(s[i][n][e], a.rule.cap);
                }
                if (biased && !edge) {
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float at = (float)(hd.slot + 8 * n + 2 * t + (e & 1));
                            s[i][n][e] = fmaf(-slope, fabsf(posf[i][e >> 1] - at), s[i][n][e]);
                        }
                }
                if (edge) {
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int r = rbase + 16 * i + g + 8 * b;
                        const long long row = hd.row0 + min(r, hd.nrows - 1);
                        const Sees sees = sees_of(a.rows, row);
#pragma unroll
                        for (int n = 0; n < 4; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int key = 8 * n + 2 * t + e, slot = hd.slot + key;
                                const bool seen = key < hd.n && sees(slot);
                                float& x = s[i][n][2 * b + e];
                                if (biased && seen) {
                                    const int at = slot < sees.base ? slot : a.rows.pos[a.rows.row0[row] + slot - sees.base];
                                    x = fmaf(-slope, fabsf(posf[i][b] - (float)at), x);
                                }
                                x = seen ? x : -INFINITY;
                            }
                    }
                }
            }
            // The running maximum, raised only by more than kRaise.
            bool raise = false;
            float mt[MT][2];
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    float x = fmaxf(s[i][0][2 * b], s[i][0][2 * b + 1]);
#pragma unroll
                    for (int n = 1; n < 4; ++n) x = fmaxf(x, fmaxf(s[i][n][2 * b], s[i][n][2 * b + 1]));
                    mt[i][b] = x;
                    raise |= x > m[i][b] + kRaise;
                }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        float x = mt[i][b];
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                        x = fmaxf(x, m[i][b]);
                        const float f = score_exp2(m[i][b] - x);
                        m[i][b] = x;
                        l[i][b] *= f;
#pragma unroll
                        for (int d = 0; d < 8; ++d) {
                            o[i][d][2 * b] *= f;
                            o[i][d][2 * b + 1] *= f;
                        }
                    }
            }
            // P as A fragments of two 16-key steps.
            uint32_t ph[MT][2][4], pl[MT][2][P2 ? 4 : 1];
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const float e0 = score_exp2(s[i][n][2 * b] - m[i][b]), e1 = score_exp2(s[i][n][2 * b + 1] - m[i][b]);
                        l[i][b] += e0 + e1;
                        const uint32_t w = pack_bf16x2(e0, e1);
                        ph[i][n >> 1][2 * (n & 1) + b] = w;
                        if constexpr (P2) pl[i][n >> 1][2 * (n & 1) + b] = pack_bf16x2(e0 - bf16lo(w), e1 - bf16hi(w));
                    }
            // O += P V: dims 8 d + 2 t (+1) in o[i][d].
            bool bad = false;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int d2 = 0; d2 < 4; ++d2) {
                    uint32_t vb[4];
                    const int key = 16 * kk + v_row;
                    ldsm_x4_t(va + key * 128 + (((2 * d2 + v_chunk) ^ (key & 7)) << 4), vb);
                    if (edge) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) bad |= drop_not_finite(vb[e]);
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        mma_bf16(o[i][2 * d2], ph[i][kk], vb[0], vb[1]);
                        mma_bf16(o[i][2 * d2 + 1], ph[i][kk], vb[2], vb[3]);
                        if constexpr (P2) {
                            mma_bf16(o[i][2 * d2], pl[i][kk], vb[0], vb[1]);
                            mma_bf16(o[i][2 * d2 + 1], pl[i][kk], vb[2], vb[3]);
                        }
                    }
                }
            if (edge && __any_sync(0xffffffffu, bad)) {
                for (int key = 0; key < hd.n; ++key) {
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const int r = rbase + 16 * i + g + 8 * b;
                            if (r >= hd.nrows || !sees_of(a.rows, hd.row0 + r)(hd.slot + key)) continue;
#pragma unroll
                            for (int d = 0; d < 8; ++d) {  // dims 8 d + 2 t, + 1: chunk d, bytes 4 t
                                const uint32_t w = *reinterpret_cast<const uint32_t*>(
                                    kt + S::kStageBytes / 2 + key * 128 + ((d ^ (key & 7)) << 4) + 4 * t);
                                if (!isfinite(bf16lo(w))) o[i][d][2 * b] += bf16lo(w);
                                if (!isfinite(bf16hi(w))) o[i][d][2 * b + 1] += bf16hi(w);
                            }
                        }
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
        if (!(hd.flags & kRLast) || !any) continue;
        // The end of this CTA's piece of the block.
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                float x = l[i][b];
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
                const int r = rbase + 16 * i + g + 8 * b;
                if (r >= hd.nrows) continue;
                if (hd.flags & kRWhole) {
                    const float inv = x == 0.f ? 0.f : 1.f / x;  // a row that sees nothing: zeros
                    const long long at = (long long)(hd.row0 + r) * a.ld + head * kHeadDim + 2 * t;
#pragma unroll
                    for (int d = 0; d < 8; ++d) {
                        const float y0 = o[i][d][2 * b] * inv, y1 = o[i][d][2 * b + 1] * inv;
                        if constexpr (P2) *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at + 8 * d) = make_float2(y0, y1);
                        else *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.out) + at + 8 * d) = pack_bf16x2(y0, y1);
                    }
                } else {
                    // Record 2 c of a piece that began before this CTA's range, 2 c + 1 of one that begins in it.
                    float* rec = a.part + (((long long)(2 * c + (hd.flags & kRBegins ? 1 : 0)) * a.heads + head) * S::kRows + r) * kPartStride;
#pragma unroll
                    for (int d = 0; d < 8; ++d)
                        *reinterpret_cast<float2*>(rec + 8 * d + 2 * t) = make_float2(o[i][d][2 * b], o[i][d][2 * b + 1]);
                    if (t == 0) *reinterpret_cast<float2*>(rec + 64) = make_float2(m[i][b], x);
                }
            }
    }
}

// Joins the pieces of the blocks that CTAs' ranges cut: one warp per row and head, lane = 2 dims.
// Every warp reads the pieces' maxima and sums lane by lane and then all records at once.
template <bool P2>
__global__ void __launch_bounds__(256) score_rows_merge_kernel(ScoreRowsArgs a, int grid, int rows_max) {
    grid_dep_wait();
    grid_dep_launch();
    const long long total = a.prefix[a.n_units];
    const int G = ctas_in_use(total, grid), u = blockIdx.x, head = blockIdx.y, lane = threadIdx.x & 31;
    const long long pb = a.prefix[u], pe = a.prefix[u + 1];
    const int c0 = cta_of(pb, total, G), c1 = cta_of(pe - 1, total, G);
    if (c0 == c1) return;
    const int2 rows = a.blocks[u];
    const int r = blockIdx.z * 8 + (threadIdx.x >> 5);
    if (r >= rows.y) return;
    auto rec = [&](int c) {
        return a.part + (((long long)(2 * c + (c == c0 ? 1 : 0)) * a.heads + head) * rows_max + r) * kPartStride;
    };
    float mx = kScoreLow;
    for (int c = c0 + lane; c <= c1; c += 32) mx = fmaxf(mx, rec(c)[64]);
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    float den = 0.f, x0 = 0.f, x1 = 0.f;
    for (int cb = c0; cb <= c1; cb += 32) {
        const int n = min(32, c1 - cb + 1);
        float w = 0.f;
        if (lane < n) {
            const float2 ml = *reinterpret_cast<const float2*>(rec(cb + lane) + 64);
            w = score_exp2(ml.x - mx);
            den += w * ml.y;
        }
#pragma unroll 8
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

template <class S, int CAP, bool P2>
void launch_shape(const ScoreRowsArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, int grid, cudaStream_t s) {
    set_max_dynamic_smem(reinterpret_cast<const void*>(score_rows_kernel<S, CAP, P2>), S::kSmem);
    launch_k(score_rows_kernel<S, CAP, P2>, dim3(grid, a.heads / S::kHeads), dim3(kThreadsR), S::kSmem, s, a, mk, mv);
    if (grid > 1) launch_k(score_rows_merge_kernel<P2>, dim3(a.n_units, a.heads, S::kRows / 8), dim3(256), 0, s, a, grid, S::kRows);
}

template <class S>
void launch_rules(const ScoreRowsArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, int grid, cudaStream_t s) {
    const int cap = score_cap_mode(a.rule.cap, !a.out_bf16);
    if (a.out_bf16) {
        if (cap == kCapNone) launch_shape<S, kCapNone, false>(a, mk, mv, grid, s);
        else if (cap == kCapFast) launch_shape<S, kCapFast, false>(a, mk, mv, grid, s);
        else launch_shape<S, kCapExact, false>(a, mk, mv, grid, s);
    } else {
        if (cap == kCapNone) launch_shape<S, kCapNone, true>(a, mk, mv, grid, s);
        else launch_shape<S, kCapExact, true>(a, mk, mv, grid, s);
    }
}

using Rows16 = Shape<1, 1>;
using Rows32 = Shape<2, 1>;
using Rows64 = Shape<2, 2>;

}  // namespace

int score_rows_block(int most_rows) { return most_rows <= Rows16::kRows ? Rows16::kRows : most_rows <= Rows32::kRows ? Rows32::kRows : Rows64::kRows; }

int score_rows_grid(int block, int heads, int sms) {
    const int slabs = heads / (block == Rows64::kRows ? Rows64::kHeads : Rows16::kHeads);
    return sms / slabs > 1 ? sms / slabs : 1;
}

size_t score_rows_part_floats(int block, int heads, int grid) { return (size_t)2 * grid * heads * block * kPartStride; }

bool launch_score_rows(const ScoreRowsArgs& a, int block, int grid, cudaStream_t s) {
    CUtensorMap mk, mv;
    const int heads = block == Rows64::kRows ? Rows64::kHeads : Rows16::kHeads;
    const long long rows = (long long)(a.heads / kGroupHeads) * a.num_streams * a.capacity;
    if (rows >= (1LL << 31) || !bf16_heads_map(&mk, a.k_cache, rows, KC, heads) || !bf16_heads_map(&mv, a.v_cache, rows, KC, heads))
        return false;
    if (block == Rows16::kRows) launch_rules<Rows16>(a, mk, mv, grid, s);
    else if (block == Rows32::kRows) launch_rules<Rows32>(a, mk, mv, grid, s);
    else launch_rules<Rows64>(a, mk, mv, grid, s);
    return true;
}

}  // namespace ptts

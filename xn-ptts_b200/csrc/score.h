// Internal launchers of attention with score rules (softcap, distance bias, spans) and of drafted
// trees: the row plan, the kernels that read it, and the acceptance of a drafted path.
//
// A row at position p of a stream sees cache slots lo..hi (slot = position); in a tree call the
// slots from `base` (the stream's length) on hold the drafted nodes, of which a row sees those in
// its lineage: bit i = node i. With s_j = q . k_j / 8 over the visible slots j:
//   t_j = cap * tanh(s_j / cap)             (s_j where cap is 0)
//   u_j = t_j - slopes[h] * |p - pos(j)|    (t_j without slopes; pos(j) = j, or a node's position)
//   out = sum_j exp(u_j) v_j / sum_j exp(u_j), zeros where nothing is visible.
#pragma once

#include "kernels.h"

namespace ptts {

constexpr int kTreeNodes = 64;  // drafted nodes per stream: one bit each

// Per row, on the device (written by the plan).
struct ScoreRows {
    int32_t* stream = nullptr;  // arena stream; -1: the plan refused the row (it sees nothing)
    int32_t* pos = nullptr;     // RoPE position, and the p of the distance bias
    int32_t* lo = nullptr;      // first visible slot
    int32_t* hi = nullptr;      // last visible slot; lo > hi: the row sees nothing
    int32_t* base = nullptr;    // tree calls: the stream's cached length
    int32_t* row0 = nullptr;    // tree calls: the row of the stream's node 0
    unsigned long long* lineage = nullptr;  // tree calls: nodes the row sees, itself among them; else nullptr
};

struct ScoreRule {
    float cap = 0.f;                // 0: none
    const float* slopes = nullptr;  // [H] or nullptr
};

struct ScorePlanArgs {
    // What the host sends: streams [n_seq], row offsets [n_seq + 1], and from blocks_at on the work
    // units or tiles as (first row, rows). An inline list is written to `list` (for the kernels after the
    // plan); else it is there.
    int32_t* list;
    int list_ints;
    int n_seq, n_rows;
    const int32_t* lengths;   // [num_streams]
    int num_streams, capacity;
    const int32_t* parents;   // [n_rows] tree calls, else nullptr
    const int32_t* first;     // [n_rows] or nullptr
    const int32_t* last;      // [n_rows] or nullptr (spans only)
    // RoPE (unless !rotate) and append, as RopeAppendArgs.
    const void* q;
    const void* k;
    const void* v;
    float* q_out;                   // [n_rows][H * 64] f32, rotated, or nullptr:
    __nv_bfloat16* q_hi = nullptr;  // q * q_scale as bf16 hi and lo planes
    __nv_bfloat16* q_lo = nullptr;
    float q_scale = 1.f;
    void* k_cache;
    void* v_cache;
    int heads, kv_heads;
    bool rotate;
    float inv_freq[kMaxPairs];
    ScoreRows rows;
    // Split kernels: the work units (single rows, or blocks of consecutive rows of one sequence:
    // (first row, rows)), their key counts (of blocks, their costs) laid end to end, and the unit each CTA
    // starts in.
    int blocks_at = -1;            // where the blocks are in the list; -1: unit u is row u
    int n_units = 0;               // 0: no units
    int32_t* prefix = nullptr;     // [n_units + 1]
    int32_t* unit_lo = nullptr;    // [n_units] first slot any row of the unit sees
    int32_t* cta_first = nullptr;  // [grid]
    int grid = 0;
    uint32_t* err;
};
// What the partition of blocks counts: a key costs 3 and 1 more for each 16 rows that score it (its bytes,
// then its softmax: 128 keys of a head pair take 1.2 us at 16 rows and 2.1 at 64), a block kScoreBlockCost
// behind its keys (rows and masks read, sums and records written, 4 to 6 us).
constexpr int kScoreBlockCost = 2560;
__host__ __device__ constexpr int score_key_cost(int rows) { return 3 + (rows + 15) / 16; }
// The CTAs that share the blocks' costs: no less than 128 keys of 64 rows for each (an item takes as long for
// fewer, and every piece is one more to join: one tree of 13 nodes on 2000 keys 31 us a call with a fourth
// of that, 22 so; of 64 nodes 38 and 28).
__host__ __device__ inline int score_ctas(long long total, int grid) {
    const int least = 128 * score_key_cost(64);
    const long long g = (total + least - 1) / least;
    return (int)(g < 1 ? 1 : (g > grid ? grid : g));
}
constexpr int kScoreInline = 768;
struct ScoreInline {  // a short list rides in the launch's parameters
    int32_t list[kScoreInline];
};
// One launch: every row's plan entry, its rotated q, its cache rows; and the units' partition.
void launch_score_plan(const ScorePlanArgs& a, const ScoreInline* list, bool in_bf16, bool cache_bf16, cudaStream_t s);

// Prompts and trees on f32 caches (attn_score_f32.cu): tiles (first row, rows) of up to kScoreF32Rows rows
// of one sequence; with splits > 1 the tiles' keys are shared out and joined through `part`.
constexpr int kScoreF32Rows = 32;
struct ScoreF32Args {
    const void* k_cache;  // the layer: kv_offset's layout
    const void* v_cache;
    const float* q;       // [n_rows][H * 64] f32, rotated
    void* out;            // [n_rows][H * 64]
    bool out_bf16;
    int n_rows, heads, num_streams, capacity;
    ScoreRows rows;
    ScoreRule rule;
    const int2* tiles;
    int n_tiles;
    int splits;
    float* part;          // [n_rows][H][splits][kPartStride] with splits > 1
};
int score_f32_splits(int tiles, int heads, int most_keys, int sms);
void launch_score_f32(const ScoreF32Args& a, cudaStream_t s);

// How the matrix-product kernels cap scores: not, by the fast form (bf16 outputs, caps from 1e-3
// to kScoreFastCap; q is then scaled by 1 / (8 cap)) or by tanhf (q scaled by log2(e) / 8, as
// without a cap).
enum { kCapNone = 0, kCapFast = 1, kCapExact = 2 };
constexpr float kScoreFastCap = 128.f;
// Caps this small bound the scores well inside f32's and bf16's exponents (32 log2(e) < 47): no maximum is
// kept (see cap_fast).
constexpr float kScoreBoundedCap = 32.f;
inline int score_cap_mode(float cap, bool out_f32) {
    return cap == 0.f ? kCapNone : (!out_f32 && cap >= 1e-3f && cap <= kScoreFastCap ? kCapFast : kCapExact);
}
inline float score_q_scale(float cap, bool out_f32) {
    constexpr float log2e = 1.4426950408889634f;
    return score_cap_mode(cap, out_f32) == kCapFast ? 0.125f / cap : 0.125f * log2e;
}

// Few rows over a whole cache, bf16 caches (attn_rows.cu): blocks of up to kTreeNodes rows of one
// sequence, the plan's units. False: the tensor maps could not be made, nothing launched.
struct ScoreRowsArgs {
    const void* k_cache;  // the layer
    const void* v_cache;
    const __nv_bfloat16* q_hi;  // [n_rows][ld], scaled by score_q_scale
    const __nv_bfloat16* q_lo;
    void* out;            // [n_rows][ld]
    bool out_bf16;
    int ld, heads, num_streams, capacity, n_rows;
    ScoreRows rows;
    ScoreRule rule;
    const int2* blocks;   // [n_units]
    int n_units;
    const int32_t* prefix;
    const int32_t* unit_lo;
    const int32_t* cta_first;
    int most_rows;        // of a block
    float* part;          // score_rows_part_floats
    uint32_t* err;
};
// CTAs along the keys (the plan's grid, and the most that the kernels use whatever the device's lengths
// are), for `keys` keys of all blocks (an upper bound).
int score_rows_grid(bool out_bf16, int heads, int sms, long long keys, int blocks);
size_t score_rows_part_floats(int heads, int grid, int most_rows);
bool launch_score_rows(const ScoreRowsArgs& a, int grid, cudaStream_t s);

// Prompts on tcgen05, bf16 caches (attn_score_prompt.cu): tiles (first row, rows) of up to 128
// rows of one sequence. False: the tensor maps could not be made, nothing launched.
struct ScorePromptArgs {
    const void* k_cache;  // the layer
    const void* v_cache;
    const __nv_bfloat16* q_hi;  // [n_rows][ld], scaled by score_q_scale
    const __nv_bfloat16* q_lo;
    void* out;            // [n_rows][ld]
    bool out_bf16;
    int ld, heads, num_streams, capacity, n_rows;
    ScoreRows rows;       // no lineages
    ScoreRule rule;
    const int2* tiles;
    int n_tiles;
    int heads_per_cta;    // 1, 2, 4 or 8
    uint32_t* err;
};
bool launch_score_prompt(const ScorePromptArgs& a, cudaStream_t s);

// Acceptance: per stream the accepted nodes' rows move from slot len + node[j] to len + j, in
// every layer and head group, and the length becomes len + their number. A stream whose length on the
// device is not `len` is refused there (DEV_ERR_BOUNDS) and stays as it is. Nodes rise, so node[j] >= j.
// The lists are one array of int32 (host or device): streams [n], lengths before [n], offsets into the
// nodes [n + 1], nodes.
constexpr int kAcceptInline = 512;
struct AcceptInline {  // a short list rides in the launch's parameters
    int32_t list[kAcceptInline];
};
struct AcceptArgs {
    void* k_cache;         // all layers
    void* v_cache;
    long long block_vec;   // 16-byte vectors of one (layer, group) block
    long long stream_vec;  // of one stream in a block
    int row_vec;           // of one row of a group
    int blocks;            // layers * groups
    int streams, capacity;
    int n;
    int32_t* lengths;
    int32_t* arrived;  // [streams] zeros: CTAs of a stream that have read its length
    uint32_t* err;
};
void launch_accept(const AcceptArgs& a, const int32_t* list_dev, cudaStream_t s);
void launch_accept_inline(const AcceptArgs& a, const AcceptInline& list, cudaStream_t s);

}  // namespace ptts

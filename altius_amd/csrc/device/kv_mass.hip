// What attention over a paged cache gave each key: mass(j) = decay mass(j) + sum over rows of 2^(x(row, j) - top(row)) / total(row), x in units of
// log2(e) as in kv_attend.h, top and 1 / total what attention leaves behind of each row.  The scores are computed again, with the rows where attention has the
// keys: a wavefront holds 32 keys in registers, as the second operand of v_mfma_f32_32x32x16_bf16, and goes through the rows, 32 at a time, which the
// block's four wavefronts share in LDS.  Accumulator register r of lane l is then row 8 (r / 4) + 4 (l / 32) + r % 4 and key l % 32: a lane adds up its own
// key's weights, and nothing is exchanged before the end.  Queries are three bf16 numbers each, whose sum they are, and so are keys of an fp32 cache, as in
// kv_attend.h.
//   Sequences of few rows (16 a block in attention) are bound by the memory that keys come from: attention leaves their scores in the workspace, 4 bytes a row
// where a key has hundreds, and a launch over the keys adds them up.  24 tokens behind 1000 to 4095 keys, 32 heads, 8 of keys, 128 channels, fp32: 130 us
// with the attention, computed again 205; in bf16 83 and 122.
//   Of many rows: 2 prompts of 1500 to 2048 (16 heads, 4 of keys, 128 channels, bf16) take 140 us of attention and 72 us
// here, bound by waits with two wavefronts a SIMD (matrix cores 28 % of the time busy); 193 us in all.  Each block splits the queries that it stages:
// split once, by a launch of its own, they take 217 in all.  In fp32 305.
//   No sum is made in an order that changes: where there are few keys the rows are cut into parts, whose sums wait in the workspace and are added in
// order by a second launch.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "kv_attend.h"

namespace altius {

using attend::AttendArgs;

namespace {

using namespace attend;

constexpr int MASS_ROWS = 32;  // of a step

struct MassArgs {
    AttendArgs at;
    float *mass;
    int32_t *positions;
    int64_t page_stride, head_stride;
    const int32_t *row_positions;
    float decay;
    uint32_t parts, max_keys;  // parts of a sequence's rows; keys of the longest sequence
    uint32_t chunks, finish_chunks;  // runs of keys of a pair (sequence, kv head) that there are blocks for: a block goes on with every chunks-th behind its own
    float *sums;               // [parts][sequence][kv head][max_keys]; null: one part
};

__device__ __forceinline__ void put_mass(const MassArgs &m, const dev::KvSequence &seq, uint32_t s, uint32_t kvh, int32_t key, float sum) {
    const uint32_t index = m.at.kv.by_page_size.div((uint32_t)key);
    const int32_t page = m.at.kv.page_of(s, index, -1);
    if (page < 0) return;
    const int64_t to = (int64_t)page * m.page_stride + (int64_t)kvh * m.head_stride + (key - (int32_t)(index * m.at.kv.page_size));
    const int32_t row = key - (seq.length - seq.n);  // its own, where it is the call's
    m.mass[to] = (row >= 0 || m.decay == 0.0f ? 0.0f : m.decay * m.mass[to]) + sum;
    if (row >= 0 && m.positions) m.positions[to] = m.row_positions ? m.row_positions[seq.start + row] : key;
}

// A sum that carries along what its last addition rounded off (Kahan's): off by two steps of itself at most, however many terms there are.  The weight that a key is
// given by many rows adds up to thousands, beside which a single one is less than a step.
struct LongSum {
    float sum = 0.0f, over = 0.0f;  // over: how much too large
    __device__ __forceinline__ void add(float x) {
        const float y = x - over, next = sum + y;
        over = (next - sum) - y, sum = next;
    }
};

template <int DP> struct MassLds {
    static constexpr int PITCH = DP + 8;  // 16-bit words; 16 rows of 16-byte reads cover all banks
    uint16_t q[2][3][MASS_ROWS * PITCH];
    float top[2][MASS_ROWS], recip[2][MASS_ROWS], slope[2][MASS_ROWS];
    int32_t low[2][MASS_ROWS], high[2][MASS_ROWS], place[2][MASS_ROWS];
};
// 32 keys a wavefront, or 64, where registers hold them: each part of a query that comes from LDS is then used twice.
template <int DP, bool BF16> constexpr int mass_tiles() { return (BF16 ? DP <= 128 : DP <= 64) ? 2 : 1; }

// A block's keys, from `first` on, and part `part` of the sequence's rows.
template <int DP, bool BF16>
__device__ __forceinline__ void weigh_run(const MassArgs &m, MassLds<DP> &lds, const dev::KvSequence &seq, uint32_t s, uint32_t kvh, uint32_t part, int32_t first) {
    constexpr int STEPS = DP / 16, PLANES = BF16 ? 1 : 3, SIZE = BF16 ? 2 : 4, TILES = mass_tiles<DP, BF16>(), KEYS = 128 * TILES;
    constexpr int PITCH = MassLds<DP>::PITCH;
    const AttendArgs &g = m.at;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31u, h = lane >> 5;
    const uint32_t pairs = g.kv.sequences * g.kv.kv_heads, pair = s * g.kv.kv_heads + kvh, rows = (uint32_t)seq.n * g.group;

    // This lane's keys.  Behind the last one that one stands in, and is left out.
    const int32_t mine = first + (int32_t)(wave * 32 * TILES), key = mine + (int32_t)col;
    int64_t k_at[TILES];
    u32x4 k[TILES][PLANES][STEPS];
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        const uint32_t read = (uint32_t)min(key + 32 * t, seq.length - 1), index = g.kv.by_page_size.div(read);
        k_at[t] = (int64_t)g.kv.page_of(s, index, 0) * g.kv.page_stride + (int64_t)(read - index * g.kv.page_size) * g.kv.slot_stride + (int64_t)kvh * g.kv.head_stride;
        const char *row = static_cast<const char *>(g.kv.keys) + k_at[t] * SIZE;
#pragma unroll
        for (int c = 0; c < STEPS; c++) {
            const uint32_t channel = 16 * c + 8 * h;
            if constexpr (BF16) {
                const u32x4 x = *reinterpret_cast<const u32x4 *>(row + SIZE * (channel < g.d ? channel : 0));
                k[t][0][c] = channel < g.d ? x : u32x4{0, 0, 0, 0};
            } else {
                const f32x4 lo = *reinterpret_cast<const f32x4 *>(row + SIZE * (channel < g.d ? channel : 0));
                const f32x4 hi = *reinterpret_cast<const f32x4 *>(row + SIZE * (channel + 4 < g.d ? channel + 4 : 0));
                const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f}, a = channel < g.d ? lo : zero, b = channel + 4 < g.d ? hi : zero;
                uint32_t w[3][4];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    split_pair(a[2 * e], a[2 * e + 1], w[0][e], w[1][e], w[2][e]);
                    split_pair(b[2 * e], b[2 * e + 1], w[0][2 + e], w[1][2 + e], w[2][2 + e]);
                }
#pragma unroll
                for (int p = 0; p < PLANES; p++) k[t][p][c] = u32x4{w[p][0], w[p][1], w[p][2], w[p][3]};
            }
        }
    }

    // The parts share the rows that can see the keys: with equal parts of all rows a causal prompt's last ones have all the work (101 us, CUs busy half of the time).
    uint32_t seen_from = 0, seen_to = (rows + MASS_ROWS - 1) / MASS_ROWS;
    const int64_t base = (int64_t)seq.length - seq.n;
    if (g.causal && !g.prefix) seen_from = (uint32_t)min((int64_t)seen_to, max((int64_t)0, first - base) * g.group / MASS_ROWS);
    if (g.window) seen_to = (uint32_t)min((int64_t)seen_to, max((int64_t)seen_from, (max((int64_t)0, (int64_t)first + KEYS + g.window - 1 - base) * g.group + MASS_ROWS - 1) / MASS_ROWS));
    const uint64_t tiles = seen_to - seen_from;
    const uint32_t from = seen_from + (uint32_t)(tiles * part / m.parts), to = seen_from + (uint32_t)(tiles * (part + 1) / m.parts);
    // Lane l's row of a tile (l % 32).  Every wavefront looks at them all.
    struct Its {
        RowRange range;
        uint32_t at;  // token times heads, and head
        int64_t query;
        bool valid;
    };
    auto row_of_tile = [&](uint32_t tile) {
        Its r;
        const uint32_t row = tile * MASS_ROWS + col;
        r.valid = row < rows;
        const uint32_t token = g.by_group.div(r.valid ? row : 0);
        const uint32_t head = kvh * g.group + (r.valid ? row : 0) - token * g.group;
        r.at = (uint32_t)(seq.start + (int32_t)token) * g.q_heads + head;
        r.query = (int64_t)(seq.start + (int32_t)token) * g.q_token + (int64_t)head * g.q_head;
        r.range = row_range(g, seq, s, token);
        if (!r.valid) r.range.low = r.range.high = 0;
        return r;
    };
    // The first tile from `tile` on any of whose rows sees any of the block's keys; the same in all wavefronts.
    auto next_tile = [&](uint32_t tile, Its &r) {
        for (; tile < to; tile++) {
            r = row_of_tile(tile);
            if (__any(r.range.low < r.range.high && r.range.low < first + KEYS && r.range.high > first)) break;
        }
        return tile;
    };
    // A tile on its way: its queries, 8 channels at a time, and what is known of its rows.
    constexpr int PIECES = MASS_ROWS * DP / 8, EACH = PIECES / 256 ? PIECES / 256 : 1;  // of a thread
    f32x4 stage[EACH][2];
    f32x2 stats;
    float its_slope;
    auto channel_of_piece = [&](int e, int half) { return (uint32_t)(8 * ((tid + 256 * e) % PIECES % (DP / 8)) + 4 * half); };
    auto fetch = [&](const Its &r) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const uint32_t row = (tid + 256 * e) % PIECES / (DP / 8), low_word = __shfl((int32_t)r.query, row), high_word = __shfl((int32_t)(r.query >> 32), row);
            const float *from = g.q + (int64_t)((uint64_t)high_word << 32 | low_word);
#pragma unroll
            for (int half = 0; half < 2; half++) stage[e][half] = *reinterpret_cast<const f32x4 *>(from + (channel_of_piece(e, half) < g.d ? channel_of_piece(e, half) : 0));
        }
        stats = *reinterpret_cast<const f32x2 *>(g.stats + 2 * (size_t)r.at);
        its_slope = g.slopes ? g.slopes[r.at % g.q_heads] * LOG2E : 0.0f;
    };
    auto park = [&](int buffer, const Its &r) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            uint32_t w[3][4];
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f}, x = channel_of_piece(e, half) < g.d ? stage[e][half] * g.scale : zero;
                split_pair(x[0], x[1], w[0][2 * half], w[1][2 * half], w[2][2 * half]);
                split_pair(x[2], x[3], w[0][2 * half + 1], w[1][2 * half + 1], w[2][2 * half + 1]);
            }
            const uint32_t row = (tid + 256 * e) % PIECES / (DP / 8);
#pragma unroll
            for (int p = 0; p < 3; p++) *reinterpret_cast<u32x4 *>(&lds.q[buffer][p][row * PITCH + channel_of_piece(e, 0)]) = u32x4{w[p][0], w[p][1], w[p][2], w[p][3]};
        }
        if (tid < MASS_ROWS) {
            lds.top[buffer][col] = stats.x, lds.recip[buffer][col] = stats.y, lds.slope[buffer][col] = its_slope;
            lds.low[buffer][col] = r.range.low, lds.high[buffer][col] = r.range.high, lds.place[buffer][col] = r.range.place;
        }
    };
    LongSum sum[TILES];
    // Weights of 16 scores of the lane's key `its` are added to `total`; whole: all rows see all of the wavefront's keys.
    auto add = [&](int buffer, float (&x)[16], int32_t its, bool whole, float &total) {
        cap_scores(g, x);
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const int at = 8 * b + 4 * (int)h;
            const f32x4 top = *reinterpret_cast<const f32x4 *>(&lds.top[buffer][at]), recip = *reinterpret_cast<const f32x4 *>(&lds.recip[buffer][at]);
            if (g.slopes) {
                const f32x4 slope = *reinterpret_cast<const f32x4 *>(&lds.slope[buffer][at]);
                const u32x4 place = *reinterpret_cast<const u32x4 *>(&lds.place[buffer][at]);
#pragma unroll
                for (int e = 0; e < 4; e++) x[4 * b + e] -= slope[e] * (float)abs((int32_t)place[e] - its);
            }
            if (whole) {
#pragma unroll
                for (int e = 0; e < 4; e++) total = __builtin_fmaf(exp2_fast(x[4 * b + e] - top[e]), recip[e], total);
            } else {
                const u32x4 low = *reinterpret_cast<const u32x4 *>(&lds.low[buffer][at]), high = *reinterpret_cast<const u32x4 *>(&lds.high[buffer][at]);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float w = exp2_fast(x[4 * b + e] - top[e]) * recip[e];
                    total += its >= (int32_t)low[e] && its < (int32_t)high[e] ? w : 0.0f;
                }
            }
        }
    };

    Its now, next;
    uint32_t tile = next_tile(from, now);
    if (tile < to) fetch(now), park(0, now);
    for (int buffer = 0; tile < to; buffer ^= 1) {
        __syncthreads();
        const uint32_t behind = next_tile(tile + 1, next);
        if (behind < to) fetch(next);
        // What all rows see, over the wavefront's lanes.
        int32_t all_low = now.range.low, all_high = now.range.high;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) all_low = max(all_low, __shfl_xor(all_low, x)), all_high = min(all_high, __shfl_xor(all_high, x));
        const bool whole = __builtin_amdgcn_readfirstlane(all_low) <= mine && __builtin_amdgcn_readfirstlane(all_high) >= mine + 32 * TILES;
        f32x16 st[TILES];
#pragma unroll
        for (int t = 0; t < TILES; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) st[t][r] = 0.0f;
#pragma unroll
        for (int c = 0; c < STEPS; c++) {
            u32x4 a[3];
#pragma unroll
            for (int p = 0; p < 3; p++) a[p] = *reinterpret_cast<const u32x4 *>(&lds.q[buffer][p][col * PITCH + 16 * c + 8 * h]);
            // Smallest terms first; the tiles in turn, so that none waits for the one before.
#pragma unroll
            for (int t = 0; t < TILES; t++) ALTIUS_MFMA32_BF16(a[2], k[t][0][c], st[t]);
            if constexpr (!BF16) {
#pragma unroll
                for (int t = 0; t < TILES; t++) ALTIUS_MFMA32_BF16(a[0], k[t][2][c], st[t]);
#pragma unroll
                for (int t = 0; t < TILES; t++) ALTIUS_MFMA32_BF16(a[1], k[t][1][c], st[t]);
            }
#pragma unroll
            for (int t = 0; t < TILES; t++) ALTIUS_MFMA32_BF16(a[1], k[t][0][c], st[t]);
            if constexpr (!BF16) {
#pragma unroll
                for (int t = 0; t < TILES; t++) ALTIUS_MFMA32_BF16(a[0], k[t][1][c], st[t]);
            }
#pragma unroll
            for (int t = 0; t < TILES; t++) ALTIUS_MFMA32_BF16(a[0], k[t][0][c], st[t]);
        }
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            float x[16];
#pragma unroll
            for (int r = 0; r < 16; r++) x[r] = st[t][r];
            float of_tile = 0.0f;
            add(buffer, x, key + 32 * t, whole, of_tile);
            sum[t].add(of_tile);
        }
        if (behind < to) park(buffer ^ 1, next);
        now = next, tile = behind;
    }

    // An infinity or NaN among the queries or keys has left NaN here, and not always where the definition has it (a key's product with parts of infinity): once
    // more then, value by value.
    float check = 0.0f;
#pragma unroll
    for (int t = 0; t < TILES; t++) check = key + 32 * t < seq.length ? __builtin_fmaf(sum[t].sum, 0.0f, check) : check;
    if (__any(check != 0.0f)) {
#pragma unroll 1
        for (int t = 0; t < TILES; t++) {
            const int32_t its = key + 32 * t;
            const int64_t at = t == 0 ? k_at[0] : k_at[TILES - 1];
            LongSum total;
            for (uint32_t row = from * MASS_ROWS + h; row < min(to * MASS_ROWS, rows); row += 2) {
                const uint32_t token = g.by_group.div(row), head = kvh * g.group + row - token * g.group;
                const RowRange range = row_range(g, seq, s, token);
                if (its < range.low || its >= range.high || its >= seq.length) continue;
                const float *q_row = g.q + (int64_t)(seq.start + (int32_t)token) * g.q_token + (int64_t)head * g.q_head;
                float x[1] = {0.0f};
                for (uint32_t c = 0; c < g.d; c++) x[0] = __builtin_fmaf(q_row[c] * g.scale, cache_value<BF16>(g.kv.keys, at + c), x[0]);
                scores(g, x, g.slopes ? g.slopes[head] * LOG2E : 0.0f, range.place - its, [](int) { return 0; });
                const f32x2 its_stats = *reinterpret_cast<const f32x2 *>(g.stats + 2 * ((size_t)(seq.start + (int32_t)token) * g.q_heads + head));
                total.add(exp2_fast(x[0] - its_stats.x) * its_stats.y);
            }
#pragma unroll
            for (int e = 0; e < TILES; e++) sum[e].sum = e == t ? total.sum : sum[e].sum;
        }
    }
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        const float total = sum[t].sum + __shfl_xor(sum[t].sum, 32);
        const int32_t its = key + 32 * t;
        if (h != 0 || its >= seq.length) continue;
        if (m.sums) m.sums[((size_t)part * pairs + pair) * m.max_keys + (size_t)its] = total;
        else put_mass(m, seq, s, kvh, its, total);
    }
}

// LONG: blocks go on with further keys.  (The loop costs registers: of 128 channels, bf16, 234 instead of 208, of fp32 some are spilled.)
template <int DP, bool BF16, bool LONG> __global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void weigh_keys(MassArgs m) {
    constexpr uint32_t KEYS = 128 * mass_tiles<DP, BF16>();
    __shared__ __align__(16) MassLds<DP> lds;
    const AttendArgs &g = m.at;
    // The first keys of a causal sequence are seen by most rows: they start first.  Blocks i, i + 8, .. share an XCD: the pairs go round, so that no XCD has the
    // long sequences to itself.
    const uint32_t pairs = g.kv.sequences * g.kv.kv_heads, outer = blockIdx.x / pairs, pair = (blockIdx.x + outer) % pairs;
    const uint32_t chunk = outer / m.parts, part = outer - chunk * m.parts, s = pair / g.kv.kv_heads, kvh = pair - s * g.kv.kv_heads;
    const dev::KvSequence seq = sequence_of(g, s);
    if (seq.n == 0) return;
    if (g.scores && (uint32_t)seq.n * g.group <= g.few_rows) return;  // finish_masses has them
    for (uint32_t at = chunk; (uint64_t)at * KEYS < (uint32_t)seq.length; at += m.chunks) {
        if (at != chunk) __syncthreads();  // behind the last reader of what is in LDS
        weigh_run<DP, BF16>(m, lds, seq, s, kvh, part, (int32_t)(at * KEYS));
        if constexpr (!LONG) break;
    }
}

// What is left to add up, a thread a key: the scores of sequences of few rows, and the parts of the others' sums, in order.
__global__ __launch_bounds__(256) void finish_masses(MassArgs m) {
    __shared__ float top[FEW_ROWS], recip[FEW_ROWS];
    __shared__ int32_t low[FEW_ROWS], high[FEW_ROWS];
    const AttendArgs &g = m.at;
    const uint32_t tid = threadIdx.x, per = m.finish_chunks, pairs = g.kv.sequences * g.kv.kv_heads, pair = blockIdx.x / per, s = pair / g.kv.kv_heads, kvh = pair - s * g.kv.kv_heads;
    const uint32_t first = (blockIdx.x - pair * per) * 256, apart_keys = per * 256;
    const dev::KvSequence seq = sequence_of(g, s);
    const uint32_t rows = (uint32_t)seq.n * g.group;
    if (rows == 0 || first >= (uint32_t)seq.length) return;
    if (!g.scores || rows > g.few_rows) {
        if (!m.sums) return;
        for (uint32_t key = first + tid; key < (uint32_t)seq.length; key += apart_keys) {
            float sum = 0.0f;
            const float *sums = m.sums + (size_t)pair * m.max_keys + key;
            const size_t apart = (size_t)pairs * m.max_keys;
            for (uint32_t part = 0; part < m.parts; part += 4) {  // a power of two of them; fewer than four read the last again
                float its[4];
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) its[e] = sums[min(part + e, m.parts - 1) * apart];
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) sum += part + e < m.parts ? its[e] : 0.0f;
            }
            put_mass(m, seq, s, kvh, (int32_t)key, sum);
        }
        return;
    }
    if (tid < rows) {
        const uint32_t token = g.by_group.div(tid), head = kvh * g.group + tid - token * g.group;
        const RowRange range = row_range(g, seq, s, token);
        const f32x2 stats = *reinterpret_cast<const f32x2 *>(g.stats + 2 * ((size_t)(seq.start + (int32_t)token) * g.q_heads + head));
        top[tid] = stats.x, recip[tid] = stats.y, low[tid] = range.low, high[tid] = range.high;
    }
    __syncthreads();
    for (uint32_t key = first + tid; key < (uint32_t)seq.length; key += apart_keys) {
        float sum = 0.0f;
        const float *scores = g.scores + (size_t)pair * g.score_rows * g.score_keys + key;
#pragma unroll 4
        for (uint32_t r = 0; r < rows; r++) {
            const float w = exp2_fast(scores[(size_t)r * g.score_keys] - top[r]) * recip[r];
            sum += (int32_t)key >= low[r] && (int32_t)key < high[r] ? w : 0.0f;
        }
        put_mass(m, seq, s, kvh, (int32_t)key, sum);
    }
}

struct MassPlan {
    uint64_t parts, chunks, finish_chunks, blocks, finish_blocks;
    size_t attend, stats, sums, scores;  // where each begins in the workspace
    uint32_t max_keys, score_rows, score_keys;  // score_rows 0: no scores are kept
    bool many;                           // sequences may have more than few rows
    bool is_long;                        // blocks go through several runs of keys
    size_t bytes;
};
// Scores are kept where they take up to this: a batch of 64 texts of 128 Ki keys and 8 kv heads needs as much.
constexpr uint64_t MOST_SCORES = (uint64_t)1 << 30;
// Blocks of a launch, where there are not more pairs: one behind its sequence's end costs 1 ns, and a page table may have room for far more keys than any sequence
// has.  24 single tokens of 1000 to 4095 keys, 8 heads of keys, in a table for 2^22: 6386 us with a block for each 128 keys of it.
constexpr uint64_t LAUNCHED = 1 << 14;
size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

MassPlan mass_plan(const DeviceCtx *ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_attend &attend) {
    MassPlan p = {};
    const size_t held = std::min((size_t)batch.table_pages * (size_t)cache.page_size, (size_t)INT32_MAX);
    const size_t max_keys = std::min(attend.max_keys ? attend.max_keys : held, held);
    const size_t max_tokens = std::min(attend.max_tokens ? attend.max_tokens : attend.tokens, attend.tokens);
    const uint64_t pairs = (uint64_t)batch.sequences * (uint64_t)cache.kv_heads, tiles = (max_tokens * (uint64_t)(attend.q_heads / cache.kv_heads) + MASS_ROWS - 1) / MASS_ROWS;
    const uint64_t block_keys = cache.head_size <= (cache.elem == AHIP_KV_BF16 ? 128 : 64) ? 256 : 128, chunks = (max_keys + block_keys - 1) / block_keys;
    const uint64_t cus = ctx && ctx->cus_per_xcd ? 8 * ctx->cus_per_xcd : 256;
    // Rows are cut until there are three blocks a CU, each of at least eight tiles of rows.
    p.parts = 1;
    while (p.parts < 16 && chunks * pairs * p.parts < 3 * cus && tiles / (2 * p.parts) >= 8) p.parts *= 2;
    p.chunks = std::min(chunks, std::max<uint64_t>(1, LAUNCHED / std::max<uint64_t>(1, pairs * p.parts)));
    p.blocks = p.chunks * pairs * p.parts, p.is_long = p.chunks < chunks;
    p.finish_chunks = std::min<uint64_t>((max_keys + 255) / 256, std::max<uint64_t>(1, LAUNCHED / std::max<uint64_t>(1, pairs)));
    p.finish_blocks = p.finish_chunks * pairs;
    const Plan attention = plan_of(ctx, cache, batch, attend);
    const uint64_t rows = max_tokens * (uint64_t)(attend.q_heads / cache.kv_heads);
    p.max_keys = (uint32_t)max_keys;
    p.many = rows > attention.few_rows;
    p.score_rows = (uint32_t)std::min<uint64_t>(rows, attention.few_rows);
    p.score_keys = (p.max_keys + 15) / 16 * 16;
    if (pairs * p.score_keys * p.score_rows * sizeof(float) > MOST_SCORES) p.score_rows = 0, p.many = true;
    p.attend = 0;
    p.stats = up16(attention.bytes);
    p.sums = up16(p.stats + 2 * attend.tokens * (size_t)attend.q_heads * sizeof(float));
    p.scores = up16(p.sums + (p.many && p.parts > 1 ? p.parts * pairs * max_keys * sizeof(float) : 0));
    p.bytes = p.scores + pairs * p.score_keys * p.score_rows * sizeof(float);
    return p;
}

template <int DP, bool BF16> void launch_weigh(hipStream_t stream, const MassPlan &plan, const MassArgs &m) {
    const dim3 grid((uint32_t)plan.blocks);
    if (plan.is_long) hipLaunchKernelGGL((weigh_keys<DP, BF16, true>), grid, dim3(256), 0, stream, m);
    else hipLaunchKernelGGL((weigh_keys<DP, BF16, false>), grid, dim3(256), 0, stream, m);
}
template <bool BF16> void launch_weigh(hipStream_t stream, const MassPlan &plan, const MassArgs &m) {
    if (m.at.d <= 64) launch_weigh<64, BF16>(stream, plan, m);
    else if (m.at.d <= 128) launch_weigh<128, BF16>(stream, plan, m);
    else launch_weigh<256, BF16>(stream, plan, m);
}

constexpr int64_t MOST_STRIDE = (int64_t)1 << 48;

}  // namespace

int kv_attention_mass_workspace(DeviceCtx *ctx, const ahip_kv_cache *cache, const ahip_kv_batch *batch, const ahip_kv_attend *attend, size_t *bytes) {
    if (!bytes) return kv_fail(ctx, AHIP_ERR_ARG, "kv attention mass: null output");
    *bytes = 0;
    dev::KvView view = {};
    if (int rc = check_attend(ctx, cache, batch, attend, &view)) return rc;
    *bytes = mass_plan(ctx, *cache, *batch, *attend).bytes;
    return AHIP_OK;
}

int launch_kv_attention_mass(DeviceCtx &ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_attend &attend, const ahip_kv_history &history,
                             float decay, const int32_t *row_positions) {
    const std::string name = "kv attention mass: ";
    if (!(decay >= 0.0f && decay <= 1.0f)) return ctx.fail(AHIP_ERR_ARG, name + "the decay is not from 0 to 1");
    if (history.page_stride < 0 || history.head_stride < 0 || history.page_stride > MOST_STRIDE || history.head_stride > MOST_STRIDE)
        return ctx.fail(AHIP_ERR_ARG, name + "a stride of the history is out of range");
    MassArgs m = {};
    if (int rc = check_attend(&ctx, &cache, &batch, &attend, &m.at.kv)) return rc;
    if (attend.tokens == 0 || batch.sequences == 0) return AHIP_OK;
    if (!history.mass) return ctx.fail(AHIP_ERR_ARG, name + "null mass");
    const MassPlan plan = mass_plan(&ctx, cache, batch, attend);
    if (!attend.workspace || attend.workspace_bytes < plan.bytes)
        return ctx.fail(AHIP_ERR_ARG, name + "the workspace holds " + std::to_string(attend.workspace ? attend.workspace_bytes : 0) + " bytes of " + std::to_string(plan.bytes));
    if ((plan.many && (plan.blocks >= MOST_BLOCKS || attend.tokens * (uint64_t)attend.q_heads > UINT32_MAX)) || plan.finish_blocks >= MOST_BLOCKS)
        return ctx.fail(AHIP_ERR_UNSUPPORTED, name + "more blocks than a grid holds");
    if (int rc = begin_attend(ctx, cache, batch, attend, false, &m.at)) return rc;
    char *space = static_cast<char *>(attend.workspace);
    m.at.stats = reinterpret_cast<float *>(space + plan.stats);
    if (plan.score_rows) {
        m.at.scores = reinterpret_cast<float *>(space + plan.scores), m.at.score_rows = plan.score_rows, m.at.score_keys = plan.score_keys;
        m.at.max_keys = plan.max_keys;
    }
    const bool bf16 = cache.elem == AHIP_KV_BF16;
    if (int rc = launch_attend_kept(ctx, m.at, bf16)) return rc;
    if (plan.max_keys == 0) return AHIP_OK;  // no page, no slot
    m.mass = history.mass, m.positions = history.positions, m.page_stride = history.page_stride, m.head_stride = history.head_stride;
    m.row_positions = row_positions, m.decay = decay;
    m.parts = (uint32_t)plan.parts, m.max_keys = plan.max_keys, m.chunks = (uint32_t)plan.chunks, m.finish_chunks = (uint32_t)plan.finish_chunks;
    m.sums = plan.many && plan.parts > 1 ? reinterpret_cast<float *>(space + plan.sums) : nullptr;
    if (plan.many) {
        if (bf16) launch_weigh<true>(ctx.stream, plan, m);
        else launch_weigh<false>(ctx.stream, plan, m);
        if (int rc = ctx.check(hipGetLastError(), "kv attention mass launch")) return rc;
    }
    if (!plan.score_rows && !m.sums) return AHIP_OK;
    hipLaunchKernelGGL(finish_masses, dim3((uint32_t)plan.finish_blocks), dim3(256), 0, ctx.stream, m);
    return ctx.check(hipGetLastError(), "kv attention mass launch");
}

}  // namespace altius

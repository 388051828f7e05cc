// Attention of a batch's newest tokens over a paged cache of keys and values:
//   x(row, j) = cap tanh(q k_j scale / cap) - slope |p - j|,   out = sum_j softmax(x)_j v_j   over low <= j < high,
// a row being one query head of one token.  The rows of one kv head -- its group of query heads, times the sequence's new
// tokens -- read the same keys, so they are computed together: row r is token r / group, head r % group of the group.
//
// One pass over the keys with a running maximum m and sum l of 2^(x log2(e)): where m rises, what has been summed is rescaled
// by 2^(old - new).  Parts of a row's keys (wavefronts of a block, blocks of a sequence) keep their own m, l and sum and are
// joined by the same rescaling.  All of it is held in fp32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv.h"
#include "math.h"

namespace altius {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.44269504088896341f;
// The maximum that weights are relative to stays until one is this much (in powers of two) above it: fp32 holds weights up to 2^8 as
// exactly as those up to 1, and most of the rescaling of what has been summed falls away.
// 3 prompts of documents (d = 128, fp32): 88 us, 91 us without the slack; a prompt of 4096 with a window, bf16: 151 and 156 us.
constexpr float SLACK = 8.0f;
// Sequences with at most so many rows for a kv head go 16 rows a block (attend_rows16, SPLIT), longer ones 128 (rows128): FEW_ROWS, or
// FEW_BESIDE_CUT in a batch whose longer ones' keys are cut as well.  4 sequences of 4000 to 8000 keys, 8 kv heads of 128 channels,
// fp32: 32 rows take 70 us by 16 rows a block and 91 us by 128, 64 rows 104 and 93 us, 128 rows 220 and 105 us; 32 sequences of
// 2000 to 4000 keys in bf16: 157 and 239, 236 and 242, 384 and 252 us.  Pieces of 57 to 333 rows (5 sequences, 8 heads of 96
// channels, fp32), the shortest by 16 rows a block, behind the others: 132 us, all by 128: 100 us.
constexpr uint32_t FEW_ROWS = 32, FEW_BESIDE_CUT = 16;
constexpr int TILE_ROWS = 128;  // a block's, of the longer ones

// How the blocks share the work on the sequences of one kind.  Not listed: a block per (sequence, kv head, row tile of the longest
// sequence).  Listed: the blocks go through the row tiles that there are (find).  Cut: so they do, and the keys of a row tile are
// cut so that at_once blocks, which are at work at once, have parts of about the same size, of split_keys keys at least; the partial results
// of a part's rows wait in the workspace in the place of its number: maximum and sum, and the weighted sum of values.
struct Share {
    uint32_t row_tiles, split_keys, rows;
    uint32_t blocks, at_once;
    bool listed, cut;
    float *part_stats, *part_out;
};

struct AttendArgs {
    dev::KvView kv;
    const float *q;
    float *out;
    int64_t q_token, q_head, out_token, out_head;
    uint32_t q_heads, group, d, few_rows;
    dev::FastDiv by_group;
    float scale, cap;  // scale: with log2(e), or by the cap where there is one; cap: 0, or the cap with log2(e)
    int causal, window;
    const float *slopes;
    const int32_t *prefix, *first_keys;
    uint32_t max_tokens, max_keys;
    Share few, many;  // of sequences with up to few_rows rows, and with more
};

// The sequence, with n == 0 where the call's bounds leave it out (too long for them: the flag is raised).
__device__ __forceinline__ dev::KvSequence sequence_of(const AttendArgs &g, uint32_t s) {
    dev::KvSequence q = dev::kv_sequence(g.kv, s);
    if ((uint32_t)q.n > g.max_tokens || (uint32_t)q.length > g.max_keys) {
        *g.kv.flag = 1;
        q.n = 0;
    }
    return q;
}

struct RowRange {
    int32_t low, high, place;
};
__device__ __forceinline__ RowRange row_range(const AttendArgs &g, const dev::KvSequence &q, uint32_t s, uint32_t token) {
    RowRange r;
    r.place = q.length - q.n + (int32_t)token;
    r.high = g.causal ? r.place + 1 : q.length;
    if (g.prefix) r.high = max(r.high, g.prefix[s]);
    r.high = min(r.high, q.length);
    r.low = g.window ? max(0, max(0, r.place) - g.window + 1) : 0;
    if (g.first_keys) r.low = max(r.low, g.first_keys[q.start + (int32_t)token]);
    return r;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float weight_of(float m, float top) { return m == -INFINITY ? 0.0f : exp2_fast(m - top); }

// tanh, as dev::rational_tanh has it, but for the division: a reciprocal and one step of Newton's, off by an fp32 step more at most.
__device__ __forceinline__ float fast_tanh(float v) {
    float p, q;
    dev::rational_tanh_parts(dev::rclamp(v, -9.0f, 9.0f), p, q);
    float r = __builtin_amdgcn_rcpf(q);
    r = __builtin_fmaf(__builtin_fmaf(-q, r, 1.0f), r, r);
    return p * r;
}

// Products of a (scaled) query and keys become scores in units of log2(e): capped, biased.  Key place(r) of the tile, which starts
// `distance` in front of the row's place, is that of x[r].
template <int N, class Place> __device__ __forceinline__ void scores(const AttendArgs &g, float (&x)[N], float slope, int32_t distance, Place place) {
    if (g.cap != 0.0f) {
        // Up to 3/4 of the cap, where nearly all scores are, tanh(x) / x is a polynomial of degree 5 in x^2, off by 2.9e-8 of
        // itself at most (a fit of the least largest error): 8 operations a score instead of 20.
        float most = fabsf(x[0]);
#pragma unroll
        for (int r = 1; r < N; r++) most = fmaxf(most, fabsf(x[r]));
        if (__any(most > 0.75f)) {
#pragma unroll
            for (int r = 0; r < N; r++) x[r] = g.cap * fast_tanh(x[r]);
        } else {
#pragma unroll
            for (int r = 0; r < N; r++) {
                const float z = x[r] * x[r], c = g.cap * x[r];
                float p = __builtin_fmaf(z, -0.004716264083981514f, 0.01958294026553631f);
                p = __builtin_fmaf(p, z, -0.05334445834159851f);
                p = __builtin_fmaf(p, z, 0.1332540661096573f);
                p = __builtin_fmaf(p, z, -0.33332958817481995f);
                x[r] = __builtin_fmaf(c * z, p, c);
            }
        }
    }
    if (g.slopes) {
#pragma unroll
        for (int r = 0; r < N; r++) x[r] -= slope * (float)abs(distance - (int32_t)place(r));
    }
}

// Two values as three pairs of bf16 whose sums they are (split3.h, without its care for infinities and what rounds up to one: those
// become NaN, and rows that see them are computed once more).
__device__ __forceinline__ void split_pair(float e0, float e1, uint32_t &p0, uint32_t &p1, uint32_t &p2) {
    p0 = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){e0, e1}, bf16x2));
    const float r0 = e0 - __uint_as_float(p0 << 16), r1 = e1 - __uint_as_float(p0 & 0xffff0000u);
    p1 = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){r0, r1}, bf16x2));
    const float s0 = r0 - __uint_as_float(p1 << 16), s1 = r1 - __uint_as_float(p1 & 0xffff0000u);
    p2 = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){s0, s1}, bf16x2));
}

// The largest of three, without the instructions that make a signalling NaN quiet in front of fmaxf.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// v of lane ^ 32 next to the lane's own, without LDS: the first is the lower half's value in both halves, the second the upper half's.
__device__ __forceinline__ void halves(float v, float &lower, float &upper) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    lower = __uint_as_float(r[0]), upper = __uint_as_float(r[1]);
}

template <bool BF16> __device__ __forceinline__ float cache_value(const void *base, int64_t at) {
    return BF16 ? __uint_as_float((uint32_t)static_cast<const uint16_t *>(base)[at] << 16) : static_cast<const float *>(base)[at];
}

// ---------------------------------------------------------------- 16 rows a wavefront, keys straight from memory
// Both products are computed transposed, S^T = K Q^T and O^T = V^T P^T, with 16 rows as columns.  The accumulator of S^T has in
// lane l, register r the score of row l % 16 and key 4 (l / 16) + r of the tile, which is where the second product wants P^T:
// the k slots of its instructions are declared to be keys in that order.  Keys and values go from memory into registers in the
// layout of the instructions' first operand, without LDS: a row of keys is read along its channels, 16 bytes a lane, a row of
// values by 16 lanes side by side, each lane's channels being rows of O^T.
// Bound by the memory that keys and values come from: no key is read twice for 16 rows.  One row of 65536 keys, 8 kv heads of 128
// channels, fp32 (537 MB): 107 us with the join of the parts, 5.0 TB/s, where a copy of 1 GiB reads and writes 5.2.  48 sequences of
// 100 to 8191 bf16 keys (401 MB), 4 kv heads of 128 channels, 8 rows each, scores capped: 99 us, 4.1 TB/s.
//   fp32 cache: v_mfma_f32_16x16x4_f32.
//   bf16 cache: v_mfma_f32_16x16x32_bf16 over the channels and _16x16x16_bf16 over the keys; q and the weights as three bf16 numbers
//   each, whose sum they are exactly, so that each of the three products is exact in the fp32 sum; a lane holds 4 keys x DP / 16
//   channels of V and turns them with v_perm.
// Tiles of 16 keys, two on their way (one for DP 256): what registers hold with two or three wavefronts a SIMD.  Tiles of 32
// keys leave one wavefront fewer.
constexpr int ROW_WAVES = 4, ROW_KEYS = 16;

template <int DP, bool BF16> struct RowTile {
    static constexpr int K_UNITS = DP * (BF16 ? 2 : 4) / 64, V_WORDS = DP * (BF16 ? 2 : 4) / 64;  // 16 bytes of keys; words of a row of values
    u32x4 k[K_UNITS];
    uint32_t v[4][V_WORDS];
};

#define ALTIUS_MFMA16_F32(A, B, C) C = __builtin_amdgcn_mfma_f32_16x16x4f32(A, B, C, 0, 0, 0)
#define ALTIUS_MFMA16_BF16(A, B, C) \
    C = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, A), __builtin_bit_cast(bf16x8, B), C, 0, 0, 0)
#define ALTIUS_MFMA16_BF16_K16(A, B, C) \
    C = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, A), __builtin_bit_cast(s16x4, B), C, 0, 0, 0)

// Row of O^T (channel) of accumulator i, register r, in lane group `part` = lane / 16.
template <int DP, bool BF16> __device__ __forceinline__ uint32_t channel_of(int i, int r, uint32_t part) {
    return BF16 ? (DP / 16) * (4 * part + r) + i : 64 * (i / 4) + 4 * (4 * part + r) + i % 4;
}

template <int DP, bool BF16> struct RowLds {
    static constexpr int PITCH = DP + 4;
    union {
        float sums[ROW_WAVES][16 * PITCH];
        // The parts of the queries, a bf16 cache's, or the queries, where registers do not hold them: all wavefronts share them.
        uint16_t q[3][16 * (DP + 8)];
        float whole_q[16 * PITCH];
    };
    float stats[ROW_WAVES][2][16];
};

// The keys of the sequences of one kind, cut into parts of about the same size, one a block, whatever the sequences' lengths.  In
// units of 64 keys: a part is as large as leaves no more parts than blocks that are at work at once, as far as the pairs (row tiles x kv
// heads of all sequences), which are cut one by one, allow.  Every block finds its part for itself, from the lengths, by a scan over the
// sequences.
constexpr uint32_t UNIT = 64;
struct SequenceWork {
    uint32_t units, pairs;  // units of one pair; pairs
    int32_t begin;          // the first unit's first key
};
template <bool FEW> __device__ __forceinline__ SequenceWork sequence_work(const AttendArgs &g, uint32_t s) {
    SequenceWork w = {0, 0, 0};
    if (s >= g.kv.sequences) return w;
    const dev::KvSequence q = sequence_of(g, s);
    const uint32_t rows = (uint32_t)q.n * g.group;
    if (rows == 0 || (rows <= g.few_rows) != FEW) return w;
    if (g.window) w.begin = max(0, max(0, q.length - q.n) - g.window + 1) & ~(int32_t)(UNIT - 1);
    w.units = max(1u, (uint32_t)(q.length - w.begin + (int32_t)UNIT - 1) / UNIT);
    w.pairs = (rows + (FEW ? 15 : TILE_ROWS - 1)) / (FEW ? 16 : TILE_ROWS) * g.kv.kv_heads;
    return w;
}
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v) {  // over the lanes up to this one
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const uint32_t t = __shfl_up(v, m);
        if (lane >= (uint32_t)m) v += t;
    }
    return v;
}
struct Found {
    uint32_t s, before, parts;  // of a pair; before: the sequence's first block
    SequenceWork work;
    __device__ __forceinline__ int32_t first_key(uint32_t part) const {
        return work.begin + (int32_t)((uint32_t)((uint64_t)part * work.units / parts) * UNIT);
    }
    __device__ __forceinline__ uint32_t part_with(int32_t key) const {  // the last part that starts at that key's unit or in front of it
        return (uint32_t)(((uint64_t)((uint32_t)(key - work.begin) / UNIT + 1) * parts - 1) / work.units);
    }
};
// The scan over the sequences: a wavefront's own of up to 64, the whole block's of more, 256 at a time.
constexpr uint32_t SCAN = 256;
struct ScanLds {
    uint32_t totals[SCAN / 64];
    Found found;
};
// Sum over the threads up to this one, and over all.
struct Sums {
    uint32_t up_to, all;
};
__device__ __forceinline__ Sums scan(bool wide, uint32_t v, ScanLds &lds) {
    Sums r;
    r.up_to = wave_prefix(v), r.all = __builtin_amdgcn_readlane(r.up_to, 63);
    if (!wide) return r;
    const uint32_t wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) lds.totals[wave] = r.all;
    __syncthreads();
    r.all = 0;
#pragma unroll
    for (uint32_t w = 0; w < SCAN / 64; w++) {
        const uint32_t total = __builtin_amdgcn_readfirstlane(lds.totals[w]);
        if (w < wave) r.up_to += total;
        r.all += total;
    }
    return r;
}
// The sequence that a block is at work on, or, by_sequence, the one asked for.  False where there is none.  For whole blocks.
template <bool FEW> __device__ __forceinline__ bool find(const AttendArgs &g, bool by_sequence, uint32_t what, Found &f) {
    __shared__ ScanLds lds;
    const Share &share = FEW ? g.few : g.many;
    const bool wide = g.kv.sequences > 64;
    const uint32_t step = wide ? SCAN : 64, index = threadIdx.x & (step - 1);
    const SequenceWork first = sequence_work<FEW>(g, index);
    auto sum = [&](auto of) {
        uint32_t total = 0;
        for (uint32_t base = 0; base < g.kv.sequences; base += step) total += scan(wide, of(base ? sequence_work<FEW>(g, base + index) : first), lds).all;
        return total;
    };
    // The units of a part: the least of a few that leave no more parts than blocks at work at once, so that few of those go without
    // one.  (More sequences than lanes leave few anyway.)
    const uint32_t units = sum([](const SequenceWork &w) { return w.units * w.pairs; });
    uint32_t part = max((units + share.at_once - 1) / share.at_once, share.split_keys / UNIT);
    for (int i = 0; i < (wide ? 0 : 4); i++) {
        if (sum([&](const SequenceWork &w) { return (w.units + part - 1) / part * w.pairs; }) <= share.at_once) break;
        part += (part + 15) / 16;
    }
    // Starts out of order can make more rows than the call has, and more blocks than were counted with: what is behind the last stays undone.
    // (The flag is raised.)
    auto fits = [&] { return f.before + (uint64_t)f.parts * f.work.pairs <= share.blocks; };
    uint32_t before = 0;
    for (uint32_t base = 0; base < g.kv.sequences; base += step) {
        const uint32_t s = base + index;
        const SequenceWork w = base ? sequence_work<FEW>(g, s) : first;
        const uint32_t parts = (w.units + part - 1) / part;
        const Sums sums = scan(wide, parts * w.pairs, lds);
        const uint32_t mine = before + sums.up_to - parts * w.pairs;
        if (by_sequence ? what - base < step : before + sums.all > what) {
            if (wide) {
                if (by_sequence ? s == what : mine <= what && what < before + sums.up_to) lds.found = {s, mine, parts, w};
                __syncthreads();
                f = lds.found;
                f.s = __builtin_amdgcn_readfirstlane(f.s), f.before = __builtin_amdgcn_readfirstlane(f.before), f.parts = __builtin_amdgcn_readfirstlane(f.parts);
                f.work.units = __builtin_amdgcn_readfirstlane(f.work.units), f.work.pairs = __builtin_amdgcn_readfirstlane(f.work.pairs);
                f.work.begin = __builtin_amdgcn_readfirstlane(f.work.begin);
                return fits();
            }
            const int lane = __builtin_ctzll(__ballot(by_sequence ? s == what : what < before + sums.up_to));
            f.s = base + lane, f.before = __builtin_amdgcn_readlane(mine, lane), f.parts = __builtin_amdgcn_readlane(parts, lane);
            f.work.units = __builtin_amdgcn_readlane(w.units, lane), f.work.pairs = __builtin_amdgcn_readlane(w.pairs, lane);
            f.work.begin = __builtin_amdgcn_readlane(w.begin, lane);
            return fits();
        }
        before += sums.all;
    }
    return false;
}

// What a block does for 16 rows of a kv head: the keys from .. to - 1, which its wavefronts share tile by tile.  whole: that is all there
// is to them; else the partial results go to place `slot`.
struct Piece {
    uint32_t s, kvh, tile;
    int32_t from, to;
    bool whole;
    uint32_t slot;
};

// UNIFORM: 16 keys that start at a multiple of 16 are in one page.  SPLIT: sequences of few rows, whose keys several blocks share.
template <int DP, bool BF16, bool UNIFORM, bool SPLIT>
__device__ __forceinline__ void piece16(const AttendArgs &g, const Piece &piece, RowLds<DP, BF16> &lds) {
    constexpr int KT = ROW_KEYS, NACC = DP / 16, PITCH = RowLds<DP, BF16>::PITCH;
    auto &sums = lds.sums;
    auto &stats = lds.stats;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t col = lane & 15u, part = lane >> 4;
    const uint32_t s = piece.s, tile = piece.tile, kvh = piece.kvh;

    const dev::KvSequence seq = sequence_of(g, s);
    const uint32_t rows = (uint32_t)seq.n * g.group;
    if ((rows <= g.few_rows) != SPLIT || tile * 16 >= rows) return;
    const uint32_t row = tile * 16 + col;
    const bool valid = row < rows;
    const uint32_t token = g.by_group.div(valid ? row : 0), head = kvh * g.group + (valid ? row : 0) - token * g.group;
    const RowRange range = row_range(g, seq, s, token);
    const int32_t low = range.low, high = range.high, place = range.place;
    const bool sees = valid && low < high;
    const float slope = g.slopes ? g.slopes[head] * LOG2E : 0.0f;

    // What any row sees, and what all see.
    int32_t any_low = sees ? low : INT32_MAX, any_high = sees ? high : 0, all_low = valid ? low : 0, all_high = valid ? high : INT32_MAX;
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) {
        any_low = min(any_low, __shfl_xor(any_low, m)), any_high = max(any_high, __shfl_xor(any_high, m));
        all_low = max(all_low, __shfl_xor(all_low, m)), all_high = min(all_high, __shfl_xor(all_high, m));
    }
    int32_t begin = max(any_low, piece.from), end = min(any_high, piece.to);
    begin = __builtin_amdgcn_readfirstlane(begin), end = __builtin_amdgcn_readfirstlane(end);
    const int32_t first = begin / KT, tiles = begin < end ? (end + KT - 1) / KT - first : 0;

    const char *keys = static_cast<const char *>(g.kv.keys), *values = static_cast<const char *>(g.kv.values);
    constexpr int SIZE = BF16 ? 2 : 4;
    const int64_t head_at = (int64_t)kvh * g.kv.head_stride;

    // fp32: channels 16 i + 4 part on; bf16: parts of channels 32 i + 8 part on.
    constexpr bool Q_HERE = DP > 128 && !BF16;
    u32x4 q[BF16 || Q_HERE ? 1 : DP / 16];
    uint32_t q_at = BF16 ? col * (DP + 8) + 8 * part : col * PITCH + 4 * part;
    constexpr int Q_PART = 16 * (DP + 8);
    const float *q_row = g.q + (int64_t)(seq.start + (int32_t)token) * g.q_token + (int64_t)head * g.q_head;
    // All loads in front of the first use, none behind a condition: a row that is not there is read as row 0, and left out below.  One
    // token behind 76, 12 heads of 64 channels: 6.6 us, 7.3 with a condition around each load.
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 read[DP / 16];
    if constexpr (BF16) {
#pragma unroll
        for (int i = 0; i < DP / 32; i++) {
            const uint32_t c = 32 * i + 8 * part, at = c < g.d ? c : 0;
            read[2 * i] = *reinterpret_cast<const f32x4 *>(q_row + at), read[2 * i + 1] = *reinterpret_cast<const f32x4 *>(q_row + at + 4);
        }
#pragma unroll
        for (int i = 0; i < DP / 32; i++) {
            const bool here = valid && 32 * i + 8 * part < g.d;
            const f32x4 lo = here ? read[2 * i] * g.scale : zero, hi = here ? read[2 * i + 1] * g.scale : zero;
            u32x4 parts[3];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                uint32_t w[3];
                split_pair(lo[2 * e], lo[2 * e + 1], w[0], w[1], w[2]);
                parts[0][e] = w[0], parts[1][e] = w[1], parts[2][e] = w[2];
                split_pair(hi[2 * e], hi[2 * e + 1], w[0], w[1], w[2]);
                parts[0][2 + e] = w[0], parts[1][2 + e] = w[1], parts[2][2 + e] = w[2];
            }
#pragma unroll
            for (int p = 0; p < 3; p++) *reinterpret_cast<u32x4 *>(&lds.q[0][q_at + p * Q_PART + 32 * i]) = parts[p];
        }
    } else {
#pragma unroll
        for (int i = 0; i < DP / 16; i++) read[i] = *reinterpret_cast<const f32x4 *>(q_row + (16 * i + 4 * part < g.d ? 16 * i + 4 * part : 0));
#pragma unroll
        for (int i = 0; i < DP / 16; i++) {
            const f32x4 x = valid && 16 * i + 4 * part < g.d ? read[i] * g.scale : zero;
            if constexpr (Q_HERE) *reinterpret_cast<f32x4 *>(&lds.whole_q[q_at + 16 * i]) = x;
            else q[i] = __builtin_bit_cast(u32x4, x);
        }
    }

    // Wavefront w takes tiles w, w + 4, ... of the block's.
    const int32_t mine = tiles > (int32_t)wave ? (tiles - (int32_t)wave + ROW_WAVES - 1) / ROW_WAVES : 0;
    auto tile_key = [&](int32_t i) { return (first + (int32_t)wave + i * ROW_WAVES) * KT; };
    auto row_at = [&](uint32_t key) {  // elements from the start of the cache
        const uint32_t index = g.kv.by_page_size.div(key);
        return (int64_t)g.kv.page_of(s, index, 0) * g.kv.page_stride + (int64_t)(key - index * g.kv.page_size) * g.kv.slot_stride + head_at;
    };
    const uint32_t slot_bytes = (uint32_t)g.kv.slot_stride * SIZE;
    // Where pages hold whole tiles: where the wavefront's next 64 tiles start, in bytes from the start of the cache, a tile a lane.  A
    // tile then starts at one address for all lanes, whose parts lie at fixed distances from it (below 2^31 bytes, or the call takes the
    // other kernel).
    int64_t starts = 0;
    auto fetch_starts = [&](int32_t from) {
        const int32_t i = from + (int32_t)lane;
        const uint32_t key = (uint32_t)tile_key(i < mine ? i : mine - 1), index = g.kv.by_page_size.div(key);
        starts = ((int64_t)g.kv.page_of(s, index, 0) * g.kv.page_stride + (int64_t)(key - index * g.kv.page_size) * g.kv.slot_stride + head_at) * SIZE;
    };
    // Where they do not: lane l has the row of key l % 16 of a tile, looked up a tile ahead of its use.  Keys in front of the first that
    // is seen and behind the last may have no page: those two stand in for them.
    int32_t page_ahead = 0;
    auto key_ahead = [&](int32_t i) { return (uint32_t)max(begin, min(tile_key(i) + (int32_t)col, end - 1)); };
    auto look_up = [&](int32_t i) { page_ahead = g.kv.table[(int64_t)s * g.kv.table_stride + g.kv.by_page_size.div(key_ahead(i))]; };
    auto row_ahead = [&](int32_t i) {  // of tile i, whose pages are known
        const uint32_t key = key_ahead(i);
        if ((uint32_t)page_ahead >= g.kv.pages) *g.kv.flag = 1;
        const int32_t page = (uint32_t)page_ahead < g.kv.pages ? page_ahead : 0;
        return ((int64_t)page * g.kv.page_stride + (int64_t)(key - g.kv.by_page_size.div(key) * g.kv.page_size) * g.kv.slot_stride + head_at) * SIZE;
    };

    // A lane's parts of a tile: of row `col` of the keys 16 bytes at 64 c + 16 part; of row 4 part + r of the values, fp32: 16 bytes at
    // 256 j + 16 col, bf16: DP / 8 bytes.  No load depends on a condition, which would have the compiler wait for those before it:
    // channels that a head does not have are read as others (their queries are 0, their sums go nowhere).
    typedef RowTile<DP, BF16> Tile;
    const uint32_t row_bytes = g.d * SIZE;
    constexpr uint32_t V_STEP = BF16 ? DP / 8 : 16;
    auto load_parts = [&](Tile &t, auto whole, const char *k_row, auto v_row) {
        constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
        for (int c = 0; c < Tile::K_UNITS; c++) {
            if (WHOLE) t.k[c] = *reinterpret_cast<const u32x4 *>(k_row + 64 * c);
            else t.k[c] = *reinterpret_cast<const u32x4 *>(k_row + (64 * c + 16 * part < row_bytes ? 64 * c : 0));
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const char *p = v_row(r);
            if constexpr (BF16 && DP == 64) {
                const u32x2 x = *reinterpret_cast<const u32x2 *>(p);
                t.v[r][0] = x.x, t.v[r][1] = x.y;
            } else {
                constexpr uint32_t APART = BF16 ? 16 : 256;
#pragma unroll
                for (int w = 0; w < Tile::V_WORDS / 4; w++) {
                    const char *at = p + (WHOLE || APART * w + V_STEP * col < row_bytes ? APART * w : 0);
                    const u32x4 x = *reinterpret_cast<const u32x4 *>(at);
#pragma unroll
                    for (int e = 0; e < 4; e++) t.v[r][4 * w + e] = x[e];
                }
            }
        }
    };
    // Lanes without channels of their own read the first ones.
    const uint32_t k_byte = 16 * part < row_bytes ? 16 * part : 0, v_byte = V_STEP * col < row_bytes ? V_STEP * col : 0;
    const uint32_t k_off = col * slot_bytes + k_byte, v_off = 4 * part * slot_bytes + v_byte;
    auto load = [&](int32_t i, Tile &t) {
        if constexpr (UNIFORM) {
            const uint32_t low_word = __builtin_amdgcn_readlane((int32_t)starts, i & 63), high_word = __builtin_amdgcn_readlane((int32_t)(starts >> 32), i & 63);
            const int64_t start = (int64_t)((uint64_t)high_word << 32 | low_word);
            const char *k_tile = keys + start, *v_tile = values + start;
            auto v_row = [&](int r) { return v_tile + (uint64_t)r * slot_bytes + v_off; };
            if (g.d == DP) load_parts(t, std::true_type(), k_tile + k_off, v_row);
            else load_parts(t, std::false_type(), k_tile + k_off, v_row);
        } else {
            const int64_t row = row_ahead(i);
            auto v_row = [&](int r) {
                const uint32_t low_word = __shfl((int32_t)row, 4 * part + r), high_word = __shfl((int32_t)(row >> 32), 4 * part + r);
                return values + (int64_t)((uint64_t)high_word << 32 | low_word) + v_byte;
            };
            load_parts(t, std::false_type(), keys + row + k_byte, v_row);
        }
    };
    auto value_key = [&](int r) { return 4 * (int32_t)part + r; };
    // Slots that no row sees may hold anything: their weight is 0, so is their value then.
    auto clear_unseen = [&](int32_t key0, Tile &t) {
        if (key0 >= begin && key0 + KT <= end) return;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int32_t key = key0 + value_key(r);
            const bool seen = key >= begin && key < end;
#pragma unroll
            for (int w = 0; w < Tile::V_WORDS; w++) t.v[r][w] = seen ? t.v[r][w] : 0;
        }
    };

    float top = -INFINITY, total = 0.0f;
    f32x4 acc[NACC];
#pragma unroll
    for (int i = 0; i < NACC; i++) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // Scores of the tile (NS registers a lane, key0 + value_key(r)), running maximum and sum, weights in their place.
    constexpr int NS = 4;
    auto weigh = [&](int32_t key0, float (&x)[NS]) {
        const bool full = key0 >= all_low && key0 + KT <= all_high && key0 >= begin && key0 + KT <= end;
        scores(g, x, slope, place - key0, value_key);
        float most = -INFINITY;
#pragma unroll
        for (int r = 0; r < NS; r++) {
            const int32_t key = key0 + value_key(r);
            if (full || (key >= low && key < high && key >= begin && key < end)) most = fmaxf(most, x[r]);
        }
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        const float now = fmaxf(top, most);
        if (__any(now > top + SLACK)) {
            const float corr = weight_of(top, now);
            total *= corr;
#pragma unroll
            for (int i = 0; i < NACC; i++) acc[i] *= corr;
            top = now;
        }
        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int r = 0; r < NS; r++) {
            const int32_t key = key0 + value_key(r);
            const bool seen = full || (key >= low && key < high && key >= begin && key < end);
            x[r] = seen ? exp2_fast(x[r] - base) : 0.0f;
            total += x[r];
        }
    };

    auto products = [&](int32_t i, Tile &t) {
        const int32_t key0 = tile_key(i);
        float x[NS];
        f32x4 large = {0.0f, 0.0f, 0.0f, 0.0f}, small = large;
        if (BF16 || Q_HERE) asm volatile("" : "+v"(q_at));  // or what is in LDS would move to registers in front of the loop
#pragma unroll
        for (int c = 0; c < Tile::K_UNITS; c++) {
            if constexpr (BF16) {
                auto part_of = [&](int p) { return *reinterpret_cast<const u32x4 *>(&lds.q[0][q_at + p * Q_PART + 32 * c]); };
                ALTIUS_MFMA16_BF16(t.k[c], part_of(2), small);
                ALTIUS_MFMA16_BF16(t.k[c], part_of(0), large);
                ALTIUS_MFMA16_BF16(t.k[c], part_of(1), small);
            } else {
                u32x4 its_q;
                if constexpr (Q_HERE) its_q = *reinterpret_cast<const u32x4 *>(&lds.whole_q[q_at + 16 * c]);
                else its_q = q[c];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (c % 2 == 0) ALTIUS_MFMA16_F32(__uint_as_float(t.k[c][e]), __uint_as_float(its_q[e]), large);
                    else ALTIUS_MFMA16_F32(__uint_as_float(t.k[c][e]), __uint_as_float(its_q[e]), small);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 4; r++) x[r] = large[r] + small[r];
        weigh(key0, x);
        clear_unseen(key0, t);
        if constexpr (BF16) {
            u32x2 p[3];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                uint32_t w[3];
                split_pair(x[2 * e], x[2 * e + 1], w[0], w[1], w[2]);
                p[0][e] = w[0], p[1][e] = w[1], p[2][e] = w[2];
            }
            u32x2 v[NACC];
#pragma unroll
            for (int c = 0; c < NACC; c++) {
                const uint32_t pick = c % 2 ? 0x07060302u : 0x05040100u;
                v[c] = u32x2{__builtin_amdgcn_perm(t.v[1][c / 2], t.v[0][c / 2], pick), __builtin_amdgcn_perm(t.v[3][c / 2], t.v[2][c / 2], pick)};
            }
#pragma unroll
            for (int e = 2; e >= 0; e--)  // a sum's next term comes after all others': none waits for the one before
#pragma unroll
                for (int c = 0; c < NACC; c++) ALTIUS_MFMA16_BF16_K16(v[c], p[e], acc[c]);
        } else {
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int w = 0; w < Tile::V_WORDS; w++) ALTIUS_MFMA16_F32(__uint_as_float(t.v[r][w]), x[r], acc[w]);
        }
    };

    // Two tiles take turns, one on its way during the other's products; heads of more than 128 channels have registers for one.
    auto load_one = [&](int32_t i, Tile &t) {
        if (UNIFORM && (i & 63) == 0) fetch_starts(i);
        load(i, t);
        if (!UNIFORM) look_up(min(i + 1, mine - 1));
    };
    Tile a;
    if (mine > 0 && !UNIFORM) look_up(0);
    if constexpr (DP > 128) {
        for (int32_t i = 0; i < mine; i++) {
            load_one(i, a);
            products(i, a);
        }
    } else if (mine > 0) {
        Tile b;
        load_one(0, a);
        for (int32_t i = 0;;) {
            load_one(min(i + 1, mine - 1), b);
            products(i, a);
            if (++i >= mine) break;
            load_one(min(i + 1, mine - 1), a);
            products(i, b);
            if (++i >= mine) break;
        }
    }
    total += __shfl_xor(total, 16);
    total += __shfl_xor(total, 32);

    // An infinity or NaN among the keys or values, or a score beyond fp32, has left one here, and not always where the
    // definition has it (0 x infinity of a key that the row does not see; parts of infinity of opposite signs).  Once more then,
    // value by value.
    float check = total * 0.0f;
#pragma unroll
    for (int i = 0; i < NACC; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) check = __builtin_fmaf(acc[i][r], 0.0f, check);
    if (__any(valid && check != 0.0f)) {
        top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int i = 0; i < NACC; i++) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int32_t i = 0; i < mine; i++) {
            const int32_t from = max(tile_key(i), begin), to = min(tile_key(i) + KT, end);
            for (int32_t key = from; key < to; key++) {
                const int64_t at = row_at((uint32_t)key);
                float dot = 0.0f;
                if (valid)
                    for (uint32_t c = part; c < g.d; c += 4) dot = __builtin_fmaf(q_row[c] * g.scale, cache_value<BF16>(keys, at + c), dot);
                dot += __shfl_xor(dot, 16);
                dot += __shfl_xor(dot, 32);
                if (!sees || key < low || key >= high) continue;
                float x[1] = {dot};
                scores(g, x, slope, place - key, [](int) { return 0; });
                const float now_top = fmaxf(top, x[0]);
                const float corr = weight_of(top, now_top), p = exp2_fast(x[0] - (now_top == -INFINITY ? 0.0f : now_top));
                top = now_top;
                total = total * corr + p;
#pragma unroll
                for (int j = 0; j < NACC; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const uint32_t c = channel_of<DP, BF16>(j, r, part);
                        if (c < g.d) acc[j][r] = acc[j][r] * corr + p * cache_value<BF16>(values, at + c);
                    }
            }
        }
    }

    // The block's wavefronts join their parts, where queries were.
    if (BF16 || Q_HERE) __syncthreads();
    if (part == 0) stats[wave][0][col] = top, stats[wave][1][col] = total;
#pragma unroll
    for (int i = 0; i < NACC; i += 4)
#pragma unroll
        for (int r = 0; r < 4; r++)
            *reinterpret_cast<f32x4 *>(&sums[wave][col * PITCH + channel_of<DP, BF16>(i, r, part)]) = f32x4{acc[i][r], acc[i + 1][r], acc[i + 2][r], acc[i + 3][r]};
    __syncthreads();

    for (uint32_t unit = threadIdx.x; unit < 16 * (DP / 4); unit += 64 * ROW_WAVES) {
        const uint32_t r = unit / (DP / 4), c = 4 * (unit % (DP / 4)), mine_row = tile * 16 + r;
        if (mine_row >= rows || c >= g.d) continue;
        float m = stats[0][0][r];
#pragma unroll
        for (int w = 1; w < ROW_WAVES; w++) m = fmaxf(m, stats[w][0][r]);
        float l = 0.0f;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < ROW_WAVES; w++) {
            const float f = weight_of(stats[w][0][r], m);
            l = __builtin_fmaf(stats[w][1][r], f, l);
            o += *reinterpret_cast<const f32x4 *>(&sums[w][r * PITCH + c]) * f;
        }
        if (SPLIT && !piece.whole) {
            const size_t at = (size_t)piece.slot * 16 + r;
            *reinterpret_cast<f32x4 *>(g.few.part_out + at * g.d + c) = o;
            if (c == 0) g.few.part_stats[2 * at] = m, g.few.part_stats[2 * at + 1] = l;
        } else {
            const uint32_t t = g.by_group.div(mine_row), h = kvh * g.group + mine_row - t * g.group;
            const RowRange of = row_range(g, seq, s, t);
            const float recip = of.low < of.high ? 1.0f / l : 0.0f;
            *reinterpret_cast<f32x4 *>(g.out + (int64_t)(seq.start + (int32_t)t) * g.out_token + (int64_t)h * g.out_head + c) =
                of.low < of.high ? o * recip : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
}

template <int DP, bool BF16, bool UNIFORM, bool SPLIT>
__device__ __forceinline__ void rows16(const AttendArgs &g, uint32_t id, RowLds<DP, BF16> &lds) {
    const Share &share = SPLIT ? g.few : g.many;
    Piece piece = {0, 0, 0, 0, INT32_MAX, true, 0};
    if (!SPLIT || !share.listed) {
        const uint32_t outer = id / g.kv.kv_heads;
        piece.kvh = id - outer * g.kv.kv_heads;
        piece.tile = outer % share.row_tiles, piece.s = outer / share.row_tiles;
        piece16<DP, BF16, UNIFORM, SPLIT>(g, piece, lds);
        return;
    }
    Found f;
    if (!find<true>(g, false, id, f)) return;
    const uint32_t inside = id - f.before, pair = inside / f.parts, part = inside - pair * f.parts;
    piece.s = f.s, piece.tile = pair / g.kv.kv_heads, piece.kvh = pair - piece.tile * g.kv.kv_heads;
    piece.from = f.first_key(part), piece.to = part + 1 == f.parts ? INT32_MAX : f.first_key(part + 1);
    piece.whole = f.parts == 1;
    piece.slot = id;
    piece16<DP, BF16, UNIFORM, SPLIT>(g, piece, lds);
}

// Heads of more than 128 channels have no tiles of 128 rows: all their rows go 16 a wavefront (SPLIT false).
template <int DP, bool BF16, bool UNIFORM, bool SPLIT>
__global__ __launch_bounds__(64 * ROW_WAVES, DP == 256 ? 1 : BF16 && DP == 128 ? 3 : 2) void attend_rows16(AttendArgs g) {
    __shared__ __align__(16) RowLds<DP, BF16> lds;
    rows16<DP, BF16, UNIFORM, SPLIT>(g, blockIdx.x, lds);
}

// ---------------------------------------------------------------- 128 rows a block, keys through LDS
// A wavefront owns 32 rows; the block's four share tiles of 32 keys in LDS.  S^T = K Q^T and O^T = V^T P^T again, by
// v_mfma_f32_32x32x16_bf16: accumulator register r of lane l holds row l % 32 and key 8 (r / 4) + 4 (l / 32) + r % 4, and the
// second product takes its k slots in that order, in which V^T lies in LDS.  Queries and weights are three bf16 numbers each, as
// above; so are the values of an fp32 cache, split on their way into LDS, and six products of the parts are what fp32 holds of the
// whole (the three left out are below 2^-24 of it).  A bf16 cache's values are one number: three products.
//   Two tiles of each operand in LDS, one barrier a tile.  A prompt of 4096 with a window of 1500 (16 heads, 4 of keys, 128
// channels, bf16, capped) takes 150 us, 275 TFLOP/s of scores and sums, 825 of the instructions' own, where a large bf16 product
// reaches 1356; 4 prompts of 1024 (12 heads of 64 channels, fp32) 58 us, 111 and 670.  The matrix cores are busy 29 and 26 % of the time, the
// vector unit 35 and 28 %: bound by waits with one or two wavefronts a SIMD and by places left empty, since blocks see different numbers of keys
// (1.25 times the mean the longest with the window, 4 to 32 tiles in the prompts).
constexpr int TILE_KEYS = 32;

#define ALTIUS_MFMA32_BF16(A, B, C) \
    C = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, A), __builtin_bit_cast(bf16x8, B), C, 0, 0, 0)

template <int DP, bool BF16> struct TileLds {
    static constexpr int PLANES = BF16 ? 1 : 3;
    static constexpr int K_PITCH = DP + 8;          // 16-bit words; 16 rows of 16-byte reads cover all banks
    static constexpr int V_PITCH = TILE_KEYS + 8;   // a row is a channel
    // The queries' third parts, read once a tile, where registers do not hold all three.
    static constexpr bool Q_HERE = DP > 64;
    uint16_t k[2][PLANES][TILE_KEYS * K_PITCH], v[2][PLANES][DP * V_PITCH];
    uint16_t q[Q_HERE ? 4 : 1][Q_HERE ? 32 * K_PITCH : 8];
    int32_t bounds[4][2];
};

template <int DP, bool BF16, bool UNIFORM>
__device__ __forceinline__ void rows128(const AttendArgs &g, uint32_t id, TileLds<DP, BF16> &lds) {
    using Lds = TileLds<DP, BF16>;
    constexpr int PLANES = Lds::PLANES, K_PITCH = Lds::K_PITCH, V_PITCH = Lds::V_PITCH;
    constexpr int STEPS = DP / 16, PARTS = DP / 32;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t col = lane & 31u, h = lane >> 5;

    const Share &share = g.many;
    uint32_t kvh, s, tile;
    int32_t from = 0, to = INT32_MAX;
    bool whole = true;
    const bool first_rows_first = g.first_keys && (g.prefix || !g.causal);
    if (!share.listed) {
        // The last rows of a causal sequence see most keys: they start first.  Of documents whose first keys are open to all rows (or
        // later ones to earlier rows) the first rows see most.  Blocks that follow each other work on different heads.
        kvh = id % g.kv.kv_heads;
        const uint32_t outer = id / g.kv.kv_heads, order = outer / g.kv.sequences;
        s = outer % g.kv.sequences;
        tile = first_rows_first ? order : share.row_tiles - 1 - order;
    } else {
        Found f;
        if (!find<false>(g, false, id, f)) return;
        const uint32_t inside = id - f.before, pair = inside / f.parts, part = inside - pair * f.parts;
        s = f.s, tile = pair / g.kv.kv_heads, kvh = pair - tile * g.kv.kv_heads;
        from = f.first_key(part), to = part + 1 == f.parts ? INT32_MAX : f.first_key(part + 1);
        whole = f.parts == 1;
        if (whole && !first_rows_first) tile = f.work.pairs / g.kv.kv_heads - 1 - tile;
    }

    const dev::KvSequence seq = sequence_of(g, s);
    const uint32_t rows = (uint32_t)seq.n * g.group;
    if (rows <= g.few_rows || tile * TILE_ROWS >= rows) return;
    const uint32_t row = tile * TILE_ROWS + wave * 32 + col;
    const bool valid = row < rows;
    const uint32_t token = g.by_group.div(valid ? row : 0), head = kvh * g.group + (valid ? row : 0) - token * g.group;
    const RowRange range = row_range(g, seq, s, token);
    const int32_t low = range.low, high = range.high, place = range.place;
    const bool sees = valid && low < high;
    const float slope = g.slopes ? g.slopes[head] * LOG2E : 0.0f;

    int32_t any_low = sees ? low : INT32_MAX, any_high = sees ? high : 0, all_low = valid ? low : 0, all_high = valid ? high : INT32_MAX;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        any_low = min(any_low, __shfl_xor(any_low, m)), any_high = max(any_high, __shfl_xor(any_high, m));
        all_low = max(all_low, __shfl_xor(all_low, m)), all_high = min(all_high, __shfl_xor(all_high, m));
    }
    if (lane == 0) lds.bounds[wave][0] = any_low, lds.bounds[wave][1] = any_high;
    __syncthreads();
    int32_t begin = INT32_MAX, end = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) begin = min(begin, lds.bounds[w][0]), end = max(end, lds.bounds[w][1]);
    begin = max(begin, from), end = min(end, to);
    begin = __builtin_amdgcn_readfirstlane(begin), end = __builtin_amdgcn_readfirstlane(end);
    any_low = max(begin, __builtin_amdgcn_readfirstlane(any_low)), any_high = min(end, __builtin_amdgcn_readfirstlane(any_high));
    all_low = max(begin, __builtin_amdgcn_readfirstlane(all_low)), all_high = min(end, __builtin_amdgcn_readfirstlane(all_high));
    const int32_t first = begin / TILE_KEYS, tiles = begin < end ? (end + TILE_KEYS - 1) / TILE_KEYS - first : 0;
    // The tiles that this wavefront's rows see.
    const int32_t mine_from = any_low < any_high ? any_low / TILE_KEYS - first : INT32_MAX - 1, mine_to = any_low < any_high ? (any_high + TILE_KEYS - 1) / TILE_KEYS - first : 0;

    const char *keys = static_cast<const char *>(g.kv.keys), *values = static_cast<const char *>(g.kv.values);
    constexpr int SIZE = BF16 ? 2 : 4;
    const int64_t head_at = (int64_t)kvh * g.kv.head_stride;

    // Staging.  Keys: 16-byte units, a row after the other.  Values: blocks of 4 keys (which lie side by side in V^T) and VC
    // channels.  All threads do the same, without a branch: where the units or blocks are fewer, some are fetched and written twice.
    constexpr int VC = DP == 64 ? 2 : 4, V_BLOCKS = 8 * (DP / VC), K_UNITS_ROW = DP * SIZE / 16, K_UNITS = TILE_KEYS * K_UNITS_ROW, K_EACH = (K_UNITS + 255) / 256;
    static_assert(V_BLOCKS <= 256 && DP % VC == 0, "staging");
    const uint32_t v_tid = V_BLOCKS == 256 ? tid : tid % V_BLOCKS, v_block = v_tid & 7u, v_channel = VC * (v_tid >> 3);
    // Keys 4 b .. 4 b + 3 of a tile are slots 16 (b / 4) + 8 (b % 2) + 4 (b / 2 % 2) on.
    const uint32_t v_slot = 16 * (v_block >> 2) + 8 * (v_block & 1u) + 4 * ((v_block >> 1) & 1u);
    // Unit e of a thread is K_ROWS keys behind the one before, in the same channels, where that divides the rows up evenly.
    constexpr bool EVEN = 256 % K_UNITS_ROW == 0 && K_UNITS % 256 == 0;
    constexpr int K_ROWS = 256 / K_UNITS_ROW;
    auto k_key = [&](int e) { return EVEN ? tid / K_UNITS_ROW + e * K_ROWS : (e * 256 + tid) % K_UNITS / K_UNITS_ROW; };
    auto k_unit = [&](int e) { return EVEN ? tid % K_UNITS_ROW : (e * 256 + tid) % K_UNITS % K_UNITS_ROW; };
    constexpr int V_WORDS = VC * SIZE / 4;  // of a key
    typedef uint32_t VWords __attribute__((ext_vector_type(V_WORDS == 1 ? 2 : V_WORDS)));
    u32x4 k_stage[K_EACH];
    VWords v_stage[4];

    // Where pages hold at least half a tile: where the next 32 tiles' halves start, in bytes from the start of the cache, a half a lane.
    int64_t starts = 0;
    auto fetch_starts = [&](int32_t from) {
        const int32_t key = (first + from) * TILE_KEYS + 16 * (int32_t)lane;
        if (!UNIFORM) return;
        // A half that nobody sees any of may have no page: it is read from the start of the cache, and left out.
        const uint32_t index = g.kv.by_page_size.div((uint32_t)max(begin, min(key, end - 1)));
        starts = ((int64_t)g.kv.page_of(s, index, 0) * g.kv.page_stride + (int64_t)((uint32_t)key - index * g.kv.page_size) * g.kv.slot_stride + head_at) * SIZE;
        if (key >= end || key + 16 <= begin) starts = 0;
    };
    auto row_at = [&](uint32_t key) {  // elements from the start of the cache
        const uint32_t index = g.kv.by_page_size.div(key);
        return (int64_t)g.kv.page_of(s, index, 0) * g.kv.page_stride + (int64_t)(key - index * g.kv.page_size) * g.kv.slot_stride + head_at;
    };
    const uint32_t slot_bytes = (uint32_t)g.kv.slot_stride * SIZE;
    // No load below depends on a condition, which would have the compiler wait for those before it.  Channels that a head does not
    // have are read as its first ones: their queries are 0, their sums go nowhere.
    auto k_byte = [&](int e) { return (16 / SIZE) * k_unit(e) < g.d ? 16 * k_unit(e) : 0u; };
    const uint32_t v_byte = v_channel < g.d ? SIZE * v_channel : 0;
    const uint32_t k_off = tid / K_UNITS_ROW % 16 * slot_bytes + k_byte(0), v_off = 4 * (v_block & 3u) * slot_bytes + v_byte;
    struct Halves {
        int64_t at[2];
    };
    auto halves_of = [&](int32_t i) {
        Halves t;
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t low_word = __builtin_amdgcn_readlane((int32_t)starts, (2 * i + half) & 63), high_word = __builtin_amdgcn_readlane((int32_t)(starts >> 32), (2 * i + half) & 63);
            t.at[half] = (int64_t)((uint64_t)high_word << 32 | low_word);
        }
        return t;
    };
    // Where they do not: lane l has the row of key l % 32 of a tile, looked up a tile ahead of its first use.  Keys in front of the first
    // that is seen and behind the last may have no page: those two stand in for them.
    int32_t page_ahead = 0;
    int64_t rows_next = 0, rows_ahead = 0;  // bytes from the start of the cache, of tiles i + 1 and i + 2 while tile i is computed
    auto key_ahead = [&](int32_t i) { return (uint32_t)max(begin, min((first + i) * TILE_KEYS + (int32_t)col, end - 1)); };
    auto look_up = [&](int32_t i) { page_ahead = g.kv.table[(int64_t)s * g.kv.table_stride + g.kv.by_page_size.div(key_ahead(i))]; };
    auto advance = [&](int32_t i) {  // to tile i, whose pages are known
        const uint32_t key = key_ahead(i);
        if ((uint32_t)page_ahead >= g.kv.pages) *g.kv.flag = 1;
        const int32_t page = (uint32_t)page_ahead < g.kv.pages ? page_ahead : 0;
        rows_next = rows_ahead;
        rows_ahead = ((int64_t)page * g.kv.page_stride + (int64_t)(key - g.kv.by_page_size.div(key) * g.kv.page_size) * g.kv.slot_stride + head_at) * SIZE;
    };
    auto row_of = [&](int64_t rows_of_tile, uint32_t key) {
        const uint32_t low_word = __shfl((int32_t)rows_of_tile, key), high_word = __shfl((int32_t)(rows_of_tile >> 32), key);
        return (int64_t)((uint64_t)high_word << 32 | low_word);
    };
    auto fetch_keys = [&](const Halves &half) {
#pragma unroll
        for (int e = 0; e < K_EACH; e++) {
            const char *p;
            if constexpr (!UNIFORM) p = keys + row_of(rows_ahead, k_key(e)) + k_byte(e);
            else if constexpr (EVEN && K_ROWS <= 16) p = keys + half.at[e * K_ROWS / 16] + (uint64_t)(e * K_ROWS % 16) * slot_bytes + k_off;
            else if constexpr (EVEN) p = keys + (k_key(e) < 16 ? half.at[0] : half.at[1]) + k_off;
            else p = keys + (k_key(e) < 16 ? half.at[0] : half.at[1]) + (k_key(e) % 16 * slot_bytes + k_byte(e));
            k_stage[e] = *reinterpret_cast<const u32x4 *>(p);
        }
    };
    auto fetch_values = [&](const Halves &half, int64_t rows_of_tile) {
        const char *base = values + (v_block < 4 ? half.at[0] : half.at[1]) + v_off;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const char *p = UNIFORM ? base + (uint64_t)e * slot_bytes : values + row_of(rows_of_tile, 4 * v_block + e) + v_byte;
            if constexpr (V_WORDS == 1) v_stage[e][0] = *reinterpret_cast<const uint32_t *>(p);
            else v_stage[e] = *reinterpret_cast<const VWords *>(p);
        }
    };
    // Slots that no row sees may hold anything: their weight is 0, so is their value then.
    auto clear_unseen = [&](int32_t i) {
        const int32_t key0 = (first + i) * TILE_KEYS;
        if (key0 >= begin && key0 + TILE_KEYS <= end) return;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int32_t key = key0 + 4 * (int32_t)v_block + e;
            const bool seen = key >= begin && key < end;
#pragma unroll
            for (int w = 0; w < V_WORDS; w++) v_stage[e][w] = seen ? v_stage[e][w] : 0;
        }
    };
    auto park_key = [&](int buffer, int e) {
        uint16_t *to = &lds.k[buffer][0][k_key(e) * K_PITCH + (16 / SIZE) * k_unit(e)];
        if constexpr (BF16) {
            *reinterpret_cast<u32x4 *>(to) = k_stage[e];
        } else {
            uint32_t p[3][2];
#pragma unroll
            for (int w = 0; w < 2; w++) split_pair(__uint_as_float(k_stage[e][2 * w]), __uint_as_float(k_stage[e][2 * w + 1]), p[0][w], p[1][w], p[2][w]);
#pragma unroll
            for (int q = 0; q < 3; q++) *reinterpret_cast<u32x2 *>(to + q * (TILE_KEYS * K_PITCH)) = u32x2{p[q][0], p[q][1]};
        }
    };
    auto park_value = [&](int buffer, int c) {
        uint16_t *to = &lds.v[buffer][0][(v_channel + c) * V_PITCH + v_slot];
        if constexpr (BF16) {
            const uint32_t pick = c % 2 ? 0x07060302u : 0x05040100u;
            *reinterpret_cast<u32x2 *>(to) =
                u32x2{__builtin_amdgcn_perm(v_stage[1][c / 2], v_stage[0][c / 2], pick), __builtin_amdgcn_perm(v_stage[3][c / 2], v_stage[2][c / 2], pick)};
        } else {
            uint32_t p[3][2];
#pragma unroll
            for (int w = 0; w < 2; w++) split_pair(__uint_as_float(v_stage[2 * w][c]), __uint_as_float(v_stage[2 * w + 1][c]), p[0][w], p[1][w], p[2][w]);
#pragma unroll
            for (int q = 0; q < 3; q++) *reinterpret_cast<u32x2 *>(to + q * (DP * V_PITCH)) = u32x2{p[q][0], p[q][1]};
        }
    };
    // Of the units of keys and channels of values that a thread puts into LDS, keys first, those from .. to - 1.
    constexpr int PARKED = K_EACH + VC;
    auto park = [&](int from, int to, int key_buffer, int value_buffer) {
#pragma unroll
        for (int n = from; n < to; n++) {
            if (n < K_EACH) park_key(key_buffer, n);
            else park_value(value_buffer, n - K_EACH);
        }
    };

    // The first tile's keys and values and the second's keys, while the queries are split.
    Halves next = {};  // of the tile whose values are fetched next: its keys were a tile ago
    if (tiles > 0) {
        if (UNIFORM) fetch_starts(0), next = halves_of(0);
        else look_up(0), advance(0), look_up(min(1, tiles - 1));
        fetch_keys(next), fetch_values(next, rows_ahead);
        if (UNIFORM) next = halves_of(1);
        else advance(min(1, tiles - 1)), look_up(min(2, tiles - 1));
    }
    const float *q_row = g.q + (int64_t)(seq.start + (int32_t)token) * g.q_token + (int64_t)head * g.q_head;
    u32x4 q[Lds::Q_HERE ? 2 : 3][STEPS];
    uint16_t *q_here = &lds.q[Lds::Q_HERE ? wave : 0][Lds::Q_HERE ? col * K_PITCH + 8 * h : 0];
    if constexpr (Lds::Q_HERE) {
        // A row of queries by DP / 4 lanes side by side, all loads on their way at once, then part by part through LDS, where the third
        // ones stay.  (A lane that reads its own row asks for 64 lines with each load.)
        constexpr int UNITS = 32 * (DP / 4) / 64;
        const int64_t mine = (int64_t)(seq.start + (int32_t)token) * g.q_token + (int64_t)head * g.q_head;
        f32x4 whole[UNITS];
        auto row_unit = [&](int e) { return (64 * e + lane) / (DP / 4); };
        auto channel_unit = [&](int e) { return 4 * ((64 * e + lane) % (DP / 4)); };
#pragma unroll
        for (int e = 0; e < UNITS; e++) {
            const uint32_t low_word = __shfl((int32_t)mine, row_unit(e)), high_word = __shfl((int32_t)(mine >> 32), row_unit(e));
            whole[e] = *reinterpret_cast<const f32x4 *>(g.q + (int64_t)((uint64_t)high_word << 32 | low_word) + (channel_unit(e) < g.d ? channel_unit(e) : 0));
        }
        const float scale = g.scale;
        u32x2 third[UNITS], second[UNITS];
        uint16_t *shared = lds.q[wave];
#pragma unroll
        for (int e = 0; e < UNITS; e++) {
            const float by = channel_unit(e) < g.d ? scale : 0.0f;
            uint32_t w[3][2];
            split_pair(whole[e][0] * by, whole[e][1] * by, w[0][0], w[1][0], w[2][0]);
            split_pair(whole[e][2] * by, whole[e][3] * by, w[0][1], w[1][1], w[2][1]);
            *reinterpret_cast<u32x2 *>(shared + row_unit(e) * K_PITCH + channel_unit(e)) = u32x2{w[0][0], w[0][1]};
            second[e] = u32x2{w[1][0], w[1][1]}, third[e] = u32x2{w[2][0], w[2][1]};
        }
        auto wait = [] { __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront"), __builtin_amdgcn_wave_barrier(); };
#pragma unroll
        for (int p = 0; p < 2; p++) {
            wait();
#pragma unroll
            for (int i = 0; i < STEPS; i++) q[p][i] = *reinterpret_cast<const u32x4 *>(q_here + 16 * i);
            wait();
#pragma unroll
            for (int e = 0; e < UNITS; e++) *reinterpret_cast<u32x2 *>(shared + row_unit(e) * K_PITCH + channel_unit(e)) = p == 0 ? second[e] : third[e];
        }
        wait();
    } else {
        f32x4 lo[STEPS], hi[STEPS];
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            const uint32_t c = 16 * i + 8 * h;
            lo[i] = *reinterpret_cast<const f32x4 *>(q_row + (c < g.d ? c : 0)), hi[i] = *reinterpret_cast<const f32x4 *>(q_row + (c + 4 < g.d ? c + 4 : 0));
        }
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            const uint32_t c = 16 * i + 8 * h;
            const float by[2] = {c < g.d ? g.scale : 0.0f, c + 4 < g.d ? g.scale : 0.0f};
            uint32_t w[3][4];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                split_pair(lo[i][2 * e] * by[0], lo[i][2 * e + 1] * by[0], w[0][e], w[1][e], w[2][e]);
                split_pair(hi[i][2 * e] * by[1], hi[i][2 * e + 1] * by[1], w[0][2 + e], w[1][2 + e], w[2][2 + e]);
            }
#pragma unroll
            for (int p = 0; p < 3; p++) q[p][i] = u32x4{w[p][0], w[p][1], w[p][2], w[p][3]};
        }
    }

    float top = -INFINITY, total = 0.0f;
    f32x16 acc[PARTS], st;
#pragma unroll
    for (int i = 0; i < PARTS; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[i][r] = 0.0f;

    auto key_of = [&](int r) { return 8 * (r >> 2) + 4 * (int32_t)h + (r & 3); };
    // Smallest terms first.
    auto multiply = [&](const u32x4 (&a)[PLANES], const u32x4 &b0, const u32x4 &b1, const u32x4 &b2, f32x16 &c) {
        if constexpr (BF16) {
            ALTIUS_MFMA32_BF16(a[0], b2, c);
            ALTIUS_MFMA32_BF16(a[0], b1, c);
            ALTIUS_MFMA32_BF16(a[0], b0, c);
        } else {
            ALTIUS_MFMA32_BF16(a[0], b2, c);
            ALTIUS_MFMA32_BF16(a[2], b0, c);
            ALTIUS_MFMA32_BF16(a[1], b1, c);
            ALTIUS_MFMA32_BF16(a[0], b1, c);
            ALTIUS_MFMA32_BF16(a[1], b0, c);
            ALTIUS_MFMA32_BF16(a[0], b0, c);
        }
    };
    // FENCED: operands are read from LDS a step before they are used, and what is done beside a step stays between its fences, where
    // the compiler deals it out among the matrix instructions.  One wavefront a SIMD has nothing else to fill the waits with: 3 prompts
    // of documents, fp32, d = 128: 108 -> 99 us; d = 64, two a SIMD: 63 -> 60 us.  A bf16 cache's kernel has no registers left for
    // it: a prompt of 4096 with a window takes 152 us without and 194 us with it.
    constexpr bool FENCED = !BF16;
    auto fence = [] { if constexpr (FENCED) __builtin_amdgcn_sched_barrier(0); };
    struct Operand {
        u32x4 of[PLANES], third;
    };
    auto key_operand = [&](int buffer, int c, Operand &a) {
#pragma unroll
        for (int p = 0; p < PLANES; p++) a.of[p] = *reinterpret_cast<const u32x4 *>(&lds.k[buffer][p][col * K_PITCH + 16 * c + 8 * h]);
        if constexpr (Lds::Q_HERE) a.third = *reinterpret_cast<const u32x4 *>(q_here + 16 * c);
    };
    auto value_operand = [&](int buffer, int step, Operand &a) {
#pragma unroll
        for (int w = 0; w < PLANES; w++)
            a.of[w] = *reinterpret_cast<const u32x4 *>(&lds.v[buffer][w][(32 * (step % PARTS) + col) * V_PITCH + 16 * (step / PARTS) + 8 * h]);
    };
    auto first_product = [&](int buffer, auto beside) {
#pragma unroll
        for (int r = 0; r < 16; r++) st[r] = 0.0f;
        Operand a[2];
        if (FENCED) key_operand(buffer, 0, a[0]);
#pragma unroll
        for (int c = 0; c < STEPS; c++) {
            if (!FENCED) key_operand(buffer, c, a[c & 1]);
            else if (c + 1 < STEPS) key_operand(buffer, c + 1, a[(c + 1) & 1]);
            if constexpr (Lds::Q_HERE) multiply(a[c & 1].of, q[0][c], q[1][c], a[c & 1].third, st);
            else multiply(a[c & 1].of, q[0][c], q[1][c], q[2][c], st);
            beside(c);
            fence();
        }
    };

    if (tiles > 0) {
        clear_unseen(0);
        park(0, PARKED, 0, 0);
        if (tiles > 1) {
            fetch_keys(next);
            park(0, K_EACH, 1, 0);
        }
        __syncthreads();
        if (mine_from == 0) first_product(0, [](int) {});
    }
    // Tile i: its scores are in registers, its values and the next tile's keys in LDS.  The next tile's first product runs beside the
    // exponentials and splits of this one's weights, this one's second product beside the staging of the tiles behind: the matrix
    // cores and the vector unit have work at the same time, in one wavefront as in two.
    for (int32_t i = 0; i < tiles; i++) {
        __syncthreads();
        const int32_t key0 = (first + i) * TILE_KEYS;
        // Tiles i + 2 and i + 1; behind the last one it is fetched again, and not read.
        const int32_t ahead = min(i + 2, tiles - 1);
        if (UNIFORM) {
            fetch_values(next, 0);
            if ((ahead & 31) == 0) fetch_starts(ahead);
            next = halves_of(ahead);
        } else {
            advance(ahead);
            fetch_values(next, rows_next);
            look_up(min(i + 3, tiles - 1));
        }
        fetch_keys(next);
        if (i >= mine_from && i < mine_to) {
            float x[16];
#pragma unroll
            for (int r = 0; r < 16; r++) x[r] = st[r];
            scores(g, x, slope, place - key0, key_of);
            if (key0 < all_low || key0 + TILE_KEYS > all_high) {
                // A score that is not there is minus infinity: its weight is 0 once a finite maximum is known, and the row that has none
                // yet takes 0 for it.
                const int32_t from = max(low, begin) - key0, to = min(high, end) - key0;
#pragma unroll
                for (int r = 0; r < 16; r++) x[r] = key_of(r) >= from && key_of(r) < to ? x[r] : -INFINITY;
            }
            float most = x[0], lower, upper;
#pragma unroll
            for (int r = 1; r < 15; r += 2) most = max3(most, x[r], x[r + 1]);
            most = max3(most, x[15], x[15]);
            halves(most, lower, upper);
            const float now = max3(top, lower, upper);
            if (__any(now > top + SLACK)) {
                const float corr = weight_of(top, now);
                total *= corr;
#pragma unroll
                for (int t = 0; t < PARTS; t++)
#pragma unroll
                    for (int r = 0; r < 16; r++) acc[t][r] *= corr;
                top = now;
            }
            const float base = top == -INFINITY ? 0.0f : top;
            if (i + 1 == tiles - 1) clear_unseen(i + 1);
            Operand v[2];
            u32x4 p[2][3];
            auto weights = [&](int from, int to) {  // pairs of them
#pragma unroll
                for (int n = from; n < to; n++) {
                    const float a = exp2_fast(x[2 * n] - base), b = exp2_fast(x[2 * n + 1] - base);
                    total += a;
                    total += b;
                    uint32_t w[3];
                    split_pair(a, b, w[0], w[1], w[2]);
#pragma unroll
                    for (int e = 0; e < 3; e++) p[n / 4][e][n % 4] = w[e];
                }
            };
            if (!FENCED) weights(0, 8);
            fence();
            first_product((i + 1) & 1, [&](int c) {
                if (!FENCED) return;
                if (c + 1 == STEPS) value_operand(i & 1, 0, v[0]);
                weights(8 * c / STEPS, 8 * (c + 1) / STEPS);
            });
#pragma unroll
            for (int step = 0; step < 2 * PARTS; step++) {
                if (!FENCED) value_operand(i & 1, step, v[step & 1]);
                else if (step + 1 < 2 * PARTS) value_operand(i & 1, step + 1, v[(step + 1) & 1]);
                const auto &w = p[step / PARTS];
                multiply(v[step & 1].of, w[0], w[1], w[2], acc[step % PARTS]);
                if (FENCED) park(step * PARKED / (2 * PARTS), (step + 1) * PARKED / (2 * PARTS), i & 1, (i + 1) & 1);
                fence();
            }
            if (!FENCED) park(0, PARKED, i & 1, (i + 1) & 1);
        } else {
            if (i + 1 == mine_from) first_product((i + 1) & 1, [](int) {});
            if (i + 1 == tiles - 1) clear_unseen(i + 1);
            park(0, PARKED, i & 1, (i + 1) & 1);
        }
    }
    {
        float lower, upper;
        halves(total, lower, upper);
        total = lower + upper;
    }

    // As in piece16: what is not finite is computed once more, value by value.
    float check = total * 0.0f;
#pragma unroll
    for (int t = 0; t < PARTS; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) check = __builtin_fmaf(acc[t][r], 0.0f, check);
    if (__any(valid && check != 0.0f)) {
        top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int t = 0; t < PARTS; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[t][r] = 0.0f;
        for (int32_t key = max(begin, any_low); key < min(end, any_high); key++) {
            const int64_t at = row_at((uint32_t)key);
            float dot = 0.0f;
            if (valid)
                for (uint32_t c = h; c < g.d; c += 2) dot = __builtin_fmaf(q_row[c] * g.scale, cache_value<BF16>(keys, at + c), dot);
            dot += __shfl_xor(dot, 32);
            if (!sees || key < low || key >= high) continue;
            float x[1] = {dot};
            scores(g, x, slope, place - key, [](int) { return 0; });
            const float now = fmaxf(top, x[0]);
            const float corr = weight_of(top, now), p = exp2_fast(x[0] - (now == -INFINITY ? 0.0f : now));
            top = now;
            total = total * corr + p;
#pragma unroll
            for (int t = 0; t < PARTS; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const uint32_t c = 32 * t + (uint32_t)key_of(r);
                    if (c < g.d) acc[t][r] = acc[t][r] * corr + p * cache_value<BF16>(values, at + c);
                }
        }
    }

    if (!valid) return;
    const size_t at = (size_t)id * TILE_ROWS + wave * 32 + col;
    float *const row_out = whole ? g.out + (int64_t)(seq.start + (int32_t)token) * g.out_token + (int64_t)head * g.out_head : share.part_out + at * g.d;
    const float factor = !whole ? 1.0f : 1.0f / total;
    if (!whole && h == 0) share.part_stats[2 * at] = top, share.part_stats[2 * at + 1] = total;
#pragma unroll
    for (int t = 0; t < PARTS; t++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const uint32_t c = 32 * t + 8 * b + 4 * h;
            if (c >= g.d) continue;
            f32x4 o = {acc[t][4 * b], acc[t][4 * b + 1], acc[t][4 * b + 2], acc[t][4 * b + 3]};
            *reinterpret_cast<f32x4 *>(row_out + c) = !whole ? o : sees ? o * factor : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
}

// Prompts, and the sequences of few rows that share a batch with them: the last blocks are the latter's, and end at once where there
// are none.
template <int DP, bool BF16, bool UNIFORM>
__global__ __launch_bounds__(256, BF16 || DP == 64 ? 2 : 1) void attend_rows128(AttendArgs g) {
    __shared__ __align__(16) union {
        RowLds<DP <= 64 ? 64 : 128, BF16> few;
        TileLds<DP, BF16> many;
    } lds;
    if (blockIdx.x < g.many.blocks) rows128<DP, BF16, UNIFORM>(g, blockIdx.x, lds.many);
    else rows16<DP <= 64 ? 64 : 128, BF16, UNIFORM, true>(g, blockIdx.x - g.many.blocks, lds.few);
}

// Joins the splits of a row, of which only those that hold keys that it sees were computed for it.  A group of lanes holds the row's
// channels, four a lane.  few: a block per row, whose groups of lanes deal the splits out among themselves; else a group per row.  Bound by
// latency: the scan for a row's parts, their statistics, their sums.  10 us behind one row's 512 parts, 10 us behind 5 pieces of 57 to 333 rows,
// 4 to 5 us where the sizes allow parts and there are none.
constexpr int JOIN = 256, MOST_SPLITS = 1024;
__global__ __launch_bounds__(JOIN) void join_splits(AttendArgs g, uint32_t few_blocks) {
    __shared__ float factors[MOST_SPLITS];
    __shared__ __align__(16) f32x4 sums[JOIN];
    __shared__ float totals[JOIN / 64];
    const bool few = blockIdx.x < few_blocks;
    const Share &share = few ? g.few : g.many;
    const uint32_t lanes = g.d / 4, groups = JOIN / lanes, lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
    const uint32_t id = few ? blockIdx.x : blockIdx.x - few_blocks, chunks = few ? share.rows : (share.rows + groups - 1) / groups;
    const uint32_t outer = id / chunks, row = few ? id - outer * chunks : (id - outer * chunks) * groups + group;
    const uint32_t kvh = outer % g.kv.kv_heads, s = outer / g.kv.kv_heads;
    const dev::KvSequence seq = sequence_of(g, s);
    const uint32_t rows = (uint32_t)seq.n * g.group;
    if ((rows <= g.few_rows) != few || row - (few ? 0 : group) >= rows) return;
    Found f;
    if (!(few ? find<true>(g, true, s, f) : find<false>(g, true, s, f)) || f.parts <= 1) return;  // one block did it all
    if (!few && (group >= groups || row >= rows)) return;
    const uint32_t t = g.by_group.div(row), h = kvh * g.group + row - t * g.group;
    const RowRange of = row_range(g, seq, s, t);
    float *to = g.out + (int64_t)(seq.start + (int32_t)t) * g.out_token + (int64_t)h * g.out_head + 4 * lane;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    if (of.low >= of.high) {
        if (!few || group == 0) *reinterpret_cast<f32x4 *>(to) = zero;
        return;
    }
    // Partial results, and how many rows they are apart.  A row of few has all; of more, those of the keys that it sees.
    uint32_t count = f.parts, apart = 16, first = 0, tile = row / 16, inside = row % 16;
    if (!few) {
        first = f.part_with(of.low), count = f.part_with(of.high - 1) + 1 - first;
        apart = TILE_ROWS, tile = row / TILE_ROWS, inside = row % TILE_ROWS;
    }
    const size_t at = (size_t)(f.before + (tile * g.kv.kv_heads + kvh) * f.parts + first) * apart + inside;
    const float *stats = share.part_stats + 2 * at;
    const f32x4 *parts = reinterpret_cast<const f32x4 *>(share.part_out + at * g.d) + lane;
    const size_t stats_apart = 2 * apart, parts_apart = (size_t)apart * lanes;

    float top = -INFINITY, total = 0.0f;
    f32x4 o = zero;
    if (!few) {
        for (uint32_t i = 0; i < count; i++) top = fmaxf(top, stats[stats_apart * i]);
        for (uint32_t i = 0; i < count; i++) {
            const float f = weight_of(stats[stats_apart * i], top);
            total = __builtin_fmaf(stats[stats_apart * i + 1], f, total);
            o += parts[i * parts_apart] * f;
        }
        *reinterpret_cast<f32x4 *>(to) = o * (1.0f / total);
        return;
    }
    // Every wavefront finds the maximum by itself; the weights of the splits wait in LDS.
    for (uint32_t i = threadIdx.x & 63u; i < count; i += 64) top = fmaxf(top, stats[stats_apart * i]);
    top = dev::wave_reduce<dev::MaxOp>(top);
    for (uint32_t i = threadIdx.x; i < count; i += JOIN) {
        factors[i] = weight_of(stats[stats_apart * i], top);
        total = __builtin_fmaf(stats[stats_apart * i + 1], factors[i], total);
    }
    total = dev::wave_reduce<dev::SumOp>(total);
    if ((threadIdx.x & 63u) == 0) totals[threadIdx.x >> 6] = total;
    __syncthreads();
    if (group < groups) {
#pragma unroll 4
        for (uint32_t i = group; i < count; i += groups) o += parts[i * parts_apart] * factors[i];
    }
    sums[threadIdx.x] = o;
    __syncthreads();
    if (group != 0) return;
    total = 0.0f;
#pragma unroll
    for (int w = 0; w < JOIN / 64; w++) total += totals[w];
    for (uint32_t i = 1; i < groups; i++) o += sums[i * lanes + lane];
    *reinterpret_cast<f32x4 *>(to) = o * (1.0f / total);
}

bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

constexpr uint64_t MOST_ROWS = (uint64_t)1 << 30, MOST_BLOCKS = (uint64_t)1 << 24;  // a grid ends at 2^32 threads

// The largest head that blocks of 128 rows are built for.
constexpr int TILE_CHANNELS = 128;

struct Plan {
    Share few, many;  // their pointers from the start of the workspace, as yet
    uint32_t few_rows;
    size_t bytes;
};

Plan plan_of(const DeviceCtx *ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_attend &attend) {
    Plan p = {};
    const uint32_t group = (uint32_t)(attend.q_heads / cache.kv_heads);
    const size_t held = std::min((size_t)batch.table_pages * (size_t)cache.page_size, (size_t)INT32_MAX);
    const size_t max_tokens = std::min(attend.max_tokens ? attend.max_tokens : attend.tokens, attend.tokens);
    const size_t max_keys = std::min(attend.max_keys ? attend.max_keys : held, held);
    const uint32_t rows = (uint32_t)(max_tokens * group);
    const uint64_t cus = ctx && ctx->cus_per_xcd ? 8 * ctx->cus_per_xcd : 256, pairs = (uint64_t)batch.sequences * (uint64_t)cache.kv_heads;
    const uint64_t key_bytes = 2 * (uint64_t)cache.head_size * (cache.elem == AHIP_KV_BF16 ? 2 : 4);
    // tiles: no batch has more row tiles of this kind, times kv heads.
    auto share = [&](Share &s, uint32_t most_rows, uint32_t tile, uint64_t tiles, bool cut, uint64_t at_once, uint64_t least) {
        s.rows = most_rows;
        s.row_tiles = (most_rows + tile - 1) / tile;
        s.split_keys = (uint32_t)((std::max<uint64_t>(UNIT, least) + UNIT - 1) / UNIT * UNIT);
        s.at_once = (uint32_t)std::min<uint64_t>(at_once, MOST_SPLITS);
        const uint64_t all = pairs * s.row_tiles, units = tiles * ((max_keys + UNIT - 1) / UNIT);
        const bool counted = tiles < MOST_BLOCKS && units < UINT32_MAX;
        s.cut = cut && max_keys > 2 * s.split_keys && counted;
        // A block without rows costs its place 1 us, the list 3 us a block: 200 single tokens of 1000 keys and a piece of 512 behind
        // 1488, bf16, 32 heads, 8 of keys, 128 channels (25728 blocks, or 1512): 280 us by all blocks, 249 us by the list; 32
        // tokens of 4000 keys and the piece (4224, or 400): 166 and 173 us.
        s.listed = s.cut || (counted && tile == TILE_ROWS && all > tiles + 16 * at_once);
        if (s.listed && !s.cut) s.split_keys = (uint32_t)1 << 31;
        s.blocks = (uint32_t)std::min<uint64_t>(s.listed ? tiles : all, UINT32_MAX);
        if (!s.cut) return;
        // No more parts than both the parts' least size and at_once allow, and one more a pair.
        s.blocks = (uint32_t)(std::min<uint64_t>(s.at_once, units * UNIT / s.split_keys) + tiles);
        const size_t parts = (size_t)s.blocks * tile;
        s.part_stats = reinterpret_cast<float *>(p.bytes);
        p.bytes += 2 * parts * sizeof(float);
        s.part_out = reinterpret_cast<float *>(p.bytes);
        p.bytes += parts * (size_t)cache.head_size * sizeof(float);
    };
    const bool bf16 = cache.elem == AHIP_KV_BF16, tiled = cache.head_size <= TILE_CHANNELS;
    const uint64_t many_at_once = cus * (bf16 || cache.head_size <= 64 ? 2 : 1);
    // A sequence of many rows has more than FEW_BESIDE_CUT, and all have no more than the call: so many tiles are full, and one a
    // sequence is not.
    const uint64_t all_rows = attend.tokens * (uint64_t)group, row_tiles = (rows + TILE_ROWS - 1) / TILE_ROWS;
    const uint64_t many_tiles = (uint64_t)cache.kv_heads * std::min(batch.sequences * row_tiles, all_rows / TILE_ROWS + std::min<uint64_t>(batch.sequences, all_rows / (FEW_BESIDE_CUT + 1)));
    // Prompts whose blocks would leave half the places empty: pieces of 57 to 333 rows, up to 4858 keys, 392 us whole and 100 us cut;
    // one prompt of 1024, 12 heads of 64 channels, 50 and 37 us.  With three quarters of the places taken (4 such prompts) this cut
    // costs (59 us whole, 78 us cut): it gives every row tile parts of the whole sequence, half of which a causal prompt does not see.  Parts of 128 keys at least: a prompt of 400, 16 heads of 128, fp32, 32 us, with 256 36 us.
    if (rows > FEW_ROWS) {
        if (tiled) share(p.many, rows, TILE_ROWS, many_tiles, many_tiles < many_at_once / 2, many_at_once, 128);
        else share(p.many, rows, 16, pairs * ((rows + 15) / 16), false, 0, 0);
    }
    p.few_rows = p.many.cut ? FEW_BESIDE_CUT : FEW_ROWS;
    // A part for each block that is at work at once (as many a CU as registers allow), none shorter than 128 KiB of keys and values or
    // 64 keys: one token of 1024 keys, 12 heads of 64 channels, fp32, takes 16 us, with parts of 256 KiB 20, of 64 KiB 14 us; of 8192
    // keys, 8 kv heads of 128: 28, 26 and 28 us.  Nothing is cut into fewer than three: 300 keys take 10 us in one and 15 us in two.
    // From two blocks a place on nothing is cut: finding the parts costs more than a last long sequence does.  bf16, 128 channels, sequences
    // of very different lengths: 48 of up to 8191 keys, 4 kv heads (192 blocks whole) 148 us, cut 98 us; with 8 kv heads 128 of up to
    // 4000 (1024) 232 and 233; 512 of up to 2000 (4096) 416 and 464; 1024 of up to 1000 422 and 559 us.
    const uint64_t few_at_once = cus * (cache.head_size <= 64 || (bf16 && tiled) ? 3 : tiled ? 2 : 1), few_most = std::min(rows, p.few_rows);
    const uint64_t few_tiles = pairs * ((few_most + 15) / 16);
    share(p.few, (uint32_t)few_most, 16, few_tiles, few_tiles < 2 * few_at_once, few_at_once, 128 * 1024 / key_bytes);
    return p;
}

int check_attend(DeviceCtx *ctx, const ahip_kv_cache *cache, const ahip_kv_batch *batch, const ahip_kv_attend *attend, dev::KvView *view) {
    const std::string name = "kv attention: ";
    if (!attend) return kv_fail(ctx, AHIP_ERR_ARG, name + "null attend");
    if (int rc = make_kv_view(ctx, "kv attention", cache, batch, attend->tokens, view)) return rc;
    if (attend->q_heads <= 0 || attend->q_heads > 65535 || attend->q_heads % cache->kv_heads)
        return kv_fail(ctx, AHIP_ERR_SHAPE, name + std::to_string(attend->q_heads) + " query heads do not share " + std::to_string(cache->kv_heads) + " heads of keys");
    if (!std::isfinite(attend->scale * LOG2E) || !std::isfinite(attend->softcap) || attend->softcap < 0 || attend->window < 0)
        return kv_fail(ctx, AHIP_ERR_ARG, name + "the scale, the cap or the window is out of range");
    // Queries are scaled by scale / cap in fp32, whose parts in bf16 reach 2^-24 below them, and scores multiplied by the cap: with a
    // quotient outside 2^-64 .. 2^64 the parts would be flushed to zero, or the quotient or the product infinite.
    const double beside_cap = attend->softcap != 0.0f ? std::fabs((double)attend->scale) / attend->softcap : 0.0;
    if (beside_cap != 0.0 && !(beside_cap >= 0x1p-64 && beside_cap <= 0x1p64)) return kv_fail(ctx, AHIP_ERR_ARG, name + "the cap is out of range beside the scale");
    if (!std::isfinite(attend->softcap * LOG2E)) return kv_fail(ctx, AHIP_ERR_ARG, name + "the cap is out of range");
    // Sizes that the plan's products and the kernels' row numbers hold.
    const uint64_t group = (uint64_t)(attend->q_heads / cache->kv_heads), most_tokens = std::min(attend->max_tokens ? attend->max_tokens : attend->tokens, attend->tokens);
    if (most_tokens * group > MOST_ROWS) return kv_fail(ctx, AHIP_ERR_UNSUPPORTED, name + "more than 2^30 rows for a head of keys");
    if ((uint64_t)batch->sequences * (uint64_t)cache->kv_heads >= MOST_BLOCKS) return kv_fail(ctx, AHIP_ERR_UNSUPPORTED, name + "more blocks than a grid holds");
    const bool bf16 = cache->elem == AHIP_KV_BF16;
    const int64_t unit = bf16 ? 8 : 4;
    if (cache->head_size > 256 || cache->head_size % unit) return kv_fail(ctx, AHIP_ERR_UNSUPPORTED, name + "no kernel for heads of " + std::to_string(cache->head_size));
    bool on = aligned16(attend->q) && aligned16(attend->out) && aligned16(cache->keys) && aligned16(cache->values) && cache->page_stride % unit == 0 &&
              cache->head_stride % unit == 0 && cache->slot_stride % unit == 0 && (!attend->workspace || aligned16(attend->workspace));
    for (int i = 0; i < 2; i++) {
        if (attend->q_strides[i] > ((size_t)1 << 48) || attend->out_strides[i] > ((size_t)1 << 48)) return kv_fail(ctx, AHIP_ERR_ARG, name + "a stride is out of range");
        on = on && attend->q_strides[i] % 4 == 0 && attend->out_strides[i] % 4 == 0;
    }
    if (!on) return kv_fail(ctx, AHIP_ERR_UNSUPPORTED, name + "a tensor or stride is not on 16-byte boundaries");
    return AHIP_OK;
}

template <int DP, bool BF16, bool UNIFORM> int launch_wide(DeviceCtx &ctx, const AttendArgs &g) {
    hipLaunchKernelGGL((attend_rows16<DP, BF16, UNIFORM, true>), dim3(g.few.blocks), dim3(64 * ROW_WAVES), 0, ctx.stream, g);
    if (int rc = ctx.check(hipGetLastError(), "kv attention launch")) return rc;
    if (!g.many.blocks) return AHIP_OK;
    hipLaunchKernelGGL((attend_rows16<DP, BF16, UNIFORM, false>), dim3(g.many.blocks), dim3(64 * ROW_WAVES), 0, ctx.stream, g);
    return ctx.check(hipGetLastError(), "kv attention launch");
}
template <int DP, bool BF16, bool UNIFORM> int launch_tiled(DeviceCtx &ctx, const AttendArgs &g) {
    if (!g.many.blocks)
        hipLaunchKernelGGL((attend_rows16<DP <= 64 ? 64 : 128, BF16, UNIFORM, true>), dim3(g.few.blocks), dim3(64 * ROW_WAVES), 0, ctx.stream, g);
    else
        hipLaunchKernelGGL((attend_rows128<DP, BF16, UNIFORM>), dim3(g.few.blocks + g.many.blocks), dim3(256), 0, ctx.stream, g);
    return ctx.check(hipGetLastError(), "kv attention launch");
}

// By the head's channels, rounded up.  Heads of 96 channels have a size of their own: 4 prompts of 512 (16 heads, 4 of keys, fp32)
// 46 us, at 128 channels 53 us; of 1024, bf16, 8 heads of keys: 63 and 72 us.
template <bool BF16, bool UNIFORM> int launch_by_size(DeviceCtx &ctx, const AttendArgs &g) {
    if (g.d <= 64) return launch_tiled<64, BF16, UNIFORM>(ctx, g);
    if (g.d <= 96) return launch_tiled<96, BF16, UNIFORM>(ctx, g);
    if (g.d <= TILE_CHANNELS) return launch_tiled<128, BF16, UNIFORM>(ctx, g);
    return launch_wide<256, BF16, UNIFORM>(ctx, g);
}

}  // namespace

int kv_attention_workspace(DeviceCtx *ctx, const ahip_kv_cache *cache, const ahip_kv_batch *batch, const ahip_kv_attend *attend, size_t *bytes) {
    if (!bytes) return kv_fail(ctx, AHIP_ERR_ARG, "kv attention: null output");
    *bytes = 0;
    dev::KvView view = {};
    // The sizes alone: neither the tensors nor the arrays on the device need exist yet.
    if (int rc = check_attend(ctx, cache, batch, attend, &view)) return rc;
    *bytes = plan_of(ctx, *cache, *batch, *attend).bytes;
    return AHIP_OK;
}

int launch_kv_attention(DeviceCtx &ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_attend &attend) {
    AttendArgs g = {};
    if (int rc = check_attend(&ctx, &cache, &batch, &attend, &g.kv)) return rc;
    if (attend.tokens == 0 || batch.sequences == 0) return AHIP_OK;
    if (int rc = require_kv_arrays(ctx, "kv attention", cache, batch)) return rc;
    if (!attend.q || !attend.out) return ctx.fail(AHIP_ERR_ARG, "kv attention: null pointer");
    if (attend.out == attend.q) return ctx.fail(AHIP_ERR_ARG, "kv attention: out is q");
    const Plan plan = plan_of(&ctx, cache, batch, attend);
    if (plan.bytes && (!attend.workspace || attend.workspace_bytes < plan.bytes))
        return ctx.fail(AHIP_ERR_ARG, "kv attention: the workspace holds " + std::to_string(attend.workspace ? attend.workspace_bytes : 0) + " bytes of " +
                                          std::to_string(plan.bytes));
    g.q = attend.q, g.out = attend.out;
    g.q_token = (int64_t)attend.q_strides[0], g.q_head = (int64_t)attend.q_strides[1];
    g.out_token = (int64_t)attend.out_strides[0], g.out_head = (int64_t)attend.out_strides[1];
    g.q_heads = (uint32_t)attend.q_heads, g.group = (uint32_t)(attend.q_heads / cache.kv_heads), g.d = (uint32_t)cache.head_size;
    g.by_group = dev::make_fastdiv(g.group);
    g.cap = attend.softcap * LOG2E;
    g.scale = attend.softcap != 0.0f ? attend.scale / attend.softcap : attend.scale * LOG2E;
    g.causal = attend.causal, g.window = attend.window, g.slopes = attend.slopes, g.prefix = attend.prefix, g.first_keys = attend.first_keys;
    g.max_tokens = (uint32_t)(attend.max_tokens ? std::min(attend.max_tokens, attend.tokens) : attend.tokens);
    g.max_keys = (uint32_t)std::min(attend.max_keys ? attend.max_keys : (size_t)INT32_MAX, (size_t)INT32_MAX);
    g.few = plan.few, g.many = plan.many, g.few_rows = plan.few_rows;
    for (Share *s : {&g.few, &g.many})
        if (s->cut) {
            s->part_stats = reinterpret_cast<float *>(static_cast<char *>(attend.workspace) + reinterpret_cast<uintptr_t>(s->part_stats));
            s->part_out = reinterpret_cast<float *>(static_cast<char *>(attend.workspace) + reinterpret_cast<uintptr_t>(s->part_out));
        }
    const uint64_t pairs = (uint64_t)g.kv.sequences * g.kv.kv_heads, groups = JOIN / (g.d / 4);
    const uint64_t few_joins = g.few.cut ? pairs * g.few.rows : 0, many_joins = g.many.cut ? pairs * ((g.many.rows + groups - 1) / groups) : 0;
    if ((uint64_t)g.few.blocks + g.many.blocks >= MOST_BLOCKS || few_joins + many_joins >= MOST_BLOCKS)
        return ctx.fail(AHIP_ERR_UNSUPPORTED, "kv attention: more blocks than a grid holds");
    // Pages of whole groups of 16 keys: a group's page is looked up once, not key by key, and its slots lie within 2^31 bytes.  Pages of
    // 64, 4 prompts of 1024 (12 heads of 64 channels, fp32): 61.7 us, key by key 67.5; a prompt of 4096 with a window, bf16:
    // 156 and 166 us; one token of 65536 keys, pages of 16: 111 and 113 us.
    const bool bf16 = cache.elem == AHIP_KV_BF16, uniform = cache.page_size % 16 == 0 && cache.slot_stride < (int64_t)1 << 23;
    int rc = bf16 ? (uniform ? launch_by_size<true, true>(ctx, g) : launch_by_size<true, false>(ctx, g))
                  : (uniform ? launch_by_size<false, true>(ctx, g) : launch_by_size<false, false>(ctx, g));
    if (rc || few_joins + many_joins == 0) return rc;
    hipLaunchKernelGGL(join_splits, dim3((uint32_t)(few_joins + many_joins)), dim3(JOIN), 0, ctx.stream, g, (uint32_t)few_joins);
    return ctx.check(hipGetLastError(), "kv attention launch");
}

}  // namespace altius

// Attention over the pages of a cache that a cheap score selects: means of the pages that fill, a score for each page from its mean, the best pages of each
// row and head of keys, and attention (kv_attend.h) over those, each row being a sequence of its own with a page table of its own for each head.
//   Scores are sums of products of fp32 values in 64 bits, where no product is rounded: of d channels they are off by d 2^-53 of the sum of |q mean| at most, and only
// pages whose scores are that near to each other may change places with another order of sums.  All kernels here add in the same order: equal means have equal scores.
//   One token behind 65535 (32 of 1024 pages of 64, 32 heads, 8 of keys, 128 channels, fp32) 31 us, bound by the chains of four launches; 48 behind 100 to 16000 (40
// pages of 32, 4 heads of keys, bf16) 61 us, 35 of them attention at 3.6 TB/s; 309 rows behind 6001 to 12000 (61 pages of 16, 16 heads, 4 of keys of 80 channels,
// fp32) 127 us, 95 of them attention, each row's pages for itself, 820 MB asked of L2.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv_attend.h"
#include "kv_rank.h"

namespace altius {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

// LARGE: of a block that makes its scores itself (48 tokens of up to 500 pages, 4 heads of keys: 20.3 us, with 256 threads 23.8; 1024 leave no registers, 63).
constexpr uint32_t BLOCK = 256, LARGE = 512;
constexpr uint32_t HELD = 8192;      // images of pages in LDS
constexpr uint32_t LISTED = 16384;   // chosen pages in LDS, of a row that has more
constexpr uint32_t SCORED = 64;      // pages of a block that does nothing but score a row
constexpr uint32_t SCORED_ROWS = 8, ROW_PAGES = 128;  // rows and pages of one that scores several
constexpr uint32_t MOST_CHANNELS = 256;

struct SparseArgs {
    dev::KvView kv;
    float *means;
    int64_t means_page, means_head;
    int32_t *chosen;
    const float *q;
    int64_t q_token, q_head;
    uint32_t d, group, q_heads, most, first, last;
    uint32_t max_tokens, max_keys, max_pages, held, chunks;
    bool bf16, fills;   // fills: as many blocks again make the mean of the page that a row fills
    double *scores;     // [row][kv head][max_pages]; null: choose_pages makes them itself
    int32_t *table, *starts, *lengths;  // of the sequences that attention sees
};

// ---------------------------------------------------------------- means
// The mean of page `page` for one head, by a block: lanes side by side take 4 channels each, groups of lanes the slots in turn; sums in 64 bits, rounded once.
template <uint32_t THREADS> __device__ __forceinline__ void page_mean(const SparseArgs &g, int32_t page, uint32_t head) {
    __shared__ double sums[THREADS][4];
    const uint32_t lanes = g.d / 4, groups = THREADS / lanes, lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
    const int64_t at = (int64_t)page * g.kv.page_stride + (int64_t)head * g.kv.head_stride + 4 * lane;
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
    if (group < groups) {
#pragma unroll 4
        for (uint32_t slot = group; slot < g.kv.page_size; slot += groups) {
            const int64_t from = at + (int64_t)slot * g.kv.slot_stride;
            if (g.bf16) {
                const u16x4 x = *reinterpret_cast<const u16x4 *>(static_cast<const uint16_t *>(g.kv.keys) + from);
#pragma unroll
                for (int e = 0; e < 4; e++) sum[e] += (double)__uint_as_float((uint32_t)x[e] << 16);
            } else {
                const f32x4 x = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(g.kv.keys) + from);
#pragma unroll
                for (int e = 0; e < 4; e++) sum[e] += (double)x[e];
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; e++) sums[threadIdx.x][e] = sum[e];
    __syncthreads();
    if (group == 0) {
        f32x4 mean;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            for (uint32_t i = 1; i < groups; i++) sum[e] += sums[i * lanes + lane][e];
            mean[e] = (float)(sum[e] / (double)g.kv.page_size);
        }
        *reinterpret_cast<f32x4 *>(g.means + (int64_t)page * g.means_page + (int64_t)head * g.means_head + 4 * lane) = mean;
    }
}

__device__ __forceinline__ dev::KvSequence within(const SparseArgs &g, dev::KvSequence q) {
    if ((uint32_t)q.n > g.max_tokens || (uint32_t)q.length > g.max_keys) {
        *g.kv.flag = 1;
        q.n = 0;
    }
    return q;
}

// A block for each sequence, page that its rows can have filled, and head; where there are not blocks for all it goes on with every chunks-th page behind its own.
__global__ __launch_bounds__(BLOCK) void mean_pages(SparseArgs g) {
    const uint32_t outer = blockIdx.x / g.kv.kv_heads, head = blockIdx.x - outer * g.kv.kv_heads, s = outer / g.chunks, i = outer - s * g.chunks;
    const dev::KvSequence q = within(g, dev::kv_sequence(g.kv, s));
    if (q.n == 0) return;
    const uint32_t base = (uint32_t)max(0, q.length - q.n);
    for (uint32_t index = g.kv.by_page_size.div(base) + i; (uint64_t)(index + 1) * g.kv.page_size <= (uint32_t)q.length; index += g.chunks) {
        const int32_t page = g.kv.page_of(s, index, -1);
        if (page >= 0) page_mean<BLOCK>(g, page, head);
    }
}

// ---------------------------------------------------------------- scores
// The larger of a lane's value and that of the lane that CONTROL names.
template <int CONTROL> __device__ __forceinline__ double larger(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    const uint32_t low = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CONTROL, 0xF, 0xF, false);
    const uint32_t high = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CONTROL, 0xF, 0xF, false);
    return fmax(v, __longlong_as_double((long long)((uint64_t)high << 32 | low)));
}

// Scores of pages of a row's sequence, by a block, 16 a wavefront: this wavefront's from `start` on and every `step` behind, below `to`, with v_mfma_f64_4x4x4_4b_f64: four blocks of 4 pages by 4 heads, 4
// channels at a time.  Lane 16 k + p has page p, lane 16 k + 4 b + j head j, and either channels 16 u + 4 k .. + 3 for u < UNITS; the result of page 4 b + i and
// head j is in lane 16 i + 4 b + j.  No sum goes from lane to lane, and 16 pages of 128 channels and 4 heads take 32 instructions; the same with the vector
// unit, 16 lanes a page, spent more on adding up the lanes than on products (one token, 48 texts, group of 8: 34.5 us, so 26).
// put(page, score, again): again: the larger of it and what is there.
template <uint32_t UNITS, int FOURS, class Put> __device__ __forceinline__ void score_range(const SparseArgs &g, uint32_t s, uint32_t row, uint32_t head, uint32_t start, uint32_t step, uint32_t to, Put put) {
    const uint32_t lane = threadIdx.x & 63u, k = lane >> 4;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t h0 = 0; h0 < g.group; h0 += 4 * FOURS) {
        double q[FOURS][UNITS][4];
#pragma unroll
        for (int f = 0; f < FOURS; f++) {
            const uint32_t its = head * g.group + min(h0 + 4 * f + (lane & 3u), g.group - 1);  // the last one more than once: the largest is the same
            const float *from_q = g.q + (int64_t)row * g.q_token + (int64_t)its * g.q_head;
#pragma unroll
            for (uint32_t u = 0; u < UNITS; u++) {
                const uint32_t c = 16 * u + 4 * k;
                const f32x4 x = c < g.d ? *reinterpret_cast<const f32x4 *>(from_q + c) : zero;
#pragma unroll
                for (int e = 0; e < 4; e++) q[f][u][e] = (double)x[e];
            }
        }
        // The means of 16 pages while those in front are multiplied.
        auto page_at = [&](uint32_t base) { return base + (lane & 15u) < to ? g.kv.page_of(s, base + (lane & 15u), 0) : 0; };
        f32x4 ahead[UNITS];
        auto fetch = [&](int32_t page) {
            const float *mean = g.means + (int64_t)page * g.means_page + (int64_t)head * g.means_head;
#pragma unroll
            for (uint32_t u = 0; u < UNITS; u++) ahead[u] = *reinterpret_cast<const f32x4 *>(mean + (16 * u + 4 * k < g.d ? 16 * u + 4 * k : 0));
        };
        fetch(page_at(start));
        int32_t page = page_at(start + step);
        for (uint32_t base = start; base < to; base += step) {
            f32x4 x[UNITS];
#pragma unroll
            for (uint32_t u = 0; u < UNITS; u++) x[u] = ahead[u];
            if (base + step < to) {
                fetch(page);
                page = page_at(base + 2 * step);
            }
            double v[FOURS];
#pragma unroll
            for (int f = 0; f < FOURS; f++) v[f] = 0.0;
#pragma unroll
            for (uint32_t u = 0; u < UNITS; u++) {
                if (16 * u >= g.d) break;
                if (16 * u + 4 * k >= g.d) x[u] = zero;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const double mine = (double)x[u][e];
#pragma unroll
                    for (int f = 0; f < FOURS; f++) v[f] = __builtin_amdgcn_mfma_f64_4x4x4f64(mine, q[f][u][e], v[f], 0, 0, 0);
                }
            }
#pragma unroll
            for (int f = 1; f < FOURS; f++) v[0] = fmax(v[0], v[f]);
            const double best = larger<dev::DPP_QUAD_XOR2>(larger<dev::DPP_QUAD_XOR1>(v[0]));
            const uint32_t its = base + (lane & 12u) + (lane >> 4);
            if ((lane & 3u) == 0 && its < to) put(its, best, h0 != 0);
        }
    }
}

// The row's place in its sequence, and the pages in front of it with its own: 0 where there is no such row.
struct Row {
    uint32_t s, pages, place;
    int32_t signed_place;  // below 0 in a sequence that is shorter than its rows
    bool live;
};
// behind: the first row behind the sequence's, where it is live.
__device__ __forceinline__ Row row_of(const SparseArgs &g, uint32_t row, uint32_t *behind = nullptr) {
    dev::KvSequence q = {0, 0, 0};
    Row r = {0, 0, 0, 0, false};
    r.s = dev::kv_sequence_of(g.kv, row, q);
    if (r.s >= g.kv.sequences) return r;
    q = within(g, q);
    const int32_t t = (int32_t)row - q.start;
    if (t < 0 || t >= q.n) return r;
    r.live = true;
    if (behind) *behind = (uint32_t)(q.start + q.n);
    const int32_t place = r.signed_place = q.length - q.n + t;
    if (place < 0) return r;
    r.place = (uint32_t)place, r.pages = g.kv.by_page_size.div(r.place) + 1;
    return r;
}

template <uint32_t UNITS, int FOURS> __global__ __launch_bounds__(BLOCK) void score_pages(SparseArgs g) {
    const uint32_t outer = blockIdx.x / g.chunks, chunk = blockIdx.x - outer * g.chunks, row = outer / g.kv.kv_heads, head = outer - row * g.kv.kv_heads;
    const Row r = row_of(g, row);
    if (r.pages <= g.most) return;  // all are chosen
    double *to_scores = g.scores + (size_t)outer * g.max_pages;
    // A run of SCORED pages, and those behind it where there are not blocks for all.  (The first pages, which are chosen anyway, among them.)
    score_range<UNITS, FOURS>(g, r.s, row, head, chunk * SCORED + 16 * (threadIdx.x >> 6), g.chunks * SCORED, r.pages - g.last,
                              [&](uint32_t page, double score, bool again) { to_scores[page] = again ? fmax(to_scores[page], score) : score; });
}
static_assert(SCORED == BLOCK / 64 * 16, "16 pages a wavefront");

// The same for SCORED_ROWS rows next to each other, whose queries wait in LDS: rows of one sequence read its means together.  309 rows behind 6001 to 12000 tokens in
// pages of 16, 4 heads of keys of 80 channels: 34 us with the choice (128 pages a block; 256 leave CUs idle, 39); each row by itself, in the block that chooses, 52.
template <uint32_t UNITS> __global__ __launch_bounds__(BLOCK) void score_rows(SparseArgs g) {
    __shared__ double queries[SCORED_ROWS][UNITS][4][16];  // [row][u][e][4 k + j]: of channel 16 u + 4 k + e and head j
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, k = lane >> 4;
    const uint32_t outer = blockIdx.x / g.chunks, chunk = blockIdx.x - outer * g.chunks, group = outer / g.kv.kv_heads, head = outer - group * g.kv.kv_heads;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t end_row = min((group + 1) * SCORED_ROWS, g.kv.tokens);
    for (uint32_t row = group * SCORED_ROWS, rows; row < end_row; row += rows) {
        uint32_t behind;  // the first row that is another sequence's
        const Row r = row_of(g, row, &behind);
        rows = r.live ? min(behind, end_row) - row : 1;
        // The last row has most pages.
        const uint32_t last_pages = r.live ? (uint32_t)max(0, (int32_t)g.kv.by_page_size.div((uint32_t)max(0, r.signed_place + (int32_t)rows - 1)) + 1) : 0;
        if (!r.live || r.signed_place + (int32_t)rows <= 0 || last_pages <= g.most) continue;
        const uint32_t most_to = last_pages - g.last;
        if (chunk * ROW_PAGES >= most_to) continue;
        for (uint32_t h0 = 0; h0 < g.group; h0 += 4) {
            __syncthreads();
            for (uint32_t i = tid; i < rows * UNITS * 16; i += BLOCK) {  // 4 channels of a query each
                const uint32_t j = i & 3u, its_k = i >> 2 & 3u, u = i / 16 % UNITS, its = i / (16 * UNITS), c = 16 * u + 4 * its_k;
                const uint32_t h = head * g.group + min(h0 + j, g.group - 1);  // the last one more than once
                const f32x4 x = c < g.d ? *reinterpret_cast<const f32x4 *>(g.q + (int64_t)(row + its) * g.q_token + (int64_t)h * g.q_head + c) : zero;
#pragma unroll
                for (int e = 0; e < 4; e++) queries[its][u][e][4 * its_k + j] = (double)x[e];
            }
            __syncthreads();
            // 16 pages of a wavefront at a time: of this block's run of ROW_PAGES, and of those behind it where there are not blocks for all.
            for (uint32_t at = chunk; at * ROW_PAGES < most_to; at += g.chunks) {
                const uint32_t from = max(at * ROW_PAGES, g.first), to = min((at + 1) * ROW_PAGES, most_to);
                for (uint32_t base = from + 16 * wave; base < to; base += BLOCK / 4) {
                    const uint32_t index = base + (lane & 15u);
                    const int32_t page = index < to ? g.kv.page_of(r.s, index, 0) : 0;
                    const float *mean = g.means + (int64_t)page * g.means_page + (int64_t)head * g.means_head;
                    double mine[UNITS][4];
#pragma unroll
                    for (uint32_t u = 0; u < UNITS; u++) {
                        const uint32_t c = 16 * u + 4 * k;
                        f32x4 x = *reinterpret_cast<const f32x4 *>(mean + (c < g.d ? c : 0));
                        if (c >= g.d) x = zero;
#pragma unroll
                        for (int e = 0; e < 4; e++) mine[u][e] = (double)x[e];
                    }
                    const uint32_t its_page = base + (lane & 12u) + (lane >> 4);
                    for (uint32_t its = 0; its < rows; its++) {
                        double v = 0.0;
#pragma unroll
                        for (uint32_t u = 0; u < UNITS; u++) {
                            if (16 * u < g.d) {
#pragma unroll
                                for (int e = 0; e < 4; e++) v = __builtin_amdgcn_mfma_f64_4x4x4f64(mine[u][e], queries[its][u][e][4 * k + (lane & 3u)], v, 0, 0, 0);
                            }
                        }
                        const double best = larger<dev::DPP_QUAD_XOR2>(larger<dev::DPP_QUAD_XOR1>(v));
                        if ((lane & 3u) == 0 && its_page < to) {
                            double *put = g.scores + ((size_t)(row + its) * g.kv.kv_heads + head) * g.max_pages + its_page;
                            *put = h0 ? fmax(*put, best) : best;
                        }
                    }
                }
            }
        }
    }
}

// ---------------------------------------------------------------- the best
// Larger for larger scores, 0 for NaN.
__device__ __forceinline__ uint64_t rank_image(double score) {
    if (score != score) return 0;
    const uint64_t u = (uint64_t)__double_as_longlong(score + 0.0);
    return u >> 63 ? ~u : u | (uint64_t)1 << 63;
}

// A block for each row and head of keys: the smallest image that is chosen (kv_rank.h), equal ones by their number, then the pages in order.
template <uint32_t UNITS, int FOURS, uint32_t THREADS> __global__ __launch_bounds__(THREADS) void choose_pages(SparseArgs g) {
    constexpr uint32_t WAVES = THREADS / 64;
    extern __shared__ uint64_t images[];
    __shared__ uint32_t totals[2][WAVES][2];
    __shared__ dev::RankLds<1> rank_lds;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t rows = g.kv.tokens * g.kv.kv_heads, id = blockIdx.x < rows ? blockIdx.x : blockIdx.x - rows, row = id / g.kv.kv_heads, head = id - row * g.kv.kv_heads;
    const Row r = row_of(g, row);
    if (blockIdx.x >= rows) {  // where rows fill pages for later calls: beside the choice (behind it, one token of 1024 pages takes 5 us more)
        const int32_t page = r.pages && r.place + 1 == r.pages * g.kv.page_size ? g.kv.page_of(r.s, r.pages - 1, -1) : -1;
        if (page >= 0) page_mean<THREADS>(g, page, head);
        return;
    }
    const int32_t first_row = g.kv.starts[0], end_row = g.kv.starts[g.kv.sequences];
    if (head == 0 && tid < 2 && (tid == 0 || row + 1 == g.kv.tokens)) {
        const int32_t at = (int32_t)(row + tid);
        g.starts[at] = max(0, min(min(max(at, first_row), end_row), (int32_t)g.kv.tokens));
    }
    if (!r.live) {
        // In front of the sequences or behind them: a sequence without rows; in one that does not fit: left out.
        if (head == 0 && tid == 0) g.lengths[row] = (int32_t)row < first_row || (int32_t)row >= end_row ? 0 : -1;
        return;
    }
    const size_t list = ((size_t)row * g.kv.kv_heads + head) * g.most;
    const uint32_t count = min(r.pages, g.most);
    if (head == 0 && tid == 0) g.lengths[row] = count ? (int32_t)((count - 1) * g.kv.page_size + (r.place - (r.pages - 1) * g.kv.page_size) + 1) : 0;
    for (uint32_t i = count + tid; i < g.most; i += THREADS) g.chosen[list + i] = -1;
    auto put = [&](uint32_t at, uint32_t page) {
        g.chosen[list + at] = (int32_t)page;
        g.table[list + at] = g.kv.page_of(r.s, page, -1);
    };
    if (r.pages <= g.most) {
        for (uint32_t i = tid; i < count; i += THREADS) put(i, i);
        return;
    }
    uint32_t *const in_order = reinterpret_cast<uint32_t *>(images + g.held);  // g.most of them

    const uint32_t from = g.first, to = r.pages - g.last, want = g.most - g.first - g.last;  // of the pages from .. to - 1, of which there are more
    const double *scores = UNITS ? nullptr : g.scores + ((size_t)row * g.kv.kv_heads + head) * g.max_pages;
    if constexpr (UNITS != 0) {
        if (want)
            score_range<UNITS, FOURS>(g, r.s, row, head, from + 16 * (tid >> 6), 16 * WAVES, to, [&](uint32_t page, double score, bool again) {
                const uint64_t v = rank_image(score);
                images[page] = again ? max(images[page], v) : v;
            });
    } else {
        const uint32_t end = min(to, g.held);
        for (uint32_t base = from + tid; base < end; base += 4 * THREADS) {  // four loads on their way at once
            double v[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; u++) v[u] = scores[min(base + u * THREADS, end - 1)];
#pragma unroll
            for (uint32_t u = 0; u < 4; u++)
                if (base + u * THREADS < end) images[base + u * THREADS] = rank_image(v[u]);
        }
    }
    __syncthreads();
    auto image = [&](uint32_t page) { return UNITS != 0 || page < g.held ? images[page] : rank_image(scores[page]); };

    dev::Ranked<uint64_t> ranked = {0, 0, true};
    if (want)
        ranked = dev::rank_largest<uint64_t>(rank_lds, want, [&](auto count_in) {
            for (uint32_t page = from + tid; page < to; page += THREADS) count_in(image(page));
        });
    const uint64_t least = ranked.least;
    const bool exact = ranked.exact;
    const uint32_t ties = ranked.ties;
    uint32_t listed = 0, tied = 0;
    const uint64_t before = ((uint64_t)1 << lane) - 1;
    for (uint32_t base = 0, turn = 0; base < r.pages; base += THREADS, turn ^= 1) {
        const uint32_t page = base + tid;
        const bool there = page < r.pages, always = there && (page < from || page >= to);
        const uint64_t v = there && !always && want ? image(page) : 0;
        bool stays = always || (there && want && (exact ? v >= least : v > least));
        if (!exact) {  // ties of the wavefronts in front count first
            const bool tie = there && !always && v == least;
            const uint64_t tie_mask = __ballot(tie);
            __syncthreads();
            if (lane == 0) totals[turn][wave][1] = (uint32_t)__popcll(tie_mask);
            __syncthreads();
            uint32_t tie_at = tied;
            for (uint32_t w = 0; w < WAVES; w++) {
                if (w < wave) tie_at += totals[turn][w][1];
                tied += totals[turn][w][1];
            }
            stays = stays || (tie && tie_at + (uint32_t)__popcll(tie_mask & before) < ties);
        }
        const uint64_t stay_mask = __ballot(stays);
        __syncthreads();
        if (lane == 0) totals[turn][wave][0] = (uint32_t)__popcll(stay_mask);
        __syncthreads();
        uint32_t at = listed;
        for (uint32_t w = 0; w < WAVES; w++) {
            if (w < wave) at += totals[turn][w][0];
            listed += totals[turn][w][0];
        }
        if (stays) in_order[at + (uint32_t)__popcll(stay_mask & before)] = page;
    }
    // Their places in the cache are looked up together, not as each is found.
    __syncthreads();
    for (uint32_t i = tid; i < g.most; i += THREADS) put(i, in_order[i]);
}

// ---------------------------------------------------------------- the host's part
bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }
constexpr int64_t MOST_STRIDE = (int64_t)1 << 48;
constexpr uint64_t MOST_GRID = (uint64_t)1 << 24, SCORES = (uint64_t)1 << 28;
// Blocks that score or make means, where there are not more rows or sequences: one without pages costs 1 ns, and a page table may have room for far more than any sequence has.
constexpr uint64_t LAUNCHED = 1 << 14;

int check_means(DeviceCtx *ctx, const std::string &name, const ahip_kv_cache &cache, const ahip_kv_sparse &sparse) {
    if (sparse.page_stride < 0 || sparse.head_stride < 0 || sparse.page_stride > MOST_STRIDE || sparse.head_stride > MOST_STRIDE)
        return kv_fail(ctx, AHIP_ERR_ARG, name + "a stride of the means is out of range");
    const int64_t unit = cache.elem == AHIP_KV_BF16 ? 8 : 4;
    if (cache.head_size > (int32_t)MOST_CHANNELS || cache.head_size % unit) return kv_fail(ctx, AHIP_ERR_UNSUPPORTED, name + "no kernel for heads of " + std::to_string(cache.head_size));
    if (!aligned16(sparse.means) || sparse.page_stride % 4 || sparse.head_stride % 4 || !aligned16(cache.keys) || cache.page_stride % unit || cache.head_stride % unit ||
        cache.slot_stride % unit)
        return kv_fail(ctx, AHIP_ERR_UNSUPPORTED, name + "a tensor or stride is not on 16-byte boundaries");
    return AHIP_OK;
}

struct SparsePlan {
    ahip_kv_batch batch;    // as attention sees it
    ahip_kv_attend attend;
    size_t attend_bytes, starts, lengths, table, scores, bytes;
    uint64_t max_pages, rows, chunks, score_blocks;  // rows: times heads of keys; chunks: of a row's pages that there are blocks for
    bool split, by_rows;                     // scores by a launch of their own, for rows next to each other at once
};

// No sequence of the call has more.
uint64_t most_pages(const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_attend &attend) {
    const size_t held = (size_t)batch.table_pages * (size_t)cache.page_size, max_keys = std::min(attend.max_keys ? attend.max_keys : held, held);
    return (max_keys + cache.page_size - 1) / cache.page_size;
}

SparsePlan sparse_plan(const DeviceCtx *ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_attend &attend, const ahip_kv_sparse &sparse) {
    SparsePlan p = {};
    p.batch = {(int32_t)attend.tokens, sparse.most, (int64_t)sparse.most * cache.kv_heads, nullptr, nullptr, nullptr};
    p.attend = attend;
    p.attend.max_tokens = 1, p.attend.max_keys = 0;
    p.max_pages = most_pages(cache, batch, attend);
    p.rows = attend.tokens * (uint64_t)cache.kv_heads;
    const uint64_t cus = ctx && ctx->cus_per_xcd ? 8 * ctx->cus_per_xcd : 256;
    // A block that chooses makes its scores itself where there are blocks for all CUs, or few pages: 48 tokens of up to 500 pages, 4 heads of keys, 61 us
    // with their attention, 76 by launches of their own; one token of 1024 pages, 8 heads, 50 us and 31.  Of pages of 64, 8 heads of keys: one token of 256 pages 29 us either
    // way, of 512 33 and 30; 8 tokens of 512 47 and 46; 24 of 512 91 and 97; 48 of 1024 178 and 188.
    p.split = p.max_pages > HELD || (p.rows < cus && p.max_pages > 8 * SCORED);
    // Rows of one sequence read its means together, as far as their scores fit into SCORES bytes.
    const size_t max_tokens = std::min(attend.max_tokens ? attend.max_tokens : attend.tokens, attend.tokens);
    p.by_rows = max_tokens >= SCORED_ROWS && p.max_pages > SCORED && (p.split || p.rows * p.max_pages * sizeof(double) <= SCORES);
    p.split = p.split || p.by_rows;
    const uint64_t scored = p.by_rows ? (attend.tokens + SCORED_ROWS - 1) / SCORED_ROWS * cache.kv_heads : p.rows, run = p.by_rows ? ROW_PAGES : SCORED;
    p.chunks = std::min((p.max_pages + run - 1) / run, std::max<uint64_t>(1, LAUNCHED / std::max<uint64_t>(1, scored)));
    p.score_blocks = scored * p.chunks;
    p.attend_bytes = attend::plan_of(ctx, cache, p.batch, p.attend).bytes;
    p.starts = up16(p.attend_bytes);
    p.lengths = up16(p.starts + (attend.tokens + 1) * sizeof(int32_t));
    p.table = up16(p.lengths + attend.tokens * sizeof(int32_t));
    p.scores = up16(p.table + p.rows * (size_t)sparse.most * sizeof(int32_t));
    p.bytes = p.split ? p.scores + p.rows * p.max_pages * sizeof(double) : p.scores;
    return p;
}

int check_sparse(DeviceCtx *ctx, const ahip_kv_cache *cache, const ahip_kv_batch *batch, const ahip_kv_attend *attend, const ahip_kv_sparse *sparse, dev::KvView *view) {
    const std::string name = "kv attention over chosen pages: ";
    if (!sparse) return kv_fail(ctx, AHIP_ERR_ARG, name + "null sparse");
    if (int rc = attend::check_attend(ctx, cache, batch, attend, view)) return rc;
    if (!attend->causal || attend->window || attend->slopes || attend->prefix || attend->first_keys)
        return kv_fail(ctx, AHIP_ERR_UNSUPPORTED, name + "causal attention without window, slopes, prefix and first keys only");
    if (sparse->first < 0 || sparse->last < 1 || (int64_t)sparse->first + sparse->last > sparse->most)
        return kv_fail(ctx, AHIP_ERR_ARG, name + "the first and the last pages, one of those at least, fit into what is chosen");
    if ((int64_t)sparse->most * cache->page_size > INT32_MAX - (1 << 16) || attend->tokens * (uint64_t)cache->kv_heads >= MOST_GRID / 2)
        return kv_fail(ctx, AHIP_ERR_UNSUPPORTED, name + "more chosen keys, or rows, than are supported");
    if (sparse->most > (int32_t)LISTED && (uint64_t)sparse->most < most_pages(*cache, *batch, *attend))
        return kv_fail(ctx, AHIP_ERR_UNSUPPORTED, name + "more than " + std::to_string(LISTED) + " pages chosen of more");
    return check_means(ctx, name, *cache, *sparse);
}

template <uint32_t UNITS, int FOURS> void launch_choice(hipStream_t stream, const SparseArgs &g, const SparsePlan &p) {
    const dim3 grid((uint32_t)(g.fills ? 2 * p.rows : p.rows)), block(BLOCK);
    // What a block holds: images, and the list of a row that has more pages than it chooses.
    const uint32_t held = (uint32_t)(g.held * sizeof(uint64_t) + (g.most < g.max_pages ? g.most * sizeof(uint32_t) : 0));
    if (p.by_rows) {
        hipLaunchKernelGGL((score_rows<UNITS>), dim3((uint32_t)p.score_blocks), block, 0, stream, g);
        hipLaunchKernelGGL((choose_pages<0, 1, BLOCK>), grid, block, held, stream, g);
    } else if (p.split) {
        hipLaunchKernelGGL((score_pages<UNITS, FOURS>), dim3((uint32_t)p.score_blocks), block, 0, stream, g);
        hipLaunchKernelGGL((choose_pages<0, 1, BLOCK>), grid, block, held, stream, g);
    } else {
        hipLaunchKernelGGL((choose_pages<UNITS, FOURS, LARGE>), grid, dim3(LARGE), held, stream, g);
    }
}

SparseArgs args_of(const dev::KvView &view, const ahip_kv_cache &cache, const ahip_kv_sparse &sparse) {
    SparseArgs g = {};
    g.kv = view;
    g.means = sparse.means, g.means_page = sparse.page_stride, g.means_head = sparse.head_stride;
    g.d = (uint32_t)cache.head_size, g.bf16 = cache.elem == AHIP_KV_BF16;
    return g;
}

// Pages that the rows of a call can fill: g.chunks, and a launch over them.
int launch_means(DeviceCtx &ctx, SparseArgs g, const std::string &name) {
    const uint64_t pairs = (uint64_t)g.kv.sequences * g.kv.kv_heads;
    g.chunks = (uint32_t)std::min<uint64_t>(g.max_tokens / g.kv.page_size + 1, std::max<uint64_t>(1, LAUNCHED / pairs));
    const uint64_t blocks = pairs * g.chunks;
    if (blocks >= MOST_GRID) return ctx.fail(AHIP_ERR_UNSUPPORTED, name + "more blocks than a grid holds");
    hipLaunchKernelGGL(mean_pages, dim3((uint32_t)blocks), dim3(BLOCK), 0, ctx.stream, g);
    return ctx.check(hipGetLastError(), "kv page means launch");
}

}  // namespace

int launch_kv_page_means(DeviceCtx &ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_sparse &sparse, size_t tokens, size_t max_tokens) {
    const std::string name = "kv page means: ";
    dev::KvView view = {};
    if (int rc = make_kv_view(&ctx, "kv page means", &cache, &batch, tokens, &view)) return rc;
    if (int rc = check_means(&ctx, name, cache, sparse)) return rc;
    if (tokens == 0 || batch.sequences == 0) return AHIP_OK;
    if (int rc = require_kv_arrays(ctx, "kv page means", cache, batch)) return rc;
    if (!sparse.means) return ctx.fail(AHIP_ERR_ARG, name + "null means");
    SparseArgs g = args_of(view, cache, sparse);
    g.max_tokens = (uint32_t)std::min(max_tokens ? max_tokens : tokens, tokens), g.max_keys = INT32_MAX;
    return launch_means(ctx, g, name);
}

int kv_attention_sparse_workspace(DeviceCtx *ctx, const ahip_kv_cache *cache, const ahip_kv_batch *batch, const ahip_kv_attend *attend, const ahip_kv_sparse *sparse,
                                  size_t *bytes) {
    if (!bytes) return kv_fail(ctx, AHIP_ERR_ARG, "kv attention over chosen pages: null output");
    *bytes = 0;
    dev::KvView view = {};
    if (int rc = check_sparse(ctx, cache, batch, attend, sparse, &view)) return rc;
    *bytes = sparse_plan(ctx, *cache, *batch, *attend, *sparse).bytes;
    return AHIP_OK;
}

int launch_kv_attention_sparse(DeviceCtx &ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_attend &attend, const ahip_kv_sparse &sparse) {
    const std::string name = "kv attention over chosen pages: ";
    dev::KvView view = {};
    if (int rc = check_sparse(&ctx, &cache, &batch, &attend, &sparse, &view)) return rc;
    if (attend.tokens == 0 || batch.sequences == 0) return AHIP_OK;
    if (int rc = require_kv_arrays(ctx, "kv attention over chosen pages", cache, batch)) return rc;
    if (!sparse.means || !sparse.chosen || !attend.q) return ctx.fail(AHIP_ERR_ARG, name + "null pointer");
    SparsePlan p = sparse_plan(&ctx, cache, batch, attend, sparse);
    if (!attend.workspace || attend.workspace_bytes < p.bytes)
        return ctx.fail(AHIP_ERR_ARG, name + "the workspace holds " + std::to_string(attend.workspace ? attend.workspace_bytes : 0) + " bytes of " + std::to_string(p.bytes));
    char *space = static_cast<char *>(attend.workspace);
    SparseArgs g = args_of(view, cache, sparse);
    g.chosen = sparse.chosen, g.q = attend.q, g.q_token = (int64_t)attend.q_strides[0], g.q_head = (int64_t)attend.q_strides[1];
    g.q_heads = (uint32_t)attend.q_heads, g.group = (uint32_t)(attend.q_heads / cache.kv_heads);
    g.most = (uint32_t)sparse.most, g.first = (uint32_t)sparse.first, g.last = (uint32_t)sparse.last;
    g.max_tokens = (uint32_t)std::min(attend.max_tokens ? attend.max_tokens : attend.tokens, attend.tokens);
    g.max_keys = (uint32_t)std::min(attend.max_keys ? attend.max_keys : (size_t)INT32_MAX, (size_t)INT32_MAX);
    g.max_pages = (uint32_t)p.max_pages, g.held = (uint32_t)std::min<uint64_t>(p.max_pages, HELD);
    g.chunks = (uint32_t)p.chunks;
    g.starts = reinterpret_cast<int32_t *>(space + p.starts), g.lengths = reinterpret_cast<int32_t *>(space + p.lengths), g.table = reinterpret_cast<int32_t *>(space + p.table);
    g.scores = p.split ? reinterpret_cast<double *>(space + p.scores) : nullptr;
    // What attention will see, before anything is launched.
    p.batch.query_starts = g.starts, p.batch.lengths = g.lengths, p.batch.page_table = g.table;
    p.attend.workspace_bytes = p.attend_bytes;
    attend::AttendArgs a = {};
    if (int rc = attend::begin_attend(ctx, cache, p.batch, p.attend, false, &a)) return rc;
    a.kv.table_head = sparse.most;

    // A single row fills a page for later calls only; several may score a page that one of them has filled.  Blocks beside the choice are as many again, as far as a
    // grid of 2^32 threads holds both.
    g.fills = g.max_tokens == 1 && 2 * p.rows * (p.split ? BLOCK : LARGE) < MOST_GRID * BLOCK;
    if (!g.fills)
        if (int rc = launch_means(ctx, g, name)) return rc;
    if (g.d <= 64) g.group <= 4 ? launch_choice<4, 1>(ctx.stream, g, p) : launch_choice<4, 2>(ctx.stream, g, p);
    else if (g.d <= 128) g.group <= 4 ? launch_choice<8, 1>(ctx.stream, g, p) : launch_choice<8, 2>(ctx.stream, g, p);
    else launch_choice<16, 1>(ctx.stream, g, p);
    if (int rc = ctx.check(hipGetLastError(), "kv attention over chosen pages launch")) return rc;
    return attend::launch_attend_kept(ctx, a, g.bf16);
}

}  // namespace altius

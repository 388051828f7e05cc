// What attention over a paged cache gave each key: mass(j) = decay mass(j) + sum over rows of 2^(x(row, j) - top(row)) / total(row), x in units of
// log2(e) as in kv_attend.h, top and 1 / total what attention leaves behind of each row.  The scores are computed again, with the rows where attention has the
// keys: a wavefront holds 32 keys in registers, as the second operand of v_mfma_f32_32x32x16_bf16, and goes through the rows, 32 at a time, which the
// block's four wavefronts share in LDS.  Accumulator register r of lane l is then row 8 (r / 4) + 4 (l / 32) + r % 4 and key l % 32: a lane adds up its own
// key's weights, and nothing is exchanged before the end.  Queries are three bf16 numbers each, whose sum they are, and so are keys of an fp32 cache, as in
// kv_attend.h.
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

constexpr int MASS_KEYS = 128, MASS_ROWS = 32;  // of a block; of a step

struct MassArgs {
    AttendArgs at;
    float *mass;
    int32_t *positions;
    int64_t page_stride, head_stride;
    const int32_t *row_positions;
    float decay;
    uint32_t chunks, parts;  // of MASS_KEYS keys a sequence, and of its rows
    float *sums;             // [parts][sequence][kv head][chunks * MASS_KEYS]; null: one part
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

template <int DP> struct MassLds {
    static constexpr int PITCH = DP + 8;
    uint16_t q[3][MASS_ROWS * PITCH];
    float top[MASS_ROWS], recip[MASS_ROWS], slope[MASS_ROWS];
    int32_t low[MASS_ROWS], high[MASS_ROWS], place[MASS_ROWS];
    int64_t q_at[MASS_ROWS];
};

template <int DP, bool BF16> __global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void weigh_keys(MassArgs m) {
    constexpr int STEPS = DP / 16, PLANES = BF16 ? 1 : 3, SIZE = BF16 ? 2 : 4;
    __shared__ __align__(16) MassLds<DP> lds;
    constexpr int PITCH = MassLds<DP>::PITCH;
    const AttendArgs &g = m.at;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31u, h = lane >> 5;
    // The first keys of a causal sequence are seen by most rows: they start first.
    uint32_t id = blockIdx.x;
    const uint32_t part = id % m.parts;
    id /= m.parts;
    const uint32_t pairs = g.kv.sequences * g.kv.kv_heads, chunk = id / pairs, pair = id - chunk * pairs, s = pair / g.kv.kv_heads, kvh = pair - s * g.kv.kv_heads;
    const dev::KvSequence seq = sequence_of(g, s);
    const int32_t first = (int32_t)(chunk * MASS_KEYS);
    if (seq.n == 0 || first >= seq.length) return;
    const uint32_t rows = (uint32_t)seq.n * g.group;

    // This lane's key.  Behind the last one that one stands in, and is left out.
    const int32_t key = first + (int32_t)(wave * 32 + col);
    const uint32_t read = (uint32_t)min(key, seq.length - 1), index = g.kv.by_page_size.div(read);
    const int64_t k_at = (int64_t)g.kv.page_of(s, index, 0) * g.kv.page_stride + (int64_t)(read - index * g.kv.page_size) * g.kv.slot_stride + (int64_t)kvh * g.kv.head_stride;
    u32x4 k[PLANES][STEPS];
    {
        const char *row = static_cast<const char *>(g.kv.keys) + k_at * SIZE;
#pragma unroll
        for (int c = 0; c < STEPS; c++) {
            const uint32_t channel = 16 * c + 8 * h;
            if constexpr (BF16) {
                const u32x4 x = *reinterpret_cast<const u32x4 *>(row + SIZE * (channel < g.d ? channel : 0));
                k[0][c] = channel < g.d ? x : u32x4{0, 0, 0, 0};
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
                for (int p = 0; p < PLANES; p++) k[p][c] = u32x4{w[p][0], w[p][1], w[p][2], w[p][3]};
            }
        }
    }

    const uint32_t tiles = (rows + MASS_ROWS - 1) / MASS_ROWS, from = (uint32_t)((uint64_t)tiles * part / m.parts), to = (uint32_t)((uint64_t)tiles * (part + 1) / m.parts);
    float sum = 0.0f;
    for (uint32_t tile = from; tile < to; tile++) {
        // Every wavefront looks at the rows' ranges: a tile none of whose rows sees any of the block's keys is left out by all.
        const uint32_t row = tile * MASS_ROWS + col;
        const bool valid = row < rows;
        const uint32_t token = g.by_group.div(valid ? row : 0), head = kvh * g.group + (valid ? row : 0) - token * g.group;
        const RowRange range = row_range(g, seq, s, token);
        if (!__any(valid && range.low < first + MASS_KEYS && range.high > first && range.low < range.high)) continue;
        __syncthreads();
        if (tid < MASS_ROWS) {
            lds.low[col] = valid ? range.low : 0, lds.high[col] = valid ? range.high : 0, lds.place[col] = range.place;
            const f32x2 stats = *reinterpret_cast<const f32x2 *>(g.stats + 2 * ((size_t)(seq.start + (int32_t)token) * g.q_heads + head));
            lds.top[col] = stats.x, lds.recip[col] = stats.y;
            lds.slope[col] = g.slopes ? g.slopes[head] * LOG2E : 0.0f;
            lds.q_at[col] = (int64_t)(seq.start + (int32_t)token) * g.q_token + (int64_t)head * g.q_head;
        }
        // Queries: 8 threads a row.
        {
            const uint32_t its = tile * MASS_ROWS + tid / 8, t = g.by_group.div(its < rows ? its : 0), its_head = kvh * g.group + (its < rows ? its : 0) - t * g.group;
            const float *q_row = g.q + (int64_t)(seq.start + (int32_t)t) * g.q_token + (int64_t)its_head * g.q_head;
            f32x4 x[DP / 32];
#pragma unroll
            for (int e = 0; e < DP / 32; e++) {
                const uint32_t c = 32 * e + 4 * (tid & 7u);
                x[e] = *reinterpret_cast<const f32x4 *>(q_row + (c < g.d ? c : 0));
            }
#pragma unroll
            for (int e = 0; e < DP / 32; e++) {
                const uint32_t c = 32 * e + 4 * (tid & 7u);
                const float by = c < g.d && its < rows ? g.scale : 0.0f;
                uint32_t w[3][2];
                split_pair(x[e][0] * by, x[e][1] * by, w[0][0], w[1][0], w[2][0]);
                split_pair(x[e][2] * by, x[e][3] * by, w[0][1], w[1][1], w[2][1]);
#pragma unroll
                for (int p = 0; p < 3; p++) *reinterpret_cast<u32x2 *>(&lds.q[p][(tid / 8) * PITCH + c]) = u32x2{w[p][0], w[p][1]};
            }
        }
        __syncthreads();
        f32x16 st;
#pragma unroll
        for (int r = 0; r < 16; r++) st[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < STEPS; c++) {
            u32x4 a[3];
#pragma unroll
            for (int p = 0; p < 3; p++) a[p] = *reinterpret_cast<const u32x4 *>(&lds.q[p][col * PITCH + 16 * c + 8 * h]);
            // Smallest terms first.
            ALTIUS_MFMA32_BF16(a[2], k[0][c], st);
            if constexpr (!BF16) {
                ALTIUS_MFMA32_BF16(a[0], k[2][c], st);
                ALTIUS_MFMA32_BF16(a[1], k[1][c], st);
            }
            ALTIUS_MFMA32_BF16(a[1], k[0][c], st);
            if constexpr (!BF16) ALTIUS_MFMA32_BF16(a[0], k[1][c], st);
            ALTIUS_MFMA32_BF16(a[0], k[0][c], st);
        }
        auto row_of = [&](int r) { return 8 * (r >> 2) + 4 * (int32_t)h + (r & 3); };
        float x[16];
        float check = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; r++) x[r] = st[r], check = __builtin_fmaf(st[r], 0.0f, check);
        // Infinity or NaN: of a row or key that is not seen, or parts of infinity of opposite signs.  Value by value then.
        if (__any(check != 0.0f)) {
#pragma unroll 1
            for (int r = 0; r < 16; r++) {
                const float *q_row = g.q + lds.q_at[row_of(r)];
                float dot = 0.0f;
                for (uint32_t c = 0; c < g.d; c++) dot = __builtin_fmaf(q_row[c] * g.scale, cache_value<BF16>(g.kv.keys, k_at + c), dot);
#pragma unroll
                for (int e = 0; e < 16; e++) x[e] = e == r ? dot : x[e];
            }
        }
        cap_scores(g, x);
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const int at = 8 * b + 4 * (int)h;
            const f32x4 top = *reinterpret_cast<const f32x4 *>(&lds.top[at]), recip = *reinterpret_cast<const f32x4 *>(&lds.recip[at]), slope = *reinterpret_cast<const f32x4 *>(&lds.slope[at]);
            const u32x4 low = *reinterpret_cast<const u32x4 *>(&lds.low[at]), high = *reinterpret_cast<const u32x4 *>(&lds.high[at]), place = *reinterpret_cast<const u32x4 *>(&lds.place[at]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float y = x[4 * b + e];
                if (g.slopes) y -= slope[e] * (float)abs((int32_t)place[e] - key);
                const float w = exp2_fast(y - top[e]) * recip[e];
                sum += key >= (int32_t)low[e] && key < (int32_t)high[e] ? w : 0.0f;
            }
        }
    }
    sum += __shfl_xor(sum, 32);
    if (h != 0 || key >= seq.length) return;
    if (m.sums) m.sums[((size_t)part * pairs + pair) * (m.chunks * MASS_KEYS) + (size_t)key] = sum;
    else put_mass(m, seq, s, kvh, key, sum);
}

// The parts of a key's sum, in order.  A thread a key.
__global__ __launch_bounds__(256) void add_masses(MassArgs m) {
    const uint32_t pairs = m.at.kv.sequences * m.at.kv.kv_heads, per = (m.chunks * MASS_KEYS + 255) / 256, pair = blockIdx.x / per;
    const uint32_t s = pair / m.at.kv.kv_heads, kvh = pair - s * m.at.kv.kv_heads, key = (blockIdx.x - pair * per) * 256 + threadIdx.x;
    const dev::KvSequence seq = sequence_of(m.at, s);
    if (seq.n == 0 || key >= (uint32_t)seq.length) return;
    float sum = 0.0f;
    for (uint32_t part = 0; part < m.parts; part++) sum += m.sums[((size_t)part * pairs + pair) * (m.chunks * MASS_KEYS) + key];
    put_mass(m, seq, s, kvh, (int32_t)key, sum);
}

struct MassPlan {
    uint64_t chunks, parts, blocks;
    size_t attend, stats, sums;  // where each begins in the workspace
    size_t bytes;
};
size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

MassPlan mass_plan(const DeviceCtx *ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_attend &attend) {
    MassPlan p = {};
    const size_t held = std::min((size_t)batch.table_pages * (size_t)cache.page_size, (size_t)INT32_MAX);
    const size_t max_keys = std::min(attend.max_keys ? attend.max_keys : held, held);
    const size_t max_tokens = std::min(attend.max_tokens ? attend.max_tokens : attend.tokens, attend.tokens);
    const uint64_t pairs = (uint64_t)batch.sequences * (uint64_t)cache.kv_heads, tiles = (max_tokens * (uint64_t)(attend.q_heads / cache.kv_heads) + MASS_ROWS - 1) / MASS_ROWS;
    p.chunks = (max_keys + MASS_KEYS - 1) / MASS_KEYS;
    const uint64_t cus = ctx && ctx->cus_per_xcd ? 8 * ctx->cus_per_xcd : 256;
    // Rows are cut until there are three blocks a CU, each of at least eight tiles of rows.
    p.parts = 1;
    while (p.parts < 16 && p.chunks * pairs * p.parts < 3 * cus && tiles / (2 * p.parts) >= 8) p.parts *= 2;
    p.blocks = p.chunks * pairs * p.parts;
    p.attend = 0;
    p.stats = up16(plan_of(ctx, cache, batch, attend).bytes);
    p.sums = up16(p.stats + 2 * attend.tokens * (size_t)attend.q_heads * sizeof(float));
    p.bytes = p.parts > 1 ? p.sums + p.parts * pairs * p.chunks * MASS_KEYS * sizeof(float) : p.sums;
    return p;
}

template <bool BF16> void launch_weigh(hipStream_t stream, uint32_t blocks, const MassArgs &m) {
    if (m.at.d <= 64) hipLaunchKernelGGL((weigh_keys<64, BF16>), dim3(blocks), dim3(256), 0, stream, m);
    else if (m.at.d <= 128) hipLaunchKernelGGL((weigh_keys<128, BF16>), dim3(blocks), dim3(256), 0, stream, m);
    else hipLaunchKernelGGL((weigh_keys<256, BF16>), dim3(blocks), dim3(256), 0, stream, m);
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
    const uint64_t joins = plan.parts > 1 ? (uint64_t)batch.sequences * cache.kv_heads * ((plan.chunks * MASS_KEYS + 255) / 256) : 0;
    if (plan.blocks >= MOST_BLOCKS || joins >= MOST_BLOCKS) return ctx.fail(AHIP_ERR_UNSUPPORTED, name + "more blocks than a grid holds");
    if (int rc = begin_attend(ctx, cache, batch, attend, &m.at)) return rc;
    char *space = static_cast<char *>(attend.workspace);
    m.at.stats = reinterpret_cast<float *>(space + plan.stats);
    const bool bf16 = cache.elem == AHIP_KV_BF16;
    if (int rc = launch_attend_rows(ctx, m.at, bf16)) return rc;
    m.mass = history.mass, m.positions = history.positions, m.page_stride = history.page_stride, m.head_stride = history.head_stride;
    m.row_positions = row_positions, m.decay = decay;
    m.chunks = (uint32_t)plan.chunks, m.parts = (uint32_t)plan.parts;
    m.sums = plan.parts > 1 ? reinterpret_cast<float *>(space + plan.sums) : nullptr;
    if (bf16) launch_weigh<true>(ctx.stream, (uint32_t)plan.blocks, m);
    else launch_weigh<false>(ctx.stream, (uint32_t)plan.blocks, m);
    if (int rc = ctx.check(hipGetLastError(), "kv attention mass launch")) return rc;
    if (!joins) return AHIP_OK;
    hipLaunchKernelGGL(add_masses, dim3((uint32_t)joins), dim3(256), 0, ctx.stream, m);
    return ctx.check(hipGetLastError(), "kv attention mass launch");
}

}  // namespace altius

// What happens to a cache that is full, or whose drafted tokens have been judged: which slots stay (ahip_kv_evict), and slots that go to other
// places of their sequence (ahip_kv_move).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv.h"

namespace altius {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct History {
    float *mass;
    int32_t *positions;
    int64_t page_stride, head_stride;
};

// ---------------------------------------------------------------- who stays
// A block for each sequence and head of keys.  The budget's smallest value is found digit by digit of an order-preserving image of the
// masses (11, 11 and 10 bits): a histogram of the values that share the digits so far, in LDS, and the bin that the rank falls into.  What is kept
// by its position is counted apart, so that it does not all meet in one bin.  The image waits in LDS as far as that goes (32768 places), what
// is behind is read anew, out of L2.  Then wavefronts take runs of places in order: one walk counts, one writes the lists.
// Bound by latency: the walks of one block, one after the other.  48 sequences of 1025 places, 8 heads: 13.4 us; 4 of 20011 to 50000: 131 us.
constexpr uint32_t EVICT = 1024, WAVES = EVICT / 64, BINS = 2048, HELD = 32768;
constexpr uint32_t KEPT = 0xffffffffu;  // by its position; above every mass

struct EvictArgs {
    dev::KvView kv;
    History history;
    uint32_t budget, most, max_keys, held;
    int32_t recent, first;
    int32_t *sources, *targets, *counts, *lengths;
};

__device__ __forceinline__ uint32_t rank_image(float mass) {
    if (mass != mass) return 0;
    const uint32_t u = __float_as_uint(mass + 0.0f);  // -0 and 0 are equal
    return u >> 31 ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(EVICT) void choose_evicted(EvictArgs g) {
    extern __shared__ uint32_t held[];
    __shared__ uint32_t bins[BINS];
    __shared__ uint32_t per_wave[WAVES][4];
    __shared__ uint32_t found[2];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t s = blockIdx.x / g.kv.kv_heads, head = blockIdx.x - s * g.kv.kv_heads;
    const int32_t length = g.kv.lengths[s];
    int32_t *const count = g.counts + (int64_t)s * g.kv.kv_heads + head;
    const bool fits = length >= 0 && (uint64_t)length <= (uint64_t)g.kv.table_pages * g.kv.page_size && (uint32_t)length <= g.max_keys;
    if (!fits || (uint32_t)length <= g.budget) {
        if (tid == 0) {
            *count = 0;
            if (!fits) *g.kv.flag = 1;
            else if (head == 0) g.lengths[s] = length;
        }
        return;
    }
    const uint32_t n = (uint32_t)length;
    if (tid == 0 && head == 0) g.lengths[s] = (int32_t)g.budget;
    auto slot_of = [&](uint32_t place) {
        const uint32_t index = g.kv.by_page_size.div(place);
        return (int64_t)g.kv.page_of(s, index, 0) * g.history.page_stride + (int64_t)head * g.history.head_stride + (place - index * g.kv.page_size);
    };

    // The newest position.
    int32_t newest = INT32_MIN;
    for (uint32_t place = tid; place < n; place += EVICT) newest = max(newest, g.history.positions[slot_of(place)]);
#pragma unroll
    for (int m = 32; m; m >>= 1) newest = max(newest, __shfl_xor(newest, m));
    if (lane == 0) per_wave[wave][0] = (uint32_t)newest;
    for (uint32_t b = tid; b < BINS; b += EVICT) bins[b] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < WAVES; w++) newest = max(newest, (int32_t)per_wave[w][0]);
    const int64_t above = (int64_t)newest - g.recent;

    auto image_of = [&](uint32_t place) {
        const int64_t at = slot_of(place);
        const int32_t position = g.history.positions[at];
        return position < g.first || position > above ? KEPT : rank_image(g.history.mass[at]);
    };
    auto image = [&](uint32_t place) { return place < g.held ? held[place] : image_of(place); };

    // The first digit's histogram, the images into LDS, and how many are kept by their position.
    uint32_t kept = 0;
    for (uint32_t place = tid; place < n; place += EVICT) {
        const uint32_t v = image_of(place);
        if (place < g.held) held[place] = v;
        if (v == KEPT) kept++;
        else atomicAdd(&bins[v >> 21], 1u);
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) kept += __shfl_xor(kept, m);
    __syncthreads();  // behind the readers of per_wave
    if (lane == 0) per_wave[wave][0] = kept;
    __syncthreads();
    kept = 0;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; w++) kept += per_wave[w][0];

    // least: the smallest image that stays; ties: how many of that image do.
    uint32_t least = KEPT, ties = g.budget;
    if (kept < g.budget) {
        uint32_t need = g.budget - kept;  // of those that share the digits so far
        least = 0;
        for (int digit = 0; digit < 3; digit++) {
            const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
            const uint32_t width = digit == 2 ? 1024 : 2048;
            if (digit) {
                __syncthreads();
                for (uint32_t b = tid; b < BINS; b += EVICT) bins[b] = 0;
                __syncthreads();
                const int known = digit == 1 ? 21 : 10;
                for (uint32_t place = tid; place < n; place += EVICT) {
                    const uint32_t v = image(place);
                    if (v != KEPT && v >> known == least >> known) atomicAdd(&bins[v >> shift & (width - 1)], 1u);
                }
                __syncthreads();
            }
            // Thread t has bins 2 t and 2 t + 1: how many values are above them.
            const uint32_t low = bins[2 * tid], high = bins[2 * tid + 1];
            uint32_t up_to = low + high;  // from this lane's bins on, within the wavefront
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const uint32_t t = __shfl_down(up_to, m);
                if (lane + m < 64) up_to += t;
            }
            __syncthreads();
            if (lane == 0) per_wave[wave][1] = up_to;
            __syncthreads();
            uint32_t over = up_to - low - high;
            for (uint32_t w = wave + 1; w < WAVES; w++) over += per_wave[w][1];
            if (over < need && need <= over + high) found[0] = 2 * tid + 1, found[1] = over;
            else if (over + high < need && need <= over + high + low) found[0] = 2 * tid, found[1] = over + high;
            __syncthreads();
            least |= found[0] << shift;
            need -= found[1];
        }
        ties = need;
    }

    // Runs of places, a wavefront each, in order: what each has above `least` and at it, below the budget and from it on.
    const uint32_t run = (n + EVICT - 1) / EVICT * 64, from = min(wave * run, n), to = min(from + run, n);
    uint32_t counts[4] = {0, 0, 0, 0};
    for (uint32_t base = from; base < to; base += 64) {
        const uint32_t place = base + lane, v = place < to ? image(place) : 0;
        const bool there = place < to, low = place < g.budget;
        counts[0] += (uint32_t)__popcll(__ballot(there && low && v > least));
        counts[1] += (uint32_t)__popcll(__ballot(there && low && v == least));
        counts[2] += (uint32_t)__popcll(__ballot(there && !low && v > least));
        counts[3] += (uint32_t)__popcll(__ballot(there && !low && v == least));
    }
    __syncthreads();
    if (lane < 4) per_wave[wave][lane] = counts[lane];
    __syncthreads();
    // What the runs in front leave: ties already kept, holes and movers already listed.
    uint32_t tied = 0, holes = 0, movers = 0;
    for (uint32_t w = 0; w < wave; w++) {
        const uint32_t start = min(w * run, n), end = min(start + run, n), lows = min(end, g.budget) - min(start, g.budget);
        const uint32_t left = ties - tied, stay_low = min(per_wave[w][1], left), stay_high = min(per_wave[w][3], left - stay_low);
        holes += lows - per_wave[w][0] - stay_low;
        movers += per_wave[w][2] + stay_high;
        tied += stay_low + stay_high;
    }
    const int64_t list = ((int64_t)s * g.kv.kv_heads + head) * g.most;
    const uint64_t before = ((uint64_t)1 << lane) - 1;
    for (uint32_t base = from; base < to; base += 64) {
        const uint32_t place = base + lane, v = place < to ? image(place) : 0;
        const bool there = place < to, low = place < g.budget, tie = there && v == least;
        const uint64_t tie_mask = __ballot(tie);
        const bool stays = there && (v > least || (tie && tied + (uint32_t)__popcll(tie_mask & before) < ties));
        const bool hole = there && low && !stays, mover = stays && !low;
        const uint64_t hole_mask = __ballot(hole), mover_mask = __ballot(mover);
        const uint32_t hole_at = holes + (uint32_t)__popcll(hole_mask & before), mover_at = movers + (uint32_t)__popcll(mover_mask & before);
        if (hole && hole_at < g.most) g.targets[list + hole_at] = (int32_t)place;
        if (mover && mover_at < g.most) g.sources[list + mover_at] = (int32_t)place;
        holes += (uint32_t)__popcll(hole_mask), movers += (uint32_t)__popcll(mover_mask);
        tied += (uint32_t)__popcll(tie_mask);
    }
    if (tid == EVICT - 64) *count = (int32_t)min(movers, g.most);  // the last run's: all of them
}

// ---------------------------------------------------------------- moves
// A slot's row of keys and row of values are units of 16 bytes (of one element where a row or stride is no multiple of that).  A block takes some
// moves of one list: their places become addresses once, in LDS, then its threads read all their units before any is written, so that a
// list that must go in order may be taken a blockful at a time.  Bound by memory: 8 caches of 1100 to 2000 moves for each of 8 heads of 128 channels, bf16,
// 30 us, 3.5 TB/s read and written.
constexpr uint32_t MOVE = 256, EACH = 8;  // threads; units that a thread holds

struct MoveArgs {
    dev::KvView kv;
    History history;
    const int32_t *sources, *targets, *counts;
    int64_t sequence_stride, head_stride, count_sequence, count_head;
    uint32_t most, row_units, moves, chunks;  // units of a slot's keys; moves of a block at a time; blocks of a list (0: one goes through it in order)
};

template <class Unit> __global__ __launch_bounds__(MOVE) void move_slots(MoveArgs g) {
    __shared__ int64_t place_of[2][MOVE];  // units from the start of the cache; -1: left out
    const uint32_t tid = threadIdx.x, chunks = g.chunks ? g.chunks : 1;
    const uint32_t pair = blockIdx.x / chunks, chunk = blockIdx.x - pair * chunks, s = pair / g.kv.kv_heads, head = pair - s * g.kv.kv_heads;
    const int32_t count = g.counts[(int64_t)s * g.count_sequence + (int64_t)head * g.count_head];
    if (count < 0 || (uint32_t)count > g.most) {
        if (tid == 0) *g.kv.flag = 1;
        return;
    }
    const int64_t list = (int64_t)s * g.sequence_stride + (int64_t)head * g.head_stride;
    const uint32_t places = g.kv.table_pages * g.kv.page_size, both = 2 * g.row_units;
    Unit *const keys = static_cast<Unit *>(g.kv.keys), *const values = static_cast<Unit *>(g.kv.values);
    const uint32_t to = g.chunks ? min((chunk + 1) * g.moves, (uint32_t)count) : (uint32_t)count;
    for (uint32_t from = chunk * g.moves; from < to; from += g.moves) {
        const uint32_t now = min(g.moves, to - from);
        int64_t remembered[2] = {-1, -1};
        float mass = 0.0f;
        int32_t position = 0;
        if (tid < now) {
            const uint32_t place[2] = {(uint32_t)g.sources[list + from + tid], (uint32_t)g.targets[list + from + tid]};
            int64_t at[2];
            bool fits = true;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                at[e] = -1;
                if (place[e] < places) {
                    const uint32_t index = g.kv.by_page_size.div(place[e]), slot = place[e] - index * g.kv.page_size;
                    const int32_t page = g.kv.page_of(s, index, -1);
                    if (page >= 0) {
                        at[e] = (int64_t)page * g.kv.page_stride + (int64_t)head * g.kv.head_stride + (int64_t)slot * g.kv.slot_stride;
                        remembered[e] = (int64_t)page * g.history.page_stride + (int64_t)head * g.history.head_stride + slot;
                    }
                } else {
                    *g.kv.flag = 1;
                }
                fits = fits && at[e] >= 0;
            }
            place_of[0][tid] = fits ? at[0] : -1, place_of[1][tid] = at[1];
            if (!fits) remembered[0] = -1;
            if (remembered[0] >= 0) {
                if (g.history.mass) mass = g.history.mass[remembered[0]];
                if (g.history.positions) position = g.history.positions[remembered[0]];
            }
        }
        __syncthreads();
        // A move's units side by side, keys then values; more than a block holds at a time in turns, each of whole moves or of one move's columns.
        const uint32_t columns = min(both, MOVE * EACH);
        for (uint32_t column = 0; column < both; column += columns) {
            const uint32_t width = min(columns, both - column), units = now * width;
            Unit x[EACH];
            auto each = [&](auto what) {
#pragma unroll
                for (uint32_t e = 0; e < EACH; e++) {
                    const uint32_t i = e * MOVE + tid;
                    if (i >= units) break;
                    const uint32_t move = i / width, unit = column + (i - move * width);
                    if (place_of[0][move] < 0) continue;
                    what(e, move, unit < g.row_units ? keys : values, unit < g.row_units ? unit : unit - g.row_units);
                }
            };
            each([&](uint32_t e, uint32_t move, Unit *base, uint32_t unit) { x[e] = base[place_of[0][move] + unit]; });
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            each([&](uint32_t e, uint32_t move, Unit *base, uint32_t unit) { base[place_of[1][move] + unit] = x[e]; });
        }
        if (remembered[0] >= 0) {
            if (g.history.mass) g.history.mass[remembered[1]] = mass;
            if (g.history.positions) g.history.positions[remembered[1]] = position;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
}

constexpr int64_t MOST_STRIDE = (int64_t)1 << 48;
constexpr uint64_t MOST_BLOCKS = (uint64_t)1 << 21;  // of up to 1024 threads: a grid ends at 2^32

int take_history(DeviceCtx &ctx, const char *who, const ahip_kv_history *history, History *to) {
    *to = {};
    if (!history) return AHIP_OK;
    if (history->page_stride < 0 || history->head_stride < 0 || history->page_stride > MOST_STRIDE || history->head_stride > MOST_STRIDE)
        return ctx.fail(AHIP_ERR_ARG, std::string(who) + ": a stride of the history is out of range");
    *to = {history->mass, history->positions, history->page_stride, history->head_stride};
    return AHIP_OK;
}

}  // namespace

int launch_kv_evict(DeviceCtx &ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_history &history, const ahip_kv_eviction &eviction) {
    const char *who = "kv evict";
    const std::string name = "kv evict: ";
    EvictArgs g = {};
    if (int rc = make_kv_view(&ctx, who, &cache, &batch, 0, &g.kv)) return rc;
    if (int rc = take_history(ctx, who, &history, &g.history)) return rc;
    if (eviction.budget < 1 || eviction.recent < 0 || eviction.first < 0 || (int64_t)eviction.recent + eviction.first > eviction.budget)
        return ctx.fail(AHIP_ERR_ARG, name + "the budget is at least 1, and the first and the recent positions fit into it");
    const size_t held = (size_t)batch.table_pages * (size_t)cache.page_size;
    const size_t max_keys = std::min(eviction.max_keys ? eviction.max_keys : held, held);
    const int64_t most = std::min<int64_t>(eviction.budget, (int64_t)max_keys - eviction.budget);
    if (eviction.most < 0 || eviction.most < most)
        return ctx.fail(AHIP_ERR_ARG, name + "lists of " + std::to_string(eviction.most) + " do not hold " + std::to_string(most) + " moves");
    if (batch.sequences == 0) return AHIP_OK;
    if (!batch.lengths || (batch.table_pages && !batch.page_table)) return ctx.fail(AHIP_ERR_ARG, name + "null batch array");
    if (cache.pages == 0) return ctx.fail(AHIP_ERR_ARG, name + "the cache has no pages");
    if (!history.mass || !history.positions || !eviction.counts || !eviction.lengths || (eviction.most && (!eviction.sources || !eviction.targets)))
        return ctx.fail(AHIP_ERR_ARG, name + "null pointer");
    const uint64_t blocks = (uint64_t)batch.sequences * (uint64_t)cache.kv_heads;
    if (blocks >= MOST_BLOCKS) return ctx.fail(AHIP_ERR_UNSUPPORTED, name + "more blocks than a grid holds");
    g.budget = (uint32_t)eviction.budget, g.most = (uint32_t)eviction.most, g.max_keys = (uint32_t)max_keys;
    g.recent = eviction.recent, g.first = eviction.first;
    g.sources = eviction.sources, g.targets = eviction.targets, g.counts = eviction.counts, g.lengths = eviction.lengths;
    g.held = (uint32_t)std::min<size_t>(max_keys, HELD);
    hipLaunchKernelGGL(choose_evicted, dim3((uint32_t)blocks), dim3(EVICT), g.held * sizeof(uint32_t), ctx.stream, g);
    return ctx.check(hipGetLastError(), "kv evict launch");
}

int launch_kv_move(DeviceCtx &ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_moves &moves, const ahip_kv_history *history) {
    const char *who = "kv move";
    const std::string name = "kv move: ";
    MoveArgs g = {};
    if (int rc = make_kv_view(&ctx, who, &cache, &batch, 0, &g.kv)) return rc;
    if (int rc = take_history(ctx, who, history, &g.history)) return rc;
    if (moves.most < 0) return ctx.fail(AHIP_ERR_ARG, name + "the length of the lists is negative");
    for (int i = 0; i < 2; i++)
        if (moves.strides[i] < 0 || moves.count_strides[i] < 0 || moves.strides[i] > MOST_STRIDE || moves.count_strides[i] > MOST_STRIDE)
            return ctx.fail(AHIP_ERR_ARG, name + "a stride of the lists is out of range");
    if (batch.sequences == 0 || moves.most == 0) return AHIP_OK;
    if (batch.table_pages && !batch.page_table) return ctx.fail(AHIP_ERR_ARG, name + "null page table");
    if (cache.pages == 0 || !cache.keys || !cache.values) return ctx.fail(AHIP_ERR_ARG, name + "the cache has no pages");
    if (!moves.sources || !moves.targets || !moves.counts) return ctx.fail(AHIP_ERR_ARG, name + "null pointer");
    const int64_t size = cache.elem == AHIP_KV_BF16 ? 2 : 4, elements = 16 / size;
    const bool wide = cache.head_size % elements == 0 && cache.page_stride % elements == 0 && cache.head_stride % elements == 0 && cache.slot_stride % elements == 0 &&
                      reinterpret_cast<uintptr_t>(cache.keys) % 16 == 0 && reinterpret_cast<uintptr_t>(cache.values) % 16 == 0;
    const int64_t unit = wide ? elements : 1;
    g.row_units = (uint32_t)(cache.head_size / unit);
    if (g.row_units > (1u << 30)) return ctx.fail(AHIP_ERR_UNSUPPORTED, name + "heads of 2^30 channels and more are not supported");
    g.kv.page_stride /= unit, g.kv.head_stride /= unit, g.kv.slot_stride /= unit;
    g.sources = moves.sources, g.targets = moves.targets, g.counts = moves.counts;
    g.sequence_stride = moves.strides[0], g.head_stride = moves.strides[1], g.count_sequence = moves.count_strides[0], g.count_head = moves.count_strides[1];
    g.most = (uint32_t)moves.most;
    g.moves = std::max(1u, std::min(MOVE, MOVE * EACH / (2 * g.row_units)));
    const uint64_t chunks = moves.apart ? ((uint64_t)g.most + g.moves - 1) / g.moves : 1, blocks = (uint64_t)batch.sequences * (uint64_t)cache.kv_heads * chunks;
    if (blocks >= 8 * MOST_BLOCKS) return ctx.fail(AHIP_ERR_UNSUPPORTED, name + "more blocks than a grid holds");
    g.chunks = moves.apart ? (uint32_t)chunks : 0;
    if (wide) hipLaunchKernelGGL(move_slots<u32x4>, dim3((uint32_t)blocks), dim3(MOVE), 0, ctx.stream, g);
    else if (size == 4) hipLaunchKernelGGL(move_slots<uint32_t>, dim3((uint32_t)blocks), dim3(MOVE), 0, ctx.stream, g);
    else hipLaunchKernelGGL(move_slots<uint16_t>, dim3((uint32_t)blocks), dim3(MOVE), 0, ctx.stream, g);
    return ctx.check(hipGetLastError(), "kv move launch");
}

}  // namespace altius

// What happens to a cache that is full, or whose drafted tokens have been judged: which slots stay (ahip_kv_evict), and slots that go to other
// places of their sequence (ahip_kv_move).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv.h"
#include "kv_rank.h"

namespace altius {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct History {
    float *mass;
    int32_t *positions;
    int64_t page_stride, head_stride;
};

// ---------------------------------------------------------------- who stays
// A block for each sequence and head of keys, a wavefront for each run of places.  Masses become an order-preserving image of 32 bits; the smallest that
// stays is found among them (kv_rank.h), then the runs are counted and listed in order.
//   Up to 2048 places 256 threads hold 8 images each.  48 sequences of 1025 places, 8 heads: 7.9 us.
//   Up to 57344 places 1024 threads hold 56.  4 sequences of 20011 to 50000 places: 55 us, bound by the latency of one block's walks over the places, a CU
// each; 4 of 57344: 63 us.  Beyond, images wait in LDS as far as that goes, and what is behind is read anew, out of L2: 4 of 57345 113 us, of 65536 119, of 131072
// 246, in pages of 16 435.
constexpr uint32_t HELD = 28672, PAGES = 4096, SMALL = 256, SMALL_EACH = 8, LARGE = 1024, LARGE_EACH = 56;
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

// EACH: images that a thread holds; 0: they are in LDS and memory.
template <uint32_t THREADS, uint32_t EACH> __global__ __launch_bounds__(THREADS) void choose_evicted(EvictArgs g) {
    constexpr uint32_t WAVES = THREADS / 64, AHEAD = 8;  // loads of a thread that are on their way at once
    constexpr bool STARTS = EACH != AHEAD;               // where pages start is looked up once
    static_assert(EACH % AHEAD == 0, "whole sweeps");
    extern __shared__ uint32_t held[];
    __shared__ int64_t page_starts[STARTS ? PAGES : 1];
    __shared__ uint32_t per_wave[WAVES][4];
    __shared__ dev::RankLds<EACH == SMALL_EACH ? 1 : 8> rank_lds;  // 50000 masses in one row of bins: 62 us; in 8: 55; 1025 have none to wait for
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t s = blockIdx.x / g.kv.kv_heads, head = blockIdx.x - s * g.kv.kv_heads;
    const int32_t length = g.kv.lengths[s];
    int32_t *const count = g.counts + (int64_t)s * g.kv.kv_heads + head;
    const bool fits = length >= 0 && (uint64_t)length <= (uint64_t)g.kv.table_pages * g.kv.page_size && (uint32_t)length <= g.max_keys;
    if (!fits || (uint32_t)length <= g.budget) {
        if (tid == 0) {
            *count = 0;
            if (!fits) *g.kv.flag = 1;
            else if (head == 0 && g.lengths) g.lengths[s] = length;
        }
        return;
    }
    const uint32_t n = (uint32_t)length;
    if (tid == 0 && head == 0 && g.lengths) g.lengths[s] = (int32_t)g.budget;
    // This wavefront's places: at most 64 EACH.
    const uint32_t run = (n + THREADS - 1) / THREADS * 64, from = min(wave * run, n), to = min(from + run, n);

    const int32_t *const table = g.kv.table + (int64_t)s * g.kv.table_stride;
    bool outside = false;  // the flag is raised in the end: no branch in front of a load
    auto start_of = [&](uint32_t index) {
        const uint32_t page = (uint32_t)table[index];
        outside = outside || page >= g.kv.pages;
        return (int64_t)(page < g.kv.pages ? page : 0) * g.history.page_stride + (int64_t)head * g.history.head_stride;
    };
    if constexpr (STARTS) {
        for (uint32_t index = tid; index < PAGES && (uint64_t)index * g.kv.page_size < n; index += THREADS) page_starts[index] = start_of(index);
        __syncthreads();
    }
    // The next AHEAD x 64 places (behind the end the last one again), all loads on their way before the first is used: left to itself the compiler
    // waits for one at a time.
    auto ahead = [&](uint32_t base, auto load) {
        int64_t at[AHEAD];
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; u++) {
            const uint32_t place = min(base + 64 * u + lane, n - 1), index = g.kv.by_page_size.div(place);
            at[u] = (!STARTS || index >= PAGES ? start_of(index) : page_starts[index]) + (place - index * g.kv.page_size);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; u++) load(u, at[u]);
        __builtin_amdgcn_sched_barrier(0);
    };
    // The newest position, and what stays for its own: above every mass.
    int32_t newest = INT32_MIN, positions[AHEAD];
    uint32_t masses[AHEAD];
    if constexpr (EACH == AHEAD) {
        ahead(from, [&](uint32_t u, int64_t at) { positions[u] = g.history.positions[at], masses[u] = __float_as_uint(g.history.mass[at]); });
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; u++) newest = max(newest, positions[u]);
    } else {  // (56 positions a thread beside as many images leave no registers: 69 us instead of 62, with one row of bins)
        for (uint32_t base = from; base < to; base += 64 * AHEAD) {
            ahead(base, [&](uint32_t u, int64_t at) { positions[u] = g.history.positions[at]; });
#pragma unroll
            for (uint32_t u = 0; u < AHEAD; u++) newest = max(newest, positions[u]);
        }
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) newest = max(newest, __shfl_xor(newest, m));
    if (lane == 0) per_wave[wave][0] = (uint32_t)newest;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < WAVES; w++) newest = max(newest, (int32_t)per_wave[w][0]);
    // How far a position is behind the newest fits 32 bits without a sign, whatever both are.
    auto image_of = [&](int32_t position, uint32_t mass) {
        return position < g.first || (uint32_t)newest - (uint32_t)position < (uint32_t)g.recent ? KEPT : rank_image(__uint_as_float(mass));
    };
    // Images of the places from `base` on, 0 behind the end.
    auto take_images = [&](uint32_t base, uint32_t *v) {
        if constexpr (EACH != AHEAD) ahead(base, [&](uint32_t u, int64_t at) { positions[u] = g.history.positions[at], masses[u] = __float_as_uint(g.history.mass[at]); });
#pragma unroll
        for (uint32_t u = 0; u < AHEAD; u++) v[u] = base + 64 * u + lane < to ? image_of(positions[u], masses[u]) : 0;
    };
    uint32_t images[EACH ? EACH : 1];
    if constexpr (EACH != 0) {
#pragma unroll
        for (uint32_t i = 0; i < EACH; i += AHEAD) {
            if (EACH > AHEAD && from + 64 * i >= to) break;
            take_images(from + 64 * i, images + i);
        }
    }
    if constexpr (EACH == 0) {
        for (uint32_t base = from; base < min(to, g.held); base += 64 * AHEAD) {
            uint32_t v[AHEAD];
            take_images(base, v);
#pragma unroll
            for (uint32_t u = 0; u < AHEAD; u++)
                if (base + 64 * u < to && base + 64 * u < g.held) held[base + 64 * u + lane] = v[u];
        }
    }
    // what(base, v) for every 64 places of the run in order: this lane's image, 0 behind the end.
    auto each = [&](auto what) {
        if constexpr (EACH != 0) {
#pragma unroll
            for (uint32_t i = 0; i < EACH; i++) {
                if (from + 64 * i >= to) break;
                what(from + 64 * i, images[i]);
            }
        } else {
            for (uint32_t base = from; base < to; base += 64 * AHEAD) {
                uint32_t v[AHEAD];
                if (base + 64 * AHEAD <= g.held) {
#pragma unroll
                    for (uint32_t u = 0; u < AHEAD; u++) v[u] = held[base + 64 * u + lane];
                } else {
                    take_images(base, v);
                }
#pragma unroll
                for (uint32_t u = 0; u < AHEAD; u++)
                    if (base + 64 * u < to) what(base + 64 * u, v[u]);
            }
        }
    };

    // The smallest image that stays, and of how many of it.  The zeros behind the end are among the values: none is larger than any, and they have no place.
    const auto ranked = dev::rank_largest<uint32_t>(rank_lds, g.budget, [&](auto count_in) { each([&](uint32_t, uint32_t v) { count_in(v); }); });
    const uint32_t least = ranked.least, ties = ranked.exact ? n : ranked.ties;

    // What each run has above `least` and at it, below the budget and from it on: masks of 64 places.
    auto first_of = [](uint32_t base, uint32_t end) { return base + 64 <= end ? ~(uint64_t)0 : base >= end ? 0 : ((uint64_t)1 << (end - base)) - 1; };
    uint32_t counts[4] = {0, 0, 0, 0};
    each([&](uint32_t base, uint32_t v) {
        const uint64_t over = __ballot(v > least), at = __ballot(v == least) & first_of(base, to);
        if (base >= g.budget) {  // nearly all of a long sequence
            counts[2] += (uint32_t)__popcll(over), counts[3] += (uint32_t)__popcll(at);
        } else {
            const uint64_t low = first_of(base, g.budget);
            counts[0] += (uint32_t)__popcll(over & low), counts[1] += (uint32_t)__popcll(at & low);
            counts[2] += (uint32_t)__popcll(over & ~low), counts[3] += (uint32_t)__popcll(at & ~low);
        }
    });
    __syncthreads();
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < 4; i++) per_wave[wave][i] = counts[i];
    }
    __syncthreads();
    // What the runs in front leave: ties already kept, holes and movers already listed.
    uint32_t tied = 0, holes = 0, movers = 0;
    for (uint32_t w = 0; w < wave; w++) {
        const uint32_t start = min(w * run, n), end = min(start + run, n), lows = min(end, g.budget) - min(start, g.budget);
        const uint32_t *of = per_wave[w], left = ties - tied, stay_low = min(of[1], left), stay_high = min(of[3], left - stay_low);
        holes += lows - of[0] - stay_low;
        movers += of[2] + stay_high;
        tied += stay_low + stay_high;
    }
    const int64_t list = ((int64_t)s * g.kv.kv_heads + head) * g.most;
    const uint64_t before = ((uint64_t)1 << lane) - 1;
    auto put = [&](int32_t *to_list, uint64_t mask, uint32_t listed, uint32_t base) {
        const uint32_t at = listed + (uint32_t)__popcll(mask & before);
        if ((mask >> lane & 1) && at < g.most) to_list[list + at] = (int32_t)(base + lane);
    };
    each([&](uint32_t base, uint32_t v) {
        uint64_t stay = __ballot(v > least);
        const uint64_t at = __ballot(v == least) & first_of(base, to);
        if (at) {
            stay |= __ballot((at >> lane & 1) && tied + (uint32_t)__popcll(at & before) < ties);
            tied += (uint32_t)__popcll(at);
        }
        uint64_t mover = stay;
        if (base < g.budget) {
            const uint64_t low = first_of(base, g.budget), hole = low & first_of(base, to) & ~stay;
            mover &= ~low;
            if (hole) put(g.targets, hole, holes, base), holes += (uint32_t)__popcll(hole);
        }
        if (mover) put(g.sources, mover, movers, base), movers += (uint32_t)__popcll(mover);
    });
    if (tid == THREADS - 64) *count = (int32_t)min(movers, g.most);  // the last run's: all of them
    if (outside) *g.kv.flag = 1;
}

// Where the new lengths go into the place of the old ones: once all blocks have read those.
__global__ __launch_bounds__(256) void shorten(EvictArgs g, int32_t *lengths) {
    const uint32_t s = blockIdx.x * 256 + threadIdx.x;
    if (s >= g.kv.sequences) return;
    const int32_t length = lengths[s];
    if (length >= 0 && (uint64_t)length <= (uint64_t)g.kv.table_pages * g.kv.page_size && (uint32_t)length <= g.max_keys && (uint32_t)length > g.budget) lengths[s] = (int32_t)g.budget;
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
    const bool in_place = eviction.lengths == batch.lengths;
    const int64_t apart = reinterpret_cast<intptr_t>(eviction.lengths) - reinterpret_cast<intptr_t>(batch.lengths), all = (int64_t)sizeof(int32_t) * batch.sequences;
    if (!in_place && apart < all && apart > -all) return ctx.fail(AHIP_ERR_ARG, name + "the new lengths overlap the batch's and are not in their place");
    g.sources = eviction.sources, g.targets = eviction.targets, g.counts = eviction.counts, g.lengths = in_place ? nullptr : eviction.lengths;
    if (max_keys <= SMALL * SMALL_EACH) {
        hipLaunchKernelGGL((choose_evicted<SMALL, SMALL_EACH>), dim3((uint32_t)blocks), dim3(SMALL), 0, ctx.stream, g);
    } else if (max_keys <= LARGE * LARGE_EACH) {
        hipLaunchKernelGGL((choose_evicted<LARGE, LARGE_EACH>), dim3((uint32_t)blocks), dim3(LARGE), 0, ctx.stream, g);
    } else {
        g.held = HELD;
        hipLaunchKernelGGL((choose_evicted<LARGE, 0>), dim3((uint32_t)blocks), dim3(LARGE), HELD * sizeof(uint32_t), ctx.stream, g);
    }
    if (int rc = ctx.check(hipGetLastError(), "kv evict launch")) return rc;
    if (!in_place) return AHIP_OK;
    hipLaunchKernelGGL(shorten, dim3(((uint32_t)batch.sequences + 255) / 256), dim3(256), 0, ctx.stream, g, eviction.lengths);
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

// Rotary positions of heads, the norm of each head in front of them, and the same on the way into a paged cache.
//
// A row is one head of one token: d adjacent channels.  Its norm is y = x gamma / sqrt(mean(x^2) + eps); pair (a, b) of its
// first `dim` channels becomes m (a cos t - b sin t, a sin t + b cos t), t = position * frequency.  8 d bytes a row for
// 6 operations a pair: bound by memory, and by launch and latency where there are few rows.
//
// t reaches 10^5 and more, where fp32 holds it to 0.01 only: t / (pi / 2) is rounded to a whole number of quarter turns in 64
// bits, and sine and cosine of the rest (at most pi / 4) are polynomials in 32.  That is a few times the work of the rotation
// itself, so a lane keeps the angles of its pairs and takes several heads of a token with them.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "kv.h"

namespace altius {

namespace {

using dev::FastDiv;
using dev::make_fastdiv;

constexpr int BLOCK = 256;

struct RowsOf {  // rows at base + token * token_stride + head * head_stride (+ batch * batch_stride)
    const float *src;
    float *dst;  // null: into the cache
    const float *gamma;
    int64_t src_batch, src_token, src_head, dst_batch, dst_token, dst_head;
};

struct RotateArgs {
    RowsOf rows[3];       // queries (or the only tensor), keys, values
    uint32_t ends[3];     // heads[0], heads[0] + heads[1], ...: which of them a head index belongs to
    uint32_t heads;       // ends[2]
    uint32_t tokens, batch;
    uint32_t d, dim;      // channels of a row, of which the first dim turn
    uint32_t interleaved;
    // Threads are lanes of rows, `threads` of them; rows of one lane group lie `groups` heads apart.  Which comes next after the lane:
    // the group of heads (then the token), or the token (then the group).
    uint32_t threads, token_next;
    FastDiv lanes, groups, by_tokens;
    const double *frequencies;
    float magnitude, epsilon;
    const void *positions;
    int32_t position_size;
    int64_t position_stride, first_position;
    dev::KvView kv;
};

// sin and cos of position * frequency.  The Taylor polynomials end where the next term is below 2^-25 of the result for
// |r| <= pi / 4: r^11 / 11! = 1.8e-9, r^12 / 12! = 1.1e-10.
__device__ __forceinline__ void turn(double position, double frequency, float magnitude, float &cos_out, float &sin_out) {
    const double quarters = position * frequency * 0.63661977236758134308;  // 2 / pi
    // A sum beyond 2^52 is whole, its lowest bits are the quarter turns.
    const double shifted = quarters + 6755399441055744.0;  // 1.5 x 2^52
    const float r = (float)((quarters - (shifted - 6755399441055744.0)) * 1.57079632679489661923);
    const uint32_t quadrant = (uint32_t)__double2loint(shifted);
    const float r2 = r * r;
    float s = __builtin_fmaf(r2, 2.75573192e-6f, -1.98412698e-4f);
    s = __builtin_fmaf(s, r2, 8.33333333e-3f);
    s = __builtin_fmaf(s, r2, -0.166666667f);
    s = __builtin_fmaf(s * r2, r, r);
    float c = __builtin_fmaf(r2, -2.75573192e-7f, 2.48015873e-5f);
    c = __builtin_fmaf(c, r2, -1.38888889e-3f);
    c = __builtin_fmaf(c, r2, 4.16666667e-2f);
    c = __builtin_fmaf(c, r2, -0.5f);
    c = __builtin_fmaf(c, r2, 1.0f);
    const float cc = quadrant & 1u ? s : c, ss = quadrant & 1u ? c : s;
    cos_out = magnitude * (((quadrant + 1u) & 2u) ? -cc : cc);
    sin_out = magnitude * ((quadrant & 2u) ? -ss : ss);
}

__device__ __forceinline__ double position_of(const RotateArgs &g, uint32_t b, uint32_t token, int64_t otherwise) {
    if (!g.positions) return (double)otherwise;
    const int64_t at = (int64_t)b * g.position_stride + token;
    return g.position_size == 8 ? (double)static_cast<const int64_t *>(g.positions)[at] : (double)static_cast<const int32_t *>(g.positions)[at];
}

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <bool BF16> __device__ __forceinline__ void cache_store4(void *base, int64_t at, const f32x4 &v) {
    // Round to nearest even: the one rounding to fewer bits here, asked for by the cache's type.
    if (BF16) *reinterpret_cast<bf16x4 *>(static_cast<uint16_t *>(base) + at) = __builtin_convertvector(v, bf16x4);
    else *reinterpret_cast<f32x4 *>(static_cast<float *>(base) + at) = v;
}
template <bool BF16> __device__ __forceinline__ void cache_store1(void *base, int64_t at, float v) {
    if (BF16) static_cast<__bf16 *>(base)[at] = (__bf16)v;
    else static_cast<float *>(base)[at] = v;
}

// Where a token's row goes in the cache (elements), and whether it goes anywhere.  For whole wavefronts.
struct Slot {
    int64_t at;
    bool live;
};
__device__ __forceinline__ Slot slot_of(const dev::KvView &kv, uint32_t token, int64_t &place) {
    Slot slot = {0, false};
    place = 0;
    dev::KvSequence q = {};
    const uint32_t s = dev::kv_sequence_of(kv, token, q);
    if (s >= kv.sequences || (s == 0 && (int64_t)token < q.start)) return slot;  // padding behind the last sequence or in front of the first
    const int64_t p = (int64_t)q.length - q.n + ((int64_t)token - q.start);
    if (q.n == 0 || (int64_t)token < q.start || (int64_t)token >= (int64_t)q.start + q.n || p < 0) {  // starts out of order, or shorter than its rows
        *kv.flag = 1;
        return slot;
    }
    place = p;
    const uint32_t index = kv.by_page_size.div((uint32_t)p);
    const int32_t page = kv.page_of(s, index, -1);
    if (page < 0) return slot;
    slot.at = (int64_t)page * kv.page_stride + (int64_t)((uint32_t)p - index * kv.page_size) * kv.slot_stride;
    slot.live = true;
    return slot;
}

// One of three arguments by selection: indexing them would read them from memory in front of every address.
#define ALTIUS_ROWS_FIELD(which, field) ((which) == 0 ? g.rows[0].field : (which) == 1 ? g.rows[1].field : g.rows[2].field)

// Eight channels a lane, in two float4 A and B: the two halves' channels (4 u, dim / 2 + 4 u) of the part that turns where
// halves turn together, neighbours (8 u, 8 u + 4) otherwise.  N heads of its token per lane, all loads in front of the first use.
// Rows that are normed have a power of two of lanes, which add up their squares; others exactly as many as they need.
//   Bound by memory: 4096 tokens x 16 heads of 128 channels, normed, 67 MB in 14.0 us, 4.8 TB/s, where a copy of 1 GiB moves 5.2;
// 9 prompts into a bf16 cache, 117 MB in 30 us, 3.9 TB/s, whose rows of 256 bytes are written out of order; interleaved pairs of half
// of 80 channels, 31 MB in 9.0 us, 3.4 TB/s, by waits: each frequency is loaded behind a condition and waited for by itself, behind the
// position's wait, five trips to memory in a row.  One token of 12 heads: 3.2 us, a launch.
template <int N, bool CACHE, bool BF16>
__global__ __launch_bounds__(BLOCK) void rotate_rows_vec4(RotateArgs g) {
    const uint32_t mine = blockIdx.x * BLOCK + threadIdx.x, thread = min(mine, g.threads - 1);
    const uint32_t of = g.lanes.div(thread), lane = thread - of * g.lanes.d;
    uint32_t group, item;
    if (g.token_next) {  // of = (batch * groups + group) * tokens + token
        const uint32_t outer = g.by_tokens.div(of), b = g.groups.div(outer);
        group = outer - b * g.groups.d;
        item = b * g.tokens + (of - outer * g.tokens);
    } else {
        item = g.groups.div(of);
        group = of - item * g.groups.d;
    }
    const uint32_t b = CACHE ? 0 : g.by_tokens.div(item), token = CACHE ? item : item - b * g.tokens;

    const uint32_t half = g.dim / 2;
    const bool split = !g.interleaved && 4 * lane < half;  // this lane's A and B are the halves of a pair
    const uint32_t offset = g.interleaved ? 8 * lane : split ? 4 * lane : g.dim + 8 * (lane - half / 4);
    const uint32_t a_at = offset, b_at = split ? half + offset : offset + 4;
    const bool has_a = a_at < g.d, has_b = b_at < g.d;

    f32x4 a[N], c[N];
    uint32_t which[N], head[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        uint32_t h = group + (uint32_t)i * g.groups.d;
        const bool live = h < g.heads && mine < g.threads;
        if (!live) h = 0;
        which[i] = CACHE ? (h >= g.ends[0]) + (h >= g.ends[1]) : 0;
        head[i] = h - (which[i] ? g.ends[which[i] - 1] : 0);
        const float *src = ALTIUS_ROWS_FIELD(which[i], src) + (int64_t)b * g.rows[0].src_batch + (int64_t)token * ALTIUS_ROWS_FIELD(which[i], src_token) +
                           (int64_t)head[i] * ALTIUS_ROWS_FIELD(which[i], src_head);
        a[i] = c[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (live && has_a) a[i] = *reinterpret_cast<const f32x4 *>(src + a_at);
        if (live && has_b) c[i] = *reinterpret_cast<const f32x4 *>(src + b_at);
        if (!live) which[i] = 3;
    }

    int64_t place = (int64_t)g.first_position + token;
    Slot slot = {0, true};
    if (CACHE) {
        slot = slot_of(g.kv, token, place);
        if (!slot.live) return;
    }

    // The angles: of pairs (4 u + j) where halves turn together, of pairs (4 u + j) of neighbours in A and B alike.
    float co[4], si[4];
    const bool turns = offset < g.dim;
    if (turns) {
        const double position = position_of(g, b, token, place);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t pair = 4 * lane + j;
            co[j] = 1.0f, si[j] = 0.0f;
            if (pair < half) turn(position, g.frequencies[pair], g.magnitude, co[j], si[j]);
        }
    }

#pragma unroll
    for (int i = 0; i < N; i++) {
        if (which[i] == 3) continue;  // alike in all lanes of a row
        const float *gamma = ALTIUS_ROWS_FIELD(which[i], gamma);
        if (gamma) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) sum = __builtin_fmaf(a[i][j], a[i][j], sum);
#pragma unroll
            for (int j = 0; j < 4; j++) sum = __builtin_fmaf(c[i][j], c[i][j], sum);
            for (uint32_t m = 1; m < g.lanes.d; m <<= 1) sum += __shfl_xor(sum, m);
            const float scale = 1.0f / sqrtf(sum / (float)g.d + g.epsilon);
            const f32x4 ones = {1.0f, 1.0f, 1.0f, 1.0f};
            const f32x4 ga = has_a ? *reinterpret_cast<const f32x4 *>(gamma + a_at) : ones, gb = has_b ? *reinterpret_cast<const f32x4 *>(gamma + b_at) : ones;
            a[i] = a[i] * scale * ga;
            c[i] = c[i] * scale * gb;
        }
        if (turns && which[i] != 2) {
            if (split) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float x = a[i][j], y = c[i][j];
                    a[i][j] = x * co[j] - y * si[j];
                    c[i][j] = x * si[j] + y * co[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float x = a[i][2 * j], y = a[i][2 * j + 1], z = c[i][2 * j], w = c[i][2 * j + 1];
                    a[i][2 * j] = x * co[j] - y * si[j];
                    a[i][2 * j + 1] = x * si[j] + y * co[j];
                    if (offset + 4 < g.dim) {
                        c[i][2 * j] = z * co[2 + j] - w * si[2 + j];
                        c[i][2 * j + 1] = z * si[2 + j] + w * co[2 + j];
                    }
                }
            }
        }
        if (CACHE && which[i] != 0) {
            void *base = which[i] == 1 ? g.kv.keys : g.kv.values;
            const int64_t at = slot.at + (int64_t)head[i] * g.kv.head_stride;
            if (has_a) cache_store4<BF16>(base, at + a_at, a[i]);
            if (has_b) cache_store4<BF16>(base, at + b_at, c[i]);
        } else {
            const RowsOf &r = g.rows[0];
            float *dst = r.dst + (int64_t)b * r.dst_batch + (int64_t)token * r.dst_token + (int64_t)head[i] * r.dst_head;
            if (has_a) *reinterpret_cast<f32x4 *>(dst + a_at) = a[i];
            if (has_b) *reinterpret_cast<f32x4 *>(dst + b_at) = c[i];
        }
    }
}

// Any sizes, strides and alignment: a wavefront per row, single channels, the angles anew for each row.
template <bool CACHE, bool BF16>
__global__ __launch_bounds__(BLOCK) void rotate_rows_any(RotateArgs g) {
    const uint32_t lane = threadIdx.x & 63u, item = blockIdx.x;
    const uint32_t h = blockIdx.y * (BLOCK / 64) + (threadIdx.x >> 6);
    if (h >= g.heads) return;
    const uint32_t b = CACHE ? 0 : item / g.tokens, token = CACHE ? item : item - b * g.tokens;
    int64_t place = (int64_t)g.first_position + token;
    Slot slot = {0, true};
    if (CACHE) {
        slot = slot_of(g.kv, token, place);
        if (!slot.live) return;
    }
    const uint32_t which = CACHE ? (h >= g.ends[0]) + (h >= g.ends[1]) : 0, head = h - (which ? g.ends[which - 1] : 0);
    const RowsOf &r = g.rows[which];
    const float *src = r.src + (int64_t)b * r.src_batch + (int64_t)token * r.src_token + (int64_t)head * r.src_head;
    const double position = position_of(g, b, token, place);
    float scale = 1.0f;
    if (r.gamma) {
        float sum = 0.0f;
        for (uint32_t i = lane; i < g.d; i += 64) sum = __builtin_fmaf(src[i], src[i], sum);
        sum = dev::wave_reduce<dev::SumOp>(sum);
        scale = 1.0f / sqrtf(sum / (float)g.d + g.epsilon);
    }
    auto value = [&](uint32_t i) { return r.gamma ? src[i] * scale * r.gamma[i] : src[i]; };
    auto put = [&](uint32_t i, float v) {
        if (CACHE && which != 0) cache_store1<BF16>(which == 1 ? g.kv.keys : g.kv.values, slot.at + (int64_t)head * g.kv.head_stride + i, v);
        else r.dst[(int64_t)b * r.dst_batch + (int64_t)token * r.dst_token + (int64_t)head * r.dst_head + i] = v;
    };
    const uint32_t dim = which == 2 ? 0 : g.dim, half = dim / 2;
    for (uint32_t p = lane; p < half; p += 64) {
        const uint32_t i = g.interleaved ? 2 * p : p, j = g.interleaved ? 2 * p + 1 : half + p;
        float co, si;
        turn(position, g.frequencies[p], g.magnitude, co, si);
        const float x = value(i), y = value(j);
        put(i, x * co - y * si);
        put(j, x * si + y * co);
    }
    for (uint32_t i = dim + lane; i < g.d; i += 64) put(i, value(i));
}

uint32_t log2_up(size_t n) {
    uint32_t l = 0;
    while (((size_t)1 << l) < n) l++;
    return l;
}

bool quads(int64_t stride) { return stride % 4 == 0; }
bool aligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Work (lanes x rows) from which a lane takes two heads and computes the angles once for both: 9 prompts of 100 to 1024 tokens
// into a bf16 cache (117 MB) take 31.7 us, 33.7 us with one head a lane; 64 single tokens (3 MB, below it) 4.7 us,
// with two heads 5.5 us.
constexpr uint64_t MANY = (uint64_t)1 << 18;

template <bool CACHE, bool BF16> int launch_rotate(DeviceCtx &ctx, const RotateArgs &g, const char *what) {
    // Float4s wherever rows and their parts allow it; a row of up to 512 channels is one lane group of a wavefront.
    bool vec = g.d % 4 == 0 && g.d <= 512 && g.dim % (g.interleaved ? 4 : 8) == 0;
    for (int i = 0; i < 3; i++) {
        const RowsOf &r = g.rows[i];
        if (!r.src) continue;
        vec = vec && aligned(r.src, 16) && (!r.gamma || aligned(r.gamma, 16)) && quads(r.src_batch) && quads(r.src_token) && quads(r.src_head);
        if (r.dst) vec = vec && aligned(r.dst, 16) && quads(r.dst_batch) && quads(r.dst_token) && quads(r.dst_head);
    }
    if (CACHE)
        vec = vec && aligned(g.kv.keys, BF16 ? 8 : 16) && aligned(g.kv.values, BF16 ? 8 : 16) && quads(g.kv.page_stride) && quads(g.kv.head_stride) &&
              quads(g.kv.slot_stride);
    const uint64_t items = (uint64_t)g.tokens * g.batch;
    const uint32_t units = g.interleaved ? (g.d + 7) / 8 : g.dim / 8 + (g.d - g.dim + 7) / 8;
    const uint32_t lanes = g.rows[0].gamma || g.rows[1].gamma ? 1u << log2_up(units) : units;
    const uint64_t work = items * g.heads * lanes;
    // Two heads a lane where there are threads enough for the whole part all the same.
    const uint32_t n = work >= MANY ? 2 : 1, groups = (g.heads + n - 1) / n;
    const uint64_t threads = items * groups * lanes;
    vec = vec && threads < ((uint64_t)1 << 31);
    if (!vec) {
        hipLaunchKernelGGL((rotate_rows_any<CACHE, BF16>), dim3((uint32_t)items, (g.heads + BLOCK / 64 - 1) / (BLOCK / 64)), dim3(BLOCK), 0, ctx.stream, g);
        return ctx.check(hipGetLastError(), what);
    }
    RotateArgs a = g;
    a.threads = (uint32_t)threads;
    // Rows next to each other in memory are next to each other in a block.
    a.token_next = !CACHE && g.rows[0].src_token < g.rows[0].src_head;
    a.lanes = make_fastdiv(lanes), a.groups = make_fastdiv(groups), a.by_tokens = make_fastdiv(g.tokens);
    const dim3 grid((a.threads + BLOCK - 1) / BLOCK);
    if (n == 2) hipLaunchKernelGGL((rotate_rows_vec4<2, CACHE, BF16>), grid, dim3(BLOCK), 0, ctx.stream, a);
    else hipLaunchKernelGGL((rotate_rows_vec4<1, CACHE, BF16>), grid, dim3(BLOCK), 0, ctx.stream, a);
    return ctx.check(hipGetLastError(), what);
}

int take_rotary(DeviceCtx &ctx, const char *who, const ahip_rotary *rotary, size_t head_size, RotateArgs *g) {
    g->dim = 0, g->interleaved = 0, g->frequencies = nullptr, g->magnitude = 1.0f;
    if (!rotary) return AHIP_OK;
    const std::string name(who);
    if (rotary->layout != AHIP_ROTARY_HALVES && rotary->layout != AHIP_ROTARY_INTERLEAVED) return ctx.fail(AHIP_ERR_ARG, name + ": unknown rotary layout");
    if (rotary->dim < 0 || rotary->dim % 2 || (size_t)rotary->dim > head_size)
        return ctx.fail(AHIP_ERR_SHAPE, name + ": " + std::to_string(rotary->dim) + " channels cannot turn in a head of " + std::to_string(head_size));
    if (rotary->dim && !rotary->frequencies) return ctx.fail(AHIP_ERR_ARG, name + ": null frequencies");
    if (!aligned(rotary->frequencies, 8)) return ctx.fail(AHIP_ERR_ARG, name + ": frequencies are not on an 8-byte boundary");
    g->dim = (uint32_t)rotary->dim;
    g->interleaved = rotary->layout == AHIP_ROTARY_INTERLEAVED;
    g->frequencies = rotary->frequencies;
    g->magnitude = rotary->magnitude;
    return AHIP_OK;
}

int take_positions(DeviceCtx &ctx, const char *who, const void *positions, int size, RotateArgs *g) {
    if (positions && size != 4 && size != 8) return ctx.fail(AHIP_ERR_ARG, std::string(who) + ": positions must be i32 or i64");
    if (positions && !aligned(positions, (size_t)size)) return ctx.fail(AHIP_ERR_ARG, std::string(who) + ": positions are not on a boundary of their size");
    g->positions = positions;
    g->position_size = size;
    return AHIP_OK;
}

// Extents and strides that 64-bit element offsets hold with room to spare.
constexpr size_t MOST = (size_t)1 << 48;

}  // namespace

int launch_rotary_heads(DeviceCtx &ctx, const ahip_head_rows &rows, const ahip_rotary *rotary) {
    const char *who = "rotary heads";
    RotateArgs g = {};
    if (int rc = take_rotary(ctx, who, rotary, rows.head_size, &g)) return rc;
    if (int rc = take_positions(ctx, who, rows.positions, rows.position_size, &g)) return rc;
    for (int i = 0; i < 3; i++)
        if (rows.x_strides[i] > MOST || rows.out_strides[i] > MOST) return ctx.fail(AHIP_ERR_ARG, "rotary heads: a stride is out of range");
    if (rows.position_stride > MOST) return ctx.fail(AHIP_ERR_ARG, "rotary heads: a stride is out of range");
    if (rows.batch == 0 || rows.tokens == 0 || rows.heads == 0 || rows.head_size == 0) return AHIP_OK;
    if (!rows.out || !rows.x) return ctx.fail(AHIP_ERR_ARG, "rotary heads: null pointer");
    constexpr size_t INDEX = (size_t)1 << 31;
    if (rows.batch >= INDEX || rows.tokens >= INDEX || rows.batch * rows.tokens >= INDEX / 256 || rows.heads > 65535 || rows.head_size >= INDEX)
        return ctx.fail(AHIP_ERR_UNSUPPORTED, "rotary heads: 2^23 tokens, 65535 heads or 2^31 channels and more are not supported");
    if (rows.out == rows.x && !std::equal(rows.out_strides, rows.out_strides + 3, rows.x_strides))
        return ctx.fail(AHIP_ERR_ARG, "rotary heads: out is x with other strides");
    g.rows[0] = {rows.x, rows.out, rows.gamma, (int64_t)rows.x_strides[0], (int64_t)rows.x_strides[1], (int64_t)rows.x_strides[2],
                 (int64_t)rows.out_strides[0], (int64_t)rows.out_strides[1], (int64_t)rows.out_strides[2]};
    g.ends[0] = g.ends[1] = g.ends[2] = g.heads = (uint32_t)rows.heads;
    g.tokens = (uint32_t)rows.tokens, g.batch = (uint32_t)rows.batch, g.d = (uint32_t)rows.head_size;
    g.epsilon = rows.epsilon;
    g.position_stride = (int64_t)rows.position_stride, g.first_position = rows.first_position;
    return launch_rotate<false, false>(ctx, g, "rotary heads launch");
}

int launch_kv_append(DeviceCtx &ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_tokens &tokens, const ahip_rotary *rotary) {
    const char *who = "kv append";
    RotateArgs g = {};
    if (int rc = make_kv_view(&ctx, who, &cache, &batch, tokens.tokens, &g.kv)) return rc;
    if (int rc = take_rotary(ctx, who, rotary, (size_t)cache.head_size, &g)) return rc;
    if (int rc = take_positions(ctx, who, tokens.positions, tokens.position_size, &g)) return rc;
    if (tokens.q_heads < 0 || tokens.q_heads > 65535 - 2 * cache.kv_heads) return ctx.fail(AHIP_ERR_ARG, "kv append: the number of query heads is out of range");
    for (int i = 0; i < 2; i++)
        if (std::max(std::max(tokens.q_strides[i], tokens.k_strides[i]), std::max(tokens.v_strides[i], tokens.q_out_strides[i])) > MOST)
            return ctx.fail(AHIP_ERR_ARG, "kv append: a stride is out of range");
    if (tokens.tokens == 0 || batch.sequences == 0) return AHIP_OK;
    if (int rc = require_kv_arrays(ctx, who, cache, batch)) return rc;
    if (!tokens.k || !tokens.v || (tokens.q_heads && (!tokens.q || !tokens.q_out))) return ctx.fail(AHIP_ERR_ARG, "kv append: null pointer");
    if (tokens.q_heads && tokens.q_out == tokens.q && !std::equal(tokens.q_strides, tokens.q_strides + 2, tokens.q_out_strides))
        return ctx.fail(AHIP_ERR_ARG, "kv append: q_out is q with other strides");
    if (tokens.q_heads)
        g.rows[0] = {tokens.q, tokens.q_out, tokens.q_gamma, 0, (int64_t)tokens.q_strides[0], (int64_t)tokens.q_strides[1],
                     0, (int64_t)tokens.q_out_strides[0], (int64_t)tokens.q_out_strides[1]};
    g.rows[1] = {tokens.k, nullptr, tokens.k_gamma, 0, (int64_t)tokens.k_strides[0], (int64_t)tokens.k_strides[1], 0, 0, 0};
    g.rows[2] = {tokens.v, nullptr, nullptr, 0, (int64_t)tokens.v_strides[0], (int64_t)tokens.v_strides[1], 0, 0, 0};
    g.ends[0] = (uint32_t)tokens.q_heads;
    g.ends[1] = g.ends[0] + (uint32_t)cache.kv_heads;
    g.ends[2] = g.heads = g.ends[1] + (uint32_t)cache.kv_heads;
    g.tokens = (uint32_t)tokens.tokens, g.batch = 1, g.d = (uint32_t)cache.head_size;
    g.epsilon = tokens.epsilon;
    return cache.elem == AHIP_KV_BF16 ? launch_rotate<true, true>(ctx, g, "kv append launch") : launch_rotate<true, false>(ctx, g, "kv append launch");
}

int kv_fail(DeviceCtx *ctx, int code, const std::string &msg) {
    if (ctx) return ctx->fail(code, msg);
    set_global_error(msg);
    return code;
}

int make_kv_view(DeviceCtx *ctx, const char *who, const ahip_kv_cache *cache, const ahip_kv_batch *batch, size_t tokens, dev::KvView *view) {
    const std::string name(who);
    if (!cache || !batch) return kv_fail(ctx, AHIP_ERR_ARG, name + ": null cache or batch");
    if (cache->elem != AHIP_KV_F32 && cache->elem != AHIP_KV_BF16) return kv_fail(ctx, AHIP_ERR_ARG, name + ": unknown type of cache");
    if (cache->kv_heads <= 0 || cache->kv_heads > 32767 || cache->head_size <= 0 || cache->page_size <= 0)
        return kv_fail(ctx, AHIP_ERR_ARG, name + ": a cache has at least one head, channel and slot per page, and at most 32767 heads");
    if (cache->pages < 0 || cache->pages > INT32_MAX) return kv_fail(ctx, AHIP_ERR_ARG, name + ": the number of pages is out of range");
    const int64_t most = (int64_t)1 << 48;
    if (cache->page_stride < 0 || cache->head_stride < 0 || cache->slot_stride < 0 || cache->page_stride > most || cache->head_stride > most ||
        cache->slot_stride > INT32_MAX)
        return kv_fail(ctx, AHIP_ERR_ARG, name + ": a stride of the cache is out of range");
    if (batch->sequences < 0 || batch->table_pages < 0 || batch->table_stride < 0 || batch->table_stride > most)
        return kv_fail(ctx, AHIP_ERR_ARG, name + ": a size of the batch is out of range");
    // Kernels look some tiles ahead of a sequence's end.
    if ((int64_t)batch->table_pages * cache->page_size > INT32_MAX - (1 << 16))
        return kv_fail(ctx, AHIP_ERR_UNSUPPORTED, name + ": sequences of 2^31 - 2^16 tokens and more are not supported");
    if (tokens >= ((size_t)1 << 23)) return kv_fail(ctx, AHIP_ERR_UNSUPPORTED, name + ": 2^23 tokens and more in a call are not supported");
    view->keys = cache->keys, view->values = cache->values;
    view->page_stride = cache->page_stride, view->head_stride = cache->head_stride, view->slot_stride = cache->slot_stride;
    view->pages = (uint32_t)cache->pages, view->page_size = (uint32_t)cache->page_size, view->kv_heads = (uint32_t)cache->kv_heads;
    view->sequences = (uint32_t)batch->sequences, view->tokens = (uint32_t)tokens;
    view->by_page_size = dev::make_fastdiv((uint32_t)cache->page_size);
    view->table = batch->page_table, view->starts = batch->query_starts, view->lengths = batch->lengths;
    view->table_stride = batch->table_stride;
    view->table_pages = (uint32_t)batch->table_pages;
    view->flag = ctx ? ctx->flags + dev::KV_FLAG : nullptr;
    return AHIP_OK;
}

int require_kv_arrays(DeviceCtx &ctx, const char *who, const ahip_kv_cache &cache, const ahip_kv_batch &batch) {
    const std::string name(who);
    if (!batch.query_starts || !batch.lengths || (batch.table_pages && !batch.page_table)) return ctx.fail(AHIP_ERR_ARG, name + ": null batch array");
    if (cache.pages == 0 || !cache.keys || !cache.values) return ctx.fail(AHIP_ERR_ARG, name + ": the cache has no pages");
    return AHIP_OK;
}

int rotary_frequencies(double *frequencies, int dim, double base, int scaling, double factor, double length, double slow_turns, double fast_turns) {
    const char *who = "rotary frequencies: ";
    if (dim < 0 || dim % 2) return kv_fail(nullptr, AHIP_ERR_ARG, std::string(who) + "the number of channels is odd or negative");
    if (dim && !frequencies) return kv_fail(nullptr, AHIP_ERR_ARG, std::string(who) + "null output");
    if (!(base > 0) || !std::isfinite(base)) return kv_fail(nullptr, AHIP_ERR_ARG, std::string(who) + "the base must be positive");
    if (scaling < AHIP_ROTARY_PLAIN || scaling > AHIP_ROTARY_TURNS) return kv_fail(nullptr, AHIP_ERR_ARG, std::string(who) + "unknown scaling");
    if (scaling != AHIP_ROTARY_PLAIN && (!(factor > 0) || !std::isfinite(factor))) return kv_fail(nullptr, AHIP_ERR_ARG, std::string(who) + "the factor must be positive");
    if (scaling == AHIP_ROTARY_BASE && dim == 2) return kv_fail(nullptr, AHIP_ERR_ARG, std::string(who) + "one pair alone has no slowest one to stretch to");
    if (scaling == AHIP_ROTARY_TURNS && (!(length > 0) || !std::isfinite(length) || !(slow_turns < fast_turns) || !std::isfinite(slow_turns) || !std::isfinite(fast_turns)))
        return kv_fail(nullptr, AHIP_ERR_ARG, std::string(who) + "turns need a length, and fewer slow turns than fast ones");
    if (scaling == AHIP_ROTARY_BASE) base *= std::pow(factor, (double)dim / (dim - 2));
    if (!(base > 0) || !std::isfinite(base)) return kv_fail(nullptr, AHIP_ERR_ARG, std::string(who) + "the stretched base is out of range");
    for (int i = 0; i < dim / 2; i++) {
        double f = std::pow(base, -2.0 * i / dim);
        if (scaling == AHIP_ROTARY_LINEAR) f /= factor;
        if (scaling == AHIP_ROTARY_TURNS) {
            const double turns = length * f / 6.283185307179586476925, keep = std::min(1.0, std::max(0.0, (turns - slow_turns) / (fast_turns - slow_turns)));
            f *= keep + (1.0 - keep) / factor;
        }
        frequencies[i] = f;
    }
    return AHIP_OK;
}

}  // namespace altius

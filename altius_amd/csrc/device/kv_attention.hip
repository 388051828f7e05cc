// Attention over a paged cache, the host's part: what is refused, how the work is cut, which kernel of kv_attend.h a call takes.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "kv_attend.h"

namespace altius {

namespace attend {

namespace {
bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
}  // namespace

Plan plan_of(const DeviceCtx *ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_attend &attend, bool tree) {
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
        // Trees see nearly all of their sequence, whatever its length: 16 of 48 tokens behind 8000 (8 heads of keys of 128 channels, bf16) 482 us whole, 347 cut, of 16 to
        // 48 behind 300 to 8000 in fp32 617 and 519.
        if (tiled) share(p.many, rows, TILE_ROWS, many_tiles, many_tiles < (tree ? 4 * many_at_once : many_at_once / 2), many_at_once, 128);
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

int begin_attend(DeviceCtx &ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_attend &attend, bool tree, AttendArgs *args) {
    AttendArgs &g = *args;
    if (int rc = check_attend(&ctx, &cache, &batch, &attend, &g.kv)) return rc;
    if (attend.tokens == 0 || batch.sequences == 0) return AHIP_OK;
    if (int rc = require_kv_arrays(ctx, "kv attention", cache, batch)) return rc;
    if (!attend.q || !attend.out) return ctx.fail(AHIP_ERR_ARG, "kv attention: null pointer");
    if (attend.out == attend.q) return ctx.fail(AHIP_ERR_ARG, "kv attention: out is q");
    const Plan plan = plan_of(&ctx, cache, batch, attend, tree);
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
    return AHIP_OK;
}

}  // namespace attend

int kv_attention_workspace(DeviceCtx *ctx, const ahip_kv_cache *cache, const ahip_kv_batch *batch, const ahip_kv_attend *attend, size_t *bytes) {
    if (!bytes) return kv_fail(ctx, AHIP_ERR_ARG, "kv attention: null output");
    *bytes = 0;
    dev::KvView view = {};
    // The sizes alone: neither the tensors nor the arrays on the device need exist yet.
    if (int rc = attend::check_attend(ctx, cache, batch, attend, &view)) return rc;
    *bytes = attend::plan_of(ctx, *cache, *batch, *attend, false).bytes;
    // The rows may be trees, whose keys are cut where a piece's are not.
    if (attend::may_be_trees(*attend)) *bytes = std::max(*bytes, attend::plan_of(ctx, *cache, *batch, *attend, true).bytes);
    return AHIP_OK;
}

int launch_kv_attention(DeviceCtx &ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_attend &attend) {
    attend::AttendArgs g = {};
    if (int rc = attend::begin_attend(ctx, cache, batch, attend, false, &g)) return rc;
    return g.q ? attend::launch_attend<attend::PLAIN>(ctx, g, cache.elem == AHIP_KV_BF16) : AHIP_OK;
}

}  // namespace altius

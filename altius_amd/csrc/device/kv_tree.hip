// Attention of trees of drafted tokens over a paged cache: the kernels of kv_attend.h, with a mask of a row's own tree beside its range of keys.
// The tree costs a load of the parents and the walk up at a block's start, and a look at the mask in the last one or two tiles of a sequence: 8 tokens behind 500 (12
// heads of 64 channels, fp32) 14.0 us, as a piece 12.6.  16 trees of 16 to 48 tokens behind 300 to 8000 (bf16, 32 heads, 8 of keys, 128 channels) 172 us, 189
// TFLOP/s; 2 of 40 to 61 behind 20011 to 30000 (fp32, 16 heads, 4 of keys, 96 channels, biased) 183 us, 81.  Bound by rows of the blocks of 128 that are not there (a
// third) and by what bounds rows128.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kv_attend.h"

namespace altius {

int launch_kv_attention_tree(DeviceCtx &ctx, const ahip_kv_cache &cache, const ahip_kv_batch &batch, const ahip_kv_attend &attend, const int32_t *parents) {
    const std::string name = "kv attention of a tree: ";
    if (!attend.causal || attend.prefix) return ctx.fail(AHIP_ERR_ARG, name + "a tree is causal and has no prefix");
    if (attend.max_tokens > attend::TREE_ROWS) return ctx.fail(AHIP_ERR_UNSUPPORTED, name + "more than 256 rows a sequence");
    attend::AttendArgs g = {};
    if (int rc = attend::begin_attend(ctx, cache, batch, attend, attend::may_be_trees(attend), &g)) return rc;
    if (!g.q) return AHIP_OK;
    if (!parents) return ctx.fail(AHIP_ERR_ARG, name + "null parents");
    g.parents = parents;
    g.max_tokens = std::min(g.max_tokens, attend::TREE_ROWS);
    return attend::launch_attend<attend::TREE>(ctx, g, cache.elem == AHIP_KV_BF16);
}

}  // namespace altius

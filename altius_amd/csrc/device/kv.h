// A paged cache of keys and values and the sequences of a call as the kernels see them (rotary.hip, kv_attention.hip).
// Everything a caller's device memory says -- where a sequence's rows start, how long it is, which page a place is in --
// is checked here before it becomes an address.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"
#include "ctx.h"

namespace altius {
namespace dev {

constexpr int KV_FLAG = 2;  // which of the context's error flags these kernels raise

struct KvView {
    void *keys, *values;
    int64_t page_stride, head_stride, slot_stride;
    uint32_t pages, page_size, kv_heads, sequences, tokens;
    FastDiv by_page_size;
    const int32_t *table, *starts, *lengths;
    int64_t table_stride;
    uint32_t table_pages;
    int *flag;

    // The page that place `j` (< table_pages * page_size, which is below 2^31) of sequence s is in.  One outside the cache
    // raises the flag and reads as `instead`.
    __device__ __forceinline__ int32_t page_of(uint32_t s, uint32_t index, int32_t instead) const {
        const int32_t page = table[(int64_t)s * table_stride + index];
        if ((uint32_t)page < pages) return page;
        *flag = 1;
        return instead;
    }
};

// The rows of one sequence in the call's tensors, and its length; n == 0 also where what the device memory says does not fit
// the tensors or the page table (then the flag is raised).
struct KvSequence {
    int32_t start, n, length;
};
__device__ __forceinline__ KvSequence kv_sequence(const KvView &kv, uint32_t s) {
    KvSequence q;
    q.start = kv.starts[s];
    const int64_t n = (int64_t)kv.starts[s + 1] - q.start;
    q.length = kv.lengths[s];
    const bool fits = q.start >= 0 && n >= 0 && q.start + n <= (int64_t)kv.tokens && q.length >= 0 &&
                      (uint64_t)q.length <= (uint64_t)kv.table_pages * kv.page_size;
    if (!fits) *kv.flag = 1;
    q.n = fits ? (int32_t)n : 0;
    return q;
}

// The sequence that row `token` belongs to, kv.sequences if it is behind the last one's.  Most calls that matter for their
// latency have one row per sequence, so that guess is tried before a search.
__device__ __forceinline__ uint32_t kv_sequence_of(const KvView &kv, uint32_t token) {
    const int32_t t = (int32_t)token;
    if (token < kv.sequences && kv.starts[token] <= t && t < kv.starts[token + 1]) return token;
    uint32_t low = 0, high = kv.sequences;  // how many of starts[1 ..] are <= t
    while (low < high) {
        const uint32_t mid = (low + high) >> 1;
        if (kv.starts[mid + 1] <= t) low = mid + 1;
        else high = mid;
    }
    return low;
}

}  // namespace dev

// Host: what both operators ask of the sizes of a cache and a batch, and of their pointers.
int require_kv_arrays(DeviceCtx &ctx, const char *who, const ahip_kv_cache &cache, const ahip_kv_batch &batch);
int make_kv_view(DeviceCtx *ctx, const char *who, const ahip_kv_cache *cache, const ahip_kv_batch *batch, size_t tokens, dev::KvView *view);
// A failure with or without a context.
int kv_fail(DeviceCtx *ctx, int code, const std::string &msg);

}  // namespace altius

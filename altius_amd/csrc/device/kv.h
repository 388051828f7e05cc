// A paged cache of keys and values and the sequences of a call as the kernels see them (rotary.hip, kv_attend.h and the other
// kv_ files).
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
    int64_t table_stride, table_head;  // entries from one sequence's row to the next's, and from one kv head's (0: all share)
    uint32_t table_pages;
    int *flag;

    // The page that place `j` (< table_pages * page_size, which is below 2^31) of sequence s is in.  One outside the cache
    // raises the flag and reads as `instead`.
    __device__ __forceinline__ int32_t page_of(uint32_t s, uint32_t index, int32_t instead, uint32_t head = 0) const {
        const int32_t page = table[(int64_t)s * table_stride + (int64_t)head * table_head + index];
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
__device__ __forceinline__ KvSequence kv_checked(const KvView &kv, int32_t start, int32_t next, int32_t length) {
    KvSequence q;
    q.start = start;
    q.length = length;
    const int64_t n = (int64_t)next - start;
    const bool fits = start >= 0 && n >= 0 && start + n <= (int64_t)kv.tokens && length >= 0 && (uint64_t)length <= (uint64_t)kv.table_pages * kv.page_size;
    if (!fits) *kv.flag = 1;
    q.n = fits ? (int32_t)n : 0;
    return q;
}
__device__ __forceinline__ KvSequence kv_sequence(const KvView &kv, uint32_t s) { return kv_checked(kv, kv.starts[s], kv.starts[s + 1], kv.lengths[s]); }

// The sequence that row `token` belongs to, kv.sequences if it is behind the last one's, 0 if it is in front of the first one's, and what
// there is to know of it.  For whole wavefronts: up to 64 sequences are read at once, a lane each.  More are searched, one row per sequence
// first, then by cutting the range in eight with loads that do not wait for each other.
__device__ __forceinline__ uint32_t kv_sequence_of(const KvView &kv, uint32_t token, KvSequence &q) {
    const int32_t t = (int32_t)token;
    if (kv.sequences <= 64) {
        const uint32_t lane = threadIdx.x & 63u;
        const int32_t first = kv.starts[0], next = lane < kv.sequences ? kv.starts[lane + 1] : INT32_MAX, length = lane < kv.sequences ? kv.lengths[lane] : 0;
        uint32_t s = 0;
        for (uint64_t left = ~(uint64_t)0; left;) {  // each row of the wavefront in turn
            const int32_t one = __builtin_amdgcn_readlane(t, __builtin_ctzll(left));
            const uint32_t before = (uint32_t)__popcll(__ballot(next <= one));
            const bool mine = t == one;
            if (mine) s = before;
            left &= ~__ballot(mine);
        }
        const int32_t before = __shfl(next, (int)s - 1), behind = __shfl(next, (int)s), its_length = __shfl(length, (int)s);
        if (s < kv.sequences) q = kv_checked(kv, s ? before : first, behind, its_length);
        return s;
    }
    uint32_t low = 0, high = kv.sequences;  // how many of starts[1 ..] are <= t: low to high
    if (token < kv.sequences && kv.starts[token] <= t && t < kv.starts[token + 1]) low = high = token;
    while (low < high) {
        const uint32_t step = (high - low + 7) / 8;
        uint32_t below = 0;
#pragma unroll
        for (uint32_t i = 1; i <= 7; i++) {
            const uint32_t at = low + i * step, in = at <= high ? at : high;
            below += at <= high && kv.starts[in] <= t ? 1u : 0u;
        }
        low += below * step;
        if (below < 7 && low + step - 1 < high) high = low + step - 1;
    }
    if (low < kv.sequences) q = kv_sequence(kv, low);
    return low;
}

}  // namespace dev

// Host: what both operators ask of the sizes of a cache and a batch, and of their pointers.
int require_kv_arrays(DeviceCtx &ctx, const char *who, const ahip_kv_cache &cache, const ahip_kv_batch &batch);
int make_kv_view(DeviceCtx *ctx, const char *who, const ahip_kv_cache *cache, const ahip_kv_batch *batch, size_t tokens, dev::KvView *view);
// A failure with or without a context.
int kv_fail(DeviceCtx *ctx, int code, const std::string &msg);

}  // namespace altius

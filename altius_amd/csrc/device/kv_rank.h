// The smallest of the `want` largest of a block's values, which are order-preserving images in whole numbers.
#pragma once

#include "common.h"

namespace altius {
namespace dev {

// Sums over the lanes up to this one: within rows of 16, then the rows in front.
template <int CONTROL, int ROWS> __device__ __forceinline__ uint32_t plus_moved(uint32_t v) {
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t lanes_up_to(uint32_t v) {
    v = plus_moved<0x111, 0xF>(v);  // row_shr by 1, 2, 4, 8
    v = plus_moved<0x112, 0xF>(v);
    v = plus_moved<0x114, 0xF>(v);
    v = plus_moved<0x118, 0xF>(v);
    v = plus_moved<0x142, 0xA>(v);  // row_bcast 15: lane 15 of a row to the next one
    return plus_moved<0x143, 0xC>(v);  // row_bcast 31: lane 31 to the upper half
}

// COPIES: bins of some lanes' own, in other banks.  Values share few first bytes, and lanes that count the same one wait for each other.
template <uint32_t COPIES> struct RankLds {
    uint32_t bins[COPIES][256 + 32 / COPIES], totals[4], found[3];
};
template <class Image> struct Ranked {
    Image least;    // all above it are among the largest
    uint32_t ties;  // and of those at it so many; all of them where exact
    bool exact;
};
// each(f) calls f with every value of the calling thread; of all threads' there are more than `want`, which is at least 1.  A byte at a time, from the top: a
// histogram in LDS of the values that share the bytes so far, and the bin that the rank falls into, until all of a bin are wanted.  For whole blocks of 256
// threads or more; lds must not be in use.
template <class Image, uint32_t COPIES, class Each> __device__ __forceinline__ Ranked<Image> rank_largest(RankLds<COPIES> &lds, uint32_t want, Each each) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tid < 256)
#pragma unroll
        for (uint32_t i = 0; i < COPIES; i++) lds.bins[i][tid] = 0;
    __syncthreads();
    Ranked<Image> r = {0, want, false};
    for (int shift = 8 * (int)sizeof(Image) - 8; shift >= 0; shift -= 8) {
        const Image known = shift == 8 * (int)sizeof(Image) - 8 ? 0 : ~(Image)0 << (shift + 8);
        each([&](Image v) {
            if ((v & known) == r.least) atomicAdd(&lds.bins[lane % COPIES][(uint32_t)(v >> shift) & 255u], 1u);
        });
        __syncthreads();
        uint32_t count = 0, up_to = 0;
        if (tid < 256) {  // the largest first
#pragma unroll
            for (uint32_t i = 0; i < COPIES; i++) count += lds.bins[i][255 - tid], lds.bins[i][255 - tid] = 0;
            up_to = lanes_up_to(count);
            if (lane == 63) lds.totals[wave] = up_to;
        }
        __syncthreads();
        if (tid < 256) {
            uint32_t before = up_to - count;
            for (uint32_t w = 0; w < wave; w++) before += lds.totals[w];
            if (before < r.ties && r.ties <= before + count) lds.found[0] = 255 - tid, lds.found[1] = before, lds.found[2] = count;
        }
        __syncthreads();
        r.least |= (Image)lds.found[0] << shift;
        r.ties -= lds.found[1];
        if (r.ties == lds.found[2]) {
            r.exact = true;
            break;
        }
    }
    return r;
}

}  // namespace dev
}  // namespace altius

// block_scan.cuh -- a prefix sum over the threads of a block of 1024.
#pragma once

#include "common.cuh"

namespace hc {

// Exclusive prefix sum over the block; `total` is the sum.  `scratch`: 33 numbers of shared memory.
template <class I>
__device__ __forceinline__ I block_scan(I x, long long* scratch, I& total) {
    const int w = threadIdx.x >> 5, l = lane_id();
    I y = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const I z = __shfl_up_sync(0xffffffffu, y, o);
        if (l >= o) y += z;
    }
    if (l == 31) scratch[w] = y;
    __syncthreads();
    if (w == 0) {
        I v = (I)scratch[l];
        const I own = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const I z = __shfl_up_sync(0xffffffffu, v, o);
            if (l >= o) v += z;
        }
        scratch[l] = v - own;
        if (l == 31) scratch[32] = v;
    }
    __syncthreads();
    total = (I)scratch[32];
    const I before = (I)scratch[w] + y - x;
    __syncthreads();
    return before;
}

}  // namespace hc

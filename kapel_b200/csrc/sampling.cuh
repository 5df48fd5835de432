// The first largest value of a block: what every choice of a token begins with.
#pragma once
#include "common.cuh"

namespace kb {

struct Best { float v; int i; };

__device__ __forceinline__ Best better(Best a, Best b) {
    // larger value wins; on a tie the smaller index; index -1 means "none yet"
    if (b.i < 0) return a;
    if (a.i < 0) return b;
    if (b.v > a.v || (b.v == a.v && b.i < a.i)) return b;
    return a;
}

__device__ inline Best block_best(Best x, Best* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Best y;
        y.v = __shfl_xor_sync(0xffffffffu, x.v, o);
        y.i = __shfl_xor_sync(0xffffffffu, x.i, o);
        x = better(x, y);
    }
    __syncthreads();
    if (lane == 0) scratch[warp] = x;
    __syncthreads();
    const int nwarps = (blockDim.x + 31) >> 5;
    Best t;
    t.v = 0.f; t.i = -1;
    if (lane < nwarps) t = scratch[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Best y;
        y.v = __shfl_xor_sync(0xffffffffu, t.v, o);
        y.i = __shfl_xor_sync(0xffffffffu, t.i, o);
        t = better(t, y);
    }
    return t;
}

}  // namespace kb

// What the bfloat16 kernels of shared attention have in common: warp-level products, a score in powers of two, the launchers.
#pragma once
#include "attention_shared.cuh"
#include "attention_tc.cuh"

namespace kb {

typedef __nv_bfloat16 bf16;

static __device__ int g_shared_attention_error = 0;          // a wait on an mbarrier ran out (one a file)

__device__ __forceinline__ void sh_ldmatrix(uint32_t (&r)[4], uint32_t saddr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(saddr));
}
__device__ __forceinline__ void sh_ldmatrix_trans(uint32_t (&r)[4], uint32_t saddr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(saddr));
}
__device__ __forceinline__ void sh_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t sh_transpose(uint32_t a) {           // an 8 x 8 matrix of 16-bit values across the warp
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// A product q.k as a score in powers of two: scale, and the soft cap where there is one. tanh x = 1 - 2 / (1 + e^2x): its error is some 1e-7
// whatever x, which a cap of 50 makes 1e-5 of a score; the hardware's own tanh is off by up to 2^-11 of its value, 0.01 of a score of 20.
struct SharedScore {
    float in, out;
    bool cap;
    __device__ __forceinline__ SharedScore(float scale, float c) {
        cap = c > 0.f;
        in = cap ? scale / c * 2.885390081777927f : scale * 1.4426950408889634f;
        out = c * 1.4426950408889634f;
    }
    __device__ __forceinline__ float operator()(float x) const {
        if (!cap) return x * in;
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + at_exp2(x * in)));
        return fmaf(-2.f * out, r, out);
    }
};

int shared_own_workers(int d);                               // warps a block
int launch_shared_tiles(const SharedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, cudaStream_t s);
int launch_shared_own(const SharedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, cudaStream_t s);

}  // namespace kb

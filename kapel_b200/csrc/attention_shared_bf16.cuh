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
    float in, out, u;
    bool cap;
    __device__ __forceinline__ SharedScore(float scale, float c) {
        cap = c > 0.f;
        in = cap ? scale / c * 2.885390081777927f : scale * 1.4426950408889634f;
        out = c * 1.4426950408889634f;
        u = cap ? scale / c : 0.f;
    }
    __device__ __forceinline__ float of_u(float x) const {   // the same of a product already divided by the cap
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + at_exp2(x * 2.885390081777927f)));
        return fmaf(-2.f * out, r, out);
    }
    __device__ __forceinline__ float operator()(float x) const {
        if (!cap) return x * in;
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + at_exp2(x * in)));
        return fmaf(-2.f * out, r, out);
    }
};

int shared_own_workers(int d);                               // warps a block
// Two 32-bit values at a time.
__device__ __forceinline__ unsigned long long sh_pair(uint32_t a, uint32_t b) {
    unsigned long long d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ unsigned long long sh_pair(float a, float b) { return sh_pair(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ void sh_split(unsigned long long x, uint32_t& a, uint32_t& b) { asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(x)); }
__device__ __forceinline__ unsigned long long sh_mul2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ unsigned long long sh_add2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ unsigned long long sh_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// Scores of a thread's N products in place, none of them masked, and their largest. Without a cap x scale; with one, where every product of the warp is
// below 3/4 of it, cap tanh(x) by an odd polynomial of degree 9 fitted to tanh x / x on [0, 9/16] of x^2 (6e-7 of the value), two
// values an instruction: the hardware's exponential, reciprocal and exponential again for each score are three of sixteen a clock and bound the
// kernel; this leaves one.
template <int N> __device__ __forceinline__ float sh_scores(uint32_t (&x)[N], const SharedScore& score) {
    const float first = score.cap ? score.u : score.in;
    const unsigned long long in = sh_pair(first, first);
    float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, fars[4] = {0.f, 0.f, 0.f, 0.f};        // four chains side by side
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        sh_split(sh_mul2(sh_pair(x[j], x[j + 1]), in), x[j], x[j + 1]);
        tops[(j >> 1) & 3] = fmaxf(fmaxf(tops[(j >> 1) & 3], __uint_as_float(x[j])), __uint_as_float(x[j + 1]));
    }
    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    if (!score.cap) return top;
#pragma unroll
    for (int j = 0; j < N; j += 2) fars[(j >> 1) & 3] = fmaxf(fmaxf(fars[(j >> 1) & 3], fabsf(__uint_as_float(x[j]))), fabsf(__uint_as_float(x[j + 1])));
    const float far = fmaxf(fmaxf(fars[0], fars[1]), fmaxf(fars[2], fars[3]));
    // (a NaN is passed over by fmaxf and goes through the polynomial as well as through the other)
    if (!__all_sync(0xffffffffu, far <= 0.75f)) {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = __float_as_uint(score.of_u(__uint_as_float(x[j])));
        return score.of_u(top);
    }
    constexpr float C0 = 0.999999463558197f, C1 = -0.3332834839820862f, C2 = 0.13259831070899963f, C3 = -0.05008019134402275f, C4 = 0.012950727716088295f;
    const float o = score.out;
    const unsigned long long c0 = sh_pair(C0 * o, C0 * o), c1 = sh_pair(C1 * o, C1 * o), c2 = sh_pair(C2 * o, C2 * o), c3 = sh_pair(C3 * o, C3 * o), c4 = sh_pair(C4 * o, C4 * o);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        const unsigned long long u = sh_pair(x[j], x[j + 1]), z = sh_mul2(u, u);
        sh_split(sh_mul2(u, sh_fma2(sh_fma2(sh_fma2(sh_fma2(c4, z, c3), z, c2), z, c1), z, c0)), x[j], x[j + 1]);
    }
    const float z = top * top;
    return top * fmaf(fmaf(fmaf(fmaf(C4 * o, z, C3 * o), z, C2 * o), z, C1 * o), z, C0 * o);
}

int launch_shared_tiles(const SharedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, cudaStream_t s);
int launch_shared_own(const SharedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, cudaStream_t s);

}  // namespace kb

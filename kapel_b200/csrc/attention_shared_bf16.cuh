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
// Tensor memory, 32 lanes x 16 or 32 words; and out of 16 or 8.
__device__ __forceinline__ void sh_ld(uint32_t taddr, uint32_t (&r)[32]) { at_ld32(taddr, r); }
__device__ __forceinline__ void sh_ld(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void sh_st(uint32_t taddr, const uint32_t (&r)[16]) { at_st16(taddr, r); }
__device__ __forceinline__ void sh_st(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}

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

__device__ __forceinline__ float sh_max_abs(float a, float b, float c) {
    float d;
    asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// A thread's N products divided by the cap (without one: as scores), in place; returns the largest magnitude.
template <int N> __device__ __forceinline__ float sh_scale(uint32_t (&x)[N], const SharedScore& score) {
    const float first = score.cap ? score.u : score.in;
    const unsigned long long in = sh_pair(first, first);
    float far[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        sh_split(sh_mul2(sh_pair(x[j], x[j + 1]), in), x[j], x[j + 1]);
        far[(j >> 1) & 1] = sh_max_abs(far[(j >> 1) & 1], __uint_as_float(x[j]), __uint_as_float(x[j + 1]));
    }
    return fmaxf(far[0], far[1]);
}
// The weights 2^(score - base) of what `sh_scale` left, rounded, two to a word; returns the sum of the rounded ones. `SMOOTH`: every product is
// below SH_NEAR of the cap, and cap tanh(x) is an odd polynomial of degree 7 fitted to tanh x / x (1.2e-6 of the value), two values an
// instruction. The hardware makes four exponentials or reciprocals a clock and scheduler: with the polynomial a weight takes one, not three, and
// the polynomial's products run beside it.
constexpr float SH_NEAR = 0.55f;
template <int N, typename F> __device__ __forceinline__ float sh_weights(const uint32_t (&x)[N], uint32_t (&out)[N / 2], float base, F score_of) {
    const unsigned long long less = sh_pair(-base, -base);
    unsigned long long sums[2] = {0ull, 0ull};
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        uint32_t a, b;
        sh_split(score_of(sh_pair(x[j], x[j + 1]), less), a, b);
        const uint32_t two = at_pack(at_exp2(__uint_as_float(a)), at_exp2(__uint_as_float(b)));
        sums[(j >> 1) & 1] = sh_add2(sums[(j >> 1) & 1], sh_pair(two << 16, two & 0xffff0000u));
        out[j >> 1] = two;
    }
    uint32_t la, lb;
    sh_split(sh_add2(sums[0], sums[1]), la, lb);
    return __uint_as_float(la) + __uint_as_float(lb);
}
template <int N> __device__ __forceinline__ float sh_weights_near(const uint32_t (&x)[N], uint32_t (&out)[N / 2], float base, const SharedScore& score) {
    constexpr float C0 = 0.999998927116394f, C1 = -0.33321505784988403f, C2 = 0.13132257759571075f, C3 = -0.042718496173620224f;
    const float o = score.out;
    const unsigned long long c0 = sh_pair(C0 * o, C0 * o), c1 = sh_pair(C1 * o, C1 * o), c2 = sh_pair(C2 * o, C2 * o), c3 = sh_pair(C3 * o, C3 * o);
    return sh_weights(x, out, base, [&](unsigned long long u, unsigned long long less) {
        const unsigned long long z = sh_mul2(u, u);
        return sh_fma2(u, sh_fma2(sh_fma2(sh_fma2(c3, z, c2), z, c1), z, c0), less);
    });
}

int launch_shared_tiles(const SharedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, cudaStream_t s);
int launch_shared_own(const SharedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, cudaStream_t s);

}  // namespace kb

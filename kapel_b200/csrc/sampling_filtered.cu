// A draw under temperature, top_k, top_p and min_p where the logits are, a row's settings and uniform number its own.
//
// The rules are the host sampler's (csrc/host/sampler_core.cpp; crates/kapel-infer/src/sampling.rs:157-260), in its order: x = logit /
// temperature; top_k keeps what is no smaller than the k-th largest (its ties stay); top_p keeps, the likeliest first and the lower index
// first among equals, the tokens before which the others hold less than top_p; min_p keeps p >= min_p p_max; the draw is the first index
// whose running total over what is left exceeds u times the whole. All three filters cut the same order (x down, index up), so what is
// left is always "above a cut (key, index)".
//
// A row is one cluster's: its blocks read the row once and keep their shares in shared memory (of a share beyond 49,152 columns the rest is read again,
// from the second-level cache); everything after works on chip.
//   1. The largest logit, whether a NaN is there.
//   2. For a top_k up to LIST / 2: as many of the threads' own largest logits lie above the cut's lower bound that a histogram of those few
//      finds (its bins reach to the least of them: where they ended at e^-24, one row in a hundred, with a token far above the rest, took 60 us for 15); what lies above it is gathered in the cluster's first block, sorted, cut and drawn from there. (Sorted logits may leave more
//      than LIST above it: then as below.)
//   3. Else a histogram of counts over 2,048 bins of equal steps of x below the largest. top_k: the bin in which the k-th lies. top_p: a
//      bin's weight lies between its count times the weights at its ends, so the histogram bounds where the cut is to a few bins, from above
//      and, all weights' sum being known, from below. The bins in question, or all down to them, are gathered and sorted for the exact cut
//      where they hold no more than LIST tokens, else counted again in 2,048 bins of their own; the same pass adds up what lies above them exactly (in
//      fixed point, 52 bits behind the point: whole numbers, whose order changes nothing; a thread's sums and a warp's fit 64 bits, a row's, of up to
//      2^19 tokens, has 72). (Weights added up by
//      atomics instead took 1.1 ms a row of 256,000: shared memory has none of 64 bits. Without the bound from below a nucleus of 0.99 took
//      three levels and 160 us where it takes one and 50.)
//   4. The draw goes over the whole share of every block: totals of warps, of the 32 rows of the warp's that the target falls in,
//      then along that row.
// e^x is in 64 bits, and so are the draw's sums, as on the host: a seed gives the tokens it gives there, but for borders within the roundings of either side. Those of
// the draw lie in the 13th digit. In the nucleus' sums a token is off by up to 2^-53 of the likeliest, where the host rounds every running total to as
// much of the whole: some 1e-13 of 256,000 tokens as roundings go, 3e-11 where all weights lie just below half a unit. e^x is
// made of 2^(n / 32) = 2^k T[n mod 32], n an integer within a roundoff of the nearest to 32 x / ln 2 (found in 32 bits), and a polynomial of degree 5 for what is left (the series' next term is below 3e-15): nine 64-bit operations, of which a multiprocessor does some 37 a
// clock. Two entries of T share a bank, so a warp's loads take two turns at most.
//
// What bounds it, over 256,000 tokens (recorded; logits of deviation 1.5 with 300 likely tokens above them, under a temperature of 0.8): one row alone
// takes 15 us under top_k 50, of which the row's load is 3 and the rest some eight cluster barriers and what lies between them; 20 without filters; 27 under a nucleus of
// 0.95, of which 10 are the pass that adds up all weights and counts them (two tokens' weights side by side were no faster). 64 rows: 34 us
// under top_k 50 (1.9 TB/s), 63 without filters, 78 under a nucleus of 0.95 or 0.99: two rounds of clusters, one block a multiprocessor, with
// nothing beside a row's chain of load, barriers, passes and sort; their 64-bit operations alone would take some 15. Where the nucleus is a third of all tokens (a normal distribution of
// deviation 2) its border lies among more than the list holds and takes two passes more: one row 57 us, 64 rows 177.
#include <cooperative_groups.h>
#include <cfloat>
#include "common.cuh"

namespace kb {
namespace cg = cooperative_groups;

constexpr int SF_THREADS = 1024, SF_WARPS = SF_THREADS / 32;
constexpr int SF_BINS = 2048, SF_LIST = 2048, SF_MAX_CLUSTER = 8;
constexpr int SF_SMALL = 256;                            // lists up to here are ordered by counting
constexpr int SF_FULL = 48;                              // entries of a bucket that are ordered among themselves
constexpr int SF_DEEP = 8, SF_BATCH = SF_DEEP * SF_THREADS;      // loads a thread asks for at once
constexpr int SF_ROWS = 64;                              // rows of 32 columns a warp has at most: a share of 2^16, a vocabulary of 2^19 over eight blocks
constexpr float SF_SPAN = 24.f;                          // the bins reach e^-24 below the largest; the last holds all that is below
constexpr double SF_FIXED = 4503599627370496.0;          // 2^52
constexpr double SF_STEP = 0.6931471805599453 / 32.0;    // ln 2 / 32
constexpr int SF_SMALLEST = -1076;                       // a weight below 2^-1075 is none

struct SfParams {
    int* tokens;
    const float* logits;
    const double* temperature;
    const int* top_k;
    const double* top_p;
    const double* min_p;
    const double* uniform;
    int rows, vocab;
    int share;                                           // columns a block of the cluster has (the last may have fewer)
    int cached;                                          // of them in shared memory, all or whole batches; the rest is read again from the row
};

// Sums of weights that decide a cut, in units of 2^-52: up to 2^19 of them. Those of a warp's share (2^11 columns) and of a list fit 64 bits.
typedef unsigned __int128 SfTotal;
__device__ __forceinline__ double sf_double(SfTotal x) {
    return fma((double)(unsigned long long)(x >> 64), 18446744073709551616.0, (double)(unsigned long long)x);
}

struct SfTop { float v; int nan; unsigned low; };       // a block's largest logit, and the smallest key of its threads' largest
struct SfCut { unsigned key; int index; };               // what is left: key above, or equal and the index no larger
struct SfFound {                                         // what the first block tells the others about a histogram
    int from, to;                                        // the bins the cut may be in
    unsigned above, upto;                                // tokens above them, and down to their end
};

struct SfShared {
    double powers[32];                                   // 2^(j / 32)
    unsigned counts[SF_BINS];
    unsigned long long list[SF_LIST];                    // first block: key << 32 | ~index, the largest first once sorted
    SfTop tops[SF_MAX_CLUSTER];
    double sums[SF_MAX_CLUSTER];
    unsigned long long fixed_sums[SF_MAX_CLUSTER][4];
    double warp_sum[SF_WARPS], warp_sum2[SF_WARPS];
    double row_sum[SF_ROWS];
    unsigned long long warp_fixed[SF_WARPS], warp_fixed2[SF_WARPS];
    unsigned warp_count[SF_WARPS];
    float warp_max[SF_WARPS];
    unsigned warp_low[SF_WARPS];
    SfFound found;
    SfCut cut;
    unsigned sort_lo, sort_hi;                           // the smallest and largest upper word of a list
    int listed;
    int owner, owner2;
    int kept;
};

// Keys that order as the values do; both zeros are one.
__device__ __forceinline__ unsigned sf_key(float v) {
    const unsigned u = __float_as_uint(v + 0.f);
    return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float sf_value(unsigned key) {
    return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

struct SfRow {
    const float* row;                                    // this block's share begins here
    const float* cache;
    const double* powers;
    int n, cached, first;                                // columns of the share, how many are in `cache`, the share's first column
    double inv, steps;                                   // 1 / temperature, and in steps of ln 2 / 32
    float largest, half, steps32;                        // the largest, half of it; twice the steps, in 32 bits
    __device__ __forceinline__ float at(int i) const { return i < cached ? cache[i] : row[i]; }
    __device__ __forceinline__ void scale(float top, double temperature, const double* table) {
        largest = top;
        inv = fmin(1.0 / temperature, 1e36);             // (of colder rows only what ties with the largest counts, as of one at 1e-36)
        steps = inv / SF_STEP;                           // below 2^126
        half = 0.5f * top;
        steps32 = (float)(2.0 * steps);
        powers = table;
    }
    // e^((v - largest) / temperature), which is at most 1. The logits are subtracted before they are divided (the host rounds each quotient first). What
    // is small is told by the exponent itself: one that 64-bit floats have no power of two for must not reach their exponent's bits.
    __device__ __forceinline__ double weight(float v) const {
        const float magic32 = 12582912.f;                // 1.5 2^23: a sum's last bits are the nearest integer
        const float at = fmaf(fmaf(0.5f, v, -half), steps32, magic32);           // (by halves: a difference may pass the largest float)
        if (at < magic32 + 32.f * SF_SMALLEST) return 0.0;
        const int n = __float_as_int(at) - __float_as_int(magic32), k = n >> 5;
        const double x = fma((double)v - (double)largest, steps, 6755399441055744.0 - __hiloint2double(0x43380000 + (n >> 31), n));      // half a step, and what 32 bits round
        constexpr double A = SF_STEP, A2 = A * A / 2, A3 = A2 * A / 3, A4 = A3 * A / 4, A5 = A4 * A / 5;
        const double e = powers[n & 31] * fma(x, fma(x, fma(x, fma(x, fma(x, A5, A4), A3), A2), A), 1.0);
        if (k < -1000) return __hiloint2double(__double2hiint(e) + ((k + 128) << 20), __double2loint(e)) * 2.938735877055719e-39;     // 2^-128: rounded where it is subnormal
        return __hiloint2double(__double2hiint(e) + (k << 20), __double2loint(e));
    }
    // Calls f(column, value) for the block's columns whose value is `floor` or more, a thread every SF_THREADS-th.
    template <typename F> __device__ __forceinline__ void each(float floor, F f) const {
        for (int first = 0; first < n; first += SF_BATCH) {
            const int base = first + threadIdx.x;
            float v[SF_DEEP];
            if (first < cached) {
#pragma unroll
                for (int k = 0; k < SF_DEEP; ++k) v[k] = base + k * SF_THREADS < n ? cache[base + k * SF_THREADS] : -INFINITY;
            } else {
#pragma unroll
                for (int k = 0; k < SF_DEEP; ++k) v[k] = base + k * SF_THREADS < n ? row[base + k * SF_THREADS] : -INFINITY;
            }
#pragma unroll
            for (int k = 0; k < SF_DEEP; ++k)
                if (v[k] >= floor) f(base + k * SF_THREADS, v[k]);
        }
    }
};
constexpr float SF_LOWEST = -FLT_MAX;                    // the floor of all that is possible

__device__ __forceinline__ bool sf_left(const SfCut& cut, unsigned key, int index) {
    return key > cut.key || (key == cut.key && index <= cut.index);
}
__device__ __forceinline__ float sf_floor(const SfCut& cut) { return cut.key == 0u ? SF_LOWEST : fmaxf(SF_LOWEST, sf_value(cut.key)); }

// A level's bins: equal steps of the value down from the largest in question, or of the key.
struct SfBins {
    bool by_key;
    float most, least, step;                             // bin = (most - v) step; the last holds all that is below too
    unsigned lo, hi;                                     // the same as keys; bin = (hi - key) >> shift
    int shift;
    __device__ __forceinline__ int of(float v) const {
        if (by_key) return (int)((hi - sf_key(v)) >> shift);
        const float x = (most - v) * step;
        return x < (float)(SF_BINS - 1) ? (int)x : (x == x ? SF_BINS - 1 : 0);
    }
    // No value above top(b), or below bottom(b), is in bin b (32-bit steps: an edge may lie a few roundings off).
    __device__ __forceinline__ float top(int b) const {
        if (by_key) return sf_value(hi - ((unsigned)b << shift));
        const float reach = (float)b / step * 0.999999f;
        return b > 0 && reach < FLT_MAX ? fminf(most, most - reach + fabsf(most) * 2.4e-7f) : most;
    }
    __device__ __forceinline__ float bottom(int b) const {
        if (b >= SF_BINS - 1) return least;
        if (by_key) {
            const unsigned span = (((unsigned)b + 1u) << shift) - 1u;
            return sf_value(hi - lo < span ? lo : hi - span);
        }
        return fmaxf(least, most - (float)(b + 1) / step * 1.000001f - fabsf(most) * 2.4e-7f);       // (infinite where the steps are nothing)
    }
    // Between two values that are in question: steps of the value (keys are sparse away from zero and crowded around it) unless those are so near one
    // another that the steps come to a few roundings.
    __device__ __forceinline__ static SfBins between(unsigned lo, unsigned hi, bool values) {
        SfBins b;
        b.lo = lo;
        b.hi = hi;
        b.most = sf_value(hi);
        b.least = sf_value(lo);
        b.step = (float)(SF_BINS - 1) / (b.most - b.least);
        b.by_key = !(values && b.most - b.least > fmaxf(fabsf(b.most), fabsf(b.least)) / 64.f && b.step > 1e-30f && b.step < 1e30f);
        b.shift = 0;
        while (((hi - lo) >> b.shift) >= (unsigned)SF_BINS) ++b.shift;
        return b;
    }
};
constexpr int SF_LEVELS = 8;                             // from here on by keys, whose number at least halves from level to level

// e in fixed point, rounded to a unit: 2^52 added, the sum's bits are the whole number above those of 2^52 (those of 2^53 too, where e is 1).
__device__ __forceinline__ unsigned long long sf_fixed(double e) {
    return (unsigned long long)__double_as_longlong(fma(e, SF_FIXED, 4503599627370496.0)) - 0x4330000000000000ull;
}
// run >= top_p all, the product not rounded before it is compared: equal weights reach a round share of the whole exactly.
__device__ __forceinline__ bool sf_reached(SfTotal run, double top_p, SfTotal all) {
    return fma(top_p, sf_double(all), -sf_double(run)) <= 0.0;
}

// Inclusive running totals over the block's first `warps` warps (the others have nothing), in thread order.
template <typename V> __device__ __forceinline__ V sf_warp_scan(V v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    return v;
}
template <typename V> __device__ __forceinline__ V sf_scan(V v, V* per_warp, V* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = sf_warp_scan(v);
    __syncthreads();
    if (lane == 31) per_warp[warp] = v;
    __syncthreads();
    const V sums = sf_warp_scan(per_warp[lane]);
    *total = __shfl_sync(0xffffffffu, sums, 31);
    const V before = __shfl_sync(0xffffffffu, sums, (warp + 31) & 31);
    return warp ? before + v : v;
}

// Sorts the list's first n entries (no two alike), largest first; n up to SF_LIST. A few go to where as many are larger. More go by their upper words
// to SF_BINS buckets of equal width between the smallest and the largest, and within those to where as many are larger; where a bucket holds more
// than SF_FULL (ties), all by exchanges, those within 64 neighbours by one warp each. 2,048 entries: 3 us by buckets, 15 by exchanges.
__device__ void sf_sort(SfShared& s, int n) {
    unsigned long long* list = s.list;
    const int tid = threadIdx.x;
    if (n > SF_SMALL) {
        if (tid == 0) { s.sort_lo = 0xffffffffu; s.sort_hi = 0u; }
        for (int i = tid; i < SF_BINS; i += SF_THREADS) s.counts[i] = 0u;
    }
    __syncthreads();
    if (n <= SF_SMALL) {
        // four threads an entry, a quarter of the others each
        const int i = tid >> 2;
        const unsigned long long mine = i < n ? list[i] : 0ull;
        int rank = 0;
        if (i < n)
            for (int j = tid & 3; j < n; j += 4) rank += list[j] > mine ? 1 : 0;
        rank += __shfl_xor_sync(0xffffffffu, rank, 1);
        rank += __shfl_xor_sync(0xffffffffu, rank, 2);
        __syncthreads();
        if (i < n && (tid & 3) == 0) list[rank] = mine;          // entries differ: their indices do
        __syncthreads();
        return;
    }
    constexpr int EACH = SF_LIST / SF_THREADS;
    unsigned long long mine[EACH];
    unsigned lo = 0xffffffffu, hi = 0u;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const int i = tid + k * SF_THREADS;
        mine[k] = i < n ? list[i] : 0ull;
        if (i < n) { lo = min(lo, (unsigned)(mine[k] >> 32)); hi = max(hi, (unsigned)(mine[k] >> 32)); }
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if ((tid & 31) == 0) { atomicMin(&s.sort_lo, lo); atomicMax(&s.sort_hi, hi); }
    __syncthreads();
    lo = s.sort_lo;
    hi = s.sort_hi;
    int shift = 0;
    while (((hi - lo) >> shift) >= (unsigned)SF_BINS) ++shift;
    unsigned bucket[EACH], slot[EACH];
    bool full = false;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        if (tid + k * SF_THREADS >= n) continue;
        bucket[k] = (hi - (unsigned)(mine[k] >> 32)) >> shift;
        slot[k] = atomicAdd(&s.counts[bucket[k]], 1u);
        full = full || slot[k] >= (unsigned)SF_FULL;
    }
    if (!__syncthreads_or(full)) {
        constexpr int BINS = SF_BINS / SF_THREADS;
        unsigned c[BINS], sum = 0, total;
#pragma unroll
        for (int k = 0; k < BINS; ++k) { c[k] = s.counts[tid * BINS + k]; sum += c[k]; }
        unsigned before = sf_scan(sum, s.warp_count, &total) - sum;          // behind its barriers every thread has its counts
#pragma unroll
        for (int k = 0; k < BINS; ++k) { s.counts[tid * BINS + k] = before; before += c[k]; }
        __syncthreads();
        unsigned first[EACH], end[EACH];
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            if (tid + k * SF_THREADS >= n) continue;
            first[k] = s.counts[bucket[k]];
            end[k] = bucket[k] + 1 < (unsigned)SF_BINS ? s.counts[bucket[k] + 1] : (unsigned)n;
            list[first[k] + slot[k]] = mine[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            if (tid + k * SF_THREADS >= n) continue;
            unsigned at = first[k];
            for (unsigned i = first[k]; i < end[k]; ++i) at += list[i] > mine[k] ? 1u : 0u;
            first[k] = at;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < EACH; ++k)
            if (tid + k * SF_THREADS < n) list[first[k]] = mine[k];
        __syncthreads();
        return;
    }
    int size = 512;
    while (size < n) size <<= 1;
    for (int i = tid; i < size; i += SF_THREADS)
        if (i >= n) list[i] = 0ull;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            if (tid < size / 2) {
                const int i = 2 * (tid & ~(j - 1)) + (tid & (j - 1));
                const unsigned long long a = list[i], b = list[i + j];
                if (((i & k) == 0) ? a < b : a > b) { list[i] = b; list[i + j] = a; }
            }
            // the next exchange's neighbours are this warp's own 64 where it and this one reach no farther than 32
            const int next = j > 1 ? j >> 1 : k;
            if (j > 32 || next > 32) __syncthreads(); else __syncwarp();
        }
    __syncthreads();
}

__device__ __forceinline__ void sf_clear(SfShared& s) {
    for (int i = threadIdx.x; i < SF_BINS; i += SF_THREADS) s.counts[i] = 0u;
    __syncthreads();
}

// The counts of every block added up in the first, and there the bins in which the cut may be: by count (`want` > 0) the one in which it reaches
// `want`; by weight from the first in which it may reach top_p of `all` to the first in which it does. `above` and `weight_above` lie above the
// level's keys; `whole`: all is in the level's bins, so what lies down to a bin is bounded by what lies below it too: the bounds are as near as a
// bin is wide, of the smaller of the two. Where nothing reaches it (fewer tokens, or rounding) the last bin that holds a token. Every block leaves with `found`.
__device__ void sf_find(cg::cluster_group& cluster, SfShared& s, const SfRow& r, const SfBins& bins, unsigned want, double top_p, unsigned above,
                        SfTotal weight_above, SfTotal all, bool whole) {
    const int tid = threadIdx.x;
    if (cluster.block_rank() == 0 && tid == 0) { s.owner = SF_BINS; s.owner2 = SF_BINS; s.kept = -1; }
    cluster.sync();
    if (cluster.block_rank() == 0) {
        constexpr int EACH = 2;
        static_assert(EACH * SF_THREADS == SF_BINS, "two bins a thread");
        const bool by_weight = want == 0u;
        unsigned c[EACH] = {0u, 0u}, count = 0, total_c;
        uint2 theirs[SF_MAX_CLUSTER];                    // fetched, not added up here by the others' atomics, which took three times as long
#pragma unroll
        for (int k = 0; k < SF_MAX_CLUSTER; ++k)
            theirs[k] = k < (int)cluster.num_blocks() ? reinterpret_cast<const uint2*>(cluster.map_shared_rank(&s, k)->counts)[tid] : make_uint2(0u, 0u);
#pragma unroll
        for (int k = 0; k < SF_MAX_CLUSTER; ++k) { c[0] += theirs[k].x; c[1] += theirs[k].y; }
        double least[EACH], most[EACH], lower = 0.0, upper = 0.0, all_lower = 0.0, all_upper = 0.0;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            count += c[j];
            least[j] = most[j] = 0.0;
            if (by_weight && c[j]) {
                most[j] = r.weight(bins.top(tid * EACH + j));
                least[j] = r.weight(bins.bottom(tid * EACH + j));
                least[j] = fmax(least[j] * c[j] * (1.0 - 1e-9) * SF_FIXED - 0.5 * c[j], 0.0);            // each rounded to a whole number
                most[j] = most[j] * c[j] * (1.0 + 1e-9) * SF_FIXED + 0.5 * c[j];
            }
            lower += least[j];
            upper += most[j];
        }
        unsigned run_c = above + sf_scan(count, s.warp_count, &total_c) - count;
        double run_l = 0.0, run_u = 0.0;
        if (by_weight) {
            run_l = sf_double(weight_above) + sf_scan(lower, s.warp_sum, &all_lower) - lower;
            run_u = sf_double(weight_above) + sf_scan(upper, s.warp_sum2, &all_upper) - upper;
        }
        const double sum = sf_double(all), target = top_p * sum, slack = 1e-12 * sum;          // (what 64-bit sums of up to 2,048 terms may be off by)
        unsigned at[EACH];                               // tokens above each bin
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            at[j] = run_c;
            run_c += c[j];
            run_l += least[j];
            run_u += most[j];
            if (c[j]) {
                const int b = tid * EACH + j;
                atomicMax(&s.kept, b);
                const double no_more = whole ? fmin(run_u, sum - (all_lower - run_l)) : run_u, no_less = whole ? fmax(run_l, sum - (all_upper - run_u)) : run_l;
                if (by_weight ? no_more + slack >= target : run_c >= want) atomicMin(&s.owner, b);
                if (by_weight ? no_less - slack >= target : run_c >= want) atomicMin(&s.owner2, b);
            }
        }
        __syncthreads();
        const int last = s.kept, from = min(s.owner, last), to = min(s.owner2, last);
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const int b = tid * EACH + j;
            if (b != from && b != to) continue;
            for (unsigned k = 0; k < cluster.num_blocks(); ++k) {
                SfFound* f = &cluster.map_shared_rank(&s, k)->found;
                if (b == from) { f->from = from; f->to = to; f->above = at[j]; }
                if (b == to) f->upto = at[j] + c[j];
            }
        }
    }
    cluster.sync();
}

// Two sums over the whole row of what each thread brings, up to 2^58.
__device__ void sf_sum(cg::cluster_group& cluster, SfShared& s, unsigned long long a, unsigned long long b, SfTotal& all_a, SfTotal& all_b) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { a += __shfl_xor_sync(0xffffffffu, a, o); b += __shfl_xor_sync(0xffffffffu, b, o); }
    if (lane == 0) { s.warp_fixed[warp] = a; s.warp_fixed2[warp] = b; }
    __syncthreads();
    if (warp == 0) {                                     // the warps' sums of up to 63 bits, upper and lower halves by themselves
        unsigned long long half[4] = {s.warp_fixed[lane] & 0xffffffffull, s.warp_fixed[lane] >> 32, s.warp_fixed2[lane] & 0xffffffffull, s.warp_fixed2[lane] >> 32};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int k = 0; k < 4; ++k) half[k] += __shfl_xor_sync(0xffffffffu, half[k], o);
        if (lane < (int)cluster.num_blocks()) {
            unsigned long long* there = cluster.map_shared_rank(&s, lane)->fixed_sums[cluster.block_rank()];
#pragma unroll
            for (int k = 0; k < 4; ++k) there[k] = half[k];
        }
    }
    cluster.sync();
    unsigned long long half[4] = {0ull, 0ull, 0ull, 0ull};
    for (unsigned k = 0; k < cluster.num_blocks(); ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) half[j] += s.fixed_sums[k][j];
    all_a = ((SfTotal)half[1] << 32) + half[0];
    all_b = ((SfTotal)half[3] << 32) + half[2];
}

// Every block's list behind the first block's (`listed` of them there, of which SF_LIST are kept): each asks the first for room once. The lists are complete.
__device__ void sf_collect(cg::cluster_group& cluster, SfShared& s) {
    if (cluster.block_rank() != 0) {
        SfShared* home = cluster.map_shared_rank(&s, 0);
        const int mine = s.listed;
        if (threadIdx.x == 0 && mine > 0) s.kept = atomicAdd(&home->listed, mine);
        __syncthreads();
        const int at = mine > 0 ? s.kept : 0;
        for (int i = threadIdx.x; i < min(mine, SF_LIST); i += SF_THREADS)
            if (at + i < SF_LIST) home->list[at + i] = s.list[i];
    }
    cluster.sync();
}
__device__ __forceinline__ void sf_list(SfShared& s, unsigned key, int index) {
    const int at = atomicAdd(&s.listed, 1);
    if (at < SF_LIST) s.list[at] = ((unsigned long long)key << 32) | (unsigned)~index;
}
// What is left in the bins down to `to` into the first block's list.
__device__ void sf_gather(cg::cluster_group& cluster, SfShared& s, const SfRow& r, const SfBins& bins, const SfCut& cut, int to) {
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    r.each(fmaxf(sf_floor(cut), bins.bottom(to)), [&](int i, float v) {
        const unsigned key = sf_key(v);
        if (sf_left(cut, key, r.first + i) && bins.of(v) <= to) sf_list(s, key, r.first + i);
    });
    cluster.sync();
    sf_collect(cluster, s);
}

// The first index, over the whole row in order, whose running total of `weight_of(column, value)` (nothing below `floor`) exceeds the target that
// `target_of` makes of the whole; the last index with a weight where rounding leaves the target at or above it. -1 in every thread but one of
// the block that has it.
template <typename W, typename T>
__device__ int sf_locate(cg::cluster_group& cluster, SfShared& s, const SfRow& r, float floor, W weight_of, T target_of) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int each = ((r.n + SF_WARPS - 1) / SF_WARPS + 31) / 32 * 32;      // a warp's columns lie together: totals follow their order
    const int begin = min(r.n, warp * each), end = min(r.n, begin + each);
    double local = 0.0;
    constexpr int DEEP = 8;
    for (int base = begin + lane; base < end; base += 32 * DEEP) {
        float v[DEEP];
#pragma unroll
        for (int k = 0; k < DEEP; ++k) v[k] = base + 32 * k < end ? r.at(base + 32 * k) : -INFINITY;
#pragma unroll
        for (int k = 0; k < DEEP; ++k)
            if (v[k] >= floor) local += weight_of(base + 32 * k, v[k]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) local += __shfl_xor_sync(0xffffffffu, local, o);
    if (lane == 0) s.warp_sum[warp] = local;
    __syncthreads();
    if (warp == 0) {
        const double mine = __shfl_sync(0xffffffffu, sf_warp_scan(s.warp_sum[lane]), 31);
        if (lane < (int)cluster.num_blocks()) cluster.map_shared_rank(&s, lane)->sums[cluster.block_rank()] = mine;
    }
    cluster.sync();
    double total = 0.0;
    for (unsigned b = 0; b < cluster.num_blocks(); ++b) total += s.sums[b];
    const double target = target_of(total);
    double run = 0.0, before = 0.0;
    int owner = -1, last = -1;
    for (unsigned b = 0; b < cluster.num_blocks(); ++b) {
        const double next = run + s.sums[b];
        if (s.sums[b] > 0.0) last = (int)b;
        if (owner < 0 && s.sums[b] > 0.0 && target < next) { owner = (int)b; before = run; }
        run = next;
    }
    const bool beyond = owner < 0;
    if (beyond) owner = last;
    if (owner != (int)cluster.block_rank()) return -1;
    // The first of the warps' ranges that holds the target; where rounding hid it, the last that holds anything.
    const double sum = s.warp_sum[lane], after = before + sf_warp_scan(sum);
    const unsigned some_warps = __ballot_sync(0xffffffffu, sum > 0.0), holds = __ballot_sync(0xffffffffu, sum > 0.0 && !beyond && target < after);
    bool to_end = holds == 0u;
    const int mine = to_end ? 31 - __clz(some_warps) : __ffs(holds) - 1;
    double upto_warp = __shfl_sync(0xffffffffu, after, (mine + 31) & 31);
    if (mine == 0) upto_warp = before;
    // Its rows of 32 columns, dealt out to all warps: their sums, then along the row that holds the target.
    const int from = min(r.n, mine * each), rows = (min(r.n, from + each) - from + 31) / 32;
    auto of = [&](int i) -> double {
        if (i >= r.n || i >= from + each) return 0.0;
        const float v = r.at(i);
        return v >= floor ? weight_of(i, v) : 0.0;
    };
    for (int k = warp; k < SF_ROWS; k += SF_WARPS) {
        double e = k < rows ? of(from + k * 32 + lane) : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) e += __shfl_xor_sync(0xffffffffu, e, o);
        if (lane == 0) s.row_sum[k] = e;
    }
    __syncthreads();
    if (warp != 0) return -1;
    const double a = s.row_sum[lane], b = s.row_sum[lane + 32];
    const double after_a = upto_warp + sf_warp_scan(a), half = __shfl_sync(0xffffffffu, after_a, 31), after_b = half + sf_warp_scan(b);
    const unsigned long long some_rows = ((unsigned long long)__ballot_sync(0xffffffffu, b > 0.0) << 32) | __ballot_sync(0xffffffffu, a > 0.0);
    const unsigned long long hold_rows = ((unsigned long long)__ballot_sync(0xffffffffu, b > 0.0 && target < after_b) << 32) |
                                         __ballot_sync(0xffffffffu, a > 0.0 && target < after_a);
    to_end = to_end || hold_rows == 0ull;
    const int k = to_end ? 63 - __clzll(some_rows) : __ffsll(hold_rows) - 1;
    const double before_a = __shfl_sync(0xffffffffu, after_a, (k + 31) & 31), before_b = __shfl_sync(0xffffffffu, after_b, (k + 31) & 31);
    const double row_before = k == 0 ? upto_warp : k <= 32 ? before_a : before_b;          // row 32 begins where row 31 ends
    const double e = of(from + k * 32 + lane), upto = row_before + sf_warp_scan(e);
    const unsigned some = __ballot_sync(0xffffffffu, e > 0.0), passed = __ballot_sync(0xffffffffu, e > 0.0 && !to_end && target < upto);
    return lane == 0 ? from + k * 32 + (passed ? __ffs(passed) - 1 : 31 - __clz(some)) : -1;
}

constexpr int SF_EACH = SF_LIST / SF_THREADS;            // entries of the list a thread has

__device__ __forceinline__ unsigned sf_key_of(unsigned long long entry) { return (unsigned)(entry >> 32); }

// Of the sorted list's first n entries, how many are left where the weight before each must be below top_p of `all` (`above` lies before the
// first).
__device__ int sf_kept_by_weight(SfShared& s, const SfRow& r, int n, SfTotal above, double top_p, SfTotal all) {
    unsigned long long w[SF_EACH], mine = 0, listed;
#pragma unroll
    for (int j = 0; j < SF_EACH; ++j) {
        const int i = threadIdx.x * SF_EACH + j;
        w[j] = i < n ? sf_fixed(r.weight(sf_value(sf_key_of(s.list[i])))) : 0ull;
        mine += w[j];
    }
    if (threadIdx.x == 0) s.kept = n;
    SfTotal run = above + (sf_scan(mine, s.warp_fixed, &listed) - mine);
#pragma unroll
    for (int j = 0; j < SF_EACH; ++j) {
        const int i = threadIdx.x * SF_EACH + j;
        run += w[j];
        if (i < n && sf_reached(run, top_p, all)) { atomicMin(&s.kept, i + 1); break; }
    }
    __syncthreads();
    const int kept = s.kept;
    __syncthreads();
    return kept;
}

// The first of the sorted list's n entries that `cuts` (a property that all behind it have too), or n.
template <typename F> __device__ int sf_first(SfShared& s, int n, F cuts) {
    if (threadIdx.x == 0) s.kept = n;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += SF_THREADS)
        if (cuts(s.list[i])) { atomicMin(&s.kept, i); break; }
    __syncthreads();
    const int kept = s.kept;
    __syncthreads();
    return kept;
}

// The whole choice from the first block's list of the n largest.
__device__ int sf_draw_from_list(SfShared& s, const SfRow& r, int n, int top_k, double top_p, double min_p, double u, SfTotal all) {
    sf_sort(s, n);
    int kept = n;
    if (top_k > 0 && top_k < n) {
        const unsigned kth = sf_key_of(s.list[top_k - 1]);
        kept = sf_first(s, n, [&](unsigned long long x) { return sf_key_of(x) < kth; });
    }
    if (top_p < 1.0) {
        if (top_k > 0) {                                 // the whole is what top_k left
            unsigned long long mine = 0, listed;
            for (int i = threadIdx.x; i < kept; i += SF_THREADS) mine += sf_fixed(r.weight(sf_value(sf_key_of(s.list[i]))));
            sf_scan(mine, s.warp_fixed, &listed);
            all = listed;
        }
        kept = sf_kept_by_weight(s, r, kept, 0, top_p, all);
    }
    if (min_p > 0.0) kept = sf_first(s, kept, [&](unsigned long long x) { return r.weight(sf_value(sf_key_of(x))) < min_p; });
    // In the vocabulary's order: the index above the key, turned around so that the largest entry is the lowest index.
    for (int i = threadIdx.x; i < kept; i += SF_THREADS) s.list[i] = (s.list[i] << 32) | (s.list[i] >> 32);
    sf_sort(s, kept);
    double e[SF_EACH], mine = 0.0, total;
#pragma unroll
    for (int j = 0; j < SF_EACH; ++j) {
        const int i = threadIdx.x * SF_EACH + j;
        e[j] = i < kept ? r.weight(sf_value((unsigned)s.list[i])) : 0.0;
        mine += e[j];
    }
    if (threadIdx.x == 0) { s.kept = kept; s.owner = -1; }
    double run = sf_scan(mine, s.warp_sum, &total) - mine;
    const double target = u * total;
#pragma unroll
    for (int j = 0; j < SF_EACH; ++j) {
        const int i = threadIdx.x * SF_EACH + j;
        run += e[j];
        if (e[j] > 0.0) {
            atomicMax(&s.owner, i);
            if (target < run) { atomicMin(&s.kept, i); break; }
        }
    }
    __syncthreads();
    const int at = s.kept < kept ? s.kept : s.owner;     // rounding left the target above the total: the last possible token
    return (int)~(unsigned)(s.list[at] >> 32);
}

// The exact cut inside the bins that a histogram found: every block leaves with it in `s.cut`. Every pass over the row adds up exactly what lies above the
// keys that are still in question (of the last pass's, that is) and lists those, or where they are too many counts them in bins of their own.
__device__ void sf_refine(cg::cluster_group& cluster, SfShared& s, const SfRow& r, SfBins bins, const SfCut cut, unsigned want, double top_p,
                          SfTotal all) {
    const bool by_weight = want == 0u;
    unsigned lo = max(cut.key, sf_key(SF_LOWEST)), hi = sf_key(r.largest);       // the keys in question; what lies above them:
    SfTotal weight_above = 0;
    unsigned above = 0;
    for (int level = 0; level < SF_LEVELS + 40; ++level) {       // (the last SF_LEVELS + 32nd has one key in question)
        const SfFound f = s.found;
        const unsigned within = f.upto - f.above;
        unsigned low = max(sf_key(bins.bottom(f.to)), lo), high = min(sf_key(bins.top(f.from)), hi);
        const float was = sf_value(hi);
        float least = sf_value(low), most = sf_value(high);
        const bool list = within <= (unsigned)SF_LIST;
        if (!list && by_weight && level > 0 && (bins.by_key ? high - low > (hi - lo) / 2 : most - least > 0.5f * (was - sf_value(lo)))) {
            // Bounds that leave more than half of what was in question (weights far apart in a bin): half of it, exactly.
            const unsigned middle = bins.by_key ? low + (high - low) / 2 : min(max(sf_key(0.5f * most + 0.5f * least), low), high - 1);
            const float half = sf_value(middle);
            unsigned long long a = 0, b = 0, na = 0, nb = 0;
            r.each(least, [&](int, float v) {
                if (v > was || v <= half) return;
                const unsigned long long w = sf_fixed(r.weight(v));
                if (v > most) { a += w; ++na; } else { b += w; ++nb; }
            });
            SfTotal wa, wb, ca, cb;
            sf_sum(cluster, s, a, b, wa, wb);
            cluster.sync();                              // the sums have been read
            sf_sum(cluster, s, na, nb, ca, cb);
            weight_above += wa;
            above += (unsigned)ca;
            if (sf_reached(weight_above + wb, top_p, all)) {
                low = middle + 1;
                least = sf_value(low);
            } else {
                weight_above += wb;
                above += (unsigned)cb;
                high = middle;
                most = half;
            }
            hi = high;
            cluster.sync();
        }
        const float top = sf_value(hi);
        bins = SfBins::between(low, high, level < SF_LEVELS);
        if (threadIdx.x == 0) s.listed = 0;
        sf_clear(s);
        unsigned long long weight = 0, number = 0;
        r.each(least, [&](int i, float v) {
            if (v > top) return;
            if (v > most) {
                if (by_weight) weight += sf_fixed(r.weight(v));
                ++number;
                return;
            }
            if (list) sf_list(s, sf_key(v), r.first + i);
            else atomicAdd(&s.counts[bins.of(v)], 1u);
        });
        SfTotal passed, count;
        sf_sum(cluster, s, weight, number, passed, count);
        weight_above += passed;
        above += (unsigned)count;
        lo = low;
        hi = high;
        if (list) {
            sf_collect(cluster, s);
            const int n = cluster.map_shared_rank(&s, 0)->listed;        // more than the bins held where their edges are not exact
            if (n <= SF_LIST) {
                if (cluster.block_rank() == 0) {
                    sf_sort(s, n);
                    int last;                            // the last entry that is left
                    if (by_weight) last = sf_kept_by_weight(s, r, n, weight_above, top_p, all) - 1;
                    else last = min(n - 1, max(0, (int)(want - above) - 1));
                    if (threadIdx.x == 0) {
                        SfCut c;
                        c.key = sf_key_of(s.list[last]);
                        c.index = by_weight ? (int)~(unsigned)s.list[last] : 0x7fffffff;
                        for (unsigned b = 0; b < cluster.num_blocks(); ++b) cluster.map_shared_rank(&s, b)->cut = c;
                    }
                }
                cluster.sync();
                return;
            }
            sf_clear(s);
            r.each(least, [&](int, float v) {
                if (v <= most) atomicAdd(&s.counts[bins.of(v)], 1u);
            });
        } else if (low == high) {                        // more equal tokens than the list holds
            SfCut c;
            c.key = low;
            c.index = 0x7fffffff;
            if (by_weight) {
                // The first `keep` of them: the smallest number that reaches top_p, one at least.
                const unsigned long long e = sf_fixed(r.weight(least));
                const int tied = (int)within;            // (after a halving fewer may be there: the count below stops at the last)
                int keep = tied;
                if (e > 0) {
                    for (int from = 1; from < keep;) {           // by halves
                        const int some = from + (keep - from) / 2;
                        if (sf_reached(weight_above + (SfTotal)some * e, top_p, all)) keep = some; else from = some + 1;
                    }
                }
                const int at = sf_locate(cluster, s, r, least, [&](int, float v) { return sf_key(v) == low ? 1.0 : 0.0; },
                                         [&](double) { return (double)keep - 0.5; });
                if (at >= 0)
                    for (unsigned b = 0; b < cluster.num_blocks(); ++b) cluster.map_shared_rank(&s, b)->cut = SfCut{low, r.first + at};
            } else if (threadIdx.x == 0) {
                s.cut = c;
            }
            cluster.sync();
            return;
        }
        sf_find(cluster, s, r, bins, want, top_p, above, weight_above, all, false);
    }
    if (threadIdx.x == 0) s.cut = SfCut{lo, 0x7fffffff};
    cluster.sync();
}

__global__ void __launch_bounds__(SF_THREADS, 1) sample_filtered_kernel(const SfParams p) {
    extern __shared__ __align__(16) unsigned char sf_smem[];
    SfShared& s = *reinterpret_cast<SfShared*>(sf_smem);
    float* cache = reinterpret_cast<float*>(sf_smem + (sizeof(SfShared) + 15) / 16 * 16);
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int row = blockIdx.x / blocks;
    const int tid = threadIdx.x;
    cluster.barrier_arrive();                            // behind the wait below every block runs and may be written to
    SfRow r;
    r.first = min(p.vocab, rank * p.share);
    r.n = min(p.vocab - r.first, p.share);
    r.cached = min(r.n, p.cached);
    r.row = p.logits + (size_t)row * p.vocab + r.first;
    const int ahead = (int)(((uintptr_t)r.row >> 2) & 3);
    cache += ahead;
    r.cache = cache;
    if (tid < 32) s.powers[tid] = exp2((double)tid / 32.0);          // before the barriers below
    const double temperature = p.temperature[row];
    const double top_p = p.top_p[row], min_p = p.min_p[row];
    const int top_k = p.top_k[row] > 0 && p.top_k[row] < p.vocab ? p.top_k[row] : 0;
    const double u = p.uniform[row];
    // The share, 16 bytes at a time where both the row and its place in shared memory allow (the cache begins as far behind a multiple of
    // 16 bytes as the share does). fmaxf passes over a NaN.
    float most = -INFINITY;
    bool nan = false;
    {
        const int head = min(r.n, (4 - ahead) & 3), fours = (r.n - head) / 4;
        const float4* src = reinterpret_cast<const float4*>(r.row + head);
        float4* dst = reinterpret_cast<float4*>(cache + head);
        const int kept = r.cached == r.n ? fours : (r.cached - head + 3) / 4;          // the last may reach three columns beyond
        for (int base = 0; base < fours; base += SF_BATCH) {
            float4 x[SF_DEEP];
#pragma unroll
            for (int k = 0; k < SF_DEEP; ++k) {
                const int i = base + k * SF_THREADS + tid;
                x[k] = i < fours ? src[i] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            }
#pragma unroll
            for (int k = 0; k < SF_DEEP; ++k) {
                const int i = base + k * SF_THREADS + tid;
                if (i < kept) dst[i] = x[k];
                most = fmaxf(fmaxf(fmaxf(most, x[k].x), fmaxf(x[k].y, x[k].z)), x[k].w);
                nan = nan || x[k].x != x[k].x || x[k].y != x[k].y || x[k].z != x[k].z || x[k].w != x[k].w;
            }
        }
        auto one = [&](int i) {
            const float v = r.row[i];
            if (i < r.cached) cache[i] = v;
            most = fmaxf(most, v);
            nan = nan || v != v;
        };
        if (tid < head) one(tid);
        for (int i = head + 4 * fours + tid; i < r.n; i += SF_THREADS) one(i);
    }
    const float own = most;                              // this thread's largest
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    unsigned low = __reduce_min_sync(0xffffffffu, own > -INFINITY ? sf_key(own) : 0xffffffffu);
    if ((tid & 31) == 0) { s.warp_max[tid >> 5] = most; s.warp_low[tid >> 5] = low; }
    nan = __syncthreads_or(nan);
    most = s.warp_max[tid & 31];
    low = __reduce_min_sync(0xffffffffu, s.warp_low[tid & 31]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    cluster.barrier_wait();
    if (tid < blocks) cluster.map_shared_rank(&s, tid)->tops[rank] = SfTop{most, nan ? 1 : 0, low};
    cluster.sync();
    for (int b = 0; b < blocks; ++b) {
        most = fmaxf(most, s.tops[b].v);
        nan = nan || s.tops[b].nan != 0;
        low = min(low, s.tops[b].low);
    }
    // Certain choices: greedy; a temperature that is no number leaves token 0, as a top_p that keeps nothing does; with a NaN among the
    // logits, an infinite one, or none above -inf the probabilities are none and the first largest stands.
    const bool greedy = temperature <= 0.0;
    if (greedy || !(temperature > 0.0) || top_p <= 0.0 || min_p > 1.0 || nan || isinf(most)) {
        const bool none = !greedy && (!(temperature > 0.0) || top_p <= 0.0 || (min_p > 1.0 && !nan && !isinf(most)));
        SfShared* home = cluster.map_shared_rank(&s, 0);
        if (rank == 0 && tid == 0) s.owner = 0x7fffffff;
        cluster.sync();
        int first = 0x7fffffff;
        for (int i = tid; i < r.n; i += SF_THREADS)
            if (r.at(i) == most) { first = r.first + i; break; }
        first = __reduce_min_sync(0xffffffffu, first);
        if ((tid & 31) == 0 && first != 0x7fffffff) atomicMin(&home->owner, first);
        cluster.sync();
        if (rank == 0 && tid == 0) p.tokens[row] = none || s.owner == 0x7fffffff ? 0 : s.owner;
        return;
    }
    r.scale(most, temperature, s.powers);
    SfCut cut;
    cut.key = 0u; cut.index = 0x7fffffff;
    SfBins bins;
    bins.by_key = false;
    bins.most = most;
    bins.least = SF_LOWEST;
    bins.step = (float)((SF_BINS - 1) * r.inv / SF_SPAN);
    bins.lo = bins.hi = 0u; bins.shift = 0;
    const bool by_p = top_p < 1.0;
    if (top_k > 0) {
        // The k-th may lie further below the largest than any weight that counts: here the bins reach down to the least of the threads' largest, or 200
        // below (some may have nothing but masked tokens).
        const float weights = bins.step;
        bins.step = (float)(SF_BINS - 1) / (most - fmaxf(sf_value(low), most - fmaxf(200.f, SF_SPAN / (float)fmax(r.inv, 1e-30))));
        if (top_k <= SF_LIST / 2) {
            sf_clear(s);
            if (own > -INFINITY) atomicAdd(&s.counts[bins.of(own)], 1u);
            sf_find(cluster, s, r, bins, (unsigned)top_k, 0.0, 0u, 0, 0, false);
            if (s.found.upto >= (unsigned)top_k) {
                const int down = s.found.to;
                sf_gather(cluster, s, r, bins, cut, down);
                const int listed = cluster.map_shared_rank(&s, 0)->listed;
                if (listed <= SF_LIST) {
                    cluster.sync();                      // the first block's count has been read
                    if (rank == 0) {
                        const int token = sf_draw_from_list(s, r, listed, top_k, by_p ? top_p : 1.0, min_p, u, 0);
                        if (tid == 0) p.tokens[row] = token;
                    }
                    return;
                }
            }
        }
        sf_clear(s);
        r.each(SF_LOWEST, [&](int, float v) { atomicAdd(&s.counts[bins.of(v)], 1u); });
        sf_find(cluster, s, r, bins, (unsigned)top_k, 0.0, 0u, 0, 0, false);
        if (s.found.upto <= (unsigned)SF_LIST) {
            const int n = (int)(s.found.upto);
            sf_gather(cluster, s, r, bins, cut, s.found.to);
            if (rank == 0) {
                const int token = sf_draw_from_list(s, r, n, top_k, by_p ? top_p : 1.0, min_p, u, 0);
                if (tid == 0) p.tokens[row] = token;
            }
            return;
        }
        sf_refine(cluster, s, r, bins, cut, (unsigned)top_k, 0.0, 0);
        cut = s.cut;
        bins.step = weights;
    }
    if (by_p) {
        sf_clear(s);
        unsigned long long mine = 0;
        SfTotal all, unused;
        const bool cuts = top_k > 0;
        r.each(sf_floor(cut), [&](int i, float v) {
            if (cuts && !sf_left(cut, sf_key(v), r.first + i)) return;
            atomicAdd(&s.counts[bins.of(v)], 1u);
            mine += sf_fixed(r.weight(v));
        });
        sf_sum(cluster, s, mine, 0ull, all, unused);
        sf_find(cluster, s, r, bins, 0u, top_p, 0u, 0, all, true);
        if (s.found.upto <= (unsigned)SF_LIST) {
            const int n = (int)(s.found.upto);
            sf_gather(cluster, s, r, bins, cut, s.found.to);
            if (rank == 0) {
                const int token = sf_draw_from_list(s, r, n, 0, top_p, min_p, u, all);
                if (tid == 0) p.tokens[row] = token;
            }
            return;
        }
        sf_refine(cluster, s, r, bins, cut, 0u, top_p, all);
        cut = s.cut;
    }
    // Below this a weight is under min_p for sure: no exponential.
    const double floor = min_p > 0.0 ? (double)most + log(min_p) / r.inv : -INFINITY;
    const float floor_v = min_p > 0.0 ? (float)(floor - 1e-5 * (fabs(floor) + fabs((double)most)) - 1e-30) : -INFINITY;
    const float sure_v = min_p > 0.0 ? (float)(floor + 1e-5 * (fabs(floor) + fabs((double)most)) + 1e-30) : -INFINITY;       // above this it is not, for sure
    const int at = sf_locate(cluster, s, r, fmaxf(sf_floor(cut), floor_v), [&](int i, float v) {
        if (!sf_left(cut, sf_key(v), r.first + i)) return 0.0;
        const double e = r.weight(v);
        return v < sure_v && e < min_p ? 0.0 : e;
    }, [&](double total) { return u * total; });
    if (at >= 0) p.tokens[row] = r.first + at;
    cluster.sync();                                      // nobody leaves while another may still write to it
}

}  // namespace kb

using namespace kb;

// No more blocks are tried for a row once half as many would have no more than this many columns each.
constexpr int SF_SHARE = 8192;

// Clusters of `blocks` blocks that run at once; asked for once a device (their blocks fill a multiprocessor whatever their share, and lie in one part of the
// chip: of eight blocks far fewer than the multiprocessors would hold).
static int active_clusters(int log_blocks, cudaLaunchConfig_t cfg, size_t smem) {
    static int known[64][4] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return 1;
    int n = device < 64 ? __atomic_load_n(&known[device][log_blocks], __ATOMIC_RELAXED) : 0;
    if (n > 0) return n;
    cfg.dynamicSmemBytes = smem;
    if (cudaOccupancyMaxActiveClusters(&n, sample_filtered_kernel, &cfg) != cudaSuccess || n < 1) { cudaGetLastError(); n = 1; }
    if (device < 64) __atomic_store_n(&known[device][log_blocks], n, __ATOMIC_RELAXED);
    return n;
}

extern "C" int kb_sample_filtered(int* tokens, const float* logits, const double* temperature, const int* top_k, const double* top_p,
                                  const double* min_p, const double* uniform, int rows, int vocab, void* stream) {
    KB_REQUIRE(rows >= 0 && vocab > 0, "sample_filtered: rows %d, vocab %d", rows, vocab);
    KB_REQUIRE(rows <= 0x7fffffff / SF_MAX_CLUSTER, "sample_filtered: %d rows is too many for one launch", rows);
    KB_REQUIRE(vocab <= (1 << 19), "sample_filtered: a vocabulary of %d (up to %d: a row's weights are added in 64 bits)", vocab, 1 << 19);
    KB_REQUIRE(rows == 0 || (tokens && logits && temperature && top_k && top_p && min_p && uniform), "sample_filtered: a null pointer");
    if (rows == 0) return 0;
    SfParams p = {};
    p.tokens = tokens; p.logits = logits; p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p; p.uniform = uniform;
    p.rows = rows; p.vocab = vocab;
    constexpr int MOST = 232448 - 1024;
    constexpr int FIXED = (int)((sizeof(SfShared) + 15) / 16 * 16) + 32;
    constexpr int CACHED = (MOST - FIXED) / 4 / SF_BATCH * SF_BATCH;
    static_assert(CACHED > 0, "the histogram and the list leave no room for a share");
    static unsigned long long done = 0;
    if (int e = allow_shared_memory((const void*)sample_filtered_kernel, MOST, &done)) return e;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(SF_THREADS);
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    // Blocks a row: as many as make the rows' time least, which is the rounds of clusters times some 16 us and 0.45 ns a column of a share (what a
    // nucleus takes). 15 clusters of eight run at once, 33 of four, 74 of two, 148 of one. As measured under a nucleus of 0.95 (us; the logits of the figures above): 256,000 columns,
    // of 12 rows 27 by eight blocks a row and 38 by four, of 16 rows 49 and 38, of 64 rows 116 and 76; 50,257 columns, of 12 rows 18, 20, 24 and 33 by
    // eight, four, two and one, of 40 rows 46, 35, 25 and 34, of 256 rows 249, 141, 94 and 66. (Blocks of 512 threads, two a multiprocessor, eight a row of
    // 256,000: 46 of 32 rows where four of 1,024 take 39, 85 of 64 where those take 76.)
    int blocks = 1;
    double least = 0.0;
    for (int log_blocks = 0; log_blocks < 4; ++log_blocks) {
        const int n = 1 << log_blocks, share = (vocab + n - 1) / n;
        if (n > 1 && n / 2 * SF_SHARE >= vocab) break;       // half as many have small shares already
        if (share > SF_ROWS * SF_THREADS) continue;
        attr[0].val.clusterDim.x = (unsigned)n;
        cfg.gridDim = dim3((unsigned)n);
        const int at_once = rows == 1 ? 1 : active_clusters(log_blocks, cfg, MOST);
        const double us = (double)((rows + at_once - 1) / at_once) * (16.0 + 0.45e-3 * share);
        if (least == 0.0 || us < least) { least = us; blocks = n; }
    }
    p.share = (vocab + blocks - 1) / blocks;
    p.cached = p.share <= (MOST - FIXED) / 4 ? p.share : CACHED;
    attr[0].val.clusterDim.x = (unsigned)blocks;
    cfg.gridDim = dim3((unsigned)(rows * blocks));
    cfg.dynamicSmemBytes = (size_t)FIXED + (size_t)p.cached * 4;
    cudaLaunchKernelEx(&cfg, sample_filtered_kernel, p);
    return check_launch("sample_filtered");
}

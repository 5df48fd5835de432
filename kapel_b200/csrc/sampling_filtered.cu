// A draw under temperature, top_k, top_p and min_p where the logits are, a row's settings and uniform number its own.
//
// The rules are the host sampler's (csrc/host/sampler_core.cpp; crates/kapel-infer/src/sampling.rs:157-260), in its order: x = logit /
// temperature; top_k keeps what is no smaller than the k-th largest (its ties stay); top_p keeps, the likeliest first and the lower index
// first among equals, the tokens before which the others hold less than top_p; min_p keeps p >= min_p p_max; the draw is the first index
// whose running total over what is left exceeds u times the whole. All three filters cut the same order (x down, index up), so what is
// left is always "above a cut (key, index)".
//
// A row is one cluster's: its blocks read the row once and keep their shares in shared memory; everything after works on chip.
//   1. The largest logit, whether a NaN is there.
//   2. For top_k or top_p a histogram over 2,048 bins of equal steps of x below the largest: counts, and for top_p the sums of e^(x - max)
//      in fixed point (44 bits behind the point: whole numbers, so the order of the atomics changes nothing; a row's sum, 2^18
//      tokens, fits 64 bits). The bins are added up in the cluster's first block, which finds the bin the cut falls in.
//   3. Where the bins down to there hold no more than LIST tokens (a top_k, a peaked nucleus), they are gathered in the first block,
//      sorted, cut and drawn from there. Otherwise only the bin of the cut is gathered and sorted to find the cut (a bin too full
//      for that is divided again between its smallest and largest key), and the draw goes over the whole share of every block.
// e^x is in 64 bits, and so are the draw's sums, as on the host: a seed gives the tokens it gave there, but for borders that lie within a
// few units of the 13th digit.
#include <cooperative_groups.h>
#include "sampling.cuh"

namespace kb {
namespace cg = cooperative_groups;

constexpr int SF_THREADS = 1024, SF_WARPS = SF_THREADS / 32;
constexpr int SF_BINS = 2048, SF_LIST = 2048, SF_MAX_CLUSTER = 8;
constexpr float SF_SPAN = 24.f;                          // the bins reach e^-24 below the largest; the last holds all that is below
constexpr double SF_FIXED = 17592186044416.0;            // 2^44

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
    int cached;                                          // of them in shared memory; the rest is read again from the row
};

struct SfTop { Best best; int nan; int unused; };
struct SfCut { unsigned key; int index; };               // what is left: key above, or equal and the index no larger
struct SfFound {                                         // what the first block tells the others about a histogram
    int bin, in_bin;                                     // the cut's bin and how many tokens it holds
    unsigned upto;                                       // tokens in the bins down to and with it
    unsigned above;                                      // tokens above it
    unsigned long long weight_above, weight_all;
};

struct SfShared {
    unsigned counts[SF_BINS];
    unsigned long long weights[SF_BINS];
    unsigned long long list[SF_LIST];                    // first block: key << 32 | ~index, the largest first once sorted
    SfTop tops[SF_MAX_CLUSTER];
    double sums[SF_MAX_CLUSTER];
    double warp_sum[SF_WARPS];
    unsigned long long warp_fixed[SF_WARPS];
    unsigned warp_count[SF_WARPS];
    SfFound found;
    SfCut cut;
    unsigned lo_key, hi_key;                             // the smallest and largest key of a bin
    int listed;
    int owner;
    int kept;
    Best best[32];
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
    int n, cached, first;                                // columns of the share, how many are in `cache`, the share's first column
    double inv;                                          // 1 / temperature
    float largest;
    __device__ __forceinline__ float at(int i) const { return i < cached ? cache[i] : row[i]; }
    __device__ __forceinline__ double weight(float v) const { return exp(((double)v - (double)largest) * inv); }
};

__device__ __forceinline__ bool sf_left(const SfCut& cut, unsigned key, int index) {
    return key > cut.key || (key == cut.key && index <= cut.index);
}

// A level's bins: equal steps below the largest at first, then equal steps of the key between two keys.
struct SfBins {
    bool by_key;
    float largest, step;                                 // bin = (largest - v) step
    unsigned lo, hi;                                     // keys that count; bin = (hi - key) >> shift
    int shift;
    __device__ __forceinline__ int of(float v, unsigned key) const {
        if (key < lo || key > hi) return -1;
        if (by_key) return (int)((hi - key) >> shift);
        const float x = (largest - v) * step;
        return x < (float)(SF_BINS - 1) ? (int)x : (x == x ? SF_BINS - 1 : 0);
    }
};

// Sorts list[0 .. n), largest first; n up to SF_LIST, padded with zeros to a power of two.
__device__ void sf_sort(unsigned long long* list, int n) {
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = threadIdx.x; i < size; i += SF_THREADS)
        if (i >= n) list[i] = 0ull;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int t = threadIdx.x; t < size / 2; t += SF_THREADS) {
                const int i = (t / j) * 2 * j + t % j;
                const unsigned long long a = list[i], b = list[i + j];
                if (((i & k) == 0) ? a < b : a > b) { list[i] = b; list[i + j] = a; }
            }
            __syncthreads();
        }
}

// run >= top_p all, the product not rounded before it is compared: equal weights reach a round share of the whole exactly.
__device__ __forceinline__ bool sf_reached(unsigned long long run, double top_p, unsigned long long all) {
    return fma(top_p, (double)all, -(double)run) <= 0.0;
}
__device__ __forceinline__ unsigned long long sf_fixed(double e) { return (unsigned long long)(e * SF_FIXED + 0.5); }

// The bins' histogram over what is left, added up in the first block; there the bin of the cut is found: the first in which the count
// down to it reaches `want`, or, by weight, in which the weight down to it reaches top_p of the whole. `base` (count, weight) lies above
// the level's keys. Every block leaves with the answer in `found`.
__device__ void sf_histogram(cg::cluster_group& cluster, SfShared& s, const SfRow& r, const SfBins& bins, const SfCut& cut, bool by_weight,
                             unsigned want, double top_p, unsigned base_count, unsigned long long base_weight, unsigned long long all_weight) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i = tid; i < SF_BINS; i += SF_THREADS) { s.counts[i] = 0u; s.weights[i] = 0ull; }
    __syncthreads();
    for (int i = tid; i < r.n; i += SF_THREADS) {
        const float v = r.at(i);
        if (!(v > -INFINITY)) continue;
        const unsigned key = sf_key(v);
        if (!sf_left(cut, key, r.first + i)) continue;
        const int b = bins.of(v, key);
        if (b < 0) continue;
        atomicAdd(&s.counts[b], 1u);
        if (by_weight) atomicAdd(&s.weights[b], sf_fixed(r.weight(v)));
    }
    cluster.sync();
    SfShared* home = cluster.map_shared_rank(&s, 0);
    if (cluster.block_rank() != 0) {
        for (int i = tid; i < SF_BINS; i += SF_THREADS) {
            const unsigned c = s.counts[i];
            if (c == 0u) continue;
            atomicAdd(&home->counts[i], c);
            if (by_weight) atomicAdd(&home->weights[i], s.weights[i]);
        }
    }
    cluster.sync();
    if (cluster.block_rank() == 0) {
        constexpr int EACH = SF_BINS / SF_THREADS;
        unsigned c[EACH], count = 0;
        unsigned long long w[EACH], weight = 0;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            c[j] = s.counts[tid * EACH + j];
            w[j] = by_weight ? s.weights[tid * EACH + j] : 0ull;
            count += c[j];
            weight += w[j];
        }
        unsigned upto_c = count;
        unsigned long long upto_w = weight;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned yc = __shfl_up_sync(0xffffffffu, upto_c, o);
            const unsigned long long yw = __shfl_up_sync(0xffffffffu, upto_w, o);
            if (lane >= o) { upto_c += yc; upto_w += yw; }
        }
        if (lane == 31) { s.warp_count[warp] = upto_c; s.warp_fixed[warp] = upto_w; }
        if (tid == 0) s.owner = SF_BINS;
        __syncthreads();
        unsigned long long all = base_weight;
        unsigned before_c = base_count;
        unsigned long long before_w = base_weight;
        for (int k = 0; k < SF_WARPS; ++k) {
            if (k < warp) { before_c += s.warp_count[k]; before_w += s.warp_fixed[k]; }
            all += s.warp_fixed[k];
        }
        if (all_weight) all = all_weight;                // a deeper level: the whole is the first level's
        before_c += upto_c - count;
        before_w += upto_w - weight;
        int mine = -1;
        unsigned above = before_c;
        unsigned long long above_w = before_w;
        unsigned run_c = before_c;
        unsigned long long run_w = before_w;
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const unsigned next_c = run_c + c[j];
            const unsigned long long next_w = run_w + w[j];
            if (mine < 0 && c[j] && (by_weight ? sf_reached(next_w, top_p, all) : next_c >= want)) { mine = tid * EACH + j; above = run_c; above_w = run_w; }
            run_c = next_c;
            run_w = next_w;
        }
        if (mine >= 0) atomicMin(&s.owner, mine);
        __syncthreads();
        // No bin reaches it (fewer tokens than `want`, or rounding): the last bin that holds a token.
        const bool none = s.owner == SF_BINS;
        __syncthreads();
        if (none) {
            int last = -1;
            run_c = before_c; run_w = before_w;
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                if (c[j]) { last = tid * EACH + j; above = run_c; above_w = run_w; }
                run_c += c[j];
                run_w += w[j];
            }
            mine = last;
            if (tid == 0) s.owner = -1;
            __syncthreads();
            if (last >= 0) atomicMax(&s.owner, last);
            __syncthreads();
        }
        if (mine >= 0 && mine == s.owner) {
            unsigned in = 0;
#pragma unroll
            for (int j = 0; j < EACH; ++j) if (tid * EACH + j == mine) in = c[j];
            SfFound f;
            f.bin = mine; f.in_bin = (int)in; f.above = above; f.upto = above + in; f.weight_above = above_w; f.weight_all = all;
            for (unsigned b = 0; b < cluster.num_blocks(); ++b) cluster.map_shared_rank(&s, b)->found = f;
        }
    }
    cluster.sync();
}

// What is left in the bins from `from` to `to` into the first block's list.
__device__ void sf_gather(cg::cluster_group& cluster, SfShared& s, const SfRow& r, const SfBins& bins, const SfCut& cut, int from, int to) {
    SfShared* home = cluster.map_shared_rank(&s, 0);
    if (cluster.block_rank() == 0 && threadIdx.x == 0) s.listed = 0;
    cluster.sync();
    const int lane = threadIdx.x & 31;
    for (int base = 0; base < r.n; base += SF_THREADS) {
        const int i = base + (int)threadIdx.x;
        bool in = false;
        unsigned key = 0;
        if (i < r.n) {
            const float v = r.at(i);
            if (v > -INFINITY) {
                key = sf_key(v);
                const int b = sf_left(cut, key, r.first + i) ? bins.of(v, key) : -1;
                in = b >= from && b <= to;
            }
        }
        const unsigned who = __ballot_sync(0xffffffffu, in);
        if (who == 0u) continue;
        int at = 0;
        if (lane == __ffs(who) - 1) at = atomicAdd(&home->listed, __popc(who));
        at = __shfl_sync(0xffffffffu, at, __ffs(who) - 1) + __popc(who & ((1u << lane) - 1u));
        if (in && at < SF_LIST) home->list[at] = ((unsigned long long)key << 32) | (unsigned)~(r.first + i);
    }
    cluster.sync();
}

// The first index, over the whole row in order, whose running total of `weight_of` exceeds the target that `target_of` makes of
// the whole; the last index with a weight where rounding leaves the target at or above it. -1 in every block but the one that has it.
template <typename W, typename T>
__device__ int sf_locate(cg::cluster_group& cluster, SfShared& s, const SfRow& r, W weight_of, T target_of) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int each = ((r.n + SF_WARPS - 1) / SF_WARPS + 31) / 32 * 32;      // a warp's columns lie together: totals follow their order
    const int begin = min(r.n, warp * each), end = min(r.n, begin + each);
    double local = 0.0;
    for (int i = begin + lane; i < end; i += 32) local += weight_of(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) local += __shfl_xor_sync(0xffffffffu, local, o);
    if (lane == 0) s.warp_sum[warp] = local;
    __syncthreads();
    if (tid == 0) {
        double mine = 0.0;
        for (int w = 0; w < SF_WARPS; ++w) mine += s.warp_sum[w];
        for (unsigned b = 0; b < cluster.num_blocks(); ++b) cluster.map_shared_rank(&s, b)->sums[cluster.block_rank()] = mine;
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
    int pick = -1;
    if (owner == (int)cluster.block_rank()) {
        int mine = -1, last_warp = -1;
        double warp_before = 0.0;
        run = before;
        for (int w = 0; w < SF_WARPS; ++w) {
            const double next = run + s.warp_sum[w];
            if (s.warp_sum[w] > 0.0) { last_warp = w; if (mine < 0 && !beyond && target < next) { mine = w; warp_before = run; } }
            run = next;
        }
        bool to_end = beyond || mine < 0;                // the crossing hid in rounding: the last possible token
        if (to_end) mine = last_warp;
        if (warp == mine) {
            run = warp_before;
            int seen = -1;
            for (int base = begin; base < end && pick < 0; base += 32) {
                const int i = base + lane;
                const double e = i < end ? weight_of(i) : 0.0;
                double upto = e;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double y = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += y;
                }
                const unsigned some = __ballot_sync(0xffffffffu, e > 0.0);
                const unsigned passed = __ballot_sync(0xffffffffu, e > 0.0 && !to_end && target < run + upto);
                if (some) seen = base + 31 - __clz(some);
                if (passed) pick = base + __ffs(passed) - 1;
                run += __shfl_sync(0xffffffffu, upto, 31);
            }
            if (pick < 0) pick = seen;
            if (lane != 0) pick = -1;
        }
    }
    return pick;
}

// Inclusive running totals over the block, in thread order.
template <typename V> __device__ V sf_scan(V v, V* per_warp, V* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    __syncthreads();
    if (lane == 31) per_warp[warp] = v;
    __syncthreads();
    V before = 0, all = 0;
    for (int w = 0; w < SF_WARPS; ++w) {
        if (w < warp) before += per_warp[w];
        all += per_warp[w];
    }
    *total = all;
    return before + v;
}

constexpr int SF_EACH = SF_LIST / SF_THREADS;            // entries of the list a thread has

__device__ __forceinline__ unsigned sf_key_of(unsigned long long entry) { return (unsigned)(entry >> 32); }

// Of the sorted list's first n entries, how many are left where the weight before each must be below top_p of `all` (`above` lies before the
// first).
__device__ int sf_kept_by_weight(SfShared& s, const SfRow& r, int n, unsigned long long above, double top_p, unsigned long long all) {
    unsigned long long w[SF_EACH], mine = 0, listed;
#pragma unroll
    for (int j = 0; j < SF_EACH; ++j) {
        const int i = threadIdx.x * SF_EACH + j;
        w[j] = i < n ? sf_fixed(r.weight(sf_value(sf_key_of(s.list[i])))) : 0ull;
        mine += w[j];
    }
    if (threadIdx.x == 0) s.kept = n;
    unsigned long long run = above + sf_scan(mine, s.warp_fixed, &listed) - mine;
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

// The whole choice from the first block's list of the n largest.
__device__ int sf_draw_from_list(SfShared& s, const SfRow& r, int n, int top_k, double top_p, double min_p, double u, unsigned long long all) {
    sf_sort(s.list, n);
    int kept = n;
    if (top_k > 0 && top_k < n) {
        const unsigned kth = sf_key_of(s.list[top_k - 1]);
        if (threadIdx.x == 0) s.kept = n;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += SF_THREADS)
            if (sf_key_of(s.list[i]) < kth) atomicMin(&s.kept, i);
        __syncthreads();
        kept = s.kept;
        __syncthreads();
    }
    if (top_p < 1.0) {
        if (top_k > 0) {                                 // the whole is what top_k left
            unsigned long long mine = 0;
            for (int i = threadIdx.x; i < kept; i += SF_THREADS) mine += sf_fixed(r.weight(sf_value(sf_key_of(s.list[i]))));
            sf_scan(mine, s.warp_fixed, &all);
        }
        kept = sf_kept_by_weight(s, r, kept, 0ull, top_p, all);
    }
    if (min_p > 0.0) {
        if (threadIdx.x == 0) s.kept = kept;
        __syncthreads();
        for (int i = threadIdx.x; i < kept; i += SF_THREADS)
            if (r.weight(sf_value(sf_key_of(s.list[i]))) < min_p) atomicMin(&s.kept, i);
        __syncthreads();
        kept = s.kept;
        __syncthreads();
    }
    // In the vocabulary's order: the index above the key, turned around so that the largest entry is the lowest index.
    for (int i = threadIdx.x; i < kept; i += SF_THREADS) s.list[i] = (s.list[i] << 32) | (s.list[i] >> 32);
    __syncthreads();
    sf_sort(s.list, kept);
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

// The exact cut inside the bin that a histogram found: every block leaves with it in `s.cut`.
__device__ void sf_refine(cg::cluster_group& cluster, SfShared& s, const SfRow& r, SfBins bins, const SfCut cut, bool by_weight, unsigned want, double top_p) {
    SfShared* home = cluster.map_shared_rank(&s, 0);
    for (;;) {
        const SfFound f = s.found;
        if (f.in_bin <= SF_LIST) {
            sf_gather(cluster, s, r, bins, cut, f.bin, f.bin);
            if (cluster.block_rank() == 0) {
                const int n = f.in_bin;
                sf_sort(s.list, n);
                int last;                                // the last entry that is left
                if (by_weight) last = sf_kept_by_weight(s, r, n, f.weight_above, top_p, f.weight_all) - 1;
                else last = min(n - 1, max(0, (int)(want - f.above) - 1));
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
        if (cluster.block_rank() == 0 && threadIdx.x == 0) { s.lo_key = 0xffffffffu; s.hi_key = 0u; }
        cluster.sync();
        unsigned lo = 0xffffffffu, hi = 0u;
        for (int i = threadIdx.x; i < r.n; i += SF_THREADS) {
            const float v = r.at(i);
            if (!(v > -INFINITY)) continue;
            const unsigned key = sf_key(v);
            if (!sf_left(cut, key, r.first + i) || bins.of(v, key) != f.bin) continue;
            lo = min(lo, key);
            hi = max(hi, key);
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        if ((threadIdx.x & 31) == 0 && lo <= hi) { atomicMin(&home->lo_key, lo); atomicMax(&home->hi_key, hi); }
        cluster.sync();
        lo = home->lo_key;
        hi = home->hi_key;
        cluster.sync();
        if (lo == hi) {                                  // more equal tokens than the list holds
            SfCut c;
            c.key = lo;
            c.index = 0x7fffffff;
            if (by_weight) {
                // The first `keep` of them: the smallest number that reaches top_p. The bin holds it, so it is one at least.
                const unsigned long long e = sf_fixed(r.weight(sf_value(lo)));
                int keep = f.in_bin;
                if (e > 0) {
                    const double some = ceil((top_p * (double)f.weight_all - (double)f.weight_above) / (double)e);
                    keep = (int)fmin(fmax(some, 1.0), (double)f.in_bin);
                    while (keep > 1 && sf_reached(f.weight_above + (unsigned long long)(keep - 1) * e, top_p, f.weight_all)) --keep;
                    while (keep < f.in_bin && !sf_reached(f.weight_above + (unsigned long long)keep * e, top_p, f.weight_all)) ++keep;
                }
                const int at = sf_locate(cluster, s, r, [&](int i) {
                    const float v = r.at(i);
                    return v > -INFINITY && sf_key(v) == lo && sf_left(cut, lo, r.first + i) ? 1.0 : 0.0;
                }, [&](double) { return (double)keep - 0.5; });
                if (at >= 0)
                    for (unsigned b = 0; b < cluster.num_blocks(); ++b) cluster.map_shared_rank(&s, b)->cut = SfCut{lo, r.first + at};
            } else if (threadIdx.x == 0) {
                s.cut = c;
            }
            cluster.sync();
            return;
        }
        bins.by_key = true;
        bins.lo = lo;
        bins.hi = hi;
        bins.shift = 0;
        while (((hi - lo) >> bins.shift) >= (unsigned)SF_BINS) ++bins.shift;
        sf_histogram(cluster, s, r, bins, cut, by_weight, want, top_p, f.above, f.weight_above, f.weight_all);
    }
}

__global__ void __launch_bounds__(SF_THREADS, 1) sample_filtered_kernel(const SfParams p) {
    extern __shared__ __align__(16) unsigned char sf_smem[];
    SfShared& s = *reinterpret_cast<SfShared*>(sf_smem);
    float* cache = reinterpret_cast<float*>(sf_smem + sizeof(SfShared));
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
    r.cache = cache;
    Best mine;
    mine.v = 0.f; mine.i = -1;
    bool nan = false;
#pragma unroll 8
    for (int i = tid; i < r.n; i += SF_THREADS) {
        const float v = r.row[i];
        if (i < r.cached) cache[i] = v;
        if (v != v) { nan = true; continue; }
        Best c;
        c.v = v; c.i = r.first + i;
        mine = better(mine, c);
    }
    nan = __syncthreads_or(nan);
    mine = block_best(mine, s.best);
    cluster.barrier_wait();
    if (tid < blocks) {
        SfTop t;
        t.best = mine; t.nan = nan ? 1 : 0; t.unused = 0;
        cluster.map_shared_rank(&s, tid)->tops[rank] = t;
    }
    cluster.sync();
    Best top;
    top.v = 0.f; top.i = -1;
    for (int b = 0; b < blocks; ++b) {
        top = better(top, s.tops[b].best);
        nan = nan || s.tops[b].nan != 0;
    }
    const double temperature = p.temperature[row];
    const double top_p = p.top_p[row], min_p = p.min_p[row];
    const int top_k = p.top_k[row] > 0 && p.top_k[row] < p.vocab ? p.top_k[row] : 0;
    const double u = p.uniform[row];
    // Certain choices: greedy; a temperature that is no number leaves token 0, as a top_p that keeps nothing does; with a NaN among the
    // logits, an infinite one, or none above -inf the probabilities are none and the first largest stands.
    const bool greedy = temperature <= 0.0;
    if (greedy || !(temperature > 0.0) || top_p <= 0.0 || min_p > 1.0 || nan || top.i < 0 || isinf(top.v)) {
        const bool none = !greedy && (!(temperature > 0.0) || top_p <= 0.0 || (min_p > 1.0 && !nan && !isinf(top.v)));
        if (rank == 0 && tid == 0) p.tokens[row] = none || top.i < 0 ? 0 : top.i;
        return;
    }
    r.largest = top.v;
    r.inv = isinf(temperature) ? 0.0 : fmin(1.0 / temperature, 1e300);
    SfCut cut;
    cut.key = 0u; cut.index = 0x7fffffff;
    SfBins bins;
    bins.by_key = false;
    bins.largest = top.v;
    bins.step = (float)((SF_BINS - 1) * r.inv / SF_SPAN);
    bins.lo = 0u; bins.hi = 0xffffffffu; bins.shift = 0;
    bool by_k = top_k > 0, by_p = top_p < 1.0;
    while (by_k || by_p) {
        const bool by_weight = !by_k;
        sf_histogram(cluster, s, r, bins, cut, by_weight, (unsigned)top_k, top_p, 0u, 0ull, 0ull);
        const SfFound f = s.found;
        if (f.upto <= (unsigned)SF_LIST) {
            sf_gather(cluster, s, r, bins, cut, 0, f.bin);
            if (rank == 0) {
                const int token = sf_draw_from_list(s, r, (int)f.upto, by_k ? top_k : 0, by_p ? top_p : 1.0, min_p, u, f.weight_all);
                if (tid == 0) p.tokens[row] = token;
            }
            return;
        }
        sf_refine(cluster, s, r, bins, cut, by_weight, (unsigned)top_k, top_p);
        cut = s.cut;
        if (by_k) by_k = false; else by_p = false;
    }
    // Below this a weight is under min_p for sure: no exponential.
    const double floor = min_p > 0.0 ? (double)top.v + log(min_p) / r.inv : -INFINITY;
    const float floor_v = min_p > 0.0 ? (float)(floor - 1e-5 * (fabs(floor) + fabs((double)top.v)) - 1e-30) : -INFINITY;
    const int at = sf_locate(cluster, s, r, [&](int i) {
        const float v = r.at(i);
        if (!(v > -INFINITY) || v < floor_v || !sf_left(cut, sf_key(v), r.first + i)) return 0.0;
        const double e = r.weight(v);
        return e < min_p ? 0.0 : e;
    }, [&](double total) { return u * total; });
    if (at >= 0) p.tokens[row] = r.first + at;
    cluster.sync();                                      // nobody leaves while another may still write to it
}

}  // namespace kb

using namespace kb;

// Blocks a row: a share of at most SF_SHARE columns each, up to a cluster of eight.
constexpr int SF_SHARE = 8192;

extern "C" int kb_sample_filtered(int* tokens, const float* logits, const double* temperature, const int* top_k, const double* top_p,
                                  const double* min_p, const double* uniform, int rows, int vocab, void* stream) {
    KB_REQUIRE(rows >= 0 && vocab > 0, "sample_filtered: rows %d, vocab %d", rows, vocab);
    KB_REQUIRE(rows <= 0x7fffffff / SF_MAX_CLUSTER, "sample_filtered: %d rows is too many for one launch", rows);
    KB_REQUIRE(vocab <= (1 << 19), "sample_filtered: a vocabulary of %d (up to %d: a row's weights are added in 64 bits)", vocab, 1 << 19);
    KB_REQUIRE(rows == 0 || (tokens && logits && temperature && top_k && top_p && min_p && uniform), "sample_filtered: a null pointer");
    if (rows == 0) return 0;
    int blocks = 1;
    while (blocks < SF_MAX_CLUSTER && (long long)blocks * SF_SHARE < vocab) blocks *= 2;
    SfParams p = {};
    p.tokens = tokens; p.logits = logits; p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p; p.uniform = uniform;
    p.rows = rows; p.vocab = vocab;
    p.share = (vocab + blocks - 1) / blocks;
    constexpr int MOST = 232448 - 1024;
    static_assert(sizeof(SfShared) + 65536 <= MOST, "the histogram and the list leave no room for a share");
    p.cached = (int)(((size_t)MOST - sizeof(SfShared)) / 4);
    if (p.cached > p.share) p.cached = p.share;
    const size_t smem = sizeof(SfShared) + (size_t)p.cached * 4;
    const cudaError_t e = cudaFuncSetAttribute(sample_filtered_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST);
    KB_REQUIRE(e == cudaSuccess, "sample_filtered: cannot have %d bytes of shared memory: %s", MOST, cudaGetErrorString(e));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * blocks));
    cfg.blockDim = dim3(SF_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)blocks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, sample_filtered_kernel, p);
    return check_launch("sample_filtered");
}

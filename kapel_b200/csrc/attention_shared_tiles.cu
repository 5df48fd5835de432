// What requests share, read once for all of them, on the fifth-generation tensor cores (bfloat16; see attention_shared.cuh for the cut).
//
// A tile is up to 128 (request, query head) pairs of one kv head; a block a multiprocessor walks its units, KEYS positions each, whatever tiles they
// belong to:
//   S = Q K^T   tcgen05.mma, Q [128 x D] and the keys [KEYS x D] K-major in shared memory (128-byte swizzle), S float32 in one of three
//               TMEM buffers;
//   P = 2^(score - m) by sixteen warps, four to each quarter of the pairs, a quarter of the unit's positions each (with eight warps the
//               multiprocessor issued 1.7 instructions a clock); written over S as bfloat16;
//   O += P V    tcgen05.mma, P from TMEM, the values [KEYS x D] an MN-major operand; O float32 stays in TMEM until the block's part of
//               the tile ends, when it goes out as a piece.
// m is a score of the pair that none seen so far passes by more than 2^ST_LAG; where a unit does, the quarter's warps wait for the product before,
// scale O in TMEM and go on. (With m the largest so far some of a warp's 32 pairs raise it in nearly every unit of the first thousands of
// positions, and scaling O of 256 components takes longer than all the rest of a unit. The weights are rounded relative to themselves, so
// larger ones lose nothing; only the largest of a pair, no longer exactly 1, is rounded as well.) The
// next tile's queries are laid out as soon as the last score product of this one is complete, so its products run while this one's O is read out.
//
// Warp 0 brings keys, 19 values (TMA, 16 positions x 64 elements a box, a box a lane); 1 allocates TMEM and issues the score products, 18
// the others; 2 to 17 are the softmax's. Every wait gives up after about a second, raises a flag and the block still frees its TMEM.
//
// What bounds it: 128 requests behind 16,384 positions, 32 heads over 16 of 128 (two tiles a kv head): 69 us, 500 Tflop/s. A unit of 128 positions takes
// 3,200 clocks where its exponentials take 1,024 and its products as many: the sixteen warps wait for the same scores, load them, agree on m
// and write their weights at the same time. In tiles of few pairs it is the softmax of the quarter that is not full: its places without a pair see no position, so its
// warps take every unit for one that not all of their pairs see, score by score (two exponentials and a reciprocal each under a soft cap). Before the first scores a block takes some 7 us (the cut, the queries), which is most of what a tile
// of few units costs.
#include "attention_shared_bf16.cuh"
#include "tensor_map.cuh"

namespace kb {

constexpr int ST_PAIRS = 128, ST_SOFT = 16, ST_THREADS = (ST_SOFT + 4) * 32, ST_S = 3;
constexpr int ST_WARP_PV = ST_SOFT + 2, ST_WARP_V = ST_SOFT + 3;
constexpr float ST_LAG = 8.f;

template <int D> struct TilesCfg {
    static constexpr int KEYS = D == 256 ? 64 : 128;
    static constexpr int CH = D / 64;                        // chunks of 64 elements
    static constexpr int Q_BYTES = ST_PAIRS * D * 2, KV_BYTES = KEYS * D * 2;
    static constexpr int RING = D == 64 ? 4 : 2;             // units of keys, and of values
    static constexpr int COL_S = D, TMEM_COLS = 512;
    static constexpr int BARS = 4 * RING + 3 * ST_S + 2;
    static constexpr int SMEM = 1024 + Q_BYTES + 2 * RING * KV_BYTES + BARS * 8 + 8 + 2 * 4 * ST_PAIRS * 4 + (int)sizeof(SharedTiles);
    static_assert(D + ST_S * KEYS <= TMEM_COLS, "O and the S buffers outgrew TMEM");
    static_assert(SMEM <= 232448, "more shared memory than a block can have");
};

// One tile and kv head's part of a block's range.
struct TilePart { int row0, n, looks, kvh, lo, hi, first, units; long long place; };
__device__ __forceinline__ TilePart st_part(const SharedParams& p, const SharedTiles& c, int u, int end) {
    TilePart w;
    const int item = shared_item(c.upto, c.tiles, p.hkv, u);
    const int units = c.upto[item + 1] - c.upto[item], in = u - c.upto[item] * p.hkv;
    w.kvh = in / units;
    w.first = in % units;
    w.units = min(units - w.first, end - u);
    w.row0 = c.row0[item]; w.n = c.n[item]; w.looks = c.looks[item]; w.lo = c.klo[item]; w.hi = c.khi[item];
    w.place = shared_tile_place(p, c.before[item], w.n, w.kvh, blockIdx.x, ST_PAIRS);
    return w;
}

// A part's queries by the softmax's warps, K-major under the swizzle: chunk c of pair r at c 16 KB + r 128, its 16-byte pieces exchanged by r mod 8.
// Eight neighbouring threads bring a pair's 128 bytes, up to eight pieces each asked for at a time. Pairs that are none keep what is there: nobody
// reads their results.
template <int D> __device__ __forceinline__ void st_queries(const SharedParams& p, const TilePart& w, unsigned char* q_smem, uint64_t* q_full) {
    constexpr int CH = TilesCfg<D>::CH, ITER = ST_PAIRS * CH * 8 / (ST_SOFT * 32), STEP = ST_SOFT * 4 / CH;
    const int st = threadIdx.x - 64, j = st & 7, ch = (st >> 3) % CH, r0 = (st >> 3) / CH;
    const int group = p.hq / p.hkv, pairs = w.n * group;
    const uint32_t by_group = (65536u + (uint32_t)group - 1u) / (uint32_t)group;          // r / group = r by_group >> 16 for r < 128
    const bf16* src = static_cast<const bf16*>(p.q) + ((size_t)w.row0 * p.hq + w.kvh * group) * D + ch * 64 + j * 8;
    unsigned char* dst = q_smem + ch * (ST_PAIRS * 128);
    uint4 x[ITER];
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
        const int r = r0 + k * STEP;
        const uint32_t row = (uint32_t)r * by_group >> 16;
        x[k] = r < pairs ? *reinterpret_cast<const uint4*>(src + (size_t)(row * p.hq + (r - row * group)) * D) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
        const int r = r0 + k * STEP;
        if (r < pairs) *reinterpret_cast<uint4*>(dst + (size_t)r * 128 + ((j ^ (r & 7)) << 4)) = x[k];
    }
    at_fence_async_smem();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) at_mbar_arrive(q_full);
}

// Lane i's word j becomes lane j's word i.
__device__ __forceinline__ void st_transpose(uint32_t (&x)[32], int lane) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
        const bool up = (lane & s) != 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            if (j & s) continue;
            const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? x[j] : x[j + s], s);
            if (up) x[j] = got; else x[j + s] = got;
        }
    }
}

template <int D>
__global__ void __launch_bounds__(ST_THREADS, 1)
shared_tiles_kernel(const SharedParams p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    using C = TilesCfg<D>;
    constexpr int KEYS = C::KEYS, CH = C::CH, RING = C::RING, PART = KEYS / 4, SB = ST_S;
    extern __shared__ unsigned char st_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)st_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* q_smem = smem;                                // [chunk][128 pairs][128 bytes]
    unsigned char* k_ring = smem + C::Q_BYTES;                   // units of [chunk][KEYS][128 bytes]
    unsigned char* v_ring = k_ring + RING * C::KV_BYTES;
    uint64_t* k_full = reinterpret_cast<uint64_t*>(v_ring + RING * C::KV_BYTES);
    uint64_t* k_empty = k_full + RING;
    uint64_t* v_full = k_empty + RING;
    uint64_t* v_empty = v_full + RING;
    uint64_t* s_full = v_empty + RING;                           // [SB] S complete
    uint64_t* p_full = s_full + SB;                              // [SB] P written, the softmax's warps arrive
    uint64_t* s_free = p_full + SB;                              // [SB] the product that read P is complete
    uint64_t* q_full = s_free + SB;                              // a part's queries are laid out, the softmax's warps arrive
    uint64_t* o_full = q_full + 1;                               // a part's products are complete
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 1);
    float* exchange = reinterpret_cast<float*>(tmem_slot + 2);   // [2][4][128]: a unit's maxima by (turn, quarter of its positions, pair)
    SharedTiles& cut = *reinterpret_cast<SharedTiles*>(exchange + 2 * 4 * ST_PAIRS);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = p.hq / p.hkv;
    dependent_wait();                                            // queries, keys and counts may be the work of the kernel before
    dependent_trigger();                                         // the kernel over rows may begin: it waits for nothing else
    shared_cut_tiles(p, cut, ST_PAIRS / group, KEYS);            // ends with a barrier
    const SharedRange range = shared_range(blockIdx.x, shared_tile_blocks(p, cut.upto[cut.tiles], cut.row_units, gridDim.x), cut.upto[cut.tiles], p.hkv);
    if (blockIdx.x == 0) shared_leave_tiles(p, cut, range.workers);
    if (range.begin == range.end) return;                        // nothing for this block: before anything is allocated
    if (tid == 0) {
        for (int s = 0; s < RING; ++s) { at_mbar_init(k_full + s, 1); at_mbar_init(k_empty + s, 1); at_mbar_init(v_full + s, 1); at_mbar_init(v_empty + s, 1); }
        for (int b = 0; b < SB; ++b) { at_mbar_init(s_full + b, 1); at_mbar_init(p_full + b, ST_SOFT); at_mbar_init(s_free + b, 1); }
        at_mbar_init(q_full, ST_SOFT);
        at_mbar_init(o_full, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(at_saddr(tmem_slot)), "r"(C::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    at_fence_before();
    __syncthreads();
    at_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool failed = false;

    if (warp == 0 || warp == ST_WARP_V) {
        // ---------------------------------------------------------------- keys or values, a box a lane
        const bool keys = warp == 0;
        constexpr int GROUPS = KEYS / 16, BATCH = 32 / GROUPS;   // groups of 16 positions a unit; units whose pages are looked up at once
        uint64_t* full = keys ? k_full : v_full;
        uint64_t* empty = keys ? k_empty : v_empty;
        const bf16* table = static_cast<const bf16*>(p.v_table);
        int c = 0;                                               // units so far
        for (int u = range.begin; u < range.end && !failed;) {
            const TilePart w = st_part(p, cut, u, range.end);
            u += w.units;
            const int k0 = (w.lo / KEYS + w.first) * KEYS;
            auto lookup = [&](int from) -> int {                 // lane GROUPS i + s: group s of unit from + i
                const int i = from + lane / GROUPS, j = k0 + i * KEYS + (lane % GROUPS) * 16;
                int page = -1;
                if (i < w.units && j < w.hi && j + 16 > w.lo) {
                    const int lp = max(j, w.lo) / p.page_size;
                    if (lp < p.table_width) page = p.block_table[(size_t)w.looks * p.table_width + lp];
                    if (page >= p.n_pages) page = -1;
                }
                return page;
            };
            int now = 0, next = lookup(0);
            for (int i = 0; i < w.units; ++i, ++c) {
                if (i % BATCH == 0) { now = next; next = lookup(i + BATCH); }
                const int s = c % RING;
                if (!__all_sync(0xffffffffu, at_mbar_wait(empty + s, ((uint32_t)(c / RING) & 1u) ^ 1u))) { failed = true; break; }
                unsigned char* dst = (keys ? k_ring : v_ring) + s * C::KV_BYTES;
                const int j0 = k0 + i * KEYS;
                const int page = __shfl_sync(0xffffffffu, now, (i % BATCH) * GROUPS + lane % GROUPS);      // lane's group: lane mod GROUPS
                const bool inner = page >= 0 && j0 + (lane % GROUPS) * 16 >= w.lo;
                // Groups that TMA brings: of keys every one with a page (a score that is not seen is replaced, whatever it is); of values those
                // that are seen from their first position on. The others are cleared, or copied as far as they are seen: 0 times garbage may be NaN.
                const uint32_t have = __ballot_sync(0xffffffffu, keys ? page >= 0 : inner) & ((1u << GROUPS) - 1u);
                if (have != (1u << GROUPS) - 1u) {
                    for (int s2 = 0; s2 < GROUPS; ++s2) {
                        if (have & (1u << s2)) continue;
                        const int pg = __shfl_sync(0xffffffffu, page, s2), j = j0 + s2 * 16;
                        const bf16* src = pg >= 0 ? table + ((size_t)((long long)pg * p.hkv + w.kvh) * p.page_size + j % p.page_size) * D : nullptr;
                        for (int e = lane; e < CH * 128; e += 32) {
                            const int chunk = e >> 7, row = (e & 127) >> 3, piece = e & 7;
                            uint4 x = make_uint4(0u, 0u, 0u, 0u);
                            if (src != nullptr && j + row >= w.lo) x = *reinterpret_cast<const uint4*>(src + (size_t)row * D + chunk * 64 + piece * 8);
                            *reinterpret_cast<uint4*>(dst + (size_t)chunk * (KEYS * 128) + s2 * 2048 + row * 128 + ((piece ^ (row & 7)) << 4)) = x;
                        }
                    }
                    at_fence_async_smem();
                    __syncwarp();
                }
                if (lane == 0) at_mbar_expect_tx(full + s, (uint32_t)(__popc(have) * CH) * 2048u);
                __syncwarp();
                const int s2 = lane % GROUPS, chunk = lane / GROUPS;
                if (chunk < CH && (have & (1u << s2))) {
                    const int row = (page * p.hkv + w.kvh) * p.page_size + (j0 + s2 * 16) % p.page_size;
                    at_tma_box(at_saddr(dst) + (uint32_t)chunk * (KEYS * 128) + (uint32_t)s2 * 2048u, keys ? &map_k : &map_v, chunk * 64, row, full + s);
                }
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- the score products
        const uint32_t one = at_elect(), tm = __shfl_sync(0xffffffffu, tmem, 0);
        constexpr uint32_t IDESC = at_idesc(ST_PAIRS, KEYS, false);
        const uint32_t q_addr = at_saddr(q_smem), ring = at_saddr(k_ring);
        int c = 0, part = 0;
        for (int u = range.begin; u < range.end && !failed; ++part) {
            const TilePart w = st_part(p, cut, u, range.end);
            u += w.units;
            if (!__all_sync(0xffffffffu, at_mbar_wait(q_full, (uint32_t)part & 1u))) { failed = true; break; }
            for (int i = 0; i < w.units; ++i, ++c) {
                const int s = c % RING, b = c % SB;
                if (!__all_sync(0xffffffffu, at_mbar_wait(k_full + s, (uint32_t)(c / RING) & 1u))) { failed = true; break; }
                if (c >= SB && !__all_sync(0xffffffffu, at_mbar_wait(s_free + b, (uint32_t)(c / SB - 1) & 1u))) { failed = true; break; }
                at_fence_after();
                const uint32_t d = tm + (uint32_t)(C::COL_S + b * KEYS);
#pragma unroll
                for (int ch = 0; ch < CH; ++ch) {
                    const uint64_t a = at_desc(q_addr + ch * (ST_PAIRS * 128), 16, 1024);
                    const uint64_t k = at_desc(ring + (uint32_t)s * C::KV_BYTES + ch * (KEYS * 128), 16, 1024);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) at_mma_ss_if(one, d, a + (uint64_t)(kk * 2), k + (uint64_t)(kk * 2), IDESC, (ch | kk) != 0 ? 1u : 0u);
                }
                if (one) at_commit(k_empty + s);
                if (one) at_commit(s_full + b);
            }
        }
    } else if (warp == ST_WARP_PV) {
        // ---------------------------------------------------------------- the P V products
        const uint32_t one = at_elect(), tm = __shfl_sync(0xffffffffu, tmem, 0);
        constexpr uint32_t IDESC = at_idesc(ST_PAIRS, D, true);
        const uint32_t ring = at_saddr(v_ring);
        int c = 0;
        for (int u = range.begin; u < range.end && !failed;) {
            const TilePart w = st_part(p, cut, u, range.end);
            u += w.units;
            for (int i = 0; i < w.units; ++i, ++c) {
                const int s = c % RING, b = c % SB;
                if (!__all_sync(0xffffffffu, at_mbar_wait(v_full + s, (uint32_t)(c / RING) & 1u))) { failed = true; break; }
                if (!__all_sync(0xffffffffu, at_mbar_wait(p_full + b, (uint32_t)(c / SB) & 1u))) { failed = true; break; }
                at_fence_after();
                const uint32_t a = tm + (uint32_t)(C::COL_S + b * KEYS);             // P lies over its S
#pragma unroll
                for (int kk = 0; kk < KEYS / 16; ++kk) {
                    const uint64_t v = at_desc(ring + (uint32_t)s * C::KV_BYTES + (uint32_t)kk * 2048u, KEYS * 128, 1024);
                    at_mma_ts_if(one, tm, a + (uint32_t)(kk * 8), v, IDESC, (i | kk) != 0 ? 1u : 0u);
                }
                if (one) at_commit(v_empty + s);
                if (one) at_commit(s_free + b);
            }
            if (!failed && one) at_commit(o_full);
        }
    } else {
        // ---------------------------------------------------------------- queries, softmax and pieces, a quarter of a pair's positions a thread
        const int quarter = warp & 3, share = (warp - 2) >> 2, pair = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const SharedScore score(p.scale, p.cap);
        auto lay_queries = [&](const TilePart& w) { st_queries<D>(p, w, q_smem, q_full); };
        int c = 0, part = 0, turns = 0;
        TilePart w = st_part(p, cut, range.begin, range.end);
        lay_queries(w);
        for (int u = range.begin; u < range.end; ++part) {
            u += w.units;
            const bool own = pair < w.n * group, idle = quarter * 32 >= w.n * group;
            const int row = w.row0 + pair / group;
            const int count = own ? p.row_count[row] : 0;
            const int lo = own ? max(shared_first(p, count), w.lo) : 0, hi = own ? min(count, w.hi) : 0;      // this pair sees [lo, hi) of the tile's
            const int lo_max = __reduce_max_sync(0xffffffffu, lo), hi_min = __reduce_min_sync(0xffffffffu, hi);
            float ref = -INFINITY, l = 0.f;
            for (int i = 0; i < w.units; ++i, ++c) {
                const int b = c % SB, j0 = (w.lo / KEYS + w.first + i) * KEYS + share * PART;
                // a wait that ran out is not repeated, but the walk goes on: the quarter's warps meet at every unit's barrier
                if (!failed && !__all_sync(0xffffffffu, at_mbar_wait(s_full + b, (uint32_t)(c / SB) & 1u))) failed = true;
                at_fence_after();
                if (!idle) {
                    uint32_t x[PART];
                    sh_ld(lanes + (uint32_t)(C::COL_S + b * KEYS + share * PART), x);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    const bool edge = j0 < lo_max || j0 + PART > hi_min;         // some pair does not see all of it (a place without one sees nothing): the same for the whole warp
                    float top = -INFINITY, far = 0.f;
                    if (edge) {
#pragma unroll
                        for (int j = 0; j < PART; ++j) {
                            float v = score(__uint_as_float(x[j]));
                            if (j0 + j < lo || j0 + j >= hi) v = -INFINITY;
                            x[j] = __float_as_uint(v);
                            top = fmaxf(top, v);
                        }
                    } else {
                        far = sh_scale(x, score);
                        top = score.cap ? score.of_u(far) : far;     // no less than the largest score
                    }
                    // The quarter's four warps tell each other their largest scores, or bounds of them; behind this barrier all have their scores in
                    // registers, so P may be written over them. Sets of places in turn. Only where a bound passes m by too much the scores
                    // themselves are looked through: the same for the four warps.
                    float* turn = exchange + (turns++ & 1) * 4 * ST_PAIRS + pair;
                    turn[share * ST_PAIRS] = top;
                    asm volatile("bar.sync %0, 128;" ::"r"(2 + quarter) : "memory");
                    float most = fmaxf(fmaxf(turn[0], turn[ST_PAIRS]), fmaxf(turn[2 * ST_PAIRS], turn[3 * ST_PAIRS]));
                    if (__any_sync(0xffffffffu, most > ref + ST_LAG)) {
                        if (!edge) {
                            top = -INFINITY;
#pragma unroll
                            for (int j = 0; j < PART; ++j) top = fmaxf(top, __uint_as_float(x[j]));
                            if (score.cap) top = score.of_u(top);
                        }
                        turn = exchange + (turns++ & 1) * 4 * ST_PAIRS + pair;
                        turn[share * ST_PAIRS] = top;
                        asm volatile("bar.sync %0, 128;" ::"r"(2 + quarter) : "memory");
                        most = fmaxf(fmaxf(turn[0], turn[ST_PAIRS]), fmaxf(turn[2 * ST_PAIRS], turn[3 * ST_PAIRS]));
                    }
                    const bool moves = most > ref + ST_LAG;          // (anything above -inf, to begin with)
                    const float was = ref;
                    if (moves) ref = most;
                    const float fade = moves ? (was == -INFINITY ? 0.f : at_exp2(was - ref)) : 1.f;
                    l *= fade;
                    if (i > 0 && __any_sync(0xffffffffu, moves && was != -INFINITY)) {
                        const int before = c - 1;
                        if (!failed && !__all_sync(0xffffffffu, at_mbar_wait(s_free + before % SB, (uint32_t)(before / SB) & 1u))) failed = true;
                        at_fence_after();
                        for (int c0 = share * 32; c0 < D; c0 += 128) {
                            uint32_t o[32];
                            __syncwarp();
                            at_ld32(lanes + (uint32_t)c0, o);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * fade);
                            at_st32(lanes + (uint32_t)c0, o);
                        }
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    }
                    const float base = ref == -INFINITY ? 0.f : ref;
                    uint32_t pr[PART / 2];
                    if (!edge && score.cap && __all_sync(0xffffffffu, far <= SH_NEAR)) {
                        l += sh_weights_near(x, pr, base, score);
                    } else {
                        if (!edge && score.cap) {
#pragma unroll
                            for (int j = 0; j < PART; ++j) x[j] = __float_as_uint(score.of_u(__uint_as_float(x[j])));
                        }
                        l += sh_weights(x, pr, base, [](unsigned long long v, unsigned long long less) { return sh_add2(v, less); });
                    }
                    sh_st(lanes + (uint32_t)(C::COL_S + b * KEYS + share * (PART / 2)), pr);
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                at_fence_before();
                __syncwarp();
                if (lane == 0) at_mbar_arrive(p_full + b);
            }
            // The last score product of this part is complete: the next part's queries take the place of this one's.
            const TilePart mine = w;
            if (u < range.end) {
                w = st_part(p, cut, u, range.end);
                lay_queries(w);
            }
            if (!idle) {
                // the pair's sum over its four shares, through shared memory
                float* turn = exchange + (turns++ & 1) * 4 * ST_PAIRS + pair;
                turn[share * ST_PAIRS] = l;
                asm volatile("bar.sync %0, 128;" ::"r"(2 + quarter) : "memory");
                l = (turn[0] + turn[ST_PAIRS]) + (turn[2 * ST_PAIRS] + turn[3 * ST_PAIRS]);
                asm volatile("bar.sync %0, 128;" ::"r"(2 + quarter) : "memory");
            }
            if (!failed && !__all_sync(0xffffffffu, at_mbar_wait(o_full, (uint32_t)part & 1u))) failed = true;
            if (!failed && !idle) {
                at_fence_after();
                // 32 pairs x 32 components a time, turned around in registers: a pair's components leave side by side, a line a store.
                float* pieces = p.tile_pieces + (mine.place + quarter * 32) * SH_PIECE(D);
                const int here = min(32, mine.n * group - quarter * 32);
                for (int c0 = share * 32; c0 < D; c0 += 128) {
                    uint32_t o[32];
                    __syncwarp();
                    at_ld32(lanes + (uint32_t)c0, o);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    st_transpose(o, lane);
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        if (j < here) pieces[(size_t)j * SH_PIECE(D) + c0 + lane] = __uint_as_float(o[j]);
                }
                if (own && share == 0)
                    *reinterpret_cast<float2*>(pieces + (size_t)lane * SH_PIECE(D) + D) = make_float2(ref == -INFINITY ? -INFINITY : ref * 0.6931471805599453f, l);
            }
            at_fence_before();
        }
    }
    if (failed) atomicExch(&g_shared_attention_error, 1);
    at_fence_before();
    __syncthreads();
    if (warp == 1) {
        at_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
    }
}

template <int D> static int launch_tiles(const SharedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, cudaStream_t s) {
    static unsigned long long done = 0;
    if (int e = allow_shared_memory((const void*)shared_tiles_kernel<D>, TilesCfg<D>::SMEM, &done)) return e;
    launch_dependent_if(p.rows <= DEPENDENT_ROWS, shared_tiles_kernel<D>, dim3(blocks), dim3(ST_THREADS), TilesCfg<D>::SMEM, s, p, mk, mv);
    return check_launch("shared_attention");
}

int launch_shared_tiles(const SharedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, cudaStream_t s) {
    return p.d == 256 ? launch_tiles<256>(p, mk, mv, blocks, s) : p.d == 128 ? launch_tiles<128>(p, mk, mv, blocks, s) : launch_tiles<64>(p, mk, mv, blocks, s);
}

}  // namespace kb

// 1 if a wait inside the kernel ever ran out (and clears the flag); synchronises the device.
extern "C" int kb_shared_tiles_error() {
    int flag = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&flag, kb::g_shared_attention_error, sizeof(int)) != cudaSuccess) return -1;
    if (flag) cudaMemcpyToSymbol(kb::g_shared_attention_error, &zero, sizeof(int));
    return flag;
}

// What each request reads by itself behind the pages it shares (bfloat16; see attention_shared.cuh for the cut): every warp a worker.
//
// The units are 16 positions of one kv head, which lie in one page: TMA brings their keys and their values as one box each of D / 64 x 16 x 64
// elements (128-byte swizzle) into a pipeline that is the warp's own (a request a lane: as eight boxes of 16 x 64 they took 1,100 clocks of the
// 2,400 that a unit of 256 components took). A warp walks its units whatever items they belong to, requests
// for the next item's keys go out while it still computes on the one before, and nothing in the loop waits for another warp: short answers of many
// requests stream like one long one. The products have the keys as the MMAs' M (S^T = K Q^T, O^T = V^T P^T), the query
// heads of the kv head as their N, eight a block, NB blocks; P^T comes out of S^T's registers by movmatrix. Scores, softmax and sums are 32-bit; the
// weights are rounded to bfloat16 for the second product, and the sum of the weights adds up the rounded ones.
//
// What bounds it: memory, at the copy's rate once under way (3 x 16 KB a warp in flight). Before that the cut is made, the block tables are read and
// the first keys and queries come, some 7 us. 64 requests of some 330 positions each, 8 kv heads of 256 (175 MB): 42 us, 4.2 TB/s.
//
// Positions of a unit that the request does not see get the weight 0, and their values are cleared in shared memory first: what another request
// left in the page may be anything.
#include "attention_shared_bf16.cuh"

namespace kb {

template <int D> struct OwnCfg {
    static constexpr int WARPS = D == 256 ? 4 : 8;
    static constexpr int STAGES = D == 64 ? 6 : 3;                       // 192 KB in flight a multiprocessor
    static constexpr int BOXES = D / 64;
    static constexpr int STAGE = 2 * BOXES * 2048;                       // bytes: keys, then values
    static constexpr int PIPES = WARPS * STAGES * STAGE;
    static constexpr int SMEM = 1024 + PIPES + WARPS * STAGES * 8 + (7 * SH_ROWS + 4) * 4;
    static_assert(SMEM <= 232448, "more shared memory than a block can have");
};

template <int D, int NB>
__global__ void __launch_bounds__(OwnCfg<D>::WARPS * 32, 1)
shared_own_kernel(const SharedParams p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    using C = OwnCfg<D>;
    constexpr int KK = D / 16, CHAINS = NB == 1 ? 4 : 2;
    extern __shared__ unsigned char so_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)so_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* all_bars = reinterpret_cast<uint64_t*>(smem + C::PIPES);
    int* upto = reinterpret_cast<int*>(all_bars + C::WARPS * C::STAGES);
    int* row_lo = upto + SH_ROWS + 1;
    int* row_hi = row_lo + SH_ROWS;
    int* length = row_hi + SH_ROWS;                          // what rows share, and with whom
    int* id = length + SH_ROWS;
    int* tile_lo = id + SH_ROWS;                            // the positions that tiles see
    int* tile_hi = tile_lo + SH_ROWS;
    int* tile_units = tile_hi + SH_ROWS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* pipe = smem + warp * C::STAGES * C::STAGE;
    uint64_t* bars = all_bars + warp * C::STAGES;
    if (lane == 0) {
        for (int s = 0; s < C::STAGES; ++s) at_mbar_init(bars + s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const int group = p.hq / p.hkv;
    int blocks = gridDim.x;
    if (p.alone) {                                           // no kernel over tiles has waited for the one before
        dependent_wait();
        dependent_trigger();
    }
    if (p.tile_cost > 0.f) {
        for (int r = threadIdx.x; r < p.rows; r += blockDim.x) { length[r] = shared_length(p, r); id[r] = p.share_id[r]; }
    }
    shared_cut_rows(p, upto, row_lo, row_hi, 16);            // ends with a barrier
    if (p.tile_cost > 0.f) {                                 // the tiles' kernel runs beside this one and has its share of the multiprocessors
        if (warp == 0) {
            const int units = shared_tile_units(p, length, id, tile_lo, tile_hi, 128 / group, D == 256 ? 64 : 128);
            if (lane == 0) *tile_units = units;
        }
        __syncthreads();
        const int theirs = shared_tile_blocks(p, *tile_units, upto[p.rows], gridDim.x);
        if (theirs < blocks) blocks -= theirs;
    }
    const SharedRange range = shared_range(blockIdx.x * C::WARPS + warp, blocks * C::WARPS, upto[p.rows], p.hkv);
    if (blockIdx.x == 0) {
        shared_leave_rows(p, upto, range.workers);
        if (p.alone) {                                       // no tiles
            for (int i = threadIdx.x; i < p.rows; i += blockDim.x) p.cut[SH_CUT_ROW_TILE + i] = -1;
            if (threadIdx.x == 0) p.cut[SH_CUT_COUNTS] = p.cut[SH_CUT_COUNTS + 1] = p.cut[SH_CUT_TILE_UNITS] = 0;
        }
    }
    const bf16* q = static_cast<const bf16*>(p.q);

    // What is asked for: unit `ask` of the worker's, the `a_in`-th of `a_units` of a request and kv head. The pages of the next
    // 32 units wait in registers, one a lane.
    int ask = range.begin, a_row = 0, a_kvh = 0, a_in = 0, a_units = 0, a_j = 0, a_batch = 0, a_lo = 0, pages = -1;
    uint32_t absent = 0;                                     // stages whose unit has no page
    auto next_unit = [&](int stage) {
        if (ask >= range.end) return;
        bool fresh = false;
        if (a_in == a_units) {
            a_row = shared_item(upto, p.rows, p.hkv, ask);
            a_units = upto[a_row + 1] - upto[a_row];
            const int in = ask - upto[a_row] * p.hkv;
            a_kvh = in / a_units;
            a_in = in % a_units;
            a_lo = row_lo[a_row];
            a_j = a_lo / 16 * 16;
            fresh = true;
        }
        if (fresh || a_in - a_batch >= 32) {
            a_batch = a_in;
            pages = -1;
            if (a_in + lane < a_units) {
                const int lp = max(a_lo, a_j + 16 * (a_in + lane)) / p.page_size;
                if (lp < p.table_width) pages = p.block_table[(size_t)a_row * p.table_width + lp];
                if (pages >= p.n_pages) pages = -1;
            }
        }
        const int page = __shfl_sync(0xffffffffu, pages, a_in - a_batch);
        if (page >= 0) {
            const int row = (page * p.hkv + a_kvh) * p.page_size + (a_j + 16 * a_in) % p.page_size;
            if (lane == 0) at_mbar_expect_tx(bars + stage, C::STAGE);
            __syncwarp();
            const uint32_t dst = at_saddr(pipe + stage * C::STAGE) + lane * (C::STAGE / 2);
            if (lane < 2) at_tma_page(dst, lane == 0 ? &map_k : &map_v, row, bars + stage);
            absent &= ~(1u << stage);
        } else {
            if (lane == 0) at_mbar_arrive(bars + stage);     // nothing to wait for
            absent |= 1u << stage;
        }
        ++ask;
        ++a_in;
    };
    if (range.begin < range.end) {                           // the first item's queries are on their way before its keys crowd the memory
        const int r = shared_item(upto, p.rows, p.hkv, range.begin), kvh = (range.begin - upto[r] * p.hkv) / (upto[r + 1] - upto[r]);
        const bf16* first = q + ((size_t)r * p.hq + kvh * group) * D;
        for (int i = lane * 64; i < group * D; i += 32 * 64) asm volatile("prefetch.global.L1 [%0];" ::"l"(first + i));
    }
    for (int s = 0; s < C::STAGES; ++s) next_unit(s);

    const SharedScore score(p.scale, p.cap);
    bool failed = false;
    int done = 0;                                            // units taken so far: stage done % STAGES, its (done / STAGES)-th use
    for (int u = range.begin; u < range.end && !failed;) {
        const int r = shared_item(upto, p.rows, p.hkv, u);
        const int units = upto[r + 1] - upto[r], in = u - upto[r] * p.hkv;
        const int kvh = in / units, first = in % units, n = min(units - first, range.end - u);
        const int lo = row_lo[r], hi = row_hi[r];
        u += n;
        uint32_t bq[KK][NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const bool has = nb * 8 + g < group;
            const uint32_t* src = reinterpret_cast<const uint32_t*>(q + ((size_t)r * p.hq + kvh * group + (has ? nb * 8 + g : 0)) * D) + t;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                bq[kk][nb][0] = has ? src[kk * 8] : 0u;
                bq[kk][nb][1] = has ? src[kk * 8 + 4] : 0u;
            }
        }
        float ot[KK][NB][4], m[NB][2], l[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m[nb][0] = m[nb][1] = -INFINITY;
            l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
            for (int i = 0; i < KK; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) ot[i][nb][c] = 0.f;
        }
        for (int i = 0; i < n; ++i, ++done) {
            const int stage = done % C::STAGES;
            if (!__all_sync(0xffffffffu, at_mbar_wait(bars + stage, (uint32_t)(done / C::STAGES) & 1u))) { failed = true; break; }
            const int j0 = lo / 16 * 16 + 16 * (first + i);
            const bool gone = (absent >> stage) & 1u, partly = j0 < lo || j0 + 16 > hi;
            unsigned char* sv = pipe + stage * C::STAGE + C::BOXES * 2048;
            const uint32_t k_at = at_saddr(pipe + stage * C::STAGE), v_at = at_saddr(sv);
            if (!gone) {
                if (partly) {
                    for (int e = lane; e < C::BOXES * 128; e += 32) {      // pieces of 16 bytes, eight a row of a box
                        const int j = j0 + (e & 127) / 8;
                        if (j < lo || j >= hi) *reinterpret_cast<uint4*>(sv + (size_t)e * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    __syncwarp();
                }
                float st[CHAINS][NB][4];                     // several chains of products: one after the other they would wait for their sums
#pragma unroll
                for (int c = 0; c < CHAINS; ++c)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int e = 0; e < 4; ++e) st[c][nb][e] = 0.f;
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    uint32_t a[4];
                    const int row = lane & 15, piece = (kk & 3) * 2 + (lane >> 4);
                    sh_ldmatrix(a, k_at + (kk >> 2) * 2048 + row * 128 + ((piece ^ (row & 7)) << 4));
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) sh_mma(st[kk % CHAINS][nb], a, bq[kk][nb][0], bq[kk][nb][1]);
                }
                uint32_t pt[NB][2];
                bool moves = false;
                float fade[NB][2];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = st[0][nb][e];
#pragma unroll
                        for (int c = 1; c < CHAINS; ++c) v += st[c][nb][e];
                        x[e] = score(v);
                        const int j = j0 + g + (e >> 1) * 8;
                        if (partly && (j < lo || j >= hi)) x[e] = -INFINITY;
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float top = fmaxf(x[h], x[h + 2]);
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                        const float next = fmaxf(m[nb][h], top);      // a unit holds a position that is seen: never -inf but for infinite scores
                        const float base = next == -INFINITY ? 0.f : next;
                        fade[nb][h] = at_exp2(m[nb][h] - base);
                        moves = moves || next > m[nb][h];
                        m[nb][h] = next;
                        x[h] = at_exp2(x[h] - base);
                        x[h + 2] = at_exp2(x[h + 2] - base);
                    }
                    const uint32_t p0 = at_pack(x[0], x[1]), p1 = at_pack(x[2], x[3]);
                    l[nb][0] = fmaf(l[nb][0], fade[nb][0], __uint_as_float(p0 << 16) + __uint_as_float(p1 << 16));
                    l[nb][1] = fmaf(l[nb][1], fade[nb][1], __uint_as_float(p0 & 0xffff0000u) + __uint_as_float(p1 & 0xffff0000u));
                    pt[nb][0] = sh_transpose(p0);
                    pt[nb][1] = sh_transpose(p1);
                }
                if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
                    for (int i2 = 0; i2 < KK; ++i2)
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            ot[i2][nb][0] *= fade[nb][0];
                            ot[i2][nb][1] *= fade[nb][1];
                            ot[i2][nb][2] *= fade[nb][0];
                            ot[i2][nb][3] *= fade[nb][1];
                        }
                }
#pragma unroll
                for (int i2 = 0; i2 < KK; ++i2) {
                    uint32_t a[4];
                    const int key = (lane & 7) + ((lane >> 4) << 3), piece = (i2 & 3) * 2 + ((lane >> 3) & 1);
                    sh_ldmatrix_trans(a, v_at + (i2 >> 2) * 2048 + key * 128 + ((piece ^ (key & 7)) << 4));
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) sh_mma(ot[i2][nb], a, pt[nb][0], pt[nb][1]);
                }
                if (partly) at_fence_async_smem();           // the cleared values lie where a copy may come next
            }
            __syncwarp();
            next_unit(stage);
        }
        if (failed) break;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[nb][h] += __shfl_xor_sync(0xffffffffu, l[nb][h], o);
                const int head = nb * 8 + 2 * t + h;
                if (head >= group) continue;
                float* piece = p.row_pieces + (shared_row_place(p, r, kvh, blockIdx.x * C::WARPS + warp) + head) * SH_PIECE(D);
#pragma unroll
                for (int i = 0; i < KK; ++i) {
                    piece[i * 16 + g] = ot[i][nb][h];
                    piece[i * 16 + 8 + g] = ot[i][nb][h + 2];
                }
                if (g == 0) { piece[D] = m[nb][h] * 0.6931471805599453f; piece[D + 1] = l[nb][h]; }
            }
    }
    dependent_wait();                                        // this grid ends behind the tiles' kernel: whoever waits for it has both
    if (failed) {
        if (lane == 0) atomicExch(&g_shared_attention_error, 1);
        // what was asked for may still come (a wait that ran out is not repeated for ever)
        for (int i = 1; i < C::STAGES && done + i < ask - range.begin; ++i) at_mbar_wait(bars + (done + i) % C::STAGES, (uint32_t)((done + i) / C::STAGES) & 1u);
    }
}

template <int D, int NB> static int launch_own(const SharedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, cudaStream_t s) {
    static unsigned long long done = 0;
    if (int e = allow_shared_memory((const void*)shared_own_kernel<D, NB>, OwnCfg<D>::SMEM, &done)) return e;
    launch_dependent_if(p.alone ? p.rows <= DEPENDENT_ROWS : p.tile_cost > 0.f, shared_own_kernel<D, NB>, dim3(blocks), dim3(OwnCfg<D>::WARPS * 32), OwnCfg<D>::SMEM, s, p, mk, mv);
    return check_launch("shared_attention");
}

int shared_own_workers(int d) { return d == 256 ? OwnCfg<256>::WARPS : d == 128 ? OwnCfg<128>::WARPS : OwnCfg<64>::WARPS; }

int launch_shared_own(const SharedParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, cudaStream_t s) {
    const bool few = p.hq / p.hkv <= 8;
    if (p.d == 256) return few ? launch_own<256, 1>(p, mk, mv, blocks, s) : launch_own<256, 2>(p, mk, mv, blocks, s);
    if (p.d == 128) return few ? launch_own<128, 1>(p, mk, mv, blocks, s) : launch_own<128, 2>(p, mk, mv, blocks, s);
    return few ? launch_own<64, 1>(p, mk, mv, blocks, s) : launch_own<64, 2>(p, mk, mv, blocks, s);
}

}  // namespace kb

// 1 if a wait inside the kernels ever ran out (and clears the flag); synchronises the device.
extern "C" int kb_shared_own_error() {
    int flag = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&flag, kb::g_shared_attention_error, sizeof(int)) != cudaSuccess) return -1;
    if (flag) cudaMemcpyToSymbol(kb::g_shared_attention_error, &zero, sizeof(int));
    return flag;
}

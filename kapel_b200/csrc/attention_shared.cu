// Attention of single tokens over shared and own pages (see attention_shared.cuh for the cut), for any element type and head size up
// to 256; and the kernel that joins the pieces.
//
// A block of 256 threads walks its units of 32 positions, lines padded with zeros to 64, 128 or 256 components. Eight threads have one (row, head) pair of the 32 that a tile takes: each
// computes every eighth position's score out of keys and queries in shared memory, and keeps every eighth group of four components of the
// sum in registers. All arithmetic is 32-bit. Where some row of the tile does not see all of a unit (its window begins there, its
// positions end there) what a row does not see is left out of its sum, not multiplied by zero: it may be anything.
//
// What bounds it: the multiply-adds and what they read of shared memory; a unit's loads are not asked for ahead of the one before. 8 requests behind
// 1,024 positions with some 70 of their own, 8 heads over 4 of 256 in 32 bits: 28 us, the joining of the pieces among them.
#include "attention_shared_bf16.cuh"
#include "tensor_map.cuh"

namespace kb {

constexpr int SR_PAIRS = 32, SR_KEYS = 32, SR_THREADS = 256, SR_DIM = 256;
static_assert(SR_PAIRS == SR_KEYS, "queries are laid out as lines are");

template <int DIM> struct SharedRowsSmem {
    float q[SR_PAIRS][DIM + 4];
    float k[SR_KEYS][DIM + 4];
    float v[SR_KEYS][DIM];
    long long line[SR_KEYS];               // a position's line of this kv head in the tables, -1 for none
    SharedTiles tiles;
    int upto[SH_ROWS + 1], lo[SH_ROWS], hi[SH_ROWS];       // units before a row, the positions it reads by itself
};

// SR_KEYS lines of `size` components into shared memory in 32 bits, zeros where a line is none and from its last component up to DIM.
template <typename T, int DIM, int STRIDE> __device__ __forceinline__ void sr_lines(float* to, const T* table, const long long* lines, int size, bool fours) {
    constexpr int WARPS = SR_THREADS / 32, ROWS = SR_KEYS / WARPS, QUADS = (DIM + 127) / 128;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (fours) {
        float4 x[ROWS][QUADS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int k = 0; k < QUADS; ++k) {
                const long long line = lines[warp + i * WARPS];
                const int c = 4 * (lane + 32 * k);
                x[i][k] = line >= 0 && c < size ? load_four(table + line * size + c) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int k = 0; k < QUADS; ++k) {
                const int c = 4 * (lane + 32 * k);
                if (c < DIM) *reinterpret_cast<float4*>(to + (warp + i * WARPS) * STRIDE + c) = x[i][k];
            }
    } else {
        for (int r = warp; r < SR_KEYS; r += WARPS)
            for (int c = lane; c < DIM; c += 32)
                to[r * STRIDE + c] = c < size && lines[r] >= 0 ? Elem<T>::load(table + lines[r] * size + c) : 0.f;
    }
}

// A unit's NI groups of eight positions from group i0 on for eight threads' pair (row `pair` of the queries): scores, the running maximum and sum, the
// weighted values.
template <int NI, int DIM>
__device__ __forceinline__ void sr_unit(const SharedRowsSmem<DIM>& s, const SharedParams& p, int pair, bool own, int i0, int j0, int first, int count, float& m, float& l,
                                        float4 (&acc)[DIM / 32]) {
    const int lane = threadIdx.x & 31, sub = threadIdx.x & 7;
    float x[NI];
    float top = -INFINITY;
    bool all = true;
#pragma unroll
    for (int i = 0; i < NI; ++i) x[i] = 0.f;
    if (own) {
#pragma unroll 8
        for (int c = 0; c < DIM / 4; ++c) {
            const float4 a = *reinterpret_cast<const float4*>(&s.q[pair][4 * c]);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const float4 b = *reinterpret_cast<const float4*>(&s.k[sub + 8 * (i0 + i)][4 * c]);
                x[i] = fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, x[i]))));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int j = sub + 8 * (i0 + i);
        float dot = x[i] * p.scale;
        if (p.cap > 0.f) dot = p.cap * tanhf(dot / p.cap);
        const bool sees = j0 + j >= first && j0 + j < count && s.line[j] >= 0;
        all = all && sees;
        x[i] = sees ? dot : -INFINITY;
        top = fmaxf(top, x[i]);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float next = fmaxf(m, top);
    const float fade = next == -INFINITY ? 1.f : expf(m - next);           // e^-inf = 0 where nothing was seen before
    m = next;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        x[i] = x[i] == -INFINITY ? 0.f : expf(x[i] - m);
        sum += x[i];
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l = l * fade + sum;
#pragma unroll
    for (int j = 0; j < DIM / 32; ++j) { acc[j].x *= fade; acc[j].y *= fade; acc[j].z *= fade; acc[j].w *= fade; }
    const bool whole = __all_sync(0xffffffffu, all || !own);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const float e = __shfl_sync(0xffffffffu, x[i], (lane & 24) + b);
            const float* v = &s.v[8 * (i0 + i) + b][4 * sub];
            if (whole || e != 0.f) {
#pragma unroll
                for (int c = 0; c < DIM / 32; ++c) {
                    const float4 y = *reinterpret_cast<const float4*>(v + 32 * c);
                    acc[c].x = fmaf(e, y.x, acc[c].x);
                    acc[c].y = fmaf(e, y.y, acc[c].y);
                    acc[c].z = fmaf(e, y.z, acc[c].z);
                    acc[c].w = fmaf(e, y.w, acc[c].w);
                }
            }
        }
}

template <typename T, int DIM>
__global__ void __launch_bounds__(SR_THREADS, 1) shared_rows_kernel(const SharedParams p) {
    extern __shared__ __align__(16) unsigned char sr_raw[];
    SharedRowsSmem<DIM>& s = *reinterpret_cast<SharedRowsSmem<DIM>*>(sr_raw);
    const int tid = threadIdx.x, slot = tid >> 3, sub = tid & 7;
    const int group = p.hq / p.hkv, rows_a_tile = SR_PAIRS / group;
    const T* q = static_cast<const T*>(p.q);
    const T* kt = static_cast<const T*>(p.k_table);
    const T* vt = static_cast<const T*>(p.v_table);
    shared_cut_tiles(p, s.tiles, rows_a_tile, SR_KEYS);
    shared_cut_rows(p, s.upto, s.lo, s.hi, SR_KEYS);
    const SharedRange over[2] = {shared_range(blockIdx.x, gridDim.x, s.tiles.upto[s.tiles.tiles], p.hkv), shared_range(blockIdx.x, gridDim.x, s.upto[p.rows], p.hkv)};
    if (blockIdx.x == 0) {
        shared_leave_tiles(p, s.tiles, over[0].workers);
        shared_leave_rows(p, s.upto, over[1].workers);
    }
    for (int kind = 0; kind < 2; ++kind)                     // what is shared, then what each row reads by itself
    for (int u = over[kind].begin; u < over[kind].end;) {
        struct { int row0, n, looks, kvh, lo, hi, first_unit, n_units; } w;
        const int* upto = kind == 0 ? s.tiles.upto : s.upto;
        const int item = shared_item(upto, kind == 0 ? s.tiles.tiles : p.rows, p.hkv, u);
        const int units = upto[item + 1] - upto[item], in = u - upto[item] * p.hkv;
        w.kvh = in / units;
        w.first_unit = in % units;
        w.n_units = min(units - w.first_unit, over[kind].end - u);
        float* pieces;
        if (kind == 0) {
            w.row0 = s.tiles.row0[item]; w.n = s.tiles.n[item]; w.looks = s.tiles.looks[item]; w.lo = s.tiles.klo[item]; w.hi = s.tiles.khi[item];
            pieces = p.tile_pieces + shared_tile_place(p, s.tiles.before[item], w.n, w.kvh, blockIdx.x, SR_PAIRS) * SH_PIECE(p.dv);
        } else {
            w.row0 = w.looks = item; w.n = 1;
            w.lo = s.lo[item]; w.hi = s.hi[item];
            pieces = p.row_pieces + shared_row_place(p, item, w.kvh, blockIdx.x) * SH_PIECE(p.dv);
        }
        u += w.n_units;
        const int pairs = w.n * group;
        // Of few pairs each has two or four of the 32 places, each with its share of a unit's positions.
        const int places = pairs <= 8 ? 8 : pairs <= 16 ? 16 : 32, shares = SR_PAIRS / places;
        const int pair = slot & (places - 1), share = slot / places;
        const int row = w.row0 + pair / group;
        const bool own = pair < pairs;
        __syncthreads();                                 // the part before is done with the queries
        if (tid < SR_KEYS) s.line[tid] = tid < pairs ? (long long)(w.row0 + tid / group) * p.hq + w.kvh * group + tid % group : -1;
        __syncthreads();
        sr_lines<T, DIM, DIM + 4>(&s.q[0][0], q, s.line, p.d, p.d % 4 == 0);
        const int count = own ? min(p.row_count[row], w.hi) : 0;
        const int first = own ? max(shared_first(p, p.row_count[row]), w.lo) : 0;
        float m = -INFINITY, l = 0.f;
        float4 acc[DIM / 32];
#pragma unroll
        for (int j = 0; j < DIM / 32; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int t = 0; t < w.n_units; ++t) {
            const int j0 = (w.lo / SR_KEYS + w.first_unit + t) * SR_KEYS;
            __syncthreads();                             // the unit before is done with keys and values
            if (tid < SR_KEYS) {
                const int j = j0 + tid;
                long long line = -1;
                if (j >= w.lo && j < w.hi) {
                    const int page = p.block_table[(size_t)w.looks * p.table_width + j / p.page_size];
                    if (page >= 0 && page < p.n_pages) line = ((long long)page * p.hkv + w.kvh) * p.page_size + j % p.page_size;
                }
                s.line[tid] = line;
            }
            __syncthreads();
            // A warp four lines, four components a lane and load (eight loads of keys, then eight of values, before the first is laid down).
            sr_lines<T, DIM, DIM + 4>(&s.k[0][0], kt, s.line, p.d, p.d % 4 == 0);
            sr_lines<T, DIM, DIM>(&s.v[0][0], vt, s.line, p.dv, p.dv % 4 == 0);
            __syncthreads();
            if (shares == 1) sr_unit<4, DIM>(s, p, pair, own, 0, j0, first, count, m, l, acc);
            else if (shares == 2) sr_unit<2, DIM>(s, p, pair, own, 2 * share, j0, first, count, m, l, acc);
            else sr_unit<1, DIM>(s, p, pair, own, share, j0, first, count, m, l, acc);
        }
        if (shares > 1) {
            // The shares' sums, through the keys' and values' places, added up in the order of the shares.
            __syncthreads();
            float* sums = &s.k[slot][0];
            float* states = &s.v[0][0];
#pragma unroll
            for (int c = 0; c < DIM / 32; ++c) *reinterpret_cast<float4*>(sums + 32 * c + 4 * sub) = acc[c];
            if (sub == 0) { states[2 * slot] = m; states[2 * slot + 1] = l; }
            __syncthreads();
            if (share > 0) continue;
            for (int k = 1; k < shares; ++k) m = fmaxf(m, states[2 * (slot + k * places)]);
            const float base = m == -INFINITY ? 0.f : m, mine = states[2 * slot] == -INFINITY ? 0.f : expf(states[2 * slot] - base);
            l *= mine;
#pragma unroll
            for (int c = 0; c < DIM / 32; ++c) { acc[c].x *= mine; acc[c].y *= mine; acc[c].z *= mine; acc[c].w *= mine; }
            for (int k = 1; k < shares; ++k) {
                const int other = slot + k * places;
                if (states[2 * other] == -INFINITY) continue;
                const float theirs = expf(states[2 * other] - base);
                l = fmaf(theirs, states[2 * other + 1], l);
#pragma unroll
                for (int c = 0; c < DIM / 32; ++c) {
                    const float4 y = *reinterpret_cast<const float4*>(&s.k[other][32 * c + 4 * sub]);
                    acc[c].x = fmaf(theirs, y.x, acc[c].x);
                    acc[c].y = fmaf(theirs, y.y, acc[c].y);
                    acc[c].z = fmaf(theirs, y.z, acc[c].z);
                    acc[c].w = fmaf(theirs, y.w, acc[c].w);
                }
            }
        }
        if (own) {
            float* piece = pieces + (size_t)pair * SH_PIECE(p.dv);
#pragma unroll
            for (int c = 0; c < DIM / 32; ++c) {
                const int at = 32 * c + 4 * sub;
                if (at < p.dv) piece[at] = acc[c].x;
                if (at + 1 < p.dv) piece[at + 1] = acc[c].y;
                if (at + 2 < p.dv) piece[at + 2] = acc[c].z;
                if (at + 3 < p.dv) piece[at + 3] = acc[c].w;
            }
            if (sub == 0) { piece[(p.dv + 3) / 4 * 4] = m; piece[(p.dv + 3) / 4 * 4 + 1] = l; }
        }
    }
}

// Joins a (row, head) pair's pieces: its tile's, worker by worker, then its own. A warp a pair: 32 pieces' references and sums at once, a lane each,
// then four (or eight) components a lane over the pieces in their order.
constexpr int SJ_WARPS = 4;
template <typename T>
__global__ void __launch_bounds__(SJ_WARPS * 32) shared_combine_kernel(const SharedParams p, int tile_pairs) {
    dependent_wait();
    dependent_trigger();
    const int pair = blockIdx.x * SJ_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (pair >= p.rows * p.hq) return;
    const int r = pair / p.hq, head = pair % p.hq;
    const int group = p.hq / p.hkv, kvh = head / group, width = SH_PIECE(p.dv);
    const int t = p.cut[SH_CUT_ROW_TILE + r], tiles = p.cut[SH_CUT_COUNTS], row_at = p.cut[SH_CUT_ROW_UNITS + r];
    const int row_units = p.cut[SH_CUT_ROW_UNITS + r + 1] - row_at;
    const int all_tiles = p.cut[SH_CUT_TILE_UNITS + tiles], all_rows = p.cut[SH_CUT_ROW_UNITS + p.rows];
    const int tile_workers = p.cut[SH_CUT_COUNTS + 1], row_workers = p.cut[SH_CUT_COUNTS + 2];
    const float sink = p.sinks ? p.sinks[head] : -INFINITY;
    const float* piece[2] = {nullptr, nullptr};          // the first of the tile's and of the row's, and the floats from one to the next
    int count[2] = {0, 0};
    const size_t step[2] = {(size_t)tile_pairs * width, (size_t)group * width};
    if (t >= 0) {
        const int at = p.cut[SH_CUT_TILE_UNITS + t], units = p.cut[SH_CUT_TILE_UNITS + t + 1] - at;
        const int* tile = p.cut + SH_CUT_TILES + 3 * t;
        const int row0 = tile[0], n = tile[1], before = tile[2];
        if (units > 0) {
            const long long u = (long long)at * p.hkv + (long long)kvh * units, all = (long long)all_tiles * p.hkv;
            const int first = shared_worker_of(u, all, tile_workers);
            count[0] = shared_worker_of(u + units - 1, all, tile_workers) - first + 1;
            piece[0] = p.tile_pieces + (shared_tile_place(p, before, n, kvh, first, tile_pairs) + (r - row0) * group + head % group) * width;
        }
    }
    if (row_units > 0) {
        const long long u = (long long)row_at * p.hkv + (long long)kvh * row_units, all = (long long)all_rows * p.hkv;
        const int first = shared_worker_of(u, all, row_workers);
        count[1] = shared_worker_of(u + row_units - 1, all, row_workers) - first + 1;
        piece[1] = p.row_pieces + (shared_row_place(p, r, kvh, first) + head % group) * width;
    }
    const int n = count[0] + count[1];
    auto at = [&](int b) { return b < count[0] ? piece[0] + b * step[0] : piece[1] + (b - count[0]) * step[1]; };
    float m = sink;
    for (int b = lane; b < n; b += 32) m = fmaxf(m, at(b)[(p.dv + 3) / 4 * 4]);
    m = warp_max(m);
    const int quads = (p.dv + 3) / 4;                    // of components: lane's, and from 128 components on 32 + lane's
    float4 sum[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    float l = 0.f;
    for (int base = 0; base < n; base += 32) {
        float mine = 0.f;
        if (base + lane < n) {
            const float2 x = *reinterpret_cast<const float2*>(at(base + lane) + (p.dv + 3) / 4 * 4);
            mine = x.x == -INFINITY ? 0.f : expf(x.x - m);           // a range of which the row sees nothing
            l = mine > 0.f ? fmaf(mine, x.y, l) : l;
        }
        const int here = min(32, n - base);
        constexpr int DEEP = 8;                          // pieces asked for before the first is used
        for (int b0 = 0; b0 < here; b0 += DEEP) {
            float4 v[DEEP][2];
#pragma unroll
            for (int b = 0; b < DEEP; ++b) {
                const float4* x = reinterpret_cast<const float4*>(at(base + min(b0 + b, here - 1)));
#pragma unroll
                for (int k = 0; k < 2; ++k) v[b][k] = lane + 32 * k < quads ? x[lane + 32 * k] : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int b = 0; b < DEEP; ++b) {
                const float w = __shfl_sync(0xffffffffu, mine, min(b0 + b, 31));
                if (w == 0.f || b0 + b >= here) continue;            // (a piece without weight may be anything)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    sum[k].x = fmaf(w, v[b][k].x, sum[k].x);
                    sum[k].y = fmaf(w, v[b][k].y, sum[k].y);
                    sum[k].z = fmaf(w, v[b][k].z, sum[k].z);
                    sum[k].w = fmaf(w, v[b][k].w, sum[k].w);
                }
            }
        }
    }
    float total = warp_sum(l);
    if (p.sinks && m != -INFINITY) total += expf(sink - m);
    const float inv = total > 0.f ? 1.f / total : 0.f;
    T* out = static_cast<T*>(p.out) + (size_t)pair * p.dv;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int c = 4 * (lane + 32 * k);
        const float v[4] = {sum[k].x * inv, sum[k].y * inv, sum[k].z * inv, sum[k].w * inv};
        if (c + 3 < p.dv && p.dv % 4 == 0) {
            store_four(out + c, make_float4(v[0], v[1], v[2], v[3]));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < p.dv) Elem<T>::store(out + c + j, v[j]);
        }
    }
}
template <typename T> static int launch_combine(const SharedParams& p, int tile_pairs, cudaStream_t s) {
    launch_dependent_if(p.rows <= DEPENDENT_ROWS, shared_combine_kernel<T>, dim3((p.rows * p.hq + SJ_WARPS - 1) / SJ_WARPS), dim3(SJ_WARPS * 32), 0, s, p, tile_pairs);
    return check_launch("shared_attention");
}

template <typename T, int DIM> static int launch_shared_rows(const SharedParams& p, int blocks, cudaStream_t s) {
    const int smem = (int)sizeof(SharedRowsSmem<DIM>);
    static unsigned long long done = 0;
    if (int e = allow_shared_memory((const void*)shared_rows_kernel<T, DIM>, smem, &done)) return e;
    shared_rows_kernel<T, DIM><<<blocks, SR_THREADS, smem, s>>>(p);
    if (int err = check_launch("shared_attention")) return err;
    return launch_combine<T>(p, SR_PAIRS, s);
}
template <typename T> static int launch_shared_rows(const SharedParams& p, int blocks, cudaStream_t s) {
    const int most = p.d > p.dv ? p.d : p.dv;
    return most <= 64 ? launch_shared_rows<T, 64>(p, blocks, s) : most <= 128 ? launch_shared_rows<T, 128>(p, blocks, s) : launch_shared_rows<T, 256>(p, blocks, s);
}

}  // namespace kb

using namespace kb;

static int shared_blocks() { return multiprocessors(); }

// Whether the tensor cores take a layer (bfloat16): one head size, whole groups of 16 positions a page, up to 16 query heads a kv head.
static bool shared_on_tensor_cores(int dtype, int hq, int hkv, int d, int dv, int page_size) {
    return dtype == KB_DT_BF16 && d == dv && (d == 64 || d == 128 || d == 256) && page_size % 16 == 0 && hq / hkv <= 16;
}

// Where all rows' block tables together have room for no more keys and values than this (the tables' width, not what lies in them: a recorded launch's choice stays
// while lengths change), every row reads what it sees by itself: the shared part comes out of
// the second-level cache for all but the first, and the kernel over tiles, some 10 us before its first product, is not launched. As measured
// (us, with tiles and without): 8 heads over 4 of 256, 2 rows sharing 64 positions (1 MB) 19 and 9, 16 sharing 1,024 (75 MB) 22 and 19, 8 sharing
// 4,096 (138 MB) 30 and 26, 32 sharing 1,024 (153 MB) 22 and 26, 16 sharing 4,096 (277 MB) 29 and 38; 32 over 16 of 128, 8 sharing 1,024 (74 MB) 27 and
// 17, 64 sharing 64 (126 MB) 46 and 22, 16 sharing 1,024 (151 MB) 26 and 25, 8 sharing 4,096 (276 MB) 30 and 37.
constexpr long long SHARED_ALONE_BYTES = 144000000;

struct SharedScratch { long long tile_places, row_places; };
static SharedScratch shared_scratch(int rows, int hq, int hkv, int d) {          // what either path needs at most
    const int blocks = shared_blocks();
    return SharedScratch{shared_tile_places(rows, hq, blocks, 128), shared_row_places(rows, hq, hkv, blocks * shared_own_workers(d))};
}
// What a unit of a tile costs a multiprocessor, counted in units of 16 positions of a row; more than its bytes say, since a block over tiles takes
// some 15 us to begin and to leave its pieces. As measured at 8, 12, 16, 24: 64 answers to 2,048 tokens, 16 heads over 8 of 256, 61, 58, 53, 54 us; 8
// to 6,144, 8 over 4 of 256, 31, 27, 31, 36; two prompts and 34 requests, 32 over 16 of 128, 84, 76, 70, 68. (These three only, and before both kernels
// counted the same units: the last takes 53 since.)
static float shared_tile_cost(int d) { return d == 256 ? 14.f : 20.f; }

// Floats of scratch memory: the tiles' pieces, the rows' pieces, then the cut.
extern "C" long long kb_shared_attention_scratch_floats(int rows, int hq, int hkv, int d, int dv) {
    if (rows <= 0 || rows > SH_ROWS || hq <= 0 || hkv <= 0 || hq % hkv || dv <= 0) return 0;
    const SharedScratch x = shared_scratch(rows, hq, hkv, d);
    return (x.tile_places + x.row_places) * SH_PIECE(dv) + SH_CUT_INTS;
}

// 1 where the kernels take these sizes, 2 where they take them on the tensor cores.
extern "C" int kb_shared_attention_takes(int dtype, int hq, int hkv, int d, int dv, int page_size) {
    if ((dtype != KB_DT_F32 && dtype != KB_DT_BF16) || hkv <= 0 || hq <= 0 || hq % hkv || hq / hkv > SR_PAIRS || d <= 0 || d > SR_DIM || dv <= 0 || dv > SR_DIM || page_size <= 0)
        return 0;
    return shared_on_tensor_cores(dtype, hq, hkv, d, dv, page_size) ? 2 : 1;
}

extern "C" int kb_shared_attention(void* out, const void* q, const void* k_table, const void* v_table, int dtype, const int* block_table,
                                   const int* row_count, const int* share_id, const int* share_len, int rows, int hq, int hkv, int d, int dv,
                                   int page_size, int table_width, int n_pages, int window, float scale, float cap, const float* sinks,
                                   float* scratch, long long scratch_floats, void* stream) {
    KB_REQUIRE(rows >= 0 && rows <= SH_ROWS, "shared_attention: %d rows (0..%d)", rows, SH_ROWS);
    KB_REQUIRE(kb_shared_attention_takes(dtype, hq, hkv, d, dv, page_size),
               "shared_attention: dtype code %d, %d heads over %d of %d / %d, pages of %d are not taken", dtype, hq, hkv, d, dv, page_size);
    KB_REQUIRE(table_width > 0 && n_pages > 0 && window >= 0 && cap >= 0.f, "shared_attention: table width %d, pages %d, window %d, soft cap %g", table_width,
               n_pages, window, cap);
    KB_REQUIRE((long long)table_width * page_size <= 0x7fffffffll / 4 && ((long long)table_width * page_size / 16 + 2) * rows * hkv <= 0x7fffffffll,
               "shared_attention: %d block tables of %d pages of %d positions are too many for one launch", rows, table_width, page_size);
    if (rows == 0) return 0;
    KB_REQUIRE(scratch != nullptr && scratch_floats >= kb_shared_attention_scratch_floats(rows, hq, hkv, d, dv), "shared_attention: scratch memory of %lld floats",
               scratch_floats);
    SharedParams p = {};
    p.q = q; p.k_table = k_table; p.v_table = v_table; p.block_table = block_table; p.row_count = row_count; p.share_id = share_id;
    p.share_len = share_len; p.sinks = sinks; p.out = out; p.rows = rows; p.hq = hq; p.hkv = hkv; p.d = d; p.dv = dv;
    p.page_size = page_size; p.table_width = table_width; p.n_pages = n_pages; p.window = window; p.scale = scale; p.cap = cap;
    const int blocks = shared_blocks();
    const SharedScratch x = shared_scratch(rows, hq, hkv, d);
    p.tile_pieces = scratch;
    p.row_pieces = scratch + x.tile_places * SH_PIECE(dv);
    p.cut = reinterpret_cast<int*>(p.row_pieces + x.row_places * SH_PIECE(dv));
    KB_REQUIRE((((uintptr_t)q | (uintptr_t)k_table | (uintptr_t)v_table | (uintptr_t)out) & 15) == 0, "shared_attention: operands must be 16-byte aligned");
    if (shared_on_tensor_cores(dtype, hq, hkv, d, dv, page_size)) {
        const unsigned long long lines = (unsigned long long)n_pages * hkv * page_size;
        KB_REQUIRE(lines <= 0x7fffffffull, "shared_attention: tables of %llu lines", lines);
        p.alone = (long long)rows * table_width * page_size * hkv * d * 4 <= SHARED_ALONE_BYTES;
        CUtensorMap mk, mv;
        // In a step of few rows the kernel over rows starts while the one over tiles runs, and takes the multiprocessors that one leaves.
        if (!p.alone) {
            const bool side = may_chain(p.rows <= DEPENDENT_ROWS);
            p.tile_cost = side ? shared_tile_cost(d) : 0.f;
            if (int e = encode_map_bf16(&mk, k_table, lines, d, d, 16)) return e;
            if (int e = encode_map_bf16(&mv, v_table, lines, d, d, 16)) return e;
            if (int e = launch_shared_tiles(p, mk, mv, blocks, (cudaStream_t)stream)) return e;
        }
        CUtensorMap ok, ov;                              // the same in boxes of all of a line's chunks
        if (int e = encode_map_bf16_chunks(&ok, k_table, lines, d, 16)) return e;
        if (int e = encode_map_bf16_chunks(&ov, v_table, lines, d, 16)) return e;
        if (int e = launch_shared_own(p, ok, ov, blocks, (cudaStream_t)stream)) return e;
        return launch_combine<__nv_bfloat16>(p, 128, (cudaStream_t)stream);
    }
    return dtype == KB_DT_F32 ? launch_shared_rows<float>(p, blocks, (cudaStream_t)stream) : launch_shared_rows<__nv_bfloat16>(p, blocks, (cudaStream_t)stream);
}

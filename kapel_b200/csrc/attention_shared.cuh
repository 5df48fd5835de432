// Attention of single tokens whose requests share the pages of a prompt: how the work is cut, for the kernels that do it.
//
// Row r is request r: it has seen row_count[r] positions, its own included, and reads those its window leaves. Rows that follow one another with
// the same share_id and share_len share the pages of their first share_len positions (whole pages, looked up in the block table of the
// row that sees furthest back: behind a window the others may have given their first pages back). Such a run is cut into tiles of at most `tile_rows` (row, query head) pairs of one kv head; a tile reads the positions that any of
// its rows sees of what they share, once. What a row has behind that is an item of its own. So
//   out = sum e^x v / (sum e^x + e^sink) over the row's positions
// is put together from pieces (sum e^(x - m) v, m, sum e^(x - m)), each over a range of positions.
//
// The cut is made on the device (lengths change from step to step, a recorded step's launch does not). An item is (a tile or a row,
// its positions); its units are `keys` positions each, times the kv heads. All items' units lie one after the other, and block b of G takes the
// units [U b / G, U (b + 1) / G), with G no more than U: every block the same number, whether a few long prompts or many short answers make them up. Where a block's
// range ends inside an item its piece is one of several; they are joined by `shared_combine_kernel`.
//
// Pieces are written by (row, head) to a place that follows from the cut alone: the items' rows before it plus `tile_rows` for each block
// before the one that writes: a block's pieces of different items cannot meet, nor those of different blocks of one item.
#pragma once
#include "common.cuh"

namespace kb {

constexpr int SH_ROWS = 512;                 // requests of one call

struct SharedParams {
    const void* q;             // [rows, hq, d]
    const void* k_table;       // [pages, hkv, page_size, d]
    const void* v_table;       // [pages, hkv, page_size, dv]
    const int* block_table;    // [rows, table_width]
    const int* row_count;      // [rows]
    const int* share_id;       // [rows]
    const int* share_len;      // [rows]
    const float* sinks;        // [hq] or null
    void* out;                 // [rows, hq, dv]
    float* pieces;             // [places, dv + 2]: (sum, m, sum of weights), m in natural units
    int* cut;                  // what block 0 leaves for the kernel that joins: see SharedCut
    int rows, hq, hkv, d, dv, page_size, table_width, n_pages, window;
    float scale, cap;
};

// The cut as the joining kernel reads it, in p.cut: [0] tiles, [1] units, [2] blocks, [3] rows in tiles; then SH_ROWS tiles of each row (-1:
// none), then for each tile {first row, rows, rows in tiles before}, then the running total of units over tiles and rows (one more than items).
constexpr int SH_CUT_HEAD = 4;
constexpr int SH_CUT_INTS = SH_CUT_HEAD + SH_ROWS + 3 * SH_ROWS + 2 * SH_ROWS + 1;

// A block's copy of the cut.
struct SharedCut {
    int tiles, units, tile_rows_total;
    int row_tile[SH_ROWS];                   // a row's tile, -1 where it shares nothing that it sees
    int row0[SH_ROWS], n[SH_ROWS], before[SH_ROWS];      // by tile
    int looks[SH_ROWS];                      // by tile: the row whose block table has the pages
    int klo[SH_ROWS], khi[SH_ROWS];          // by tile: the positions [klo, khi) that any row sees of what they share
    int upto[2 * SH_ROWS + 1];               // units (of one kv head) before item i: tiles, then rows
};

__device__ __forceinline__ int shared_first(const SharedParams& p, int count) {      // the first position a row sees
    return (p.window > 0 && count > p.window) ? count - p.window : 0;
}
// What a row shares, as the launcher's limits let it stand: whole pages, no more than its block table holds and than it has seen.
__device__ __forceinline__ int shared_length(const SharedParams& p, int r) {
    const int n = min(min(p.share_len[r], p.row_count[r]), p.table_width * p.page_size);
    return n > 0 ? n / p.page_size * p.page_size : 0;
}
__device__ __forceinline__ int shared_own_units(const SharedParams& p, int r, int length, int keys, int& lo, int& hi) {
    hi = min(p.row_count[r], p.table_width * p.page_size);
    lo = max(length, shared_first(p, p.row_count[r]));
    return lo < hi ? (hi - lo / keys * keys + keys - 1) / keys : 0;
}

// Makes the cut with the whole block (any number of warps); `rows_a_tile` requests to a tile, `keys` positions to a unit.
__device__ void shared_make_cut(const SharedParams& p, SharedCut& c, int rows_a_tile, int keys) {
    const int tid = threadIdx.x, lane = tid & 31, nt = blockDim.x;
    for (int i = tid; i < p.rows; i += nt) { c.klo[i] = 0x7fffffff; c.khi[i] = 0; c.n[i] = 0; c.row0[i] = 0x7fffffff; c.looks[i] = 0x7fffffff; }
    if (tid < 32) {
        // Where each row's run begins, and with it the row's place in the run: rows_a_tile of them to a tile.
        int run = 0, tiles = 0;
        for (int base = 0; base < p.rows; base += 32) {
            const int r = base + lane;
            const bool in = r < p.rows;
            const int length = in ? shared_length(p, r) : 0;
            const bool starts = in && (r == 0 || length == 0 || shared_length(p, r - 1) != length || p.share_id[r] != p.share_id[r - 1]);
            const unsigned who = __ballot_sync(0xffffffffu, starts);
            const unsigned mine = who & (0xffffffffu >> (31 - lane));
            const int begins = mine ? base + 31 - __clz(mine) : run;
            const bool opens = in && length > 0 && (r - begins) % rows_a_tile == 0;
            const unsigned opened = __ballot_sync(0xffffffffu, opens);
            if (in) c.row_tile[r] = length > 0 ? tiles + __popc(opened & (0xffffffffu >> (31 - lane))) - 1 : -1;
            tiles += __popc(opened);
            if (who) run = base + 31 - __clz(who);
        }
        if (lane == 0) c.tiles = tiles;
    }
    __syncthreads();
    for (int r = tid; r < p.rows; r += nt) {
        const int t = c.row_tile[r];
        if (t < 0) continue;
        atomicMin(&c.row0[t], r);
        atomicAdd(&c.n[t], 1);
        const int length = shared_length(p, r), first = shared_first(p, p.row_count[r]);
        if (first < length) {                            // else the window has passed what it shares
            atomicMin(&c.klo[t], first);
            atomicMax(&c.khi[t], length);
        }
    }
    __syncthreads();
    for (int r = tid; r < p.rows; r += nt) {
        const int t = c.row_tile[r];
        if (t >= 0 && shared_first(p, p.row_count[r]) <= c.klo[t]) atomicMin(&c.looks[t], r);
    }
    if (tid < 32) {
        int units = 0, rows_before = 0;
        const int tiles = c.tiles, items = tiles + p.rows;
        for (int base = 0; base < items; base += 32) {
            const int i = base + lane;
            int u = 0, n = 0;
            if (i < tiles) {
                n = c.n[i];
                if (c.klo[i] < c.khi[i]) u = (c.khi[i] - c.klo[i] / keys * keys + keys - 1) / keys;
            } else if (i < items) {
                int lo, hi;
                u = shared_own_units(p, i - tiles, shared_length(p, i - tiles), keys, lo, hi);
            }
            int uu = u, nn = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int a = __shfl_up_sync(0xffffffffu, uu, o), b = __shfl_up_sync(0xffffffffu, nn, o);
                if (lane >= o) { uu += a; nn += b; }
            }
            if (i < items) c.upto[i] = units + uu - u;
            if (i < tiles) c.before[i] = rows_before + nn - n;
            units += __shfl_sync(0xffffffffu, uu, 31);
            rows_before += __shfl_sync(0xffffffffu, nn, 31);
        }
        if (lane == 0) { c.upto[items] = units; c.units = units; c.tile_rows_total = rows_before; }
    }
    __syncthreads();
}

// Blocks that have work: one a unit at least, so that no block between two that share an item is without a piece of it.
__device__ __forceinline__ int shared_workers(long long units) { return (int)min((long long)gridDim.x, units); }

// Block 0 leaves the cut for the joining kernel.
__device__ void shared_leave_cut(const SharedParams& p, const SharedCut& c) {
    int* out = p.cut;
    if (threadIdx.x == 0) { out[0] = c.tiles; out[1] = c.units; out[2] = shared_workers((long long)c.units * p.hkv); out[3] = c.tile_rows_total; }
    for (int i = threadIdx.x; i < p.rows; i += blockDim.x) out[SH_CUT_HEAD + i] = c.row_tile[i];
    for (int i = threadIdx.x; i < c.tiles; i += blockDim.x) {
        int* t = out + SH_CUT_HEAD + SH_ROWS + 3 * i;
        t[0] = c.row0[i]; t[1] = c.n[i]; t[2] = c.before[i];
    }
    for (int i = threadIdx.x; i <= c.tiles + p.rows; i += blockDim.x) out[SH_CUT_HEAD + 4 * SH_ROWS + i] = c.upto[i];
}

// The block that has unit u of U, and a block's first unit.
__device__ __forceinline__ int shared_block_of(long long u, int units, int blocks) { return (int)(((u + 1) * blocks - 1) / units); }
__device__ __forceinline__ int shared_begin(int b, long long units, int blocks) { return (int)(units * b / blocks); }

// One item's part of a block's range.
struct SharedPart {
    int item, kvh;             // tiles first, then rows
    int row0, n;               // its requests
    int looks;                 // the one whose block table has the pages
    int lo, hi;                // positions of the item
    int first_unit, n_units;   // of the item's units those that this block takes (n_units of them)
    int whole;                 // whether that is all of them
    long long place;           // where this block's pieces of it go
};

// The part that holds the block's unit u (u < end); `tile_pairs` the (row, head) pairs of a full tile.
__device__ SharedPart shared_part(const SharedParams& p, const SharedCut& c, int u, int end, int keys, int tile_pairs) {
    SharedPart s;
    const int items = c.tiles + p.rows;
    int lo = 0, hi = items;                              // the last item that begins at or before u
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((long long)c.upto[mid] * p.hkv <= u) lo = mid; else hi = mid;
    }
    s.item = lo;
    const int units = c.upto[lo + 1] - c.upto[lo];       // of a kv head; not 0, or a later item would begin here too
    const int in = u - c.upto[lo] * p.hkv;
    s.kvh = in / units;
    s.first_unit = in % units;
    s.n_units = min(units - s.first_unit, end - u);
    s.whole = s.n_units == units;
    const int group = p.hq / p.hkv;
    long long rows_before;
    if (lo < c.tiles) {
        s.row0 = c.row0[lo]; s.n = c.n[lo]; s.looks = c.looks[lo]; s.lo = c.klo[lo]; s.hi = c.khi[lo];
        rows_before = (long long)c.before[lo] * p.hkv + (long long)s.kvh * s.n;
    } else {
        s.row0 = s.looks = lo - c.tiles; s.n = 1;
        shared_own_units(p, s.row0, shared_length(p, s.row0), keys, s.lo, s.hi);
        rows_before = (long long)(c.tile_rows_total + s.row0) * p.hkv + s.kvh;
    }
    s.place = rows_before * group + (long long)blockIdx.x * tile_pairs;
    return s;
}

// Places for pieces: every (row, head) once as a tile's and once as its own, and a full tile for each block.
__host__ __device__ inline long long shared_places(int rows, int hq, int blocks, int tile_pairs) {
    return 2ll * rows * hq + (long long)blocks * tile_pairs;
}

}  // namespace kb

// Attention of single tokens whose requests share the pages of a prompt: how the work is cut, for the kernels that do it.
//
// Row r is request r: it has seen row_count[r] positions, its own included, and reads those its window leaves. Rows that follow one another with
// the same share_id and share_len share the pages of their first share_len positions (whole pages, looked up in the block table of the
// row that sees furthest back: behind a window the others may have given their first pages back). Such a run is cut into tiles of at most
// `tile_pairs` (row, query head) pairs of one kv head; a tile reads the positions that any of its rows sees of what they share, once. What a
// row has behind that it reads by itself. So
//   out = sum e^x v / (sum e^x + e^sink) over the row's positions
// is put together from pieces (sum e^(x - m) v, m, sum e^(x - m)), each over a range of positions, which `shared_combine_kernel` joins.
//
// The cut is made on the device (lengths change from step to step, a recorded step's launch does not), for tiles and for rows alike. An
// item is a tile or a row with its positions; its units are so many positions each, times the kv heads. All items' units lie one
// after the other, and worker w of W (a block, or a warp) takes the units [U w / W, U (w + 1) / W), with W no more than U: every worker the
// same number, whether a few long prompts or many short answers make them up. Where a worker's range ends inside an item its piece is
// one of several.
//
// Pieces go to a place that follows from the cut alone: the pairs of the items before, plus a full item's pairs for each worker before the
// one that writes: a worker's pieces of different items cannot meet, nor those of different workers of one item.
#pragma once
#include "common.cuh"

namespace kb {

constexpr int SH_ROWS = 512;                 // requests of one call
__host__ __device__ constexpr int SH_PIECE(int dv) { return (dv + 3) / 4 * 4 + 4; }      // floats of a piece: dv (up to a multiple of four), then m and the sum of weights

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
    float* tile_pieces;        // [places, SH_PIECE]: (sum, m, sum of weights), m in natural units; of tiles,
    float* row_pieces;         // ... and of rows
    int* cut;                  // what the kernels leave for the one that joins: see SH_CUT_*
    int rows, hq, hkv, d, dv, page_size, table_width, n_pages, window;
    float scale, cap;
    int alone;                 // every row reads all it sees by itself (there is little to read)
    float tile_cost;           // > 0: the kernels over tiles and over rows run side by side; what a tile's unit costs, counted in a row's units
};

// The cut as the joining kernel reads it, in p.cut: the tile of each row (-1: none), for each tile {first row, rows, rows in tiles before}, and for tiles
// and rows the running total of their units (of one kv head; one more than there are), the number of items and of workers.
constexpr int SH_CUT_ROW_TILE = 0, SH_CUT_TILES = SH_ROWS, SH_CUT_TILE_UNITS = 4 * SH_ROWS, SH_CUT_ROW_UNITS = 5 * SH_ROWS + 1;
constexpr int SH_CUT_COUNTS = 6 * SH_ROWS + 2;           // tiles, workers over tiles, workers over rows
constexpr int SH_CUT_INTS = SH_CUT_COUNTS + 3;

// A block's copy of the cut into tiles.
struct SharedTiles {
    int tiles, row_units;                    // tiles, and units of 16 positions that the rows read by themselves
    int row_tile[SH_ROWS];                   // a row's tile, -1 where it shares nothing
    int length[SH_ROWS], id[SH_ROWS], first[SH_ROWS];    // by row: positions it shares, with whom, the first it sees
    int row0[SH_ROWS], n[SH_ROWS], before[SH_ROWS + 1];      // by tile
    int looks[SH_ROWS];                      // by tile: the row whose block table has the pages
    int klo[SH_ROWS], khi[SH_ROWS];          // by tile: the positions [klo, khi) that any row sees of what they share
    int upto[SH_ROWS + 1];                   // units before tile i
};

__device__ __forceinline__ int shared_first(const SharedParams& p, int count) {      // the first position a row sees
    return (p.window > 0 && count > p.window) ? count - p.window : 0;
}
// What a row shares, as the launcher's limits let it stand: whole pages, no more than its block table holds and than it has seen.
__device__ __forceinline__ int shared_length(const SharedParams& p, int r) {
    if (p.alone) return 0;
    const int n = min(min(p.share_len[r], p.row_count[r]), p.table_width * p.page_size);
    return n > 0 ? n / p.page_size * p.page_size : 0;
}
// The positions [lo, hi) that a row reads by itself; returns their units of `keys`, counted from a multiple of `keys`.
__device__ __forceinline__ int shared_own(const SharedParams& p, int r, int keys, int& lo, int& hi) {
    hi = min(p.row_count[r], p.table_width * p.page_size);
    lo = max(shared_length(p, r), shared_first(p, p.row_count[r]));
    return lo < hi ? (hi - lo / keys * keys + keys - 1) / keys : 0;
}

// upto[0 .. n] holds n numbers and becomes their running totals (what lies before each, then all), by one warp. No barrier.
static __device__ __noinline__ void shared_totals(int* upto, int n) {
    const int lane = threadIdx.x & 31;
    int total = 0;
#pragma unroll 1
    for (int base = 0; base < n; base += 32) {
        const int i = base + lane;
        const int mine = i < n ? upto[i] : 0;
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        if (i < n) upto[i] = total + sum - mine;
        total += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) upto[n] = total;
}

// The cut into tiles, by the whole block; `rows_a_tile` requests to a tile, `keys` positions to a unit.
__device__ inline void shared_cut_tiles(const SharedParams& p, SharedTiles& c, int rows_a_tile, int keys) {
    const int tid = threadIdx.x, lane = tid & 31, nt = blockDim.x;
#pragma unroll 1
    for (int i = tid; i < p.rows; i += nt) {
        c.klo[i] = 0x7fffffff; c.khi[i] = 0; c.before[i] = 0; c.row0[i] = 0x7fffffff; c.looks[i] = 0x7fffffff;
        c.length[i] = shared_length(p, i);               // every load of the cut is asked for here, all rows at once
        c.id[i] = p.share_id[i];
        c.first[i] = shared_first(p, p.row_count[i]);
    }
    __syncthreads();
    if (tid < 32) {
        // Where each row's run begins, and with it the row's place in the run: rows_a_tile of them to a tile.
        int run = 0, tiles = 0;
#pragma unroll 1
        for (int base = 0; base < p.rows; base += 32) {
            const int r = base + lane;
            const bool in = r < p.rows;
            const int length = in ? c.length[r] : 0;
            const bool starts = in && (r == 0 || length == 0 || c.length[r - 1] != length || c.id[r] != c.id[r - 1]);
            const unsigned who = __ballot_sync(0xffffffffu, starts);
            const unsigned mine = who & (0xffffffffu >> (31 - lane));
            const int begins = mine ? base + 31 - __clz(mine) : run;
            const bool opens = in && length > 0 && (r - begins) % rows_a_tile == 0;
            const unsigned opened = __ballot_sync(0xffffffffu, opens);
            if (in) c.row_tile[r] = length > 0 ? tiles + __popc(opened & (0xffffffffu >> (31 - lane))) - 1 : -1;
            tiles += __popc(opened);
            if (who) run = base + 31 - __clz(who);
        }
        if (lane == 0) { c.tiles = tiles; c.row_units = 0; }
    }
    __syncthreads();
#pragma unroll 1
    for (int r = tid; r < p.rows; r += nt) {
        const int t = c.row_tile[r];
        if (p.tile_cost > 0.f) {
            int lo, hi;
            atomicAdd(&c.row_units, shared_own(p, r, 16, lo, hi));
        }
        if (t < 0) continue;
        atomicMin(&c.row0[t], r);
        atomicAdd(&c.before[t], 1);
        if (c.first[r] < c.length[r]) {                  // else the window has passed what it shares
            atomicMin(&c.klo[t], c.first[r]);
            atomicMax(&c.khi[t], c.length[r]);
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int r = tid; r < p.rows; r += nt) {
        const int t = c.row_tile[r];
        if (t >= 0 && c.first[r] <= c.klo[t]) atomicMin(&c.looks[t], r);
    }
#pragma unroll 1
    for (int i = tid; i < c.tiles; i += nt) {
        c.n[i] = c.before[i];
        c.upto[i] = c.klo[i] < c.khi[i] ? (c.khi[i] - c.klo[i] / keys * keys + keys - 1) / keys : 0;
    }
    __syncthreads();
    if (tid < 32) {
        shared_totals(c.before, c.tiles);
        shared_totals(c.upto, c.tiles);
    }
    __syncthreads();
}

// The cut into rows: upto[r] = units before row r, which reads positions [lo[r], hi[r]) by itself. By the whole block.
__device__ inline void shared_cut_rows(const SharedParams& p, int* upto, int* lo, int* hi, int keys) {
#pragma unroll 1
    for (int r = threadIdx.x; r < p.rows; r += blockDim.x) upto[r] = shared_own(p, r, keys, lo[r], hi[r]);
    __syncthreads();
    if (threadIdx.x < 32) shared_totals(upto, p.rows);
    __syncthreads();
}

// The units of all tiles of one kv head, the number that shared_cut_tiles comes to, for the kernel over rows, which needs no more of that cut: both kernels
// divide the multiprocessors by it. `length` and `id` by row; klo and khi [SH_ROWS] are scratch. By one warp.
__device__ __forceinline__ int shared_tile_units(const SharedParams& p, const int* length, const int* id, int* klo, int* khi, int rows_a_tile, int keys) {
    const int lane = threadIdx.x & 31;
    int run = 0, tiles = 0;
#pragma unroll 1
    for (int base = 0; base < p.rows; base += 32) {
        const int r = base + lane, n = r < p.rows ? length[r] : 0;
        const bool starts = r < p.rows && (r == 0 || n == 0 || length[r - 1] != n || id[r - 1] != id[r]);
        const unsigned upto_here = 0xffffffffu >> (31 - lane), who = __ballot_sync(0xffffffffu, starts), mine = who & upto_here;
        const int begins = mine ? base + 31 - __clz(mine) : run;
        const bool opens = n > 0 && (r - begins) % rows_a_tile == 0;
        const unsigned opened = __ballot_sync(0xffffffffu, opens);
        const int tile = tiles + __popc(opened & upto_here) - 1;
        if (opens) { klo[tile] = 0x7fffffff; khi[tile] = n; }
        __syncwarp();
        if (n > 0) atomicMin(klo + tile, shared_first(p, p.row_count[r]));
        tiles += __popc(opened);
        if (who) run = base + 31 - __clz(who);
    }
    __syncwarp();
    int units = 0;
    for (int i = lane; i < tiles; i += 32)
        if (klo[i] < khi[i]) units += (khi[i] - klo[i] / keys * keys + keys - 1) / keys;
    return __reduce_add_sync(0xffffffffu, units);
}

// Blocks over tiles where both kernels run side by side, of `blocks` in all: as many as the tiles' share of the work, and of the rest the rows get
// one at least. `tile_units` and `row_units` of one kv head.
__device__ __forceinline__ int shared_tile_blocks(const SharedParams& p, int tile_units, int row_units, int blocks) {
    if (p.tile_cost <= 0.f || row_units == 0) return blocks;
    const float tiles = p.tile_cost * (float)tile_units, all = tiles + (float)row_units;
    return tile_units == 0 ? 0 : min(max((int)(tiles / all * (float)blocks + 0.5f), 1), blocks - 1);
}

// A worker's units, the items' one after the other and each item's kv head by kv head.
struct SharedRange { int begin, end, workers; };
__device__ __forceinline__ SharedRange shared_range(int worker, int most, int units, int hkv) {
    const long long all = (long long)units * hkv;
    SharedRange r;
    r.workers = (int)min((long long)most, all);
    r.begin = worker < r.workers ? (int)(all * worker / r.workers) : 0;
    r.end = worker < r.workers ? (int)(all * (worker + 1) / r.workers) : 0;
    return r;
}
__device__ __forceinline__ int shared_worker_of(long long u, long long units, int workers) { return (int)(((u + 1) * workers - 1) / units); }
// The item that unit u belongs to: the last that begins at or before it (one without units ends where it begins).
__device__ __forceinline__ int shared_item(const int* upto, int items, int hkv, int u) {
    int lo = 0, hi = items;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((long long)upto[mid] * hkv <= u) lo = mid; else hi = mid;
    }
    return lo;
}

// One block leaves what it knows of the cut for the joining kernel.
__device__ inline void shared_leave_tiles(const SharedParams& p, const SharedTiles& c, int workers) {
    for (int i = threadIdx.x; i < p.rows; i += blockDim.x) p.cut[SH_CUT_ROW_TILE + i] = c.row_tile[i];
    for (int i = threadIdx.x; i < c.tiles; i += blockDim.x) {
        int* t = p.cut + SH_CUT_TILES + 3 * i;
        t[0] = c.row0[i]; t[1] = c.n[i]; t[2] = c.before[i];
    }
    for (int i = threadIdx.x; i <= c.tiles; i += blockDim.x) p.cut[SH_CUT_TILE_UNITS + i] = c.upto[i];
    if (threadIdx.x == 0) { p.cut[SH_CUT_COUNTS] = c.tiles; p.cut[SH_CUT_COUNTS + 1] = workers; }
}
__device__ inline void shared_leave_rows(const SharedParams& p, const int* upto, int workers) {
    for (int i = threadIdx.x; i <= p.rows; i += blockDim.x) p.cut[SH_CUT_ROW_UNITS + i] = upto[i];
    if (threadIdx.x == 0) p.cut[SH_CUT_COUNTS + 2] = workers;
}

// Where worker w's pieces of an item go.
__device__ __forceinline__ long long shared_tile_place(const SharedParams& p, int before, int n, int kvh, int worker, int tile_pairs) {
    return ((long long)before * p.hkv + (long long)kvh * n) * (p.hq / p.hkv) + (long long)worker * tile_pairs;
}
__device__ __forceinline__ long long shared_row_place(const SharedParams& p, int r, int kvh, int worker) {
    return ((long long)r * p.hkv + kvh + worker) * (p.hq / p.hkv);
}
inline long long shared_tile_places(int rows, int hq, int workers, int tile_pairs) { return (long long)rows * hq + (long long)workers * tile_pairs; }
inline long long shared_row_places(int rows, int hq, int hkv, int workers) { return (long long)rows * hq + (long long)workers * (hq / hkv); }

}  // namespace kb

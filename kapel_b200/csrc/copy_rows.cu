// Rows of a table copied to other rows of it: what a forked request takes of the one it goes on from (the lines of a page that is not full yet,
// the state of its slot).
#include "common.cuh"

namespace kb {

constexpr int CR_THREADS = 256;

// blockIdx.y: the pair; the row in pieces of V. Rows outside the table are not touched.
template <typename V>
__global__ void __launch_bounds__(CR_THREADS) copy_rows_kernel(V* __restrict__ table, const int* __restrict__ from, const int* __restrict__ to, int rows, long long width) {
    const int a = from[blockIdx.y], b = to[blockIdx.y];
    if (a < 0 || a >= rows || b < 0 || b >= rows || a == b) return;
    const V* src = table + (long long)a * width;
    V* dst = table + (long long)b * width;
    for (long long i = (long long)blockIdx.x * CR_THREADS + threadIdx.x; i < width; i += (long long)gridDim.x * CR_THREADS) dst[i] = src[i];
}

}  // namespace kb

using namespace kb;

// table [rows, row_bytes]: row to[i] becomes row from[i], i < n. No row is both copied from and to.
extern "C" int kb_copy_rows(void* table, const int* from, const int* to, int n, int rows, long long row_bytes, void* stream) {
    KB_REQUIRE(n >= 0 && n <= 65535 && rows > 0 && row_bytes > 0, "copy_rows: %d of %d rows of %lld bytes", n, rows, row_bytes);
    KB_REQUIRE(row_bytes % 2 == 0 && ((uintptr_t)table & 15) == 0, "copy_rows: rows of %lld bytes at an address that is no multiple of 16", row_bytes);
    if (n == 0) return 0;
    KB_REQUIRE(from != nullptr && to != nullptr, "copy_rows: a null pointer");
    const bool wide = row_bytes % 16 == 0;
    const long long pieces = row_bytes / (wide ? 16 : 2);
    const long long want = (pieces + CR_THREADS - 1) / CR_THREADS;
    const dim3 grid((unsigned)(want > 64 ? 64 : want), (unsigned)n);
    if (wide) copy_rows_kernel<uint4><<<grid, CR_THREADS, 0, (cudaStream_t)stream>>>((uint4*)table, from, to, rows, pieces);
    else copy_rows_kernel<uint16_t><<<grid, CR_THREADS, 0, (cudaStream_t)stream>>>((uint16_t*)table, from, to, rows, pieces);
    return check_launch("copy_rows");
}

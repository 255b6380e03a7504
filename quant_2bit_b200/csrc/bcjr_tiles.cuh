// How the rows of a group are cut into column tiles (bcjr_mm.cuh, bcjr_fp8.cu):
// plain integer arithmetic, for the kernels, the launches and tests without a
// GPU.  Row counts go up to kMaxRows; nothing here may pass 32 bits below that.
#pragma once

#ifdef __CUDACC__
#define BCJR_TILES_FN __host__ __device__ __forceinline__
#else
#define BCJR_TILES_FN inline
#endif

namespace bcjr {
namespace mm {

constexpr long kMaxRows = 0x7fffff00L;            // 2^31 - 256: a tile behind the last row still counts

template <int COLS>
BCJR_TILES_FN int col_tiles(int rows) { return (rows + (COLS - 1)) / COLS; }

// Columns of each of a group's `tiles` tiles but the last: equal shares, so that
// there is no small tile at the end, in whole steps of the matrix instruction.
// (Not (rows + tiles - 1) / tiles: that sum passes 32 bits from 2.1e9 rows on.)
BCJR_TILES_FN int tile_share(int rows, int tiles, int step) {
    return (1 + (rows - 1) / tiles + step - 1) & ~(step - 1);
}

// No more column tiles than this can T rows in E groups make.
template <int COLS>
BCJR_TILES_FN long max_col_tiles(int T, int E) {
    if (E == 1) return col_tiles<COLS>(T);
    return T / COLS + (E < T ? E : T);
}

}  // namespace mm
}  // namespace bcjr

// Which kernel a 4-bit product runs on, from its sizes. Host code only.
#pragma once

#include <algorithm>
#include <cstdint>

namespace mb {

// Row tiles of 16 (0: gemm_w4_kernel, up to 16 rows a block, whose waves split
// K; else gemm_w4_rows_kernel), column tiles of 16 per wave (RT 0: per block)
// and waves per block.
struct W4Config {
    int rt, ct, waves;
};
constexpr W4Config kW4Configs[] = {{0, 1, 8}, {0, 2, 8}, {0, 2, 4}, {1, 2, 8}, {2, 1, 8},
                                   {2, 1, 4}, {4, 1, 16}, {4, 1, 8}, {4, 1, 4}};
constexpr int kW4ConfigCount = 9;

// Row tiles of `rows` there are if total_rows are spread over the experts.
inline int64_t w4_likely_tiles(int64_t total_rows, int experts, int rows) {
    return std::max<int64_t>(std::min<int64_t>(experts, total_rows), (total_rows + rows - 1) / rows);
}

// Rows of an expert, were they even: tiles of 16, 32 or 64 of them share one
// pass over the weights.
//
// Up to 16: blocks of 32 columns whose waves split K; with more of them than
// CUs, fewer waves a block (more blocks at once: 128 rows over 16 experts of
// 2048 x 4096 20.5 against 23.3 us; 16 x 8192 x 8192, one block a CU, 18.7
// against 16.0). Once there are enough columns for a wave to take whole ones,
// that is faster (256 rows over 64 experts of 2048 x 4096: 58 against 68 us).
//
// More: 16 columns a wave. 64 rows: blocks of 256 columns (16 waves share a
// stage of x) while there are enough of them for 2 in 5 CUs (64 x 28672 x 8192:
// 67 us, 72 on 128 columns). Else 128 columns, which leave more to split K over
// (64 x 8192 x 8192: 27 us, 39 on 64 columns; 32 rows of 50257 x 4096: 41, 44
// on 256), and 64 for a handful. Two column tiles a wave lost: half the waves,
// twice the registers (64 x 50257 x 4096: 61 for 58 us).
inline int w4_config(int64_t total_rows, int experts, int64_t N, int cu_count) {
    const int64_t rows = (total_rows + experts - 1) / experts;
    if (rows <= 16) {
        const int64_t blocks = w4_likely_tiles(total_rows, experts, 16) * ((N + 31) / 32);
        if (blocks < cu_count) return 0;
        if (2 * blocks < 3 * cu_count) return 1;
        return blocks < 8 * cu_count ? 2 : 3;
    }
    const bool tall = rows > 32;
    const int64_t tiles = w4_likely_tiles(total_rows, experts, tall ? 64 : 32);
    if (tall && tiles * ((N + 255) / 256) * 5 >= 2 * cu_count) return 6;
    const bool wide = tiles * ((N + 127) / 128) >= 16;
    return tall ? (wide ? 7 : 8) : (wide ? 4 : 5);
}

}  // namespace mb

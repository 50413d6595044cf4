// Which kernel an MX4 product runs on, from its sizes. Host code only.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstdint>

namespace mb {

// Kernels by number: tiles of kMx4Tiles (gemm_mx4_kernel), then the kernel for few rows by 8 and by 32 rows
// (gemm_mx4_rows_kernel), then the one for any size.
struct Mx4Tile {
    int size, slots;   // rows and columns; pairs of units in the LDS ring
    int per_cu;        // blocks that a CU holds
    // us of a block with at most one on every CU, and of a round of per_cu blocks on every CU: fixed, and per unit
    // of K (128). Measured at K = 4096 and 2048: 256 x 256 36.5 us (4096^3); 128 x 128 15.9 us (1024 x 4096 x 4096, a
    // block a CU) and 23.4 (2048 x 4096 x 4096, two), four slots 14.3 and two rounds 26.3; 64 x 64 7.2 us (256 x
    // 4096 x 4096), 11.3 (512 x ..., two a CU).
    double one_us, one_unit_us, round_us, round_unit_us;
};
constexpr int kMx4TileCount = 4;
constexpr Mx4Tile kMx4Tiles[kMx4TileCount] = {{256, 2, 1, 7, 0.78, 7, 0.78},
                                              {128, 2, 2, 4, 0.36, 4, 0.56},
                                              {128, 4, 1, 5, 0.29, 5, 0.29},
                                              {64, 4, 2, 3, 0.13, 3, 0.26}};
constexpr int kMx4Rows8 = kMx4TileCount, kMx4Rows32 = kMx4TileCount + 1, kMx4Any = kMx4TileCount + 2;
constexpr int kMx4ConfigCount = kMx4TileCount + 3;
constexpr int kMx4MostSplits = 16;

struct Mx4Plan {
    int config;
    int splits;   // of K, over fp32 planes in the workspace (tiles without 256)
};

struct Mx4Shape {
    int64_t total_rows, N, units, x_rows;
    int experts;
    bool by_expert, listed;   // listed: x read through a list of its rows
};

// Row tiles of `size` in all experts, were their rows spread evenly but for where they end.
inline double mx4_row_tiles(const Mx4Shape& s, int size) {
    if (!s.by_expert) return (double)((s.total_rows + size - 1) / size);
    const double hit = (double)std::min<int64_t>(s.experts, s.total_rows), tiles = (double)s.total_rows / s.experts / size;
    return hit * std::max(1.0 + 0.55 * std::max(0.0, tiles - 0.35), tiles + 0.45);
}

// `config`, `splits`: forced, or negative.
inline Mx4Plan mx4_plan(const Mx4Shape& s, size_t workspace_bytes, int cus, int64_t config, int64_t splits) {
    // Rows read through a list lie within the 2^31 bytes that a buffer offset spans.
    if (s.listed && s.x_rows > ((1ll << 31) - 1) / (s.units * 64)) return {kMx4Any, 1};
    const double plane = 4.0 * (double)s.total_rows * (double)((s.N + 3) / 4 * 4);
    auto fits = [&](int n) { return plane * n <= (double)workspace_bytes; };
    if (config < 0) {
        // Few rows stream w past x: a wave has 16 KB of its 32 columns in flight, and no barriers. 64 tokens x 4 of 64
        // experts, 4096 -> 2048: 51 us, on 64 x 64 tiles 54; 32 x 14336 x 4096 9 us for 13. From 33 rows on every 32
        // read w again: only where that leaves CUs idle otherwise (64 x 4096 x 4096 5.3 us for 6.8; 64 x 50257 x
        // 4096 51 for 32).
        const int64_t rows = s.by_expert ? (s.total_rows + s.experts - 1) / s.experts : s.total_rows;
        const int64_t columns = (s.N + 31) / 32;
        if (rows <= 8) return {kMx4Rows8, 1};
        if (!s.by_expert && (rows <= 32 || (rows <= 64 && 2 * columns <= cus))) return {kMx4Rows32, 1};
    }
    if (config >= kMx4TileCount) {
        const double rows8 = std::ceil((double)s.total_rows / 8) + s.experts, columns = (double)(s.N / 32 + 8);
        return {config == kMx4Rows8 && rows8 * columns >= (double)(1 << 30) ? kMx4Rows32 : (int)config, 1};   // int32
    }

    // The tile and split count whose predicted time is least. Splits cost a second launch and their planes, written
    // and read, and none has less than 16 units; each smaller tile or further split has to gain 3%.
    constexpr double kSumUs = 3.5, kBytesPerUs = 5e6;
    Mx4Plan best{-1, 1};
    double best_us = 0;
    for (int i = 0; i < kMx4TileCount; ++i) {
        if (config >= 0 && config != i) continue;
        const Mx4Tile& tile = kMx4Tiles[i];
        const double tiles = mx4_row_tiles(s, tile.size) * (double)((s.N + tile.size - 1) / tile.size);
        for (int n = 1; n <= kMx4MostSplits; ++n) {
            if (splits >= 0 ? n != splits && n != 1 : (n & (n - 1)) != 0) continue;
            if (n > 1 && (tile.size == 256 || !fits(n) || (splits < 0 && s.units < 16 * n))) continue;
            const double blocks = tiles * n, units = (double)s.units / n;
            double us = blocks <= cus ? tile.one_us + units * tile.one_unit_us
                                      : std::ceil(blocks / (cus * tile.per_cu)) *
                                            (tile.round_us + units * tile.round_unit_us);
            if (n > 1) us += kSumUs + 2 * n * plane / kBytesPerUs;
            if (best.config < 0 || us < 0.97 * best_us || (n > 1 && n == splits && best.config == i)) {
                best = {i, n};
                best_us = us;
            }
        }
    }
    return best;
}

}  // namespace mb

// Which kernel an MX4 product runs on, from its sizes. Host code only.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstdint>

namespace mb {

// Kernels by number: LDS-DMA pipelines (gemm_mx4_kernel), the kernels for few rows (gemm_mx4_rows_kernel), and the one
// for any size.
struct Mx4Tile {
    int rows, columns;
    int slots;    // pairs of units in the LDS ring (few rows: a wave's)
    int per_cu;   // blocks that a CU holds
    // us of a round of blocks, one at most on every CU or per_cu: fixed, and per unit of K (128). Measured, less a
    // launch, at K = 4096 and other K: 256 x 256 36.5 us (4096^3); 128 x 128 15.9 (1024 x 4096 x 4096, a block a CU)
    // and 23.4 (2048 x 4096 x 4096, two), four slots 14.3; 64 x 128 16.2 (64 x 14336 x 4096) and 16.3 (1024 x 4096 x
    // 4096, two); 64 x 64 7.2 (256 x 4096 x 4096), 14.8 (128 x 8192 x 8192) and 23.1 (256 x ..., two); 8 x 32 8.5 (16 x
    // 4096 x 14336); 32 x 32 5.2 (64 x 4096 x 4096), 12.2 (64 x 4096 x 14336) and 13.4 (64 x 8192 x 8192, two).
    double one_us, one_unit_us, round_us, round_unit_us;
    double w_us, w_rate;   // a round that w's bytes bound: fixed us, bytes a us
};
constexpr int kMx4TileCount = 5, kMx4Rows8 = 5, kMx4Rows32 = 6, kMx4Any = 7, kMx4ConfigCount = 8;
constexpr Mx4Tile kMx4Tiles[kMx4Any] = {{256, 256, 2, 1, 7, 0.78, 7, 0.78, 7, 5.0e6},
                                        {128, 128, 2, 2, 3, 0.43, 4, 0.56, 4, 5.0e6},
                                        {128, 128, 4, 1, 5, 0.29, 5, 0.29, 4, 5.3e6},
                                        {64, 128, 2, 2, 3.4, 0.40, 3, 0.42, 3, 5.0e6},
                                        {64, 64, 4, 2, 1.5, 0.18, 0.5, 0.35, 3, 5.3e6},
                                        {8, 32, 4, 3, 2.4, 0.055, 2.4, 0.18, 1, 5.5e6},
                                        {32, 32, 4, 2, 2.4, 0.09, 2.4, 0.17, 2, 5.3e6}};
constexpr int kMx4MostSplits = 16;

struct Mx4Plan {
    int config;
    int splits;   // of K, over fp32 planes in the workspace (tiles without 256)
    bool stream;  // w is loaded nontemporal
};

struct Mx4Shape {
    int64_t total_rows, N, units, x_rows;
    int experts;
    bool by_expert, listed;   // listed: x read through a list of its rows
};

// Row tiles of `size` in all experts, were their rows spread evenly but for where they end.
inline double mx4_row_tiles(const Mx4Shape& s, int size) {
    if (!s.by_expert) return (double)((s.total_rows + size - 1) / size);
    const double hit = (double)std::min<int64_t>(s.experts, s.total_rows);
    const double tiles = (double)s.total_rows / s.experts / size;
    return hit * std::max(1.0 + 0.55 * std::max(0.0, tiles - 0.35), tiles + 0.45);
}

// Row tiles of `size` that read one part of w, on average.
inline double mx4_w_reads(const Mx4Shape& s, int size) {
    return mx4_row_tiles(s, size) / (s.by_expert ? (double)std::min<int64_t>(s.experts, s.total_rows) : 1.0);
}

// w read once, and too much of it for the 256 MB Infinity Cache to hold from one call to the next beside what else runs.
// What it gains where w comes from HBM (several matrices in turn), and costs where the same w still lies in the cache, us
// (8 and 64 rows by 4096, then 512 rows by expert, 4096 -> 2048):
//   w, MiB    64                    72                    80                    96                    104
//   8 rows    16.8->15.6 13.1->14.2 18.8->17.6 15.0->15.9 19.6->18.3 16.0->17.2 21.6->19.4 18.0->18.0 24.1->22.3 18.5->21.0
//   64 rows   19.9->17.5 14.1->17.0 24.2->23.6 16.5->23.1 24.7->23.8 17.2->23.5 25.8->24.2 18.7->23.7 29.2->25.3 20.3->24.5
//   experts   68: 20.9->18.7 16.3->16.7; 85: 25.5->23.9 18.0->22.4; 102: 26.3->24.2 20.3->23.6; 272: 56.8->51.0 50.3->51.3
// From HBM it gains at every size, by the most from about 96 MiB on; below, w more often lies in the cache still, and there
// it costs up to 7 us. Read more than once: 8192^3 236 -> 258.
inline bool mx4_stream(const Mx4Shape& s, int size) {
    const double hit = s.by_expert ? (double)std::min<int64_t>(s.experts, s.total_rows) : 1.0;
    return mx4_w_reads(s, size) <= 1.2 && hit * (double)s.N * (double)s.units * 68 >= (double)(96 << 20);
}

// `config`, `splits`: forced, or negative.
inline Mx4Plan mx4_plan(const Mx4Shape& s, size_t workspace_bytes, int cus, int64_t config, int64_t splits) {
    // Rows read through a list lie within the 2^31 bytes that a buffer offset spans.
    if (s.listed && s.x_rows > ((1ll << 31) - 1) / (s.units * 64)) return {kMx4Any, 1, false};
    const double plane = 4.0 * (double)s.total_rows * (double)((s.N + 3) / 4 * 4);
    auto fits = [&](int n) { return plane * n <= (double)workspace_bytes; };
    if (config >= kMx4TileCount) {
        const double rows8 = std::ceil((double)s.total_rows / 8) + s.experts, columns = (double)(s.N / 32 + 8);
        if (config == kMx4Rows8 && rows8 * columns >= (double)(1 << 30)) config = kMx4Rows32;   // int32
        return {(int)config, 1, config != kMx4Any && mx4_stream(s, kMx4Tiles[config].rows)};
    }

    // The tile and split count whose predicted time is least. Splits cost a second launch and their planes, written
    // and read, and none has less than 16 units; each smaller tile or further split has to gain 3%. Few rows by 8 or
    // 32, whose waves stream w with no barriers: 64 tokens x 4 of 64 experts, 4096 -> 2048: 49 us, on 64 x 128
    // tiles 49.5; with 128 tokens 63 and 52. 32 x 8192 x 8192: 8.4 us, 10.1 on 64 x 64; 16 x 50257 x 4096: 29 us, 23 on
    // 64 x 128.
    constexpr double kSumUs = 3.5, kBytesPerUs = 5e6;
    Mx4Plan best{-1, 1, false};
    double best_us = 0;
    for (int i = 0; i < kMx4Any; ++i) {
        if (config >= 0 && config != i) continue;
        const Mx4Tile& tile = kMx4Tiles[i];
        const double row_tiles = mx4_row_tiles(s, tile.rows);
        const double tiles = row_tiles * (double)((s.N + tile.columns - 1) / tile.columns);
        const double w_reads = mx4_w_reads(s, tile.rows);
        for (int n = 1; n <= kMx4MostSplits; ++n) {
            if (splits >= 0 ? n != splits && n != 1 : (n & (n - 1)) != 0) continue;
            if (n > 1 && (tile.rows == 256 || i >= kMx4TileCount)) continue;
            if (n > 1 && (!fits(n) || (splits < 0 && s.units < 16 * n))) continue;
            const double blocks = tiles * n, units = (double)s.units / n, whole = cus * tile.per_cu;
            // Matrix cores and LDS, or w's bytes: a round of 64 x 128 tiles takes 28 us at K = 4096 where each tile has
            // columns of its own (128 tokens x 4 of 64 experts, 4096 -> 2048), 16 where 16 share them.
            auto round = [&](double b) {
                const double one = tile.one_us + units * tile.one_unit_us;
                const double more = tile.round_us + units * tile.round_unit_us - one, on_cu = std::ceil(b / cus);
                const double busy = on_cu <= 1 ? one : one + more * (on_cu - 1) / (tile.per_cu - 1);
                return std::max(busy, tile.w_us + b / w_reads * tile.columns * units * 68 / tile.w_rate);
            };
            const double rounds = std::floor(blocks / whole), rest = blocks - rounds * whole;
            double us = rounds * (rounds > 0 ? round(whole) : 0) + (rest > 0 ? round(rest) : 0);
            if (n > 1) us += kSumUs + 2 * n * plane / kBytesPerUs;
            if (best.config < 0 || us < 0.97 * best_us || (n > 1 && n == splits && best.config == i)) {
                best = {i, n, mx4_stream(s, tile.rows)};
                best_us = us;
            }
        }
    }
    return best;
}

}  // namespace mb

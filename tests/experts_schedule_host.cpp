// Prints the vmcnt waits that the grouped products' kernels derive from their
// load order, one line "x_pairs x_slots x_loads y_pairs y_slots y_loads odd
// even prologue" per ring of every operation and tile. Host code, compiled
// from the kernels' own header by tests/test_experts_schedule.py.
#include <cstdio>

#include "../teamredbench_amd/csrc/gemm_grouped_kernels.hpp"

int main() {
    using namespace mb;
    for (int i = 0; i < kGroupedTileCount; ++i)
        for (int op = 0; op < 3; ++op) {
            const int tile = kGroupedTiles[i], nx = kGroupedConfigs[i].nx[op], ny = kGroupedConfigs[i].ny[op];
            const bool px = op != MB_GROUPED_GRAD_WEIGHTS, py = op == MB_GROUPED_GRAD_ROWS;
            const int pair = 2 * tile * kStageK / 1024 / 4, stage = 32 * tile * 2 / 1024 / 4;
            const int ix = px ? pair : stage, iy = py ? pair : stage;
            const StepWaits w = step_schedule(px, nx, ix, py, ny, iy);
            std::printf("%d %d %d %d %d %d %d %d %d\n", px, nx, ix, py, ny, iy, w.odd, w.even, w.prologue);
        }
    return 0;
}

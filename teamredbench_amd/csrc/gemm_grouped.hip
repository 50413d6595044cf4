// Products of ragged groups of rows: one K x N matrix per expert, sorted rows
// grouped by expert (offsets in device memory), forward and both gradients.
//
// Written as out(m, n) = sum over c of X(m, c) Y(c, n) per expert:
//   op            m          c          n     X                Y
//   FORWARD       sorted row K          N     A, c in a row    B, n in a row
//   GRAD_ROWS     sorted row N          K     dC, c in a row   B, c in a row
//   GRAD_WEIGHTS  K          sorted row N     A, m in a row    dC, n in a row
//
// Rows on 16 bytes go to the LDS-DMA pipelines of gemm_grouped_kernels.hpp.
// gemm_grouped_any_kernel takes any size, stride and alignment: 128 x 128
// tiles, 4 waves of 64 x 64 on v_mfma_f32_32x32x16, a stage of 32 c, through
// registers into one of two LDS buffers while the other is computed. Global
// loads are 16 bytes at any element (the hardware takes them; element by
// element it took twice as long, 645 against 324 us for 12004 rows over 60
// experts, 2057 -> 1411). An operand whose rows run along c is kept as [m or
// n][32 c] in rows of 80 bytes, one whose rows run across it as [32 c][m or n],
// swizzled, and read with the transposing LDS reads. Rows of c past the
// expert's and c past the end load as zeros; nothing past a row's last element
// is read. Bound by the loads' latency: one stage ahead, two blocks a CU.
#include "gemm_grouped_kernels.hpp"

#include <algorithm>
#include <cmath>

namespace mb {
namespace {

constexpr int kTile = 128;
constexpr int kStage = 32;                      // c per stage
constexpr int kPitch = kStage * 2 + 16;         // bytes per LDS row along c
constexpr int kAnyBuffer = kTile * kPitch;      // bytes per operand and buffer (an operand across c takes less)

// Elements c .. c + 7 of a row of `n`; zeros past its end, none of which is read.
__device__ __forceinline__ u32x4 row_window(const uint16_t* row, int c, int n) {
    if (c + 8 <= n) return *reinterpret_cast<const u32x4_any*>(row + c);
    if (c >= n) return u32x4{0u, 0u, 0u, 0u};
    if (n >= 8) {   // the row's last 8, shifted down
        const u32x4 v = *reinterpret_cast<const u32x4_any*>(row + n - 8);
        return __builtin_bit_cast(u32x4, __builtin_bit_cast(__uint128_t, v) >> (16 * (c + 8 - n)));
    }
    __uint128_t wide = 0;
#pragma unroll 1
    for (int i = n - 1; i >= c; --i) wide = (wide << 16) | row[i];
    return __builtin_bit_cast(u32x4, wide);
}

template <int DT, int OP>
__global__ void __launch_bounds__(256)
gemm_grouped_any_kernel(const uint16_t* __restrict__ x, int64_t ldx, int64_t x_rows, const int32_t* __restrict__ rows,
                        const uint16_t* __restrict__ y, int64_t ldy, uint16_t* __restrict__ out, int64_t ldo,
                        const int32_t* __restrict__ offsets, int experts, int total, int N, int K, int tiles_n) {
    constexpr bool XC = OP != MB_GROUPED_GRAD_WEIGHTS;   // X's rows run along c
    constexpr bool YC = OP == MB_GROUPED_GRAD_ROWS;      // Y's rows run along c
    __shared__ __attribute__((aligned(1024))) unsigned char lds[2][2][kAnyBuffer];   // buffer, operand
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave >> 1, wn = wave & 1;
    const int block = (int)block_number(), tile = block / tiles_n, n0 = (block - tile * tiles_n) * kTile;
    ExpertRows ex;
    int m0;
    if constexpr (OP == MB_GROUPED_GRAD_WEIGHTS) {
        const int tiles_m = (K + kTile - 1) / kTile;
        const int e = tile / tiles_m;
        if (e >= experts) return;
        ex = expert_rows(offsets, e, total);
        m0 = (tile - e * tiles_m) * kTile;
    } else {
        int in_expert;
        if (!find_row_tile(offsets, experts, total, tile, kTile, &ex, &in_expert)) return;
        m0 = in_expert * kTile;
    }
    const int M = OP == MB_GROUPED_GRAD_WEIGHTS ? K : ex.count;
    const int NN = OP == MB_GROUPED_GRAD_ROWS ? K : N;
    const int C = OP == MB_GROUPED_FORWARD ? K : OP == MB_GROUPED_GRAD_ROWS ? N : ex.count;

    // Sorted row p of the expert -> its row of x, -1 for none.
    auto x_row = [&](int p) -> int64_t {
        const int64_t r = rows ? rows[ex.first + p] : ex.first + p;
        return r < x_rows ? r : -1;
    };
    const uint16_t* yb = OP == MB_GROUPED_GRAD_WEIGHTS ? y + ex.first * ldy : y + (int64_t)ex.expert * K * ldy;

    // A thread brings two 16-byte pieces of each operand's stage. Along c: 16 c of tile row tid / 2.
    // Across: 8 columns from 8 (tid % 16) on, of c tid / 16 and + 16.
    const int along_row = tid >> 1, along_c = (tid & 1) * 16;
    const int across_c = tid >> 4, across_col = (tid & 15) * 8;
    const uint16_t *x_along = nullptr, *y_along = nullptr;
    if constexpr (XC) {
        const int64_t r = m0 + along_row < M ? x_row(m0 + along_row) : -1;
        if (r >= 0) x_along = x + r * ldx;
    }
    if constexpr (YC) {
        if (n0 + along_row < NN) y_along = yb + (int64_t)(n0 + along_row) * ldy;
    }
    auto load_along = [&](const uint16_t* row, int c, u32x4 (&v)[2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            v[h] = row != nullptr ? row_window(row, c + along_c + 8 * h, C) : u32x4{0u, 0u, 0u, 0u};
    };
    auto load_x = [&](int c, u32x4 (&v)[2]) {
        if constexpr (XC) {
            load_along(x_along, c, v);
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int p = c + across_c + 16 * h;
                const int64_t r = p < C ? x_row(p) : -1;
                v[h] = r >= 0 ? row_window(x + r * ldx, m0 + across_col, M) : u32x4{0u, 0u, 0u, 0u};
            }
        }
    };
    auto load_y = [&](int c, u32x4 (&v)[2]) {
        if constexpr (YC) {
            load_along(y_along, c, v);
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int p = c + across_c + 16 * h;
                v[h] = p < C ? row_window(yb + p * ldy, n0 + across_col, NN) : u32x4{0u, 0u, 0u, 0u};
            }
        }
    };
    auto store = [&](unsigned char* to, bool along, const u32x4 (&v)[2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = across_c + 16 * h;
            const int at = along ? along_row * kPitch + along_c * 2 + 16 * h
                                 : c * kTile * 2 + (((across_col >> 3) ^ b_swizzle<2, kTile * 2>(c)) << 4);
            *reinterpret_cast<u32x4*>(to + at) = v[h];
        }
    };
    // Fragment of 32 rows (columns) from `base` on, substep s.
    auto fragment = [&](const unsigned char* from, bool along, int base, int s) {
        if (along)
            return *reinterpret_cast<const u32x4*>(from + (base + (lane & 31)) * kPitch + 32 * s + 16 * (lane >> 5));
        const u32x2 lo = read_b_piece<DT, kTile>(from, base, s, 0, lane);
        const u32x2 hi = read_b_piece<DT, kTile>(from, base, s, 1, lane);
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };

    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    u32x4 xv[2], yv[2];
    if (C > 0) {
        load_x(0, xv);
        load_y(0, yv);
    }
    int buf = 0;
    for (int c = 0; c < C; c += kStage, buf ^= 1) {
        store(lds[buf][0], XC, xv);
        store(lds[buf][1], YC, yv);
        __syncthreads();   // the other buffer was left by every wave before this barrier
        if (c + kStage < C) {
            load_x(c + kStage, xv);
            load_y(c + kStage, yv);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4 xf[2], yf[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                xf[i] = fragment(lds[buf][0], XC, 64 * wm + 32 * i, s);
                yf[i] = fragment(lds[buf][1], YC, 64 * wn + 32 * i, s);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = Traits<DT>::mfma(yf[j], xf[i], acc[i][j]);
        }
    }

    // Register 4g + q of lane l holds out(32i + l % 32, 32j + 8g + 4 (l / 32) + q).
    uint16_t* ob = OP == MB_GROUPED_GRAD_WEIGHTS ? out + (int64_t)ex.expert * K * ldo : out + ex.first * ldo;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int m = m0 + 64 * wm + 32 * i + (lane & 31);
        if (m >= M) continue;
        uint16_t* row = ob + m * ldo;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                typedef u32x2 u32x2_any __attribute__((aligned(2)));
                const int n = n0 + 64 * wn + 32 * j + 8 * g + 4 * (lane >> 5);
                const f32x16& v = acc[i][j];
                if (n + 4 <= NN) {
                    *reinterpret_cast<u32x2_any*>(row + n) =
                        pack4<DT>(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
                } else {
#pragma unroll
                    for (int r = 0; r < 3; ++r)
                        if (n + r < NN) row[n + r] = to_bits<DT>(v[4 * g + r]);
                }
            }
    }
}

template <int DT, int OP>
int launch_any(const GroupedCall& c, hipStream_t stream) {
    const int64_t NN = OP == MB_GROUPED_GRAD_ROWS ? c.K : c.N;
    const int tiles_n = (int)((NN + kTile - 1) / kTile);
    const int64_t tiles_m = OP == MB_GROUPED_GRAD_WEIGHTS
                                ? c.experts * ((c.K + kTile - 1) / kTile)
                                : c.total_rows / kTile + std::min<int64_t>(c.experts, c.total_rows);
    hipLaunchKernelGGL((gemm_grouped_any_kernel<DT, OP>), launch_grid(tiles_m * tiles_n), dim3(256), 0, stream,
                       static_cast<const uint16_t*>(c.x), c.ldx, c.x_rows, c.rows, static_cast<const uint16_t*>(c.y),
                       c.ldy, static_cast<uint16_t*>(c.out), c.ldo, c.offsets, c.experts, (int)c.total_rows, (int)c.N,
                       (int)c.K, tiles_n);
    MB_HIP_TRY(hipGetLastError());
    return MB_OK;
}

template <int DT>
int launch_any_op(const GroupedCall& c, hipStream_t stream) {
    if (c.op == MB_GROUPED_FORWARD) return launch_any<DT, MB_GROUPED_FORWARD>(c, stream);
    if (c.op == MB_GROUPED_GRAD_ROWS) return launch_any<DT, MB_GROUPED_GRAD_ROWS>(c, stream);
    return launch_any<DT, MB_GROUPED_GRAD_WEIGHTS>(c, stream);
}

// How a call runs. The pipelined kernels do not take rows off 16 bytes, nor an
// operand (one expert's matrix, x read through `rows`, a tile's rows) that
// passes the 2^31 bytes a buffer offset spans.
GroupedPlan grouped_plan(const GroupedCall& c, size_t workspace_bytes, const DeviceProps& props) {
    constexpr GroupedPlan kAny{-1, 1};
    const uintptr_t base = reinterpret_cast<uintptr_t>(c.x) | reinterpret_cast<uintptr_t>(c.y) |
                           reinterpret_cast<uintptr_t>(c.out);
    if ((base & 15) != 0 || ((c.ldx | c.ldy | c.ldo | c.N | c.K) & 7) != 0 || c.total_rows == 0 || c.x_rows == 0)
        return kAny;
    // Every row a tile can address, those past its operand's end too, stays below 2^30 elements.
    constexpr int64_t kMost = (1ll << 30) - 1, kTileRows = 256;
    const bool weights = c.op == MB_GROUPED_GRAD_WEIGHTS;
    const int64_t x_rows = c.rows ? c.x_rows : weights ? c.total_rows : 0;
    const int64_t y_rows = weights ? c.total_rows : c.K;
    if (std::max(x_rows, kTileRows) > kMost / c.ldx - kTileRows ||
        std::max(y_rows, kTileRows) > kMost / c.ldy - kTileRows)
        return kAny;
    const int64_t forced = tuning(MB_TUNE_GROUPED_CONFIG);
    if (forced >= kGroupedTileCount) return kAny;

    // The tile and split count whose predicted time is least; each smaller
    // tile or further split has to gain 3%. A block takes an overhead (its
    // first loads and its stores) and a time per 32 of the contraction,
    // measured at 16384 rows x 4096 x 14336 over 8 experts with every CU full:
    // 0.75 us on 256 x 256 tiles (one a CU), 0.535 on 128 x 128 (two) and
    // 0.386 on 64 x 64 (three). Nothing beats the bytes, at 5.2 TB/s. An
    // expert's row tiles: its rows, were they even, and half a tile; with
    // fewer rows than a tile one, and a share of experts that pass it. Splits cost a second
    // launch and their planes, written and read.
    constexpr double kStageUs[kGroupedTileCount] = {0.75, 0.535, 0.386};
    constexpr double kBlockUs[kGroupedTileCount] = {8, 4, 4};
    constexpr int kPerCu[kGroupedTileCount] = {1, 2, 3};
    constexpr double kSumUs = 5, kBytesPerUs = 5.2e6;
    const int64_t hit = std::min<int64_t>(c.experts, c.total_rows);   // experts with rows, at most
    const double per_expert = (double)c.total_rows / c.experts;
    const int64_t NN = c.op == MB_GROUPED_GRAD_ROWS ? c.K : c.N, C = c.op == MB_GROUPED_GRAD_ROWS ? c.N : c.K;
    const double plane = 4.0 * (double)(weights ? c.experts * c.K : c.total_rows) * (double)NN;
    const double bytes_us = 2.0 * ((double)hit * c.K * c.N + (double)c.total_rows * (c.K + c.N)) / kBytesPerUs;
    GroupedPlan best = kAny;
    double best_us = 0;
    for (int i = 0; i < kGroupedTileCount; ++i) {
        if (forced >= 0 && forced != i) continue;
        const int tile = kGroupedTiles[i];
        const double wide = (double)((NN + tile - 1) / tile);
        double blocks, stages;
        if (weights) {
            blocks = (double)c.experts * ((c.K + tile - 1) / tile) * wide;
            stages = std::max(1.0, per_expert / 32);
        } else {
            const double tiles = per_expert / tile;
            blocks = hit * wide * std::max(1.0 + 0.55 * std::max(0.0, tiles - 0.35), tiles + 0.45);
            stages = (double)((C + 31) / 32);
        }
        for (int splits = 1; splits <= 16; splits *= 2) {
            if (splits > 1 && (i == 0 || stages < 4.0 * splits || plane * splits > (double)workspace_bytes)) break;
            const double rounds = std::ceil(blocks * splits / props.cu_count) / kPerCu[i];
            double us = std::max(bytes_us, rounds * (kBlockUs[i] + stages / splits * kStageUs[i]));
            if (splits > 1) us += kSumUs + 2 * splits * plane / kBytesPerUs;
            if (best.config < 0 || us < 0.97 * best_us) {
                best = {i, splits};
                best_us = us;
            }
        }
    }
    return best;
}

}  // namespace

int gemm_grouped_launch(const GroupedCall& c, void* workspace, size_t workspace_bytes, const DeviceProps& props,
                        hipStream_t stream) {
    // The workspace only makes small calls faster: one off 16 bytes is left alone.
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) workspace_bytes = 0;
    const GroupedPlan plan = grouped_plan(c, workspace_bytes, props);
    if (plan.config >= 0)
        return c.dtype == MB_DT_FLOAT16 ? gemm_grouped_tiled_f16(c, plan, workspace, stream)
                                        : gemm_grouped_tiled_bf16(c, plan, workspace, stream);
    if (c.dtype == MB_DT_FLOAT16) return launch_any_op<MB_DT_FLOAT16>(c, stream);
    return launch_any_op<MB_DT_BFLOAT16>(c, stream);
}

}  // namespace mb

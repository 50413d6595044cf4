// Products of ragged groups of rows: one K x N matrix per expert, sorted rows
// grouped by expert (offsets in device memory), forward and both gradients.
//
// Written as out(m, n) = sum over c of X(m, c) Y(c, n) per expert:
//   op            m          c          n     X                Y
//   FORWARD       sorted row K          N     A, c in a row    B, n in a row
//   GRAD_ROWS     sorted row N          K     dC, c in a row   B, c in a row
//   GRAD_WEIGHTS  K          sorted row N     A, m in a row    dC, n in a row
//
// gemm_grouped_any_kernel takes any size, stride and alignment: 128 x 128
// tiles, 4 waves of 64 x 64 on v_mfma_f32_32x32x16, a stage of 32 c. Both
// operands go through registers into LDS as [m or n][32 c] (rows padded to 80
// bytes), every element checked against its expert's bounds and zero outside, so rows
// of neighbouring experts and whatever lies past K or N never enter a sum.
#include "experts_common.hpp"

#include <algorithm>

namespace mb {
namespace {

constexpr int kTile = 128;
constexpr int kStage = 32;                 // c per stage
constexpr int kPitch = kStage * 2 + 16;    // LDS row pitch, bytes

template <int DT>
__device__ __forceinline__ f32x16 mfma32(const u32x4& a, const u32x4& b, f32x16 c) {
    if constexpr (DT == MB_DT_FLOAT16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                       0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                        0, 0, 0);
}

template <int DT, int OP>
__global__ void __launch_bounds__(256)
gemm_grouped_any_kernel(const uint16_t* __restrict__ x, int64_t ldx, int64_t x_rows, const int32_t* __restrict__ rows,
                        const uint16_t* __restrict__ y, int64_t ldy, uint16_t* __restrict__ out, int64_t ldo,
                        const int32_t* __restrict__ offsets, int experts, int total, int N, int K, int tiles_n) {
    constexpr bool XC = OP != MB_GROUPED_GRAD_WEIGHTS;   // X's rows run along c (else along m)
    constexpr bool YC = OP == MB_GROUPED_GRAD_ROWS;      // Y's rows run along c (else along n)
    __shared__ __attribute__((aligned(16))) unsigned char lds_x[kTile * kPitch], lds_y[kTile * kPitch];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave >> 1, wn = wave & 1;
    const int tile = (int)blockIdx.x / tiles_n, n0 = ((int)blockIdx.x - tile * tiles_n) * kTile;
    ExpertRows ex;
    int m0;
    if constexpr (OP == MB_GROUPED_GRAD_WEIGHTS) {
        const int tiles_m = (K + kTile - 1) / kTile;
        const int e = tile / tiles_m;
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

    // This thread's 16 elements of a stage: row (column) of the tile and half of the stage when c runs in a
    // row, else a column of the tile and 16 of the stage's c.
    auto load_c = [&](const uint16_t* row, int c, u32x4* v) {   // 16 elements of a row from c on
        if (row != nullptr && c + 16 <= C) {
            v[0] = *reinterpret_cast<const u32x4_any*>(row + c);
            v[1] = *reinterpret_cast<const u32x4_any*>(row + c + 8);
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned lo = row != nullptr && c + 2 * i < C ? row[c + 2 * i] : 0u;
            const unsigned hi = row != nullptr && c + 2 * i + 1 < C ? row[c + 2 * i + 1] : 0u;
            v[i >> 2][i & 3] = lo | (hi << 16);
        }
    };
    const int cr = tid >> 1, ch = (tid & 1) * 16;       // c runs in a row
    const int mr = tid & 127, mh = (tid >> 7) * 16;     // it does not
    const uint16_t* x_ptr = nullptr;
    if constexpr (XC) {
        const int64_t r = m0 + cr < M ? x_row(m0 + cr) : -1;
        if (r >= 0) x_ptr = x + r * ldx;
    }
    const uint16_t* y_ptr = nullptr;
    if constexpr (YC) {
        if (n0 + cr < NN) y_ptr = yb + (int64_t)(n0 + cr) * ldy;
    }
    auto load_x = [&](int c, u32x4* v) {
        if constexpr (XC) {
            load_c(x_ptr, c + ch, v);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int p = c + mh + i;
                const int64_t r = p < C ? x_row(p) : -1;
                const unsigned e = r >= 0 && m0 + mr < M ? x[r * ldx + m0 + mr] : 0u;
                v[i >> 3][(i >> 1) & 3] = (i & 1) ? v[i >> 3][(i >> 1) & 3] | (e << 16) : e;
            }
        }
    };
    auto load_y = [&](int c, u32x4* v) {
        if constexpr (YC) {
            load_c(y_ptr, c + ch, v);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int p = c + mh + i;
                const unsigned e = p < C && n0 + mr < NN ? yb[p * ldy + n0 + mr] : 0u;
                v[i >> 3][(i >> 1) & 3] = (i & 1) ? v[i >> 3][(i >> 1) & 3] | (e << 16) : e;
            }
        }
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
    for (int c = 0; c < C; c += kStage) {
        unsigned char* px = XC ? lds_x + cr * kPitch + ch * 2 : lds_x + mr * kPitch + mh * 2;
        unsigned char* py = YC ? lds_y + cr * kPitch + ch * 2 : lds_y + mr * kPitch + mh * 2;
        *reinterpret_cast<u32x4*>(px) = xv[0];
        *reinterpret_cast<u32x4*>(px + 16) = xv[1];
        *reinterpret_cast<u32x4*>(py) = yv[0];
        *reinterpret_cast<u32x4*>(py + 16) = yv[1];
        __syncthreads();
        if (c + kStage < C) {
            load_x(c + kStage, xv);
            load_y(c + kStage, yv);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4 xf[2], yf[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = 32 * s + 16 * (lane >> 5);
                xf[i] = *reinterpret_cast<const u32x4*>(lds_x + (64 * wm + 32 * i + (lane & 31)) * kPitch + at);
                yf[i] = *reinterpret_cast<const u32x4*>(lds_y + (64 * wn + 32 * i + (lane & 31)) * kPitch + at);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = mfma32<DT>(yf[j], xf[i], acc[i][j]);
        }
        __syncthreads();
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
            for (int r = 0; r < 16; ++r) {
                const int n = n0 + 64 * wn + 32 * j + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                if (n < NN) row[n] = to_bits<DT>(acc[i][j][r]);
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
    hipLaunchKernelGGL((gemm_grouped_any_kernel<DT, OP>), dim3((unsigned)(tiles_m * tiles_n)), dim3(256), 0, stream,
                       static_cast<const uint16_t*>(c.x), c.ldx, c.x_rows, c.rows, static_cast<const uint16_t*>(c.y),
                       c.ldy, static_cast<uint16_t*>(c.out), c.ldo, c.offsets, c.experts, (int)c.total_rows, (int)c.N,
                       (int)c.K, tiles_n);
    MB_HIP_TRY(hipGetLastError());
    return MB_OK;
}

template <int DT>
int launch_dtype(const GroupedCall& c, hipStream_t stream) {
    if (c.op == MB_GROUPED_FORWARD) return launch_any<DT, MB_GROUPED_FORWARD>(c, stream);
    if (c.op == MB_GROUPED_GRAD_ROWS) return launch_any<DT, MB_GROUPED_GRAD_ROWS>(c, stream);
    return launch_any<DT, MB_GROUPED_GRAD_WEIGHTS>(c, stream);
}

// The tile configuration of the pipelined kernels, -1 for what they do not
// take: rows off 16 bytes, or an operand (one expert's matrix, x read through
// `rows`, a tile's rows) that passes the 2^31 bytes a buffer offset spans.
int tiled_config(const GroupedCall& c) {
    const uintptr_t base = reinterpret_cast<uintptr_t>(c.x) | reinterpret_cast<uintptr_t>(c.y) |
                           reinterpret_cast<uintptr_t>(c.out);
    if ((base & 15) != 0 || ((c.ldx | c.ldy | c.ldo | c.N | c.K) & 7) != 0 || c.total_rows == 0 || c.x_rows == 0)
        return -1;
    constexpr int64_t kMost = 1ll << 30;   // elements
    const bool weights = c.op == MB_GROUPED_GRAD_WEIGHTS;
    const int64_t x_rows = c.rows ? c.x_rows : weights ? c.total_rows : 256;
    if (x_rows > kMost / c.ldx || (weights ? c.total_rows : c.K) > kMost / c.ldy) return -1;
    if (const int64_t forced = tuning(MB_TUNE_GROUPED_CONFIG); forced >= 0) return forced > 4 ? -1 : (int)forced;
    if (weights) return 0;
    const int64_t rows = (c.total_rows + c.experts - 1) / c.experts;
    return rows > 256 ? 0 : rows > 64 ? 2 : 3;
}

}  // namespace

int gemm_grouped_launch(const GroupedCall& c, void* workspace, size_t workspace_bytes, const DeviceProps& props,
                        hipStream_t stream) {
    const int config = tiled_config(c);
    if (config >= 0)
        return c.dtype == MB_DT_FLOAT16 ? gemm_grouped_tiled_f16(c, config, stream)
                                        : gemm_grouped_tiled_bf16(c, config, stream);
    if (c.dtype == MB_DT_FLOAT16) return launch_dtype<MB_DT_FLOAT16>(c, stream);
    return launch_dtype<MB_DT_BFLOAT16>(c, stream);
}

}  // namespace mb

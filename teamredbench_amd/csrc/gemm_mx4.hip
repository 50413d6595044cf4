// Products of MX4 matrices: out[p][n] = sum over k of x[rows[p]][k] w[e][n][k],
// both operands in rows along k (layout: mx4_common.hpp), dense or by expert.
//
// gemm_mx4_any_kernel: a wave makes 32 rows x 32 columns from operands that go
// from global memory straight into the matrix cores' registers. 64-bit addresses, any size.
#include "gemm_mx4_kernels.hpp"

namespace mb {
namespace {

constexpr int kTile = 32;

__global__ void __launch_bounds__(64)
gemm_mx4_any_kernel(Mx4Call c, int tiles_n) {
    const int lane = threadIdx.x, half = lane >> 5, r32 = lane & 31;
    const int64_t block = block_number();
    int tm = (int)(block / tiles_n);
    const int64_t n0 = (block - (int64_t)tm * tiles_n) * kTile;
    ExpertRows ex{0, 0, (int)c.total_rows};
    if (c.offsets != nullptr && !find_row_tile(c.offsets, c.experts, (int)c.total_rows, tm, kTile, &ex, &tm)) return;
    const int m = tm * kTile + r32;   // this lane's row of the expert
    if (tm * kTile >= ex.count) return;
    int64_t row = m < ex.count ? (int64_t)ex.first + m : -1;
    if (row >= 0 && c.rows != nullptr) {
        row = c.rows[row];
        if (row >= c.x_rows) row = -1;
    }
    const int64_t n = min(n0 + r32, c.N - 1);   // columns past N are not stored
    const int64_t wrow = (int64_t)ex.expert * c.N + n;
    const auto* xp = static_cast<const u32x4*>(c.x) + max(row, (int64_t)0) * c.units * 4 + 2 * half;
    const auto* wp = static_cast<const u32x4*>(c.w) + wrow * c.units * 4 + 2 * half;
    const auto* xs = static_cast<const uint16_t*>(c.x_scales) + max(row, (int64_t)0) * c.units * 2 + half;
    const auto* ws = static_cast<const uint16_t*>(c.w_scales) + wrow * c.units * 2 + half;
    f32x16 acc;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    for (int64_t u = 0; u < c.units; ++u) {   // lane half h takes blocks 2h and 2h + 1 of the unit
        u32x4 a0 = {0, 0, 0, 0}, a1 = {0, 0, 0, 0};
        unsigned sa = 0;
        if (row >= 0) {
            a0 = xp[4 * u];
            a1 = xp[4 * u + 1];
            sa = xs[2 * u];
        }
        const unsigned sb = ws[2 * u];
        acc = mfma_mx4<0, 0>(wp[4 * u], sb, a0, sa, acc);
        acc = mfma_mx4<1, 1>(wp[4 * u + 1], sb, a1, sa, acc);
    }
    // Register 4g + q of lane l: row l % 32, column 8g + 4 (l / 32) + q.
    if (m >= ex.count) return;
    auto* out = static_cast<uint16_t*>(c.out) + (int64_t)(ex.first + m) * c.ldo + n0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int col = 8 * (i >> 2) + 4 * half + (i & 3);
        if (n0 + col < c.N)
            out[col] = c.dtype == MB_DT_FLOAT16 ? to_bits<MB_DT_FLOAT16>(acc[i]) : to_bits<MB_DT_BFLOAT16>(acc[i]);
    }
}

int launch_any(const Mx4Call& c, hipStream_t stream) {
    const int64_t tiles_m = c.offsets ? c.total_rows / kTile + std::min<int64_t>(c.experts, c.total_rows)
                                      : (c.total_rows + kTile - 1) / kTile;
    const int64_t tiles_n = (c.N + kTile - 1) / kTile;
    hipLaunchKernelGGL(gemm_mx4_any_kernel, launch_grid(tiles_m * tiles_n), dim3(64), 0, stream, c, (int)tiles_n);
    MB_HIP_TRY(hipGetLastError());
    return MB_OK;
}

Mx4Plan mx4_plan(const Mx4Call& c, size_t workspace_bytes, const DeviceProps& props) {
    // Rows read through a list lie within the 2^31 bytes that a buffer offset spans.
    if (c.rows != nullptr && c.x_rows > ((1ll << 31) - 1) / (c.units * kMx4UnitBytes)) return {-1, 1};
    const int64_t forced = tuning(MB_TUNE_MX4_CONFIG);
    int config = forced >= 0 ? (forced == 3 ? -1 : (int)forced) : c.total_rows <= 32 ? -1 : c.total_rows > 512 ? 0 : 1;
    int splits = 1;
    if (config > 0) {
        const int64_t want = tuning(MB_TUNE_MX4_SPLITS);
        const size_t plane = (size_t)c.total_rows * ((c.N + 3) / 4 * 4) * 4;
        splits = want > 0 ? (int)want : 1;
        while (splits > 1 && plane * splits > workspace_bytes) --splits;
    }
    return {config, splits};
}

}  // namespace

int gemm_mx4_launch(const Mx4Call& c, void* workspace, size_t workspace_bytes, const DeviceProps& props,
                    hipStream_t stream) {
    // The workspace only makes small calls faster: one off 16 bytes is left alone.
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) workspace_bytes = 0;
    const Mx4Plan plan = mx4_plan(c, workspace_bytes, props);
    if (plan.config < 0) return launch_any(c, stream);
    return c.dtype == MB_DT_FLOAT16 ? gemm_mx4_tiled_f16(c, plan, workspace, stream)
                                    : gemm_mx4_tiled_bf16(c, plan, workspace, stream);
}

}  // namespace mb

// Products with 4-bit weights: out[p][n] = sum over k of x[p][k] s (q - z), one
// scale s and zero point z per column n and group of k.
//
// One wave per column n and tile of 8 rows: lane l takes bytes l, l + 64, ...
// of the column's packed weights, two k a byte, and accumulates 8 rows in fp32.
#include "experts_common.hpp"

#include <algorithm>

namespace mb {
namespace {

constexpr int kRows = 8;

template <int DT>
__global__ void __launch_bounds__(256)
gemm_w4_kernel(const uint16_t* __restrict__ x, int64_t ldx, int64_t x_rows, const int32_t* __restrict__ rows,
               const uint8_t* __restrict__ q, const uint16_t* __restrict__ scales, const uint16_t* __restrict__ zeros,
               int group, uint16_t* __restrict__ out, int64_t ldo, const int32_t* __restrict__ offsets, int experts,
               int total, int N, int K, int blocks_n) {
    const int lane = threadIdx.x & 63;
    const int tile = (int)blockIdx.x / blocks_n;
    const int n = ((int)blockIdx.x - tile * blocks_n) * 4 + (threadIdx.x >> 6);
    ExpertRows ex{0, 0, total};
    int in_expert = tile;
    if (offsets != nullptr && !find_row_tile(offsets, experts, total, tile, kRows, &ex, &in_expert)) return;
    if (n >= N) return;
    const int p0 = ex.first + in_expert * kRows, count = min(kRows, ex.count - in_expert * kRows);
    const int bytes = (K + 1) / 2, groups = (K + group - 1) / group;
    const int64_t column = (int64_t)ex.expert * N + n;
    const uint8_t* qc = q + column * bytes;
    const uint16_t* sc = scales + column * groups;
    const uint16_t* zc = zeros ? zeros + column * groups : nullptr;
    const uint16_t* xp[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        xp[r] = nullptr;
        if (r < count) {
            const int64_t row = rows ? rows[p0 + r] : p0 + r;
            if (row >= 0 && row < x_rows) xp[r] = x + row * ldx;
        }
    }
    float sum[kRows] = {};
    for (int b = lane; b < bytes; b += 64) {
        const int g = 2 * b / group;
        const float s = from_bits<DT>(sc[g]), z = zc ? from_bits<DT>(zc[g]) : 8.f;
        const float w0 = s * ((float)(qc[b] & 15) - z);
        const float w1 = 2 * b + 1 < K ? s * ((float)(qc[b] >> 4) - z) : 0.f;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            if (xp[r] == nullptr) continue;
            sum[r] = fmaf(from_bits<DT>(xp[r][2 * b]), w0, sum[r]);
            if (2 * b + 1 < K) sum[r] = fmaf(from_bits<DT>(xp[r][2 * b + 1]), w1, sum[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) sum[r] += __shfl_xor(sum[r], d);
        if (lane == 0 && r < count) out[(p0 + r) * ldo + n] = to_bits<DT>(sum[r]);
    }
}

}  // namespace

int gemm_w4_launch(const W4Call& c, void* workspace, size_t workspace_bytes, const DeviceProps& props,
                   hipStream_t stream) {
    const int blocks_n = (int)((c.N + 3) / 4);
    const int64_t tiles = c.offsets ? c.total_rows / kRows + std::min<int64_t>(c.experts, c.total_rows)
                                    : (c.total_rows + kRows - 1) / kRows;
    auto kernel = c.dtype == MB_DT_FLOAT16 ? gemm_w4_kernel<MB_DT_FLOAT16> : gemm_w4_kernel<MB_DT_BFLOAT16>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles * blocks_n)), dim3(256), 0, stream,
                       static_cast<const uint16_t*>(c.x), c.ldx, c.x_rows, c.rows, static_cast<const uint8_t*>(c.q),
                       static_cast<const uint16_t*>(c.scales), static_cast<const uint16_t*>(c.zeros), c.group,
                       static_cast<uint16_t*>(c.out), c.ldo, c.offsets, c.experts, (int)c.total_rows, (int)c.N,
                       (int)c.K, blocks_n);
    MB_HIP_TRY(hipGetLastError());
    return MB_OK;
}

}  // namespace mb

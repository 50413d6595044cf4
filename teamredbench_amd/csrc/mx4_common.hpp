// Pieces shared by the microscaled 4-bit (MX4) kernels: the layout, one call of
// each operator, and the matrix instruction.
//
// MX4 holds a row in blocks of 32 elements: e2m1 floats (0, 0.5, 1, 1.5, 2, 3, 4,
// 6 and their negatives) times 2^(scale - 127), one scale byte per block (255:
// the block is NaN). Rows are padded with zeros to whole units of 128 elements, what
// a lane group of the matrix cores and one scale dword span: 64 bytes of
// elements (the even one in a byte's low half) and 4 of scales. So every row
// starts on 64 bytes, no kernel sees a partial unit, and scales go as dwords.
#pragma once

#include "experts_common.hpp"

namespace mb {

constexpr int kMx4Unit = 128;          // elements
constexpr int kMx4UnitBytes = 64;      // of elements
constexpr int kMx4UnitScales = 4;      // bytes

inline int64_t mx4_units(int64_t columns) { return (columns + kMx4Unit - 1) / kMx4Unit; }

struct Mx4Quantize {
    int dtype;
    bool fit;                          // scale rule
    const void* x;
    int64_t ldx, rows, columns;
    void *q, *scales, *qt, *scales_t;  // along rows, along columns; either pair may be null
};
int mx4_quantize_launch(const Mx4Quantize& c, hipStream_t stream);
int mx4_dequantize_launch(int dtype, const void* q, const void* scales, int64_t rows, int64_t columns, void* out,
                          int64_t ldo, hipStream_t stream);

// One call of mb_gemm_mx4, checked. offsets NULL: one expert with total_rows rows.
struct Mx4Call {
    int dtype, experts;                // dtype: of the output
    const void *x, *x_scales, *w, *w_scales;
    void* out;
    const int32_t *rows, *offsets;
    int64_t ldo, x_rows, total_rows, N, units;   // units: of K
};
int gemm_mx4_launch(const Mx4Call& c, void* workspace, size_t workspace_bytes, const DeviceProps& props,
                    hipStream_t stream);

namespace {

// acc += b a^T over 64 elements of K (32 columns of b, 32 rows of a). Lane l holds 32 elements of row l % 32 of
// each; A and B may spread K over l / 32 and the calls in any order they share. Byte SEL of the scale dwords is used.
// Alone on random operands, under the power limit, 32 x 32 x 64 sustains 6.5 to 6.7 PFLOP/s on the GPUs seen, 16 x 16 x 128
// 5.3 to 5.5.
template <int SEL_B, int SEL_A>
__device__ __forceinline__ f32x16 mfma_mx4(const u32x4& b, unsigned scale_b, const u32x4& a, unsigned scale_a,
                                           f32x16 acc) {
    constexpr int kE2M1 = 4;
    const i32x8 wide_b = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};   // e2m1 takes the first half
    const i32x8 wide_a = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide_b, wide_a, acc, kE2M1, kE2M1, SEL_B, (int)scale_b,
                                                           SEL_A, (int)scale_a);
}

}  // namespace
}  // namespace mb

// C ABI of the microscaled 4-bit operators (declared in include/mi355bench.h):
// argument checks and dispatch. C++ never throws through here: nothing below
// allocates.
#include "capi_checks.hpp"
#include "mx4_common.hpp"

using namespace mb;

namespace {

int check_values(const char* what, int dtype) {
    if (dtype == MB_DT_FLOAT32 || is_half(dtype)) return MB_OK;
    return refuse(MB_ERR_UNSUPPORTED, "%s takes float32, bfloat16 and float16, not %s", what, dtype_name(dtype));
}

// Rows x columns of a matrix, and of its MX4 forms.
int check_matrix(const char* what, int64_t rows, int64_t columns, int64_t* ld) {
    if (rows < 0 || columns < 1 || rows >= kMostRows || columns >= kMostRows)
        return refuse(MB_ERR_INVALID_ARG, "%s: needs 0 <= rows, 1 <= columns, both below 2^31 (got %lld, %lld)", what,
                      (long long)rows, (long long)columns);
    if (!leading(ld, columns, rows))
        return refuse(MB_ERR_INVALID_ARG, "%s: leading dimension %lld is below %lld columns", what, (long long)*ld,
                      (long long)columns);
    if (rows > 0 && mx4_units(rows) > (1ll << 26) / mx4_units(columns))   // 2^40 elements
        return refuse(MB_ERR_SHAPE, "%s: too large for one launch", what);
    return MB_OK;
}

int check_mx4(const char* what, const void* q, const void* scales) {
    if (off_element(q, 16) || off_element(scales, 4))
        return refuse(MB_ERR_SHAPE, "%s: elements must be on 16 bytes and scales on 4 (%p, %p)", what, q, scales);
    return MB_OK;
}

}  // namespace

extern "C" {

int mb_mx4_quantize(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t columns, int scale_rule, void* q,
                    void* scales, void* qt, void* scales_t, void* stream) {
    clear_error();
    MB_CHECK(check_values("mb_mx4_quantize", dtype));
    if (scale_rule != MB_MX4_SCALE_FLOOR && scale_rule != MB_MX4_SCALE_FIT)
        return refuse(MB_ERR_INVALID_ARG, "mb_mx4_quantize: unknown scale rule %d", scale_rule);
    MB_CHECK(check_matrix("mb_mx4_quantize", rows, columns, &ldx));
    if ((q == nullptr) != (scales == nullptr) || (qt == nullptr) != (scales_t == nullptr))
        return refuse(MB_ERR_INVALID_ARG, "mb_mx4_quantize: elements and scales come in pairs");
    MB_CHECK(check_mx4("mb_mx4_quantize", q, scales));
    MB_CHECK(check_mx4("mb_mx4_quantize", qt, scales_t));
    const DeviceProps* props = nullptr;
    if (rows == 0) return device_for_launch(&props);
    if (!x || (!q && !qt)) return refuse(MB_ERR_INVALID_ARG, "mb_mx4_quantize: null buffer pointer");
    if (off_element(x, dtype_size(dtype)))
        return refuse(MB_ERR_SHAPE, "mb_mx4_quantize: x must be on its element size (%p)", x);
    MB_CHECK(device_for_launch(&props));
    const Mx4Quantize c{dtype, scale_rule == MB_MX4_SCALE_FIT, x, ldx, rows, columns, q, scales, qt, scales_t};
    return mx4_quantize_launch(c, static_cast<hipStream_t>(stream));
}

int mb_mx4_dequantize(int dtype, const void* q, const void* scales, int64_t rows, int64_t columns, void* out,
                      int64_t ldo, void* stream) {
    clear_error();
    MB_CHECK(check_values("mb_mx4_dequantize", dtype));
    MB_CHECK(check_matrix("mb_mx4_dequantize", rows, columns, &ldo));
    const DeviceProps* props = nullptr;
    if (rows == 0) return device_for_launch(&props);
    if (!q || !scales || !out) return refuse(MB_ERR_INVALID_ARG, "mb_mx4_dequantize: null buffer pointer");
    MB_CHECK(check_mx4("mb_mx4_dequantize", q, scales));
    if (off_element(out, dtype_size(dtype)))
        return refuse(MB_ERR_SHAPE, "mb_mx4_dequantize: out must be on its element size (%p)", out);
    MB_CHECK(device_for_launch(&props));
    return mx4_dequantize_launch(dtype, q, scales, rows, columns, out, ldo, static_cast<hipStream_t>(stream));
}

int mb_gemm_mx4(int dtype, const void* x, const void* x_scales, int64_t x_rows, const int32_t* rows, const void* w,
                const void* w_scales, void* out, int64_t ldo, const int32_t* offsets, int experts, int64_t total_rows,
                int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    MB_CHECK(check_half("mb_gemm_mx4", dtype));
    MB_CHECK(check_rows("mb_gemm_mx4", rows, offsets, experts, total_rows, x_rows));
    if (offsets == nullptr && experts != 1)
        return refuse(MB_ERR_INVALID_ARG, "mb_gemm_mx4: %d experts need offsets", experts);
    if (N < 1 || K < 1 || N >= kMostRows / 2)
        return refuse(MB_ERR_INVALID_ARG, "mb_gemm_mx4: needs 1 <= N < 2^30 and K >= 1 (got %lld, %lld)",
                      (long long)N, (long long)K);
    if (K > MB_MX4_MAX_K)
        return refuse(MB_ERR_SHAPE, "mb_gemm_mx4: K must be at most %d (got %lld)", MB_MX4_MAX_K, (long long)K);
    if (!leading(&ldo, N, total_rows))
        return refuse(MB_ERR_INVALID_ARG, "mb_gemm_mx4: leading dimension %lld is below N = %lld", (long long)ldo,
                      (long long)N);
    // Ends of tiles of up to 256 rows are int32 too.
    if (total_rows > kMostRows - 256 || total_rows / 32 + experts >= kMostBlocks / ((N + 31) / 32))
        return refuse(MB_ERR_SHAPE, "mb_gemm_mx4: too many tiles for one launch");
    const DeviceProps* props = nullptr;
    if (total_rows == 0) return device_for_launch(&props);
    if (!x || !x_scales || !w || !w_scales || !out)
        return refuse(MB_ERR_INVALID_ARG, "mb_gemm_mx4: null buffer pointer");
    MB_CHECK(check_mx4("mb_gemm_mx4", x, x_scales));
    MB_CHECK(check_mx4("mb_gemm_mx4", w, w_scales));
    if (off_element(out, 2)) return refuse(MB_ERR_SHAPE, "mb_gemm_mx4: out must be on 2 bytes (%p)", out);
    MB_CHECK(device_for_launch(&props));
    const Mx4Call c{dtype, experts, x, x_scales, w, w_scales, out, rows, offsets, ldo, x_rows, total_rows, N,
                    mx4_units(K)};
    return gemm_mx4_launch(c, workspace, workspace_bytes, *props, static_cast<hipStream_t>(stream));
}

}  // extern "C"

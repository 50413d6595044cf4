// C ABI of the expert layer's operators (declared in include/mi355bench.h):
// argument checks and dispatch. C++ never throws through here: nothing below
// allocates.
#include "capi_checks.hpp"
#include "experts_common.hpp"

using namespace mb;

namespace {

bool route_counts(int64_t tokens, int experts, int top_k) {
    return tokens >= 0 && experts >= 1 && experts <= MB_ROUTE_MAX_EXPERTS && top_k >= 1 &&
           top_k <= MB_ROUTE_MAX_TOP_K && top_k <= experts;
}
bool route_slots_fit(int64_t tokens, int top_k) { return tokens <= (kMostRows - 1) / top_k; }

int check_route(const char* what, int dtype, int64_t tokens, int experts, int top_k) {
    if (dtype != MB_DT_FLOAT32 && !is_half(dtype))
        return refuse(MB_ERR_UNSUPPORTED, "%s takes float32, bfloat16 and float16, not %s", what, dtype_name(dtype));
    if (!route_counts(tokens, experts, top_k))
        return refuse(MB_ERR_INVALID_ARG,
                      "%s: needs tokens >= 0, 1 <= experts <= %d, 1 <= top_k <= min(experts, %d) (got %lld, %d, %d)",
                      what, MB_ROUTE_MAX_EXPERTS, MB_ROUTE_MAX_TOP_K, (long long)tokens, experts, top_k);
    if (!route_slots_fit(tokens, top_k))
        return refuse(MB_ERR_SHAPE, "%s: tokens * top_k must be below 2^31 (%lld * %d)", what, (long long)tokens,
                      top_k);
    return MB_OK;
}

}  // namespace

extern "C" {

size_t mb_route_workspace_size(int64_t tokens, int experts, int top_k) {
    if (!route_counts(tokens, experts, top_k) || !route_slots_fit(tokens, top_k)) return 0;
    return route_workspace(tokens, experts);
}

int mb_route(int dtype, const void* logits, int64_t ld, int64_t tokens, int experts, int top_k, int normalize,
             float* weights, int32_t* expert_ids, int32_t* offsets, int32_t* rows, int32_t* slots, void* workspace,
             size_t workspace_bytes, void* stream) {
    clear_error();
    MB_CHECK(check_route("mb_route", dtype, tokens, experts, top_k));
    if (offsets == nullptr ||
        (tokens > 0 && (!logits || !weights || !expert_ids || !rows || !slots)))
        return refuse(MB_ERR_INVALID_ARG, "mb_route: null buffer pointer");
    if (!leading(&ld, experts, tokens))
        return refuse(MB_ERR_INVALID_ARG, "mb_route: ld %lld is below %d experts", (long long)ld, experts);
    if (off_element(logits, dtype_size(dtype)) || off_element(weights, 4) || off_element(expert_ids, 4) ||
        off_element(offsets, 4) || off_element(rows, 4) || off_element(slots, 4))
        return refuse(MB_ERR_SHAPE, "mb_route: buffers must be on their element size");
    const size_t need = route_workspace(tokens, experts);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || off_element(workspace, 4)))
        return refuse(MB_ERR_WORKSPACE, "mb_route: needs %zu workspace bytes on 4 bytes (got %zu at %p)", need,
                      workspace_bytes, workspace);
    const DeviceProps* props = nullptr;
    MB_CHECK(device_for_launch(&props));
    return route_launch(dtype, logits, ld, tokens, experts, top_k, normalize != 0, weights, expert_ids, offsets, rows,
                        slots, workspace, static_cast<hipStream_t>(stream));
}

int mb_route_grad(int dtype, const void* logits, int64_t ld, const int32_t* expert_ids, const float* grad_weights,
                  int64_t tokens, int experts, int top_k, int normalize, void* grad_logits, int64_t ld_grad,
                  void* stream) {
    clear_error();
    MB_CHECK(check_route("mb_route_grad", dtype, tokens, experts, top_k));
    if (!leading(&ld, experts, tokens) || !leading(&ld_grad, experts, tokens))
        return refuse(MB_ERR_INVALID_ARG, "mb_route_grad: ld %lld / %lld is below %d experts", (long long)ld,
                      (long long)ld_grad, experts);
    const DeviceProps* props = nullptr;
    if (tokens == 0) return device_for_launch(&props);
    if (!logits || !expert_ids || !grad_weights || !grad_logits)
        return refuse(MB_ERR_INVALID_ARG, "mb_route_grad: null buffer pointer");
    if (off_element(logits, dtype_size(dtype)) || off_element(grad_logits, dtype_size(dtype)) ||
        off_element(expert_ids, 4) || off_element(grad_weights, 4))
        return refuse(MB_ERR_SHAPE, "mb_route_grad: buffers must be on their element size");
    MB_CHECK(device_for_launch(&props));
    return route_grad_launch(dtype, logits, ld, expert_ids, grad_weights, tokens, experts, top_k, normalize != 0,
                             grad_logits, ld_grad, static_cast<hipStream_t>(stream));
}

int mb_gemm_grouped(int op, int dtype, const void* x, int64_t ldx, int64_t x_rows, const int32_t* rows, const void* y,
                    int64_t ldy, void* out, int64_t ldo, const int32_t* offsets, int experts, int64_t total_rows,
                    int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    if (op < MB_GROUPED_FORWARD || op > MB_GROUPED_GRAD_WEIGHTS)
        return refuse(MB_ERR_INVALID_ARG, "mb_gemm_grouped: unknown op %d", op);
    MB_CHECK(check_half("mb_gemm_grouped", dtype));
    MB_CHECK(check_rows("mb_gemm_grouped", rows, offsets, experts, total_rows, x_rows));
    if (N < 1 || K < 1 || N >= kMostRows || K >= kMostRows)
        return refuse(MB_ERR_INVALID_ARG, "mb_gemm_grouped: N and K must be 1 .. 2^31 - 1 (got %lld, %lld)",
                      (long long)N, (long long)K);
    const bool weights = op == MB_GROUPED_GRAD_WEIGHTS;
    const int64_t matrices = experts * K;   // rows of all B (dB)
    if (!leading(&ldx, op == MB_GROUPED_GRAD_ROWS ? N : K, x_rows) ||
        !leading(&ldy, N, weights ? total_rows : matrices) ||
        !leading(&ldo, op == MB_GROUPED_GRAD_ROWS ? K : N, weights ? matrices : total_rows))
        return refuse(MB_ERR_INVALID_ARG, "mb_gemm_grouped: a leading dimension (%lld, %lld, %lld) is below its rows",
                      (long long)ldx, (long long)ldy, (long long)ldo);
    if (K > (kMostRows / 2 - 1) / (weights ? ldo : ldy))
        return refuse(MB_ERR_SHAPE, "mb_gemm_grouped: a matrix of %lld rows of %lld elements passes 2^31 bytes",
                      (long long)K, (long long)(weights ? ldo : ldy));
    const int64_t tiles_n = ((op == MB_GROUPED_GRAD_ROWS ? K : N) + 63) / 64;
    const int64_t tiles_m = weights ? experts * ((K + 63) / 64) : total_rows / 64 + experts;
    if (tiles_m >= kMostBlocks / tiles_n)
        return refuse(MB_ERR_SHAPE, "mb_gemm_grouped: too many tiles for one launch");
    const DeviceProps* props = nullptr;
    if (total_rows == 0 && !weights) return device_for_launch(&props);
    if (!out || !offsets || (total_rows > 0 && (!x || !y)))
        return refuse(MB_ERR_INVALID_ARG, "mb_gemm_grouped: null buffer pointer");
    if (off_element(x, 2) || off_element(y, 2) || off_element(out, 2))
        return refuse(MB_ERR_SHAPE, "mb_gemm_grouped: matrices must be on 2 bytes");
    MB_CHECK(device_for_launch(&props));
    GroupedCall c{op, dtype, experts, x, y, out, rows, offsets, ldx, ldy, ldo, x_rows, total_rows, N, K};
    return gemm_grouped_launch(c, workspace, workspace_bytes, *props, static_cast<hipStream_t>(stream));
}

int mb_gemm_w4(int dtype, const void* x, int64_t ldx, int64_t x_rows, const int32_t* rows, const void* q,
               const void* scales, const void* zeros, int group, void* out, int64_t ldo, const int32_t* offsets,
               int experts, int64_t total_rows, int64_t N, int64_t K, void* workspace, size_t workspace_bytes,
               void* stream) {
    clear_error();
    MB_CHECK(check_half("mb_gemm_w4", dtype));
    MB_CHECK(check_rows("mb_gemm_w4", rows, offsets, experts, total_rows, x_rows));
    if (offsets == nullptr && experts != 1)
        return refuse(MB_ERR_INVALID_ARG, "mb_gemm_w4: %d experts need offsets", experts);
    if (N < 1 || K < 1 || N >= kMostRows / 2 || K >= kMostRows / 2)
        return refuse(MB_ERR_INVALID_ARG, "mb_gemm_w4: N and K must be 1 .. 2^30 - 1 (got %lld, %lld)", (long long)N,
                      (long long)K);
    if (group < 32 || group % 32 != 0)
        return refuse(MB_ERR_SHAPE, "mb_gemm_w4: group must be a positive multiple of 32 (got %d)", group);
    if (!leading(&ldx, K, x_rows) || !leading(&ldo, N, total_rows))
        return refuse(MB_ERR_INVALID_ARG, "mb_gemm_w4: a leading dimension (%lld, %lld) is below its rows",
                      (long long)ldx, (long long)ldo);
    if (total_rows / 16 + experts >= kMostBlocks / ((N + 15) / 16))
        return refuse(MB_ERR_SHAPE, "mb_gemm_w4: too many tiles for one launch");
    const DeviceProps* props = nullptr;
    if (total_rows == 0) return device_for_launch(&props);
    if (!x || !q || !scales || !out) return refuse(MB_ERR_INVALID_ARG, "mb_gemm_w4: null buffer pointer");
    if (off_element(x, 2) || off_element(scales, 2) || off_element(zeros, 2) || off_element(out, 2))
        return refuse(MB_ERR_SHAPE, "mb_gemm_w4: x, scales, zeros and out must be on 2 bytes");
    MB_CHECK(device_for_launch(&props));
    W4Call c{dtype, experts, group, x, q, scales, zeros, out, rows, offsets, ldx, ldo, x_rows, total_rows, N, K};
    return gemm_w4_launch(c, workspace, workspace_bytes, *props, static_cast<hipStream_t>(stream));
}

namespace {

int check_combine(const char* what, int dtype, int64_t y_rows, int64_t tokens, int top_k, int64_t N) {
    MB_CHECK(check_half(what, dtype));
    if (tokens < 0 || y_rows < 0 || y_rows >= kMostRows || top_k < 1 || top_k > MB_ROUTE_MAX_TOP_K || N < 1 ||
        N >= kMostRows)
        return refuse(MB_ERR_INVALID_ARG,
                      "%s: needs tokens >= 0, 0 <= y_rows < 2^31, 1 <= top_k <= %d, N >= 1 (got %lld, %lld, %d, %lld)",
                      what, MB_ROUTE_MAX_TOP_K, (long long)tokens, (long long)y_rows, top_k, (long long)N);
    if (tokens >= kMostRows / ((N + 2047) / 2048))   // runs of 2048 columns are int32
        return refuse(MB_ERR_SHAPE, "%s: too many tokens for one launch (%lld)", what, (long long)tokens);
    return MB_OK;
}

}  // namespace

int mb_combine(int dtype, const void* y, int64_t ldy, int64_t y_rows, const float* weights, const int32_t* slots,
               int64_t tokens, int top_k, int64_t N, void* out, int64_t ldo, void* stream) {
    clear_error();
    MB_CHECK(check_combine("mb_combine", dtype, y_rows, tokens, top_k, N));
    if (!leading(&ldy, N, y_rows) || !leading(&ldo, N, tokens))
        return refuse(MB_ERR_INVALID_ARG, "mb_combine: a leading dimension (%lld, %lld) is below N = %lld",
                      (long long)ldy, (long long)ldo, (long long)N);
    const DeviceProps* props = nullptr;
    if (tokens == 0) return device_for_launch(&props);
    if ((!y && y_rows > 0) || !slots || !out) return refuse(MB_ERR_INVALID_ARG, "mb_combine: null buffer pointer");
    if (off_element(y, 2) || off_element(out, 2) || off_element(slots, 4) || off_element(weights, 4))
        return refuse(MB_ERR_SHAPE, "mb_combine: buffers must be on their element size");
    MB_CHECK(device_for_launch(&props));
    return combine_launch(dtype, y, ldy, y_rows, weights, slots, tokens, top_k, N, out, ldo,
                          static_cast<hipStream_t>(stream));
}

int mb_combine_grad(int dtype, const void* grad_out, int64_t ldg, const void* y, int64_t ldy, int64_t y_rows,
                    const float* weights, const int32_t* slots, int64_t tokens, int top_k, int64_t N, void* grad_y,
                    int64_t ld_grad_y, float* grad_weights, void* stream) {
    clear_error();
    MB_CHECK(check_combine("mb_combine_grad", dtype, y_rows, tokens, top_k, N));
    if (!leading(&ldg, N, tokens) || !leading(&ldy, N, y_rows) || !leading(&ld_grad_y, N, y_rows))
        return refuse(MB_ERR_INVALID_ARG, "mb_combine_grad: a leading dimension (%lld, %lld, %lld) is below N = %lld",
                      (long long)ldg, (long long)ldy, (long long)ld_grad_y, (long long)N);
    const DeviceProps* props = nullptr;
    if (tokens == 0 || (!grad_y && !grad_weights)) return device_for_launch(&props);
    if (!grad_out || !slots || (grad_weights && !y && y_rows > 0))
        return refuse(MB_ERR_INVALID_ARG, "mb_combine_grad: null buffer pointer");
    if (off_element(grad_out, 2) || off_element(y, 2) || off_element(grad_y, 2) || off_element(slots, 4) ||
        off_element(weights, 4) || off_element(grad_weights, 4))
        return refuse(MB_ERR_SHAPE, "mb_combine_grad: buffers must be on their element size");
    MB_CHECK(device_for_launch(&props));
    return combine_grad_launch(dtype, grad_out, ldg, y, ldy, y_rows, weights, slots, tokens, top_k, N, grad_y,
                               ld_grad_y, grad_weights, static_cast<hipStream_t>(stream));
}

}  // extern "C"

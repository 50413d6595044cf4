// Argument checks shared by the C ABI's translation units. Nothing here allocates,
// so nothing throws through the C entry points.
#pragma once

#include "mb_common.hpp"

namespace mb {
namespace {

constexpr int64_t kMostRows = 1ll << 31;      // rows and slots are int32
constexpr int64_t kMostBlocks = 1ll << 30;    // of a launch, in tiles of the smallest size

inline bool is_half(int dtype) { return dtype == MB_DT_BFLOAT16 || dtype == MB_DT_FLOAT16; }

inline int refuse(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
inline int refuse(int status, const char* fmt, ...) {
    char text[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof(text), fmt, ap);
    va_end(ap);
    set_error("%s", text);
    return status;
}

// Elements sit on their own size.
inline bool off_element(const void* p, size_t size) { return (reinterpret_cast<uintptr_t>(p) & (size - 1)) != 0; }

// 0 -> packed rows of `columns`; false if shorter than that, or the matrix passes 2^62 bytes.
inline bool leading(int64_t* ld, int64_t columns, int64_t rows) {
    if (*ld == 0) *ld = columns;
    return *ld >= columns && *ld <= (1ll << 40) && (rows <= 0 || *ld <= (1ll << 61) / rows);
}

inline int check_half(const char* what, int dtype) {
    if (is_half(dtype)) return MB_OK;
    return refuse(MB_ERR_UNSUPPORTED, "%s takes bfloat16 and float16, not %s", what, dtype_name(dtype));
}

// rows / offsets of the products over sorted rows.
inline int check_rows(const char* what, const int32_t* rows, const int32_t* offsets, int experts, int64_t total_rows,
                      int64_t x_rows) {
    if (experts < 1 || experts > MB_ROUTE_MAX_EXPERTS)
        return refuse(MB_ERR_INVALID_ARG, "%s: 1 <= experts <= %d (got %d)", what, MB_ROUTE_MAX_EXPERTS, experts);
    if (total_rows < 0 || x_rows < 0 || total_rows >= kMostRows || x_rows >= kMostRows)
        return refuse(MB_ERR_INVALID_ARG, "%s: needs 0 <= total_rows, x_rows < 2^31 (got %lld, %lld)", what,
                      (long long)total_rows, (long long)x_rows);
    if (rows == nullptr && x_rows < total_rows)
        return refuse(MB_ERR_INVALID_ARG, "%s: without rows x needs total_rows rows (%lld < %lld)", what,
                      (long long)x_rows, (long long)total_rows);
    if (off_element(rows, 4) || off_element(offsets, 4))
        return refuse(MB_ERR_SHAPE, "%s: rows and offsets must be on 4 bytes (%p, %p)", what, (const void*)rows,
                      (const void*)offsets);
    return MB_OK;
}

#define MB_CHECK(expr)              \
    do {                            \
        const int rc_ = (expr);     \
        if (rc_ != MB_OK) return rc_; \
    } while (0)

}  // namespace
}  // namespace mb

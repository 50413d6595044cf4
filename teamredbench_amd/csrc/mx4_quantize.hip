// Quantisation to MX4 and back (layout: mx4_common.hpp).
//
// A block's scale goes by its largest magnitude a = m 2^e, 1 <= m < 2:
//   FLOOR  2^(e - 2): a lands in [4, 8), and what lies above 6 saturates
//   FIT    2^(e - 1) where m > 1.5, so that nothing saturates
// not below 2^-127. a's exponent is read off its fp32 bits (subnormal a: 2^-127
// either way). Elements are x / scale, rounded to the nearest e2m1 value, ties to the even code,
// by v_cvt_scalef32_pk_fp4_*: checked against the definition for every bf16
// value under 15 scales, and for fp32 at and next to every border. A block that holds an infinity or a
// NaN has no scale: it becomes NaN as a whole (scale 255, elements 0).
//
// Bytes bound all of it: x is read once, whichever forms are written.
#include "mx4_common.hpp"

namespace mb {
namespace {

template <int DT>
struct Source {                        // elements as raw bits, two to a dword (fp32: one)
    typedef uint16_t Element;
    static constexpr int kWords = 4;   // dwords of 8 elements
};
template <>
struct Source<MB_DT_FLOAT32> {
    typedef uint32_t Element;
    static constexpr int kWords = 8;
};

typedef u32x4 u32x4_2 __attribute__((aligned(2)));
typedef u32x4 u32x4_4 __attribute__((aligned(4)));

// 8 elements from `column` on of a row of `columns`, as bits; zeros past its end, none of which is read.
template <int DT>
__device__ __forceinline__ void load8(const void* row, int64_t column, int64_t columns,
                                      unsigned (&v)[Source<DT>::kWords]) {
    typedef typename Source<DT>::Element Element;
    const Element* p = static_cast<const Element*>(row) + column;
    if (column + 8 <= columns) {
        const u32x4 a = *reinterpret_cast<const u32x4_2*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = a[i];
        if constexpr (DT == MB_DT_FLOAT32) {
            const u32x4 b = *reinterpret_cast<const u32x4_2*>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 + i] = b[i];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < Source<DT>::kWords; ++i) v[i] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (column + i < columns) {
            if constexpr (DT == MB_DT_FLOAT32) v[i] = p[i];
            else v[i / 2] |= (unsigned)p[i] << (16 * (i & 1));
        }
}

// The fp32 bits of a magnitude given as its own type's bits.
template <int DT>
__device__ __forceinline__ unsigned magnitude_bits(unsigned m) {
    if constexpr (DT == MB_DT_FLOAT32) return m;
    else if constexpr (DT == MB_DT_BFLOAT16) return m << 16;
    else return __builtin_bit_cast(unsigned, (float)__builtin_bit_cast(_Float16, (uint16_t)m));
}

// The scale byte of a block whose largest magnitude has these fp32 bits; 255 if that is no finite number.
__device__ __forceinline__ unsigned scale_byte(unsigned bits, bool fit) {
    const unsigned e = bits >> 23;
    if (e == 255) return 255;
    unsigned s = e > 2 ? e - 2 : 0;
    if (fit && e >= 2 && (bits & 0x7FFFFFu) > 0x400000u) ++s;
    return s;
}

// 8 elements (4 dwords of 16-bit bits, or 8 of fp32) as 8 nibbles under scale byte s; zeros if s is 255.
template <int DT>
__device__ __forceinline__ unsigned encode8(const unsigned* v, unsigned s) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const float scale = __builtin_bit_cast(float, s << 23);   // the instruction reads the exponent alone
    unsigned q = 0;
    if constexpr (DT == MB_DT_FLOAT32) {
        auto f = [&](int i) { return __builtin_bit_cast(float, v[i]); };
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f(0), f(1), scale, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f(2), f(3), scale, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f(4), f(5), scale, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f(6), f(7), scale, 3);
    } else if constexpr (DT == MB_DT_BFLOAT16) {
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, v[0]), scale, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, v[1]), scale, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, v[2]), scale, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, v[3]), scale, 3);
    } else {
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, v[0]), scale, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, v[1]), scale, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, v[2]), scale, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, v[3]), scale, 3);
    }
    return s == 255 ? 0u : q;
}

// The largest magnitude of 8 elements, as their own type's bits.
template <int DT>
__device__ __forceinline__ unsigned largest8(const unsigned (&v)[Source<DT>::kWords]) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < Source<DT>::kWords; ++i) {
        if constexpr (DT == MB_DT_FLOAT32) m = max(m, v[i] & 0x7FFFFFFFu);
        else m = max(m, max(v[i] & 0x7FFFu, (v[i] >> 16) & 0x7FFFu));
    }
    return m;
}

__device__ __forceinline__ unsigned lane_xor1(unsigned v) { return __builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true); }
__device__ __forceinline__ unsigned lane_xor2(unsigned v) { return __builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true); }
__device__ __forceinline__ unsigned max4(unsigned v) {   // over each four lanes
    v = max(v, lane_xor1(v));
    return max(v, lane_xor2(v));
}

// Along rows: 16 lanes per unit of a row, 8 elements a lane, four lanes a block.
template <int DT, bool FIT>
__global__ void __launch_bounds__(256)
mx4_quantize_rows_kernel(const void* __restrict__ x, int64_t ldx, int64_t rows, int64_t columns, int64_t units,
                         unsigned* __restrict__ q, unsigned char* __restrict__ scales) {
    const int64_t i = (int64_t)block_number() * 256 + threadIdx.x;
    const int64_t unit = i >> 4;
    const int64_t row = unit / units;
    if (row >= rows) return;
    const int64_t column = (unit - row * units) * kMx4Unit + 8 * (i & 15);
    unsigned v[Source<DT>::kWords];
    load8<DT>(static_cast<const typename Source<DT>::Element*>(x) + row * ldx, column, columns, v);
    const unsigned s = scale_byte(magnitude_bits<DT>(max4(largest8<DT>(v))), FIT);
    q[i] = encode8<DT>(v, s);
    if ((i & 3) == 0) scales[i >> 2] = (unsigned char)s;
}

// Along columns: a lane holds 32 rows of one column.
template <int DT, bool FIT>
__global__ void __launch_bounds__(256)
mx4_quantize_columns_kernel(const void* __restrict__ x, int64_t ldx, int64_t rows, int64_t columns, int64_t units,
                            u32x4* __restrict__ qt, unsigned char* __restrict__ scales_t) {
    typedef typename Source<DT>::Element Element;
    const int64_t i = (int64_t)block_number() * 256 + threadIdx.x;
    const int64_t blocks = 4 * units, block = i / columns, column = i - block * columns;
    if (block >= blocks) return;
    unsigned v[32], most = 0;
    const Element* p = static_cast<const Element*>(x) + column;
#pragma unroll
    for (int r = 0; r < 32; ++r) v[r] = block * 32 + r < rows ? p[(block * 32 + r) * ldx] : 0;
#pragma unroll
    for (int r = 0; r < 32; ++r) most = max(most, v[r] & (DT == MB_DT_FLOAT32 ? 0x7FFFFFFFu : 0x7FFFu));
    const unsigned s = scale_byte(magnitude_bits<DT>(most), FIT);
    u32x4 out;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        unsigned w[Source<DT>::kWords];
#pragma unroll
        for (int j = 0; j < Source<DT>::kWords; ++j) {
            if constexpr (DT == MB_DT_FLOAT32) w[j] = v[8 * d + j];
            else w[j] = v[8 * d + 2 * j] | (v[8 * d + 2 * j + 1] << 16);
        }
        out[d] = encode8<DT>(w, s);
    }
    qt[column * blocks + block] = out;
    scales_t[column * blocks + block] = (unsigned char)s;
}

// 8 elements a lane.
template <int DT>
__global__ void __launch_bounds__(256)
mx4_dequantize_kernel(const unsigned* __restrict__ q, const unsigned char* __restrict__ scales, int64_t rows,
                      int64_t columns, int64_t units, typename Source<DT>::Element* __restrict__ out, int64_t ldo) {
    const int64_t i = (int64_t)block_number() * 256 + threadIdx.x;
    const int64_t unit = i >> 4;
    const int64_t row = unit / units;
    if (row >= rows) return;
    const int64_t column = (unit - row * units) * kMx4Unit + 8 * (i & 15);
    if (column >= columns) return;
    const unsigned codes = q[i];
    const float scale = __builtin_bit_cast(float, (unsigned)scales[i >> 2] << 23);
    unsigned v[Source<DT>::kWords];
    auto two = [&](auto sel) {
        constexpr int s = decltype(sel)::value;
        if constexpr (DT == MB_DT_FLOAT32) {
            const auto f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, s);
            v[2 * s] = __builtin_bit_cast(unsigned, (float)f[0]);
            v[2 * s + 1] = __builtin_bit_cast(unsigned, (float)f[1]);
        } else if constexpr (DT == MB_DT_BFLOAT16) {
            v[s] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, s));
        } else {
            v[s] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, s));
        }
    };
    two(std::integral_constant<int, 0>{});
    two(std::integral_constant<int, 1>{});
    two(std::integral_constant<int, 2>{});
    two(std::integral_constant<int, 3>{});
    auto* p = out + row * ldo + column;
    if (column + 8 <= columns) {
        *reinterpret_cast<u32x4_2*>(p) = u32x4{v[0], v[1], v[2], v[3]};
        if constexpr (DT == MB_DT_FLOAT32) *reinterpret_cast<u32x4_2*>(p + 4) = u32x4{v[4], v[5], v[6], v[7]};
        return;
    }
#pragma unroll
    for (int e = 0; e < 7; ++e)
        if (column + e < columns) {
            if constexpr (DT == MB_DT_FLOAT32) p[e] = v[e];
            else p[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
        }
}

template <int DT, bool FIT>
int quantize(const Mx4Quantize& c, hipStream_t stream) {
    if (c.q != nullptr) {
        const int64_t units = mx4_units(c.columns);
        hipLaunchKernelGGL((mx4_quantize_rows_kernel<DT, FIT>), launch_grid((c.rows * units + 15) / 16), dim3(256), 0,
                           stream, c.x, c.ldx, c.rows, c.columns, units, static_cast<unsigned*>(c.q),
                           static_cast<unsigned char*>(c.scales));
        MB_HIP_TRY(hipGetLastError());
    }
    if (c.qt != nullptr) {
        const int64_t units = mx4_units(c.rows);
        hipLaunchKernelGGL((mx4_quantize_columns_kernel<DT, FIT>), launch_grid((c.columns * units * 4 + 255) / 256),
                           dim3(256), 0, stream, c.x, c.ldx, c.rows, c.columns, units, static_cast<u32x4*>(c.qt),
                           static_cast<unsigned char*>(c.scales_t));
        MB_HIP_TRY(hipGetLastError());
    }
    return MB_OK;
}

template <int DT>
int dequantize(const void* q, const void* scales, int64_t rows, int64_t columns, void* out, int64_t ldo,
               hipStream_t stream) {
    typedef typename Source<DT>::Element Element;
    const int64_t units = mx4_units(columns);
    hipLaunchKernelGGL((mx4_dequantize_kernel<DT>), launch_grid((rows * units + 15) / 16), dim3(256), 0, stream,
                       static_cast<const unsigned*>(q), static_cast<const unsigned char*>(scales), rows, columns, units,
                       static_cast<Element*>(out), ldo);
    MB_HIP_TRY(hipGetLastError());
    return MB_OK;
}

}  // namespace

int mx4_quantize_launch(const Mx4Quantize& c, hipStream_t stream) {
    if (c.dtype == MB_DT_FLOAT32)
        return c.fit ? quantize<MB_DT_FLOAT32, true>(c, stream) : quantize<MB_DT_FLOAT32, false>(c, stream);
    if (c.dtype == MB_DT_BFLOAT16)
        return c.fit ? quantize<MB_DT_BFLOAT16, true>(c, stream) : quantize<MB_DT_BFLOAT16, false>(c, stream);
    return c.fit ? quantize<MB_DT_FLOAT16, true>(c, stream) : quantize<MB_DT_FLOAT16, false>(c, stream);
}

int mx4_dequantize_launch(int dtype, const void* q, const void* scales, int64_t rows, int64_t columns, void* out,
                          int64_t ldo, hipStream_t stream) {
    if (dtype == MB_DT_FLOAT32) return dequantize<MB_DT_FLOAT32>(q, scales, rows, columns, out, ldo, stream);
    if (dtype == MB_DT_BFLOAT16) return dequantize<MB_DT_BFLOAT16>(q, scales, rows, columns, out, ldo, stream);
    return dequantize<MB_DT_FLOAT16>(q, scales, rows, columns, out, ldo, stream);
}

}  // namespace mb

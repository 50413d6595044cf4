// Quantisation to MX4 and back (layout: mx4_common.hpp).
//
// A block's scale goes by its largest magnitude a = m 2^e, 1 <= m < 2:
//   FLOOR  2^(e - 2): a lands in [4, 8), and what lies above 6 saturates
//   FIT    2^(e - 1) where m > 1.5, so that nothing saturates
// not below 2^-127. a's exponent is read off its fp32 bits (subnormal a: 2^-127
// either way). Elements are x / scale, rounded to the nearest e2m1 value, ties to the even code,
// by v_cvt_scalef32_pk_fp4_*, which the tests compare with the definition for every 16-bit
// value under scales from its own to 5 binades above, and for the fp32 values next to them. A block that holds an
// infinity or a NaN has no scale: it becomes NaN as a whole (scale 255, elements 0).
//
// Bytes bound all of it: x is read once, whichever forms are written. bf16 8192 x 8192, inputs and outputs not in the
// caches: rows 31 us (5.4 TB/s), columns 37 (4.6), both 49 (4.2), values back 25 (6.7; 30 over nine and more outputs in
// turn); fp32 57, 61, 75 and 44 (54). From the Infinity Cache rows take 25 us and both 37.
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

// The first 4 of them, 16 bits.
template <int DT>
__device__ __forceinline__ unsigned encode4(const unsigned* v, unsigned s) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const float scale = __builtin_bit_cast(float, s << 23);
    unsigned q = 0;
    if constexpr (DT == MB_DT_FLOAT32) {
        auto f = [&](int i) { return __builtin_bit_cast(float, v[i]); };
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f(0), f(1), scale, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f(2), f(3), scale, 1);
    } else if constexpr (DT == MB_DT_BFLOAT16) {
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, v[0]), scale, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, v[1]), scale, 1);
    } else {
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, v[0]), scale, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(f16x2, v[1]), scale, 1);
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

// Along rows: 16 lanes per unit of a row, 8 elements a lane, four lanes a block; UNITS units a lane group, loaded before
// any of them is used. The units of a matrix follow each other in q and in scales, whatever its rows.
template <int DT, int UNITS>
__global__ void __launch_bounds__(256)
mx4_quantize_rows_kernel(const void* __restrict__ x, int64_t ldx, int64_t rows, int64_t columns, int64_t units,
                         bool fit, unsigned* __restrict__ q, unsigned char* __restrict__ scales) {
    typedef typename Source<DT>::Element Element;
    const int64_t first = (int64_t)block_number() * (16 * UNITS) + threadIdx.x / 16;
    const int lane16 = threadIdx.x % 16;
    unsigned v[UNITS][Source<DT>::kWords];
    const int64_t total = rows * units;
#pragma unroll
    for (int k = 0; k < UNITS; ++k) {
        const int64_t unit = min(first + 16 * k, total - 1);
        const int64_t row = unit / units, column = (unit - row * units) * kMx4Unit + 8 * lane16;
        load8<DT>(static_cast<const Element*>(x) + row * ldx, column, columns, v[k]);
    }
#pragma unroll
    for (int k = 0; k < UNITS; ++k) {
        const int64_t unit = first + 16 * k;
        if (unit >= total) return;
        const unsigned s = scale_byte(magnitude_bits<DT>(max4(largest8<DT>(v[k]))), fit);
        q[unit * 16 + lane16] = encode8<DT>(v[k], s);
        if (lane16 % 4 == 0) scales[unit * 4 + lane16 / 4] = (unsigned char)s;
    }
}

// The largest of both 16-bit halves (fp32: of the whole).
template <int DT>
__device__ __forceinline__ unsigned max_bits(unsigned a, unsigned b) {
    if constexpr (DT == MB_DT_FLOAT32) {
        return max(a, b);
    } else {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned,
                                  __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
    }
}

// 16 bytes of elements without the first n of them, zeros behind; n < 4 (fp32) or 8.
template <int DT>
__device__ __forceinline__ u32x4 drop_first(u32x4 v, int n) {
    if constexpr (DT != MB_DT_FLOAT32) {
        if (n & 1) v = {v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
        n >>= 1;
    }
    if (n & 1) v = {v[1], v[2], v[3], 0};
    if (n & 2) v = {v[2], v[3], 0, 0};
    return v;
}

// Along columns, or along both: 128 rows x 256 bytes of each a block, through LDS. Lanes take 16 bytes of a row (16 lanes
// a row), so a row's blocks span four lanes (fp32: eight); then a lane takes 32 rows of one dword's columns. Four
// neighbouring lanes take the four blocks of 128 rows, and store 64 bytes; 16-byte chunk c of row r lies at chunk
// c ^ 4 (r / 32), which spreads their reads over the banks. (Both forms from registers, a lane holding 32 rows x 4 or 8
// columns, took 72 us for bf16 8192 x 8192: two waves a SIMD, and long chains of lane exchanges. Tiles of 256 rows, which
// store whole lines of the columns' form, took 50: what binds is the memory's turning between reads and writes.)
template <int DT, bool ROWS>
__global__ void __launch_bounds__(256)
mx4_quantize_tile_kernel(const void* __restrict__ x, int64_t ldx, int64_t rows, int64_t columns, bool fit,
                         int64_t tiles_n, unsigned char* __restrict__ q, unsigned char* __restrict__ scales,
                         unsigned char* __restrict__ qt, unsigned char* __restrict__ scales_t) {
    typedef typename Source<DT>::Element Element;
    constexpr bool WIDE = DT == MB_DT_FLOAT32;
    constexpr int EACH = WIDE ? 4 : 8, COLUMNS = 16 * EACH;   // columns of a lane's 16 bytes, of a tile
    constexpr unsigned kMagnitude = WIDE ? 0x7FFFFFFFu : 0x7FFF7FFFu;
    __shared__ u32x4 tile[128 * 16];
    const int tid = threadIdx.x, l16 = tid % 16;
    // Tiles in squares of 256 x 256: those of one XCD (block b runs on XCD b % 8), one after the other, so that its L2
    // joins their halves (fp32: quarters) of both forms' lines of 128 bytes: fp32 8192 x 8192 90 -> 76 us, 1.54 million
    // write requests where tile by tile makes 2.11 (whole ones of 64 bytes: 1.11). Squares along x's
    // rows: in panels of 2 to 16 squares' width down x both forms took 52 to 62 us for 49.
    constexpr int WIDTH = 256 / COLUMNS, SQUARE = 2 * WIDTH;
    const int64_t block = block_number(), local = block / 8, square = local / SQUARE * 8 + block % 8;
    const int64_t squares_n = (tiles_n + WIDTH - 1) / WIDTH, square_r = square / squares_n;
    const int within = (int)(local % SQUARE);
    const int64_t unit_r = 2 * square_r + within / WIDTH;
    const int64_t tile_c = (square - square_r * squares_n) * WIDTH + within % WIDTH;
    const int64_t units = (columns + kMx4Unit - 1) / kMx4Unit, units_t = (rows + kMx4Unit - 1) / kMx4Unit;
    const int64_t r0 = unit_r * kMx4Unit, c0 = tile_c * COLUMNS;
    if (unit_r >= units_t || tile_c >= tiles_n) return;
    const int row_count = (int)min(rows - r0, (int64_t)kMx4Unit);
    auto piece = [&](int k) -> u32x4& {   // this lane's of row tid / 16 + 16 k
        const int r = tid / 16 + 16 * k;
        return tile[r * 16 + (l16 ^ 4 * (r / 32))];
    };
    {
        const Element* p = static_cast<const Element*>(x) + (r0 + tid / 16) * ldx + c0 + EACH * l16;
        if (row_count == kMx4Unit && c0 + COLUMNS <= columns) {
            u32x4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const u32x4_2*>(p + 16 * k * ldx);
#pragma unroll
            for (int k = 0; k < 8; ++k) piece(k) = v[k];
        } else if (columns >= EACH) {   // an edge: pieces of the last rows and columns, less what lies before
            // them, so that eight loads are in flight here too (guarded one by one: fp32 3001 x 2057 11.9 us, this 10.8)
            const int64_t past = max(c0 + EACH * l16 - (columns - EACH), (int64_t)0);
            u32x4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                v[k] = *reinterpret_cast<const u32x4_2*>(p + min(16 * k, row_count - 1 - tid / 16) * ldx - past);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                piece(k) = past < EACH && tid / 16 + 16 * k < row_count ? drop_first<DT>(v[k], (int)past)
                                                                        : u32x4{0, 0, 0, 0};
        } else {
            const int64_t left = columns - (c0 + EACH * l16);
            for (int k = 0; k < 8; ++k) {
                u32x4 v = {0, 0, 0, 0};
                if (tid / 16 + 16 * k < row_count) {
#pragma unroll
                    for (int i = 0; i < EACH - 1; ++i)
                        if (i < left) {
                            if constexpr (WIDE) v[i] = p[16 * k * ldx + i];
                            else v[i / 2] |= (unsigned)p[16 * k * ldx + i] << 16 * (i & 1);
                        }
                }
                piece(k) = v;
            }
        }
        if constexpr (ROWS) {
            // fp32: a tile is half a unit wide, and past the last column's unit there is nothing to write.
            const int64_t unit_c = WIDE ? tile_c / 2 : tile_c;
            const int part = WIDE ? (int)(tile_c % 2) : 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const u32x4 v = piece(k);
                unsigned m = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) m = max_bits<DT>(m, v[i] & kMagnitude);
                if constexpr (!WIDE) m = max(m & 0xFFFFu, m >> 16);
                m = max4(m);
                if constexpr (WIDE) m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xF, 0xF, true));   // 7 - l
                const unsigned s = scale_byte(magnitude_bits<DT>(m), fit);
                unsigned w[Source<DT>::kWords] = {};
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = v[i];
                const int r = tid / 16 + 16 * k;
                if (r < row_count) {
                    const int64_t unit = (r0 + r) * units + unit_c;
                    if constexpr (WIDE) {
                        *reinterpret_cast<uint16_t*>(q + unit * kMx4UnitBytes + 32 * part + 2 * l16) =
                            (uint16_t)encode4<DT>(w, s);
                        if (l16 % 8 == 0) scales[unit * kMx4UnitScales + 2 * part + l16 / 8] = (unsigned char)s;
                    } else {
                        *reinterpret_cast<unsigned*>(q + unit * kMx4UnitBytes + 4 * l16) = encode8<DT>(w, s);
                        if (l16 % 4 == 0) scales[unit * kMx4UnitScales + l16 / 4] = (unsigned char)s;
                    }
                }
            }
        }
    }
    __syncthreads();
    const int group = tid % 4, at = tid / 4;   // 32 rows, dword of a row
    const int64_t c = c0 + (WIDE ? at : 2 * at);
    const unsigned* from = reinterpret_cast<const unsigned*>(tile) + 32 * group * 64 + (at ^ 16 * group);
    unsigned v[32], most = 0;
#pragma unroll
    for (int r = 0; r < 32; ++r) v[r] = from[r * 64];
#pragma unroll
    for (int r = 0; r < 32; ++r) most = max_bits<DT>(most, v[r] & kMagnitude);
#pragma unroll
    for (int j = 0; j < (WIDE ? 1 : 2); ++j) {
        constexpr unsigned kPick[2] = {0x05040100u, 0x07060302u};   // low halves of two dwords, high halves
        const unsigned s = scale_byte(magnitude_bits<DT>(WIDE ? most : most >> 16 * j & 0xFFFFu), fit);
        u32x4 out;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            unsigned w[Source<DT>::kWords];
#pragma unroll
            for (int i = 0; i < Source<DT>::kWords; ++i) {
                if constexpr (WIDE) w[i] = v[8 * d + i];
                else w[i] = __builtin_amdgcn_perm(v[8 * d + 2 * i + 1], v[8 * d + 2 * i], kPick[j]);
            }
            out[d] = encode8<DT>(w, s);
        }
        unsigned four = s << 8 * group;   // the scales of a column's four blocks
        four |= lane_xor1(four);
        four |= lane_xor2(four);
        if (c + j < columns) {
            *reinterpret_cast<u32x4*>(qt + ((c + j) * units_t + unit_r) * kMx4UnitBytes + 16 * group) = out;
            if (group == 0) *reinterpret_cast<unsigned*>(scales_t + ((c + j) * units_t + unit_r) * kMx4UnitScales) = four;
        }
    }
}

// 16 bytes of values a lane (8 elements, fp32: 4), RUNS of them, whose codes and scales are loaded before any is used.
// Whole lines are stored nontemporal where the values take half of the 256 MB Infinity Cache or more, which keeps little
// of them for who reads them next. bf16, us over three to six outputs in turn (over nine and more), and with a product of
// 1, 64 and 1024 rows behind it:
//    32 MiB ( 4096 x  4096)   8.0 ->  6.5 ( 9.9 ->  7.7), 22.4 -> 23.1, 22.7 -> 23.2, 48.5 -> 51.0
//   112 MiB (14336 x  4096)  28.6 -> 22.4 (28.6 -> 26.7), 51.7 -> 54.5, 55.5 -> 53.8, 116.5 -> 121.4
//   112 MiB ( 4096 x 14336)  28.6 -> 22.3 (28.6 -> 26.6), 51.0 -> 51.7, 65.5 -> 66.2, 160.8 -> 156.4
//   128 MiB ( 8192 x  8192)  31.8 -> 25.3 (31.8 -> 30.1), 62.5 -> 58.7, 67.0 -> 62.3, 146.5 -> 145.2
//   160 MiB (10240 x  8192)  38.5 -> 33.4 (38.5 -> 36.7), 71.7 -> 70.6, 85.4 -> 77.8, 174.2 -> 175.3
//   448 MiB (28672 x  8192)  99.9 -> 97.4 (99.9 -> 97.5), 222.2 -> 204.4, 214.4 -> 191.2, 472.4 -> 489.3
// Alone it always gains; with a reader behind it from 128 MiB on, at 112 as often as not.
template <int DT, int RUNS>
__global__ void __launch_bounds__(256)
mx4_dequantize_kernel(const unsigned char* __restrict__ q, const unsigned char* __restrict__ scales, int64_t rows,
                      int64_t columns, int64_t units, typename Source<DT>::Element* __restrict__ out, int64_t ldo,
                      bool nontemporal) {
    constexpr bool WIDE = DT == MB_DT_FLOAT32;
    constexpr int EACH = WIDE ? 4 : 8, LANES = kMx4Unit / EACH;   // elements per lane, lanes per unit
    const int64_t first = (int64_t)block_number() * (256 * RUNS) + threadIdx.x, total = rows * units * LANES;
    unsigned codes[RUNS], bytes[RUNS];
#pragma unroll
    for (int k = 0; k < RUNS; ++k) {
        const int64_t i = min(first + 256 * k, total - 1);
        codes[k] = WIDE ? reinterpret_cast<const uint16_t*>(q)[i] : reinterpret_cast<const unsigned*>(q)[i];
        bytes[k] = scales[i / (LANES / 4)];
    }
#pragma unroll
    for (int k = 0; k < RUNS; ++k) {
        const int64_t i = first + 256 * k;
        if (i >= total) return;
        const int64_t unit = i / LANES, row = unit / units;
        const int64_t column = (unit - row * units) * kMx4Unit + EACH * (i % LANES);
        if (column >= columns) continue;
        const float scale = __builtin_bit_cast(float, bytes[k] << 23);
        u32x4 v;
        auto two = [&](auto sel) {
            constexpr int s = decltype(sel)::value;
            if constexpr (WIDE) {
                if constexpr (s < 2) {
                    const auto f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[k], scale, s);
                    v[2 * s] = __builtin_bit_cast(unsigned, (float)f[0]);
                    v[2 * s + 1] = __builtin_bit_cast(unsigned, (float)f[1]);
                }
            } else if constexpr (DT == MB_DT_BFLOAT16) {
                v[s] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[k], scale, s));
            } else {
                v[s] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes[k], scale, s));
            }
        };
        two(std::integral_constant<int, 0>{});
        two(std::integral_constant<int, 1>{});
        two(std::integral_constant<int, 2>{});
        two(std::integral_constant<int, 3>{});
        auto* p = out + row * ldo + column;
        if (column + EACH <= columns) {
            if (nontemporal) __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p));
            else *reinterpret_cast<u32x4_2*>(p) = v;
            continue;
        }
#pragma unroll
        for (int e = 0; e < EACH - 1; ++e)
            if (column + e < columns) {
                if constexpr (WIDE) p[e] = v[e];
                else p[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
            }
    }
}

// Units a lane group takes: several in flight, while that leaves a block for every CU.
constexpr int64_t kManyUnits = 4 * 16 * 256;
constexpr int64_t kStreamedBytes = 128ll << 20;   // of values

template <int DT>
int quantize(const Mx4Quantize& c, hipStream_t stream) {
    const int64_t units = mx4_units(c.columns);
    auto* q = static_cast<unsigned char*>(c.q);
    auto* scales = static_cast<unsigned char*>(c.scales);
    if (c.qt == nullptr) {
        const int64_t total = c.rows * units;
        auto launch = [&](auto many) {
            constexpr int N = decltype(many)::value;
            hipLaunchKernelGGL((mx4_quantize_rows_kernel<DT, N>), launch_grid((total + 16 * N - 1) / (16 * N)),
                               dim3(256), 0, stream, c.x, c.ldx, c.rows, c.columns, units, c.fit,
                               reinterpret_cast<unsigned*>(q), scales);
        };
        if (total >= kManyUnits) launch(std::integral_constant<int, 4>{});
        else launch(std::integral_constant<int, 1>{});
    } else {
        const int64_t tiles_n = DT == MB_DT_FLOAT32 ? 2 * units : units;   // whole units
        const int64_t squares = ((mx4_units(c.rows) + 1) / 2) * ((units + 1) / 2);
        const int64_t blocks = (squares + 7) / 8 * 8 * (DT == MB_DT_FLOAT32 ? 8 : 4);
        auto kernel = q != nullptr ? mx4_quantize_tile_kernel<DT, true> : mx4_quantize_tile_kernel<DT, false>;
        hipLaunchKernelGGL(kernel, launch_grid(blocks), dim3(256), 0, stream, c.x, c.ldx, c.rows, c.columns, c.fit,
                           tiles_n, q, scales, static_cast<unsigned char*>(c.qt),
                           static_cast<unsigned char*>(c.scales_t));
    }
    MB_HIP_TRY(hipGetLastError());
    return MB_OK;
}

template <int DT>
int dequantize(const void* q, const void* scales, int64_t rows, int64_t columns, void* out, int64_t ldo,
               hipStream_t stream) {
    typedef typename Source<DT>::Element Element;
    const int64_t units = mx4_units(columns), total = rows * units;
    const int64_t lanes = total * (DT == MB_DT_FLOAT32 ? 32 : 16);
    const bool lines = ((reinterpret_cast<uintptr_t>(out) | (uintptr_t)(ldo * sizeof(Element))) & 127) == 0;
    const bool nontemporal = lines && rows * columns * (int64_t)sizeof(Element) >= kStreamedBytes;
    auto launch = [&](auto many) {
        constexpr int N = decltype(many)::value;
        hipLaunchKernelGGL((mx4_dequantize_kernel<DT, N>), launch_grid((lanes + 256 * N - 1) / (256 * N)), dim3(256), 0,
                           stream, static_cast<const unsigned char*>(q), static_cast<const unsigned char*>(scales), rows,
                           columns, units, static_cast<Element*>(out), ldo, nontemporal);
    };
    if (total >= kManyUnits) launch(std::integral_constant<int, 4>{});
    else launch(std::integral_constant<int, 1>{});
    MB_HIP_TRY(hipGetLastError());
    return MB_OK;
}

}  // namespace

int mx4_quantize_launch(const Mx4Quantize& c, hipStream_t stream) {
    if (c.dtype == MB_DT_FLOAT32) return quantize<MB_DT_FLOAT32>(c, stream);
    if (c.dtype == MB_DT_BFLOAT16) return quantize<MB_DT_BFLOAT16>(c, stream);
    return quantize<MB_DT_FLOAT16>(c, stream);
}

int mx4_dequantize_launch(int dtype, const void* q, const void* scales, int64_t rows, int64_t columns, void* out,
                          int64_t ldo, hipStream_t stream) {
    if (dtype == MB_DT_FLOAT32) return dequantize<MB_DT_FLOAT32>(q, scales, rows, columns, out, ldo, stream);
    if (dtype == MB_DT_BFLOAT16) return dequantize<MB_DT_BFLOAT16>(q, scales, rows, columns, out, ldo, stream);
    return dequantize<MB_DT_FLOAT16>(q, scales, rows, columns, out, ldo, stream);
}

}  // namespace mb

// Products with 4-bit weights: out[p][n] = sum over k of x[p][k] s (q - z), one
// scale s and zero point z per column n and group of k.
//
// For few rows the weights' bytes bound this (K N / 2 and their scales), so
// they go from HBM into registers once, 16 bytes a lane, and straight to the
// matrix cores (v_mfma_f32_16x16x32: 16 rows x 16 columns x 32 k).
//
// Integers to 16-bit floats. A dword holds k .. k + 7 of one column. (w >> 4i)
// & 0x000F000F leaves nibbles i and i + 4 in its halves; with the exponent of
// 128 (bf16) or 1024 (fp16) ORed in, each half is the float 128 + q or 1024 + q.
// That puts k in the order 0 4 1 5 2 6 3 7, which x's operand takes too (four
// byte permutes). bf16 multiplies 128 + q and an MFMA against ones gives the
// group's sum of x, so group by group, in fp32,
//   out += s * (sum x (128 + q)) - s (128 + z) * (sum x);
// the offset costs 5 of fp32's 24 bits beside a bf16 result's 8. fp16, which keeps 11, subtracts 1032
// first (exact), and needs the sum of x only for z - 8.
//
// Lanes. Lane l reads column l % 16; its 16 bytes are k 32 (l / 16) .. + 31 of a
// chunk of 128, so a column's reads are 64 contiguous bytes. The MFMA wants k
// 8 (l / 16) .. + 7 of 32 consecutive ones, so that one MFMA never mixes two
// groups: a 4 x 4 transpose between the four 16-lane groups, four
// lane-swap instructions per 16 bytes.
//
// Waves of a block split K in units of 256 (whole 128-byte lines of a column)
// and add their fp32 sums through LDS, in wave order. Rows that are not there
// multiply some other row's x and are stored as zeros; units that run past K
// take zeros for x and whatever weights lie there in bounds.
#include "experts_common.hpp"

#include <algorithm>
#include <type_traits>

namespace mb {
namespace {

typedef u32x4 u32x4_byte __attribute__((aligned(1)));   // 16 bytes at any address
constexpr int kUnit = 256;   // k per step of a wave

template <int DT>
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, f32x4 c) {
    if constexpr (DT == MB_DT_FLOAT16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                       0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                        0, 0, 0);
}

// Dword j of 16-lane group g <-> dword g of group j.
__device__ __forceinline__ u32x4 transpose_groups(u32x4 v) {
    const auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
    const auto lo = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

// 8 weights of a dword as floats, in k order 0 4 1 5 2 6 3 7: 128 + q (bf16), q - 8 (fp16).
template <int DT>
__device__ __forceinline__ u32x4 widen(unsigned w) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned pair = (w >> (4 * i)) & 0x000F000Fu;
        if constexpr (DT == MB_DT_FLOAT16) {
            typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
            const f16x2 f = __builtin_bit_cast(f16x2, pair | 0x64006400u) - (f16x2){(_Float16)1032.f, (_Float16)1032.f};
            v[i] = __builtin_bit_cast(unsigned, f);
        } else {
            v[i] = pair | 0x43004300u;
        }
    }
    return v;
}

// 8 consecutive k of x into the same order.
__device__ __forceinline__ u32x4 reorder(const u32x4& v) {
    return u32x4{__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
                 __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
}

// SPU: scales per unit and column when groups divide a unit evenly (256 / group), or 1 for groups of
// whole units; 0 for any other group: one scale looked up per 32 k.
template <int DT, bool ZEROS, int RT, int CT, int SPU, int W>
__global__ void __launch_bounds__(64 * W)
gemm_w4_kernel(const uint16_t* __restrict__ x, int64_t ldx, int64_t x_rows, const int32_t* __restrict__ rows,
               const uint8_t* __restrict__ q, const uint16_t* __restrict__ scales, const uint16_t* __restrict__ zeros,
               int group, uint16_t* __restrict__ out, int64_t ldo, const int32_t* __restrict__ offsets, int experts,
               int total, int N, int K, int blocks_n) {
    constexpr bool SUMS = DT == MB_DT_BFLOAT16 || ZEROS;     // the group's sum of x is needed
    constexpr int STEPS = kUnit / 32;                         // MFMA steps of 32 k per unit
    constexpr int PER = SPU > 0 ? STEPS / SPU : 1;            // steps per scale
    constexpr int NS = STEPS / PER;
    constexpr float kOffset = DT == MB_DT_BFLOAT16 ? 128.f : -8.f;   // the float of q is q + kOffset
    __shared__ f32x4 red[W][RT * CT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int tile = (int)blockIdx.x / blocks_n;
    const int n0 = ((int)blockIdx.x - tile * blocks_n) * 16 * CT;
    ExpertRows ex{0, 0, total};
    int in_expert = tile;
    if (offsets != nullptr && !find_row_tile(offsets, experts, total, tile, 16 * RT, &ex, &in_expert)) return;
    const int p0 = ex.first + in_expert * 16 * RT, count = min(16 * RT, ex.count - in_expert * 16 * RT);
    const int bytes = (K + 1) / 2, groups = (K + group - 1) / group;

    // Columns past N read the last one's weights and are not stored.
    const uint8_t* qp[CT];
    int64_t sp[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const int64_t column = (int64_t)ex.expert * N + min(n0 + 16 * t + c, N - 1);
        qp[t] = q + column * bytes;
        sp[t] = column * groups;
    }
    const uint16_t* xp[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int r = min(16 * t + c, count - 1);
        const int64_t row = rows ? rows[p0 + r] : p0 + r;
        xp[t] = x + (row >= 0 && row < x_rows ? row : 0) * ldx;
    }

    auto load_q = [&](int k0, u32x4 (&v)[CT][2]) {
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = k0 / 2 + 64 * h + 16 * g;
                if (at + 16 <= bytes) {
                    v[t][h] = *reinterpret_cast<const u32x4_byte*>(qp[t] + at);
                } else {
                    u32x4 p = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int b = 0; b < 15; ++b)
                        if (at + b < bytes) p[b >> 2] |= (unsigned)qp[t][at + b] << (8 * (b & 3));
                    v[t][h] = p;
                }
            }
    };
    auto load_x = [&](int t, int k, auto whole) -> u32x4 {   // k .. k + 7 of row tile t's row
        if (decltype(whole)::value || k + 8 <= K) return *reinterpret_cast<const u32x4_any*>(xp[t] + k);
        u32x4 p = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < K) p[e >> 1] |= (unsigned)xp[t][k + e] << (16 * (e & 1));
        return p;
    };
    // Scale (zero point) number i of a unit and column tile t.
    auto load_scales = [&](const uint16_t* from, int t, int k0, auto whole, uint16_t (&v)[NS]) {
        if constexpr (SPU > 1) {
            if (decltype(whole)::value) {
                typedef uint16_t vec __attribute__((ext_vector_type(SPU)));
                typedef vec vec_any __attribute__((aligned(2)));
                const vec s = *reinterpret_cast<const vec_any*>(from + sp[t] + k0 / kUnit * SPU);
#pragma unroll
                for (int i = 0; i < NS; ++i) v[i] = s[i];
                return;
            }
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) v[i] = from[sp[t] + min((k0 + i * PER * 32) / group, groups - 1)];
    };

    f32x4 acc[RT][CT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const u32x4 ones = DT == MB_DT_FLOAT16 ? u32x4{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u}
                                           : u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};

    auto unit = [&](int k0, u32x4 (&w)[CT][2], auto whole) {
        uint16_t sv[CT][NS], zv[CT][NS];
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            load_scales(scales, t, k0, whole, sv[t]);
            if constexpr (ZEROS) load_scales(zeros, t, k0, whole, zv[t]);
        }
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) w[t][h] = transpose_groups(w[t][h]);
        f32x4 dot[RT][CT], sum[RT];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (s % PER == 0) {
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < CT; ++j) dot[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
            }
            u32x4 xv[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i) xv[i] = reorder(load_x(i, k0 + 32 * s + 8 * g, whole));
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                const u32x4 wv = widen<DT>(w[j][s >> 2][s & 3]);
#pragma unroll
                for (int i = 0; i < RT; ++i) dot[i][j] = mfma16<DT>(xv[i], wv, dot[i][j]);
            }
            if constexpr (SUMS) {
#pragma unroll
                for (int i = 0; i < RT; ++i) sum[i] = mfma16<DT>(xv[i], ones, sum[i]);
            }
            if (s % PER == PER - 1) {
#pragma unroll
                for (int j = 0; j < CT; ++j) {
                    const float sc = from_bits<DT>(sv[j][s / PER]);
                    const float z = ZEROS ? from_bits<DT>(zv[j][s / PER]) : 8.f;
                    const float off = -sc * (kOffset + z);
#pragma unroll
                    for (int i = 0; i < RT; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            acc[i][j][r] = fmaf(sc, dot[i][j][r], acc[i][j][r]);
                            if constexpr (SUMS) acc[i][j][r] = fmaf(off, sum[i][r], acc[i][j][r]);
                        }
                }
            }
        }
    };

    const int units = x_rows > 0 ? (K + kUnit - 1) / kUnit : 0;
    u32x4 w[CT][2];
    if (wave < units) load_q(wave * kUnit, w);
    for (int u = wave; u < units; u += W) {
        u32x4 next[CT][2];
        if (u + W < units) load_q((u + W) * kUnit, next);
        if ((u + 1) * kUnit <= K) unit(u * kUnit, w, std::true_type{});
        else unit(u * kUnit, w, std::false_type{});
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) w[t][h] = next[t][h];
    }

    // Register r of lane l holds row 4 (l / 16) + r, column l % 16.
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) red[wave][i * CT + j][lane] = acc[i][j];
    __syncthreads();
    for (int t = wave; t < RT * CT; t += W) {
        f32x4 v = red[0][t][lane];
#pragma unroll
        for (int u = 1; u < W; ++u) v += red[u][t][lane];
        const int n = n0 + 16 * (t % CT) + c;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int p = 16 * (t / CT) + 4 * g + r;
            if (p >= count || n >= N) continue;
            const int64_t row = rows ? rows[p0 + p] : p0 + p;
            out[(p0 + p) * ldo + n] = row >= 0 && row < x_rows ? to_bits<DT>(v[r]) : 0;
        }
    }
}

template <int DT, bool ZEROS, int RT, int CT, int SPU, int W>
int launch_w4(const W4Call& c, hipStream_t stream) {
    const int blocks_n = (int)((c.N + 16 * CT - 1) / (16 * CT));
    const int64_t tiles = c.offsets ? c.total_rows / (16 * RT) + std::min<int64_t>(c.experts, c.total_rows)
                                    : (c.total_rows + 16 * RT - 1) / (16 * RT);
    hipLaunchKernelGGL((gemm_w4_kernel<DT, ZEROS, RT, CT, SPU, W>), dim3((unsigned)(tiles * blocks_n)), dim3(64 * W), 0,
                       stream, static_cast<const uint16_t*>(c.x), c.ldx, c.x_rows, c.rows,
                       static_cast<const uint8_t*>(c.q), static_cast<const uint16_t*>(c.scales),
                       static_cast<const uint16_t*>(c.zeros), c.group, static_cast<uint16_t*>(c.out), c.ldo, c.offsets,
                       c.experts, (int)c.total_rows, (int)c.N, (int)c.K, blocks_n);
    MB_HIP_TRY(hipGetLastError());
    return MB_OK;
}

template <int DT, bool ZEROS, int RT, int CT, int W>
int launch_group(const W4Call& c, hipStream_t stream) {
    if (c.group == 32) return launch_w4<DT, ZEROS, RT, CT, 8, W>(c, stream);
    if (c.group == 64) return launch_w4<DT, ZEROS, RT, CT, 4, W>(c, stream);
    if (c.group == 128) return launch_w4<DT, ZEROS, RT, CT, 2, W>(c, stream);
    if (c.group % kUnit == 0) return launch_w4<DT, ZEROS, RT, CT, 1, W>(c, stream);
    return launch_w4<DT, ZEROS, RT, CT, 0, W>(c, stream);
}

template <int DT, bool ZEROS>
int launch_rows(const W4Call& c, hipStream_t stream) {
    // Rows of an expert, were they even: tiles of 16, 32 or 64 of them share one pass over the weights.
    const int64_t rows = (c.total_rows + c.experts - 1) / c.experts;
    if (rows <= 16) return launch_group<DT, ZEROS, 1, 2, 8>(c, stream);
    if (rows <= 32) return launch_group<DT, ZEROS, 2, 2, 8>(c, stream);
    return launch_group<DT, ZEROS, 4, 2, 4>(c, stream);
}

}  // namespace

int gemm_w4_launch(const W4Call& c, void* workspace, size_t workspace_bytes, const DeviceProps& props,
                   hipStream_t stream) {
    if (c.dtype == MB_DT_FLOAT16)
        return c.zeros ? launch_rows<MB_DT_FLOAT16, true>(c, stream) : launch_rows<MB_DT_FLOAT16, false>(c, stream);
    return c.zeros ? launch_rows<MB_DT_BFLOAT16, true>(c, stream) : launch_rows<MB_DT_BFLOAT16, false>(c, stream);
}

}  // namespace mb

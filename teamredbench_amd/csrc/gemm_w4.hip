// Products with 4-bit weights: out[p][n] = sum over k of x[p][k] s (q - z), one
// scale s and zero point z per column n and group of k.
//
// For few rows the weights' bytes bound this (K N / 2 and their scales), so
// they go from HBM into registers once, 16 bytes a lane, and straight to the
// matrix cores (v_mfma_f32_16x16x32: 16 rows x 16 columns x 32 k).
//
// Integers to 16-bit floats. A dword holds k .. k + 7 of one column. Shifted and
// masked, it leaves nibbles i and i + 4 in its halves; with an exponent ORed in,
// each half is a float: 1 + q / 16 (bf16: the nibble on bits 3 .. 6) or 1024 + q
// (fp16: on the lowest). That puts k in the order 0 4 1 5 2 6 3 7, which x's
// operand takes too (four byte permutes). bf16 multiplies 1 + q / 16 and an MFMA
// against ones gives the group's sum of x, so group by group, in fp32,
//   out / 16 += s * (sum x (1 + q / 16) - (1 + z / 16) * (sum x)).
// An offset of 16 q's is the least under which four bits fit bf16's seven (the nibble on
// the lowest bits makes it 128: one shift in eight instructions less, but a
// group's sums some 30 times the result, where these are 5). bf16's x may be as
// large as fp32's range: both operands against it carry 2^-9, so that no sum
// over a unit of 256 k leaves it, and the stores take 2^13 back. fp16
// subtracts 1032 first (exact), and needs the sum of x only for z - 8.
//
// Lanes. Lane l reads column l % 16; its 16 bytes are k 32 (l / 16) .. + 31 of a
// chunk of 128, so a column's reads are 64 contiguous bytes. The MFMA wants k
// 8 (l / 16) .. + 7 of 32 consecutive ones, so that one MFMA never mixes two
// groups: a 4 x 4 transpose between the four 16-lane groups, four
// lane-swap instructions per 16 bytes. (Few rows: lane l reads column l / 4, and
// a second transpose follows within each four lanes; see Columns.)
//
// Up to 16 rows per expert (gemm_w4_kernel): the waves of a block share 32
// columns and split K in units of 256; weights come one unit ahead, x straight
// from L2, and the waves add their fp32 sums through LDS, in wave order. L1
// bounds it: a 16-byte load takes it 16 cycles if each four lanes read 64
// contiguous bytes and 64 if a quarter wave's 16 lanes read as many lines. So
// weights come in the first way and a unit's scales by one load (16 x 8192 x
// 8192, groups of 32 with zero points: 18.8 -> 16.0 us; weights alone 8); x, in
// rows as the MFMA takes them, is what is left. 10.2 us at 1 x 14336 x 4096, of which
// the bytes are 5.9.
//
// More rows, or columns enough without (gemm_w4_rows_kernel): the waves split
// the block's columns and share x through LDS, 256 k at a time, with the sums of
// x made on the way in: 59 us (4.7 TB/s) for 256 rows over 64 experts, 4096 ->
// 2048, and 58.7 us at 64 x 50257 x 4096, where widening and scaling take 34 on
// the 197 CUs that have a block. Few columns: blocks split K too, into fp32 planes that a second kernel adds.
//
// Rows that are not there multiply some other row's x and are stored as zeros;
// units that run past K take zeros for x and whatever weights lie there in bounds.
#include "experts_common.hpp"
#include "gemm_w4_plan.hpp"

#include <algorithm>
#include <type_traits>

namespace mb {
namespace {

typedef u32x4 u32x4_byte __attribute__((aligned(1)));   // 16 bytes at any address
constexpr int kUnit = 256;   // k per step of a wave: whole 128-byte lines of a column

// How weights are held: a float h (q + kOffset), h = kStep times the operand that stands for 1 in the sums of x
// (kOnes, two of them). Sums are h times what they stand for, and the stores take kBack = 1 / h.
template <int DT>
struct Held {
    static constexpr float kOffset = 16.f, kStep = 1.f / 16, kBack = 8192.f;
    static constexpr unsigned kOnes = 0x3B003B00u;                                   // 2^-9
    static constexpr unsigned kMask = 0x00780078u, kExponent = 0x3B003B00u;          // 2^-9 (1 + q / 16)
};
template <>
struct Held<MB_DT_FLOAT16> {
    static constexpr float kOffset = -8.f, kStep = 1.f, kBack = 1.f;
    static constexpr unsigned kOnes = 0x3C003C00u;
    static constexpr unsigned kMask = 0x000F000Fu, kExponent = 0x64006400u;          // 1024 + q, less 1032
};

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

// Dword j of lane l <-> dword l % 4 of lane j, among each four lanes.
__device__ __forceinline__ u32x4 transpose_quads(u32x4 v) {
    const bool odd = __lane_id() & 1, high = __lane_id() & 2;
    auto lane1 = [](unsigned x) { return (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true); };   // l ^ 1
    auto lane2 = [](unsigned x) { return (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true); };   // l ^ 2
    const u32x4 from1{lane1(v[1]), lane1(v[0]), lane1(v[3]), lane1(v[2])};
    const u32x4 a{odd ? from1[0] : v[0], odd ? v[1] : from1[1], odd ? from1[2] : v[2], odd ? v[3] : from1[3]};
    const u32x4 from2{lane2(a[2]), lane2(a[3]), lane2(a[0]), lane2(a[1])};
    return u32x4{high ? from2[0] : a[0], high ? from2[1] : a[1], high ? a[2] : from2[2], high ? a[3] : from2[3]};
}

// 8 weights of a dword as floats (see Held), in k order 0 4 1 5 2 6 3 7. `mask` and `exponent` are Held's in
// registers the compiler cannot see through: it then ANDs and ORs in one instruction, where literals take two.
template <int DT>
__device__ __forceinline__ u32x4 widen(unsigned w, unsigned mask, unsigned exponent) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        constexpr int kLowest = DT == MB_DT_FLOAT16 ? 0 : 3;   // bit of the float that the nibble's lowest takes
        const unsigned nibbles = 4 * i < kLowest ? w << kLowest : w >> (4 * i - kLowest);
        const unsigned pair = (nibbles & mask) | exponent;
        if constexpr (DT == MB_DT_FLOAT16) {
            typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
            const f16x2 f = __builtin_bit_cast(f16x2, pair) - (f16x2){(_Float16)1032.f, (_Float16)1032.f};
            v[i] = __builtin_bit_cast(unsigned, f);
        } else {
            v[i] = pair;
        }
    }
    return v;
}

// 8 consecutive k of x into the same order.
__device__ __forceinline__ u32x4 reorder(const u32x4& v) {
    return u32x4{__builtin_amdgcn_perm(v[2], v[0], 0x05040100u), __builtin_amdgcn_perm(v[2], v[0], 0x07060302u),
                 __builtin_amdgcn_perm(v[3], v[1], 0x05040100u), __builtin_amdgcn_perm(v[3], v[1], 0x07060302u)};
}

// sum + the two 16-bit floats of a dword, each times the ones of Held, in fp32.
template <int DT>
__device__ __forceinline__ float add_pair(unsigned v, float sum) {
    if constexpr (DT == MB_DT_FLOAT16) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, v), __builtin_bit_cast(f16x2, Held<DT>::kOnes), sum,
                                      false);
    } else {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, v),
                                               __builtin_bit_cast(bf16x2, Held<DT>::kOnes), sum, false);
    }
}
template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}

// Bytes `at` .. + 15 of `bytes` bytes at p, zeros past their end: the last 16
// of them shifted down, since nothing past the end may be read.
__device__ __forceinline__ u32x4 window16(const uint8_t* p, int at, int bytes) {
    if (bytes >= 16) {
        const int from = min(at, bytes - 16), shift = at - from;
        const u32x4 v = *reinterpret_cast<const u32x4_byte*>(p + from);
        const __uint128_t wide = __builtin_bit_cast(__uint128_t, v);
        return shift < 16 ? __builtin_bit_cast(u32x4, wide >> (8 * shift)) : u32x4{0u, 0u, 0u, 0u};
    }
    __uint128_t wide = 0;
#pragma unroll 1
    for (int b = bytes - 1; b >= at; --b) wide = (wide << 8) | p[b];
    return __builtin_bit_cast(u32x4, wide);
}

// 8 consecutive elements of x's row from k on, zeros past K.
__device__ __forceinline__ u32x4 load_x(const uint16_t* row, int k, int K) {
    return window16(reinterpret_cast<const uint8_t*>(row), 2 * k, 2 * K);
}

// One operand pointer set of a block, and the loads every kernel here makes.
// Where a unit's scales are. SPU: scales per unit and column when groups divide a unit evenly (kUnit /
// group), or 1 for groups of whole units; 0 for any other group: one scale looked up per 32 k.
template <int DT, bool ZEROS, int SPU>
struct Groups {
    static constexpr int STEPS = kUnit / 32;                     // MFMA steps of 32 k per unit
    static constexpr int PER = SPU > 0 ? STEPS / SPU : 1;        // steps per scale
    static constexpr int NS = STEPS / PER;                       // scales per unit and column
    static constexpr bool SUMS = DT == MB_DT_BFLOAT16 || ZEROS;  // the group's sum of x is needed
    typedef uint16_t Scales __attribute__((ext_vector_type(NS)));

    int group, groups;
    // Number of the unit's first scale (SPU > 0).
    __device__ __forceinline__ int first(int k0) const { return SPU > 1 ? k0 / kUnit * SPU : k0 / group; }
    // A unit's scales of a column, one load on any element where the unit has them all.
    __device__ __forceinline__ Scales load(const uint16_t* from, int k0) const {
        Scales v;
        if constexpr (SPU > 1) {
            const int at = first(k0);
            if (at + NS <= groups) {   // uniform
                typedef Scales Any __attribute__((aligned(2)));
                v = *reinterpret_cast<const Any*>(from + at);
            } else {
#pragma unroll
                for (int i = 0; i < NS; ++i) v[i] = from[min(at + i, groups - 1)];
            }
        } else {
#pragma unroll
            for (int i = 0; i < NS; ++i) v[i] = from[min((k0 + i * 32) / group, groups - 1)];
        }
        return v;
    }
    // Scales 8 block .. + 7 of a column, zeros past its last; for any group, those of each 32 k of a unit.
    __device__ __forceinline__ u32x4 eight(const uint16_t* from, int k0) const {
        if constexpr (SPU > 0) {
            const int at = first(k0) & ~7;
            if (at + 8 <= groups) return *reinterpret_cast<const u32x4_any*>(from + at);
            return window16(reinterpret_cast<const uint8_t*>(from), 2 * at, 2 * groups);
        } else {
            return __builtin_bit_cast(u32x4, load(from, k0));
        }
    }
};

// The columns n0 + 16 t + c of an expert; those past N read the last one's weights and are not stored.
// QUADS: lane l reads 16-byte piece l % 4 of column l / 4's 64 bytes, which costs L1 a quarter of the time, and
// transpose_quads() after transpose_groups() leaves it the k of column_of(l). Where the vector unit bounds, not L1
// (gemm_w4_rows_kernel: 1 to 4% slower with it), piece l / 16 of column l % 16.
__device__ __forceinline__ int column_of(int lane) { return 4 * (lane & 3) + ((lane >> 2) & 3); }
template <int CT, bool QUADS>
struct Columns {
    static constexpr int CHUNKS = kUnit / 128;   // 16-byte loads per unit and column tile
    const uint8_t* qp[CT];
    int bytes, K, g;

    __device__ __forceinline__ Columns(const uint8_t* q, int expert, int n0, int N, int K_, int lane)
        : bytes((K_ + 1) / 2), K(K_), g(QUADS ? lane & 3 : lane >> 4) {
#pragma unroll
        for (int t = 0; t < CT; ++t)
            qp[t] = q + ((int64_t)expert * N + min(n0 + 16 * t + (QUADS ? lane >> 2 : lane & 15), N - 1)) * bytes;
    }
    __device__ __forceinline__ void load(int k0, u32x4 (&q)[CT][CHUNKS]) const {
        const bool whole = k0 + kUnit <= K;   // uniform
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int h = 0; h < CHUNKS; ++h) {
                const int at = k0 / 2 + 64 * h + 16 * g;
                q[t][h] = whole ? *reinterpret_cast<const u32x4_byte*>(qp[t] + at) : window16(qp[t], at, bytes);
            }
    }
};

// The mask and exponent of widen().
template <int DT>
struct Widen {
    unsigned mask = Held<DT>::kMask, exponent = Held<DT>::kExponent;
    __device__ __forceinline__ Widen() {
        asm("" : "+s"(mask));
        asm("" : "+v"(exponent));
    }
    __device__ __forceinline__ u32x4 operator()(unsigned w) const { return widen<DT>(w, mask, exponent); }
};

// Row of x of sorted row p; -1 for none.
__device__ __forceinline__ int64_t x_row(const int32_t* rows, int64_t x_rows, int p) {
    const int64_t r = rows ? rows[p] : p;
    return r < x_rows ? r : -1;
}

struct W4Args {
    const uint16_t* x;
    const int32_t *rows, *offsets;
    const uint8_t* q;
    const uint16_t *scales, *zeros;
    uint16_t* out;
    float* planes;       // K splits' partial sums, [split][total][ldp]; NULL without
    int64_t ldx, ldo, x_rows;
    int group, experts, total, N, K, blocks_n, splits, ldp;
};

// The tile of a block: its rows, first column and units of K. False if there is none.
struct W4Tile {
    int expert, p0, count, n0, split, first_unit, units, turn;

    // Unit number i of the block: neighbouring blocks start elsewhere in their columns (whose length is often a
    // power of two), or all would read the same few memory channels at a time.
    __device__ __forceinline__ int unit(int i) const {
        const int u = i + turn;
        return first_unit + (u < units ? u : u - units);
    }
};
__device__ __forceinline__ bool w4_tile(const W4Args& a, int rows_per_tile, int columns, W4Tile* t) {
    int b = (int)block_number();
    t->split = b % a.splits;
    b /= a.splits;
    const int tile = b / a.blocks_n;
    t->n0 = (b - tile * a.blocks_n) * columns;
    ExpertRows ex{0, 0, a.total};
    int in_expert = tile;
    if (a.offsets == nullptr ? tile > (a.total - 1) / rows_per_tile
                             : !find_row_tile(a.offsets, a.experts, a.total, tile, rows_per_tile, &ex, &in_expert))
        return false;
    t->expert = ex.expert;
    t->p0 = ex.first + in_expert * rows_per_tile;
    t->count = min(rows_per_tile, ex.count - in_expert * rows_per_tile);
    const int units = a.x_rows > 0 ? (a.K + kUnit - 1) / kUnit : 0;   // without any row of x there is nothing to add
    t->first_unit = (int)((int64_t)units * t->split / a.splits);
    t->units = (int)((int64_t)units * (t->split + 1) / a.splits) - t->first_unit;
    t->turn = t->units > 0 ? b % t->units : 0;
    return true;
}

// Rows 4 (l / 16) + r of row tile i, column 16 j + c: rounded to out, or in fp32 to the split's plane.
template <int DT>
__device__ __forceinline__ void w4_store(const W4Args& a, const W4Tile& t, int i, int j, int c, const f32x4& v,
                                         int lane) {
    const int n = t.n0 + 16 * j + c;
    if (n >= a.N) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int p = 16 * i + 4 * (lane >> 4) + r;
        if (p >= t.count) continue;
        const float sum = x_row(a.rows, a.x_rows, t.p0 + p) >= 0 ? v[r] * Held<DT>::kBack : 0.f;
        if (a.planes != nullptr)
            a.planes[((int64_t)t.split * a.total + t.p0 + p) * a.ldp + n] = sum;
        else
            a.out[(t.p0 + p) * a.ldo + n] = to_bits<DT>(sum);
    }
}

template <int DT, bool ZEROS, int CT, int SPU, int WAVES>
__global__ void __launch_bounds__(64 * WAVES)
gemm_w4_kernel(W4Args a) {
    typedef Groups<DT, ZEROS, SPU> G;
    typedef Columns<CT, true> Cols;
    __shared__ f32x4 red[WAVES][CT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    W4Tile tile;
    if (!w4_tile(a, 16, 16 * CT, &tile)) return;
    const Cols columns(a.q, tile.expert, tile.n0, a.N, a.K, lane);
    const G groups{a.group, (a.K + a.group - 1) / a.group};
    const Widen<DT> widened;
    // Scales: lane group 0 brings those of column tile 0, group 1 of tile 1, groups 2 and 3 the zero points.
    const int held = lane >> 4;
    const uint16_t* sp = (ZEROS && held >= 2 ? a.zeros : a.scales) +
                         ((int64_t)tile.expert * a.N +
                          min(tile.n0 + 16 * (CT == 1 ? 0 : held & 1) + column_of(lane), a.N - 1)) * groups.groups;
    const int64_t row = x_row(a.rows, a.x_rows, tile.p0 + min(lane & 15, tile.count - 1));
    const uint16_t* xp = a.x + max(row, (int64_t)0) * a.ldx;
    const u32x4 ones{Held<DT>::kOnes, Held<DT>::kOnes, Held<DT>::kOnes, Held<DT>::kOnes};
    struct Unit {
        u32x4 q[CT][Cols::CHUNKS];
        typename G::Scales s;
    };
    auto load = [&](int k0, Unit& u) {
        columns.load(k0, u.q);
        u.s = groups.load(sp, k0);
    };
    f32x4 acc[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto compute = [&](Unit& w, const u32x4 (&xv)[G::STEPS]) {
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int h = 0; h < Cols::CHUNKS; ++h) w.q[t][h] = transpose_quads(transpose_groups(w.q[t][h]));
        u32x4 held_by[(G::NS + 1) / 2];   // two scales of each lane group, in every lane
#pragma unroll
        for (int i = 0; i < (G::NS + 1) / 2; ++i) {
            const unsigned pair = w.s[2 * i] | (unsigned)w.s[G::NS > 1 ? 2 * i + 1 : 0] << 16;
            held_by[i] = transpose_groups(u32x4{pair, pair, pair, pair});
        }
        f32x4 dot[CT], sum;
#pragma unroll
        for (int s = 0; s < G::STEPS; ++s) {
            if (s % G::PER == 0) {
                sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int t = 0; t < CT; ++t) dot[t] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            const u32x4 x = reorder(xv[s]);
#pragma unroll
            for (int t = 0; t < CT; ++t) dot[t] = mfma16<DT>(x, widened(w.q[t][s >> 2][s & 3]), dot[t]);
            if constexpr (G::SUMS) sum = mfma16<DT>(x, ones, sum);
            if (s % G::PER == G::PER - 1) {
#pragma unroll
                for (int t = 0; t < CT; ++t) {
                    const int n = s / G::PER;
                    auto of = [&](int group) { return from_bits<DT>((uint16_t)(held_by[n / 2][group] >> (n % 2 * 16))); };
                    const float scale = of(t);
                    const float off = -Held<DT>::kStep * (Held<DT>::kOffset + (ZEROS ? of(2 + t) : 8.f));
#pragma unroll
                    for (int r = 0; r < 4; ++r)   // the offset comes off the group's sum before its scale
                        acc[t][r] = fmaf(scale, G::SUMS ? fmaf(off, sum[r], dot[t][r]) : dot[t][r], acc[t][r]);
                }
            }
        }
    };
    // A unit's weights go out before the one ahead of it is computed.
    Unit now, next;
    if (wave < tile.units) load(tile.unit(wave) * kUnit, next);
#pragma unroll 1
    for (int u = wave; u < tile.units; u += WAVES) {
        const int k0 = tile.unit(u) * kUnit, k = k0 + 8 * (lane >> 4);
        u32x4 xv[G::STEPS];
        now = next;
        if (k0 + kUnit <= a.K) {
#pragma unroll
            for (int s = 0; s < G::STEPS; ++s) xv[s] = *reinterpret_cast<const u32x4_any*>(xp + k + 32 * s);
        } else {
#pragma unroll
            for (int s = 0; s < G::STEPS; ++s) xv[s] = load_x(xp, k + 32 * s, a.K);
        }
        if (u + WAVES < tile.units) load(tile.unit(u + WAVES) * kUnit, next);
        compute(now, xv);
    }
#pragma unroll
    for (int t = 0; t < CT; ++t) red[wave][t][lane] = acc[t];
    __syncthreads();
    if (wave < CT) {
        f32x4 v = red[0][wave][lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v += red[w][wave][lane];
        w4_store<DT>(a, tile, 0, wave, column_of(lane), v, lane);
    }
}

// 16 RT rows; WAVES waves of CT x 16 columns each. The scales (zero points) of
// the block's columns go through LDS too, 8 of a column at a time, which last 8 / NS
// units: taken by each wave unit by unit, a few bytes of every column's line each time, they cost 15 of 74 us at
// 64 x 50257 x 4096 and 23 of 76 us at 64 experts of 2048 x 4096. The terms in
// the sums of x are one fp32 MFMA per tile and 4 groups: rows x groups times groups x columns.
template <int DT, bool ZEROS, int RT, int CT, int SPU, int WAVES>
__global__ void __launch_bounds__(64 * WAVES)
gemm_w4_rows_kernel(W4Args a) {
    typedef Groups<DT, ZEROS, SPU> G;
    typedef Columns<CT, false> Cols;
    constexpr int ROWS = 16 * RT, COLUMNS = 16 * CT * WAVES;
    constexpr int PITCH = kUnit * 2 + 16;             // bytes per row: 16 rows' 16-byte reads hit all banks once
    constexpr int PIECES = kUnit / 8;                 // 16-byte pieces per row and unit
    constexpr int STRIDE = 64 * WAVES / PIECES;       // rows staged at once
    constexpr int LOADS = ROWS / STRIDE;
    constexpr int QUADS = (G::NS + 3) / 4;            // fours of groups
    static_assert(ROWS % STRIDE == 0, "rows must split over the threads");
    static_assert(2 * COLUMNS <= 64 * WAVES, "one thread per column's scales, one per its zero points");
    __shared__ __attribute__((aligned(16))) unsigned char xs[2][ROWS * PITCH];
    __shared__ __attribute__((aligned(16))) float sums[2][4 * QUADS][ROWS];   // groups past NS stay zero
    __shared__ __attribute__((aligned(16))) uint16_t scales[2][ZEROS ? 2 : 1][COLUMNS][8];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    W4Tile tile;
    if (!w4_tile(a, ROWS, COLUMNS, &tile)) return;
    const int block_n0 = tile.n0;
    tile.n0 += 16 * CT * wave;
    const Cols columns(a.q, tile.expert, tile.n0, a.N, a.K, lane);
    const G groups{a.group, (a.K + a.group - 1) / a.group};
    const Widen<DT> widened;

    // Staging of x: thread t brings piece t % PIECES of rows t / PIECES + STRIDE i.
    const int piece = tid % PIECES, first_row = tid / PIECES;
    const uint16_t* xp[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int64_t row = x_row(a.rows, a.x_rows, tile.p0 + min(first_row + STRIDE * i, tile.count - 1));
        xp[i] = a.x + max(row, (int64_t)0) * a.ldx;
    }
    auto fetch = [&](int k0, u32x4 (&v)[LOADS]) {
        const int k = k0 + 8 * piece;
        const bool whole = k0 + kUnit <= a.K;   // uniform
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            v[i] = whole ? *reinterpret_cast<const u32x4_any*>(xp[i] + k) : load_x(xp[i], k, a.K);
    };
    auto stage = [&](int slot, const u32x4 (&v)[LOADS]) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int row = first_row + STRIDE * i;
            *reinterpret_cast<u32x4*>(xs[slot] + row * PITCH + 16 * piece) = reorder(v[i]);
            if constexpr (G::SUMS) {
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) sum = add_pair<DT>(v[i][e], sum);
                // A group's 4 PER pieces lie in neighbouring lanes: rotations within them add up in each.
                sum += dpp_move<0xB1>(sum);                               // quad_perm 1 0 3 2
                sum += dpp_move<0x4E>(sum);                               // quad_perm 2 3 0 1
                if constexpr (G::PER >= 2) sum += dpp_move<0x141>(sum);   // row_half_mirror
                if constexpr (G::PER >= 4) sum += dpp_move<0x140>(sum);   // row_mirror
                if constexpr (G::PER >= 8) sum += __shfl_xor(sum, 16);
                if (piece % (4 * G::PER) == 0) sums[slot][piece / (4 * G::PER)][row] = sum;
            }
        }
    };
    // Scales: thread t those of column t, thread COLUMNS + t its zero points.
    const int of = tid / COLUMNS, column = tid % COLUMNS;
    const bool brings = of < (ZEROS ? 2 : 1);
    const uint16_t* scale_row = (of == 1 && ZEROS ? a.zeros : a.scales) +
                                ((int64_t)tile.expert * a.N + min(block_n0 + column, a.N - 1)) * groups.groups;

    f32x4 acc[RT][CT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // x in `slot`; the unit's scales from `at` on in `held`.
    auto compute = [&](int slot, int held, int at, u32x4 (&q)[CT][Cols::CHUNKS]) {
        typename G::Scales s[CT];
#pragma unroll
        for (int j = 0; j < CT; ++j)
            s[j] = *reinterpret_cast<const typename G::Scales*>(&scales[held][0][16 * (CT * wave + j) + c][at]);
        // The offset's terms of groups 4 m .. + 3.
        auto offsets = [&](int m) {
            float off[CT];
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                const int col = 16 * (CT * wave + j) + c, n = min(at + 4 * m + g, 7);
                const float z = ZEROS ? from_bits<DT>(scales[held][ZEROS][col][n]) : 8.f;
                off[j] = 4 * m + g < G::NS ? -from_bits<DT>(scales[held][0][col][n]) *
                                                 (Held<DT>::kStep * (Held<DT>::kOffset + z))
                                           : 0.f;
            }
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const float sum = sums[slot][4 * m + g][16 * i + c];
#pragma unroll
                for (int j = 0; j < CT; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(sum, off[j], acc[i][j], 0, 0, 0);
            }
        };
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int h = 0; h < Cols::CHUNKS; ++h) q[t][h] = transpose_groups(q[t][h]);
        f32x4 dot[RT][CT];
#pragma unroll
        for (int st = 0; st < G::STEPS; ++st) {
            // Just before the groups that take them off again: acc stays near the result.
            if (G::SUMS && st % (4 * G::PER) == 0) offsets(st / (4 * G::PER));
            if (st % G::PER == 0) {
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int j = 0; j < CT; ++j) dot[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            u32x4 x[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i)
                x[i] = *reinterpret_cast<const u32x4*>(xs[slot] + (16 * i + c) * PITCH + 64 * st + 16 * g);
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                const u32x4 wv = widened(q[j][st >> 2][st & 3]);
#pragma unroll
                for (int i = 0; i < RT; ++i) dot[i][j] = mfma16<DT>(x[i], wv, dot[i][j]);
            }
            if (st % G::PER == G::PER - 1) {
#pragma unroll
                for (int j = 0; j < CT; ++j) {
                    const float scale = from_bits<DT>(s[j][st / G::PER]);
#pragma unroll
                    for (int i = 0; i < RT; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(scale, dot[i][j][r], acc[i][j][r]);
                }
            }
        }
    };

    if constexpr (G::SUMS && G::NS % 4 != 0) {
        for (int i = tid; i < 2 * 4 * QUADS * ROWS; i += 64 * WAVES) (&sums[0][0][0])[i] = 0.f;
        __syncthreads();
    }
    // Round u loads unit u and computes unit u - 1; one barrier a round. x of unit u (and scales, when it starts
    // another eight) go into the slots that every wave left before this round's barrier.
    u32x4 now[CT][Cols::CHUNKS], next[CT][Cols::CHUNKS];
    u32x4 xv[LOADS], eight;
    int held = 0, block = -1, at = 0;   // of unit u - 1: slot of its scales, which eight, its first among them
#pragma unroll 1
    for (int u = 0; u <= tile.units; ++u) {
        __syncthreads();
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int h = 0; h < Cols::CHUNKS; ++h) now[t][h] = next[t][h];
        bool fresh = false;
        int next_block = 0, next_at = 0;
        if (u < tile.units) {
            const int k0 = tile.unit(u) * kUnit;
            if constexpr (SPU > 0) {
                next_block = groups.first(k0) >> 3;
                next_at = groups.first(k0) & 7;
                fresh = next_block != block;
            } else {
                fresh = true;
            }
            fetch(k0, xv);
            if (fresh && brings) eight = groups.eight(scale_row, k0);
            columns.load(k0, next);
        }
        if (u > 0) compute((u - 1) & 1, held, at, now);
        if (u < tile.units) {
            stage(u & 1, xv);
            if (fresh) {
                held ^= 1;
                if (brings) *reinterpret_cast<u32x4*>(scales[held][of][column]) = eight;
            }
            block = next_block;
            at = next_at;
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) w4_store<DT>(a, tile, i, j, c, acc[i][j], lane);
}

// out = the sum of the K splits' planes, in split order, for the rows of any expert.
template <int DT>
__global__ void __launch_bounds__(256)
gemm_w4_sum_kernel(W4Args a) {
    const int quads = a.ldp / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t p = i / quads;
    if (p >= a.total) return;
    if (a.offsets != nullptr && (p < a.offsets[0] || p >= a.offsets[a.experts])) return;
    const int n = 4 * (int)(i - p * quads);
    const float* from = a.planes + p * a.ldp + n;
    f32x4 v = *reinterpret_cast<const f32x4*>(from);
    for (int s = 1; s < a.splits; ++s) v += *reinterpret_cast<const f32x4*>(from + (int64_t)s * a.total * a.ldp);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n + e < a.N) a.out[p * a.ldo + n + e] = to_bits<DT>(v[e]);
}

// K splits: as many as give every CU one of the `blocks`, keep `least` units
// of K in each, and fit the workspace. Two blocks a CU cost more than they gave (16 x 8192 x
// 8192: 25 against 19 us: the planes and their sum).
int w4_splits(const W4Call& c, int64_t blocks, int least, size_t workspace_bytes, const DeviceProps& props) {
    const int64_t units = (c.K + kUnit - 1) / kUnit;
    const int64_t plane = c.total_rows * ((c.N + 3) / 4 * 4) * (int64_t)sizeof(float);
    int64_t splits = std::min<int64_t>(props.cu_count / blocks, units / least);
    splits = std::min(splits, (int64_t)(workspace_bytes / plane));
    return (int)std::max<int64_t>(1, splits);
}

// RT 0: gemm_w4_kernel (up to 16 rows, K split over the waves); else row tiles of 16 RT.
template <int DT, bool ZEROS, int RT, int CT, int WAVES, int SPU>
int launch_w4(const W4Call& c, void* workspace, size_t workspace_bytes, const DeviceProps& props, hipStream_t stream) {
    constexpr int COLUMNS = RT == 0 ? 16 * CT : 16 * CT * WAVES, ROWS = RT == 0 ? 16 : 16 * RT;
    const int blocks_n = (int)((c.N + COLUMNS - 1) / COLUMNS);
    const int64_t tiles = c.offsets ? c.total_rows / ROWS + std::min<int64_t>(c.experts, c.total_rows)
                                    : (c.total_rows + ROWS - 1) / ROWS;
    const int splits = w4_splits(c, w4_likely_tiles(c.total_rows, c.experts, ROWS) * blocks_n, RT == 0 ? 2 * WAVES : 2, workspace_bytes, props);
    W4Args a{static_cast<const uint16_t*>(c.x), c.rows, c.offsets, static_cast<const uint8_t*>(c.q),
             static_cast<const uint16_t*>(c.scales), static_cast<const uint16_t*>(c.zeros),
             static_cast<uint16_t*>(c.out), splits > 1 ? static_cast<float*>(workspace) : nullptr, c.ldx, c.ldo,
             c.x_rows, c.group, c.experts, (int)c.total_rows, (int)c.N, (int)c.K, blocks_n, splits,
             (int)((c.N + 3) / 4 * 4)};
    const dim3 grid = launch_grid(tiles * blocks_n * splits);
    if constexpr (RT == 0)
        hipLaunchKernelGGL((gemm_w4_kernel<DT, ZEROS, CT, SPU, WAVES>), grid, dim3(64 * WAVES), 0, stream, a);
    else
        hipLaunchKernelGGL((gemm_w4_rows_kernel<DT, ZEROS, RT, CT, SPU, WAVES>), grid, dim3(64 * WAVES), 0,
                           stream, a);
    MB_HIP_TRY(hipGetLastError());
    if (splits > 1) {
        const int64_t quads = c.total_rows * (a.ldp / 4);
        hipLaunchKernelGGL((gemm_w4_sum_kernel<DT>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, stream, a);
        MB_HIP_TRY(hipGetLastError());
    }
    return MB_OK;
}

template <int DT, bool ZEROS, int RT, int CT, int WAVES>
int launch_group(const W4Call& c, void* workspace, size_t bytes, const DeviceProps& props, hipStream_t stream) {
    if (c.group == 32) return launch_w4<DT, ZEROS, RT, CT, WAVES, kUnit / 32>(c, workspace, bytes, props, stream);
    if (c.group == 64) return launch_w4<DT, ZEROS, RT, CT, WAVES, kUnit / 64>(c, workspace, bytes, props, stream);
    if (c.group == 128) return launch_w4<DT, ZEROS, RT, CT, WAVES, kUnit / 128>(c, workspace, bytes, props, stream);
    if (c.group % kUnit == 0) return launch_w4<DT, ZEROS, RT, CT, WAVES, 1>(c, workspace, bytes, props, stream);
    return launch_w4<DT, ZEROS, RT, CT, WAVES, 0>(c, workspace, bytes, props, stream);
}

template <int DT, bool ZEROS>
int launch_config(const W4Call& c, void* workspace, size_t bytes, const DeviceProps& props, hipStream_t stream) {
    const int64_t forced = tuning(MB_TUNE_W4_CONFIG);
    const int config = forced >= 0 ? (int)forced : w4_config(c.total_rows, c.experts, c.N, props.cu_count);
    int rc = MB_ERR_INVALID_ARG;   // every config below kW4ConfigCount is taken
    [&]<int... I>(std::integer_sequence<int, I...>) {
        ([&] {
            constexpr W4Config w = kW4Configs[I];
            if (config == I) rc = launch_group<DT, ZEROS, w.rt, w.ct, w.waves>(c, workspace, bytes, props, stream);
        }(), ...);
    }(std::make_integer_sequence<int, kW4ConfigCount>{});
    return rc;
}

}  // namespace

int gemm_w4_launch(const W4Call& c, void* workspace, size_t workspace_bytes, const DeviceProps& props,
                   hipStream_t stream) {
    // The workspace only makes small calls faster: one off 16 bytes is left alone.
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) workspace_bytes = 0;
    if (c.dtype == MB_DT_FLOAT16)
        return c.zeros ? launch_config<MB_DT_FLOAT16, true>(c, workspace, workspace_bytes, props, stream)
                       : launch_config<MB_DT_FLOAT16, false>(c, workspace, workspace_bytes, props, stream);
    return c.zeros ? launch_config<MB_DT_BFLOAT16, true>(c, workspace, workspace_bytes, props, stream)
                   : launch_config<MB_DT_BFLOAT16, false>(c, workspace, workspace_bytes, props, stream);
}

}  // namespace mb

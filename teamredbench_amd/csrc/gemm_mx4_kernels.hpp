// LDS-DMA pipelined products of MX4 matrices for gfx950: out(m, n) = sum over k of
// X(m, k) W(n, k), both operands in rows along k (layout: mx4_common.hpp), dense
// or by expert, on v_mfma_scale_f32_32x32x64_f8f6f4.
#pragma once

#include "gemm_grouped_kernels.hpp"
#include "mx4_common.hpp"

namespace mb {

struct Mx4Plan {
    int config;   // tiles of kMx4Tiles[config]; -1: gemm_mx4_any_kernel
    int splits;   // of K, over fp32 planes in the workspace
};
int gemm_mx4_tiled_bf16(const Mx4Call& c, const Mx4Plan& plan, void* workspace, hipStream_t stream);
int gemm_mx4_tiled_f16(const Mx4Call& c, const Mx4Plan& plan, void* workspace, hipStream_t stream);

constexpr int kMx4TileCount = 3;
constexpr int kMx4Tiles[kMx4TileCount] = {256, 128, 64};

namespace {

struct Mx4Args {
    const unsigned char *x, *xs, *w, *ws;
    unsigned char* out;
    const int32_t *rows, *offsets;
    int64_t ldo;                          // bytes per row
    int ld, lds, units;                   // bytes of elements and of scales per row of x and w
    int x_rows, experts, total, N;
    float* planes;                        // K splits: [split][total][ldp]
    int splits, split_units, ldp;
    bool out_16;                          // out's rows start on 16 bytes
};

// Ring slots: elements two slots of a pair of units (whole 128-byte lines of every row), scales two slots of 8
// units (32 bytes of every row).
constexpr int kPairBytes = 128, kChunkUnits = 8, kChunkBytes = 32;

// Loads of step j: pair (j - 1) / 2 + 2 of x and w on odd j, then scale chunk (j - 7) / 8 + 2 where j % 8 == 7,
// `pair` and `chunk` instructions per wave; the prologue runs the same rule over the steps before 0. Step j reads
// unit j + 1, so its wait leaves only the loads issued after that unit's. By j % 8, the least of all steps.
struct Mx4Waits {
    int step[kChunkUnits], prologue;
};
constexpr Mx4Waits mx4_schedule(int pair, int chunk) {
    constexpr int kSteps = 64, kFirst = -(kChunkUnits + 1);
    int pair_end[kSteps] = {}, chunk_end[kSteps] = {}, before[kSteps] = {};
    int total = 0;
    for (int v = kFirst; v < kSteps; ++v) {
        if (v >= 0) before[v] = total;
        if ((v & 1) != 0 && (v - 1) / 2 + 2 >= 0 && (v - 1) / 2 + 2 < kSteps) pair_end[(v - 1) / 2 + 2] = (total += pair);
        if ((v & 7) == 7) chunk_end[(v + 1) / kChunkUnits + 1] = (total += chunk);
    }
    Mx4Waits r{};
    r.prologue = before[0] - (pair_end[0] > chunk_end[0] ? pair_end[0] : chunk_end[0]);
    for (int i = 0; i < kChunkUnits; ++i) r.step[i] = 63;
    for (int j = 0; j + 1 < kSteps; ++j) {
        const int p = pair_end[(j + 1) / 2], c = chunk_end[(j + 1) / kChunkUnits];
        const int wait = before[j] - (p > c ? p : c);
        if (wait < r.step[j % kChunkUnits]) r.step[j % kChunkUnits] = wait;
    }
    return r;
}

template <int DT, int TILE>
__global__ void __launch_bounds__(256)
gemm_mx4_kernel(Mx4Args args, int tiles_n, int group_m) {
    constexpr int BM = TILE, BN = TILE;
    constexpr int WTM = BM / 2, WTN = BN / 2;
    constexpr int FM = WTM / 32, FN = WTN / 32;
    constexpr int SLOT = TILE * kPairBytes, SCALE_SLOT = TILE * kChunkBytes;   // one operand's
    constexpr int W0 = 2 * SLOT;                          // x's elements, w's, x's scales, w's: two slots each
    constexpr int XS0 = 4 * SLOT, WS0 = XS0 + 2 * SCALE_SLOT;
    constexpr int LDS_BYTES = WS0 + 2 * SCALE_SLOT;
    constexpr int INSTR = SLOT / 1024 / 4;                // DMA instructions per wave, operand and pair
    constexpr int SCALE_INSTR = 2 * SCALE_SLOT / 1024 / 4;   // ... per wave and chunk, both operands
    static_assert(LDS_BYTES <= 160 * 1024 && SLOT % 4096 == 0 && SCALE_INSTR >= 1, "LDS rings");
    constexpr Mx4Waits kWaits = mx4_schedule(2 * INSTR, SCALE_INSTR);
    static_assert([&] {
        for (int w : kWaits.step)
            if (w < 0) return false;
        return kWaits.prologue >= 0 && kWaits.prologue < 64;
    }(), "a needed unit is unissued, or vmcnt overflows");
    __shared__ __attribute__((aligned(1024))) unsigned char lds[LDS_BYTES];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int half = lane >> 5, r32 = lane & 31;

    ExpertRows ex{0, 0, args.total};
    const int block = (int)block_number();
    int tm, tn, split;
    const bool by_expert = args.offsets != nullptr;
    const int tiles_m = by_expert ? count_row_tiles(args.offsets, args.experts, args.total, BM)
                                  : (args.total + BM - 1) / BM;
    if (block >= tiles_m * tiles_n * args.splits) return;
    block_coords(block, tiles_m, tiles_n, args.splits, group_m, &tm, &tn, &split);
    if (by_expert && !find_row_tile(args.offsets, args.experts, args.total, tm, BM, &ex, &tm)) return;
    const int M = ex.count, m0 = tm * BM, n0 = tn * BN;
    // Units of K of this block, in whole pairs: the second unit of a last pair that has but one is zeros.
    const int u0 = split * args.split_units, k_units = min(args.units - u0, args.split_units);
    const int ksteps = (k_units + 1) & ~1, half_pair = k_units & 1 ? k_units / 2 : -1;

    // Buffer resources over the tile's rows (gathered: all of x): rows and units past them read as zeros.
    const bool gather = args.rows != nullptr;
    const int64_t x_first = gather ? 0 : (int64_t)ex.first + m0;
    const int64_t w_first = (int64_t)ex.expert * args.N + n0;
    const int x_count = gather ? args.x_rows : min(M - m0, BM), w_count = min(args.N - n0, BN);
    auto resource = [](const unsigned char* p, int64_t first, int ld, int count) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p) + first * ld, (short)0, count * ld,
                                                 kBufferFlags);
    };
    const __amdgpu_buffer_rsrc_t rx = resource(args.x, x_first, args.ld, x_count);
    const __amdgpu_buffer_rsrc_t rw = resource(args.w, w_first, args.ld, w_count);

    auto x_row = [&](int r) {
        if (m0 + r >= M) return -1;
        if (!gather) return r;
        const int listed = args.rows[ex.first + m0 + r];
        return listed < args.x_rows ? listed : -1;
    };
    auto w_row = [&](int r) { return n0 + r < args.N ? r : -1; };

    // This lane's byte offsets of its 16-byte pieces: an instruction fills 8 rows of a pair, or the scales of 32
    // rows. Waves 0 and 1 load x's scales, 2 and 3 w's.
    int x_off[INSTR], w_off[INSTR], s_off[SCALE_INSTR];
    bool x_second[2];   // the piece lies in its pair's second unit (the swizzle repeats every 16 rows)
#pragma unroll
    for (int q = 0; q < INSTR; ++q) {
        const int r = (wave * INSTR + q) * 8 + (lane >> 3);
        const int byte = ((lane & 7) ^ swz_a2(r)) << 4;
        const int xr = x_row(r), wr = w_row(r);
        if (q < 2) x_second[q] = byte >= kMx4UnitBytes;
        x_off[q] = xr < 0 ? kNowhere : xr * args.ld + byte;
        w_off[q] = wr < 0 ? kNowhere : wr * args.ld + byte;
    }
    const bool scales_of_x = wave < 2;
#pragma unroll
    for (int q = 0; q < SCALE_INSTR; ++q) {
        const int r = ((wave & 1) * SCALE_INSTR + q) * 32 + (lane >> 1);
        const int row = scales_of_x ? x_row(r) : w_row(r);
        s_off[q] = row < 0 ? kNowhere : row * args.lds + (((lane & 1) ^ ((r >> 3) & 1)) << 4);
    }
    const __amdgpu_buffer_rsrc_t rs = scales_of_x ? resource(args.xs, x_first, args.lds, x_count)
                                                  : resource(args.ws, w_first, args.lds, w_count);

    const unsigned lds0 = (unsigned)(uintptr_t)(MB_LDS unsigned char*)lds;
    auto issue_x = [&](int pair, int at, auto idx) {
        constexpr int q = decltype(idx)::value;
        const int off = pair == half_pair && x_second[q & 1] ? kNowhere : x_off[q];
        lds_dma16(rx, lds0 + at + (wave * INSTR + q) * 1024, off, u0 * kMx4UnitBytes + pair * kPairBytes);
    };
    auto issue_w = [&](int pair, int at, auto idx) {
        constexpr int q = decltype(idx)::value;
        lds_dma16(rw, lds0 + W0 + at + (wave * INSTR + q) * 1024, w_off[q], u0 * kMx4UnitBytes + pair * kPairBytes);
    };
    auto issue_scales = [&](int chunk, auto idx) {
        constexpr int q = decltype(idx)::value;
        const unsigned to = lds0 + (scales_of_x ? XS0 : WS0) + (chunk & 1) * SCALE_SLOT;
        lds_dma16(rs, to + ((wave & 1) * SCALE_INSTR + q) * 1024, s_off[q],
                  u0 * kMx4UnitScales + chunk * kChunkBytes);
    };

    f32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    // Operands of a unit: two substeps of 64 k. Of the 8 blocks of a pair, lane half h takes 4h .. 4h + 3, two a
    // unit, so one dword brings its scales of a pair, a byte for each MFMA.
    struct UnitOps {
        u32x4 a[2][FM], b[2][FN];
    };
    struct PairScales {
        unsigned a[FM], b[FN];
    };
    constexpr int N_MFMA = 2 * FM * FN;
    // Byte offsets of this lane's reads from a slot's start.
    const int x_lane = wm * WTM + r32, w_lane = wn * WTN + r32;
    auto piece_at = [&](int row, int chunk) { return row * kPairBytes + ((chunk ^ swz_a2(row)) << 4); };
    auto scales_at = [&](int row, int unit) {   // 16 bytes hold 4 units; unit: the even one of the pair, modulo 8
        return row * kChunkBytes + (((unit >> 2) ^ ((row >> 3) & 1)) << 4) + 4 * (unit & 2) + 4 * half;
    };
    int slot_flip = 0;   // SCALE_SLOT while the current chunk's number is odd
    // Read number r of unit u (its number modulo 8, 8 for the next chunk's first), in the order the MFMAs consume
    // operands: x fragment 0, w's, x's others; a pair's first unit brings the pair's scales too.
    auto read_op = [&](auto unit, auto idx, UnitOps& o, PairScales& s) {
        constexpr int u = decltype(unit)::value, r = decltype(idx)::value;
        constexpr int FIRST = (u % 2 ? 1 : 2) * (FM + FN);   // reads of substep 0
        constexpr int t = r < FIRST ? 0 : 1;
        constexpr int f = t == 1 ? r - FIRST : u % 2 ? r : r / 2;
        constexpr bool scales = u % 2 == 0 && t == 0 && r % 2 == 1;
        constexpr int at = (u / 2) % 2 * SLOT, chunk = 2 * (u % 2) + t;
        constexpr bool is_w = f >= 1 && f <= FN;
        constexpr int frag = is_w ? f - 1 : f == 0 ? 0 : f - FN;
        const int row = (is_w ? w_lane : x_lane) + 32 * frag;
        if constexpr (scales) {
            const int flip = u == kChunkUnits ? slot_flip ^ SCALE_SLOT : slot_flip;
            const unsigned v =
                *reinterpret_cast<const unsigned*>(lds + (is_w ? WS0 : XS0) + flip + scales_at(row, u % kChunkUnits));
            if constexpr (is_w) s.b[frag] = v;
            else s.a[frag] = v;
        } else {
            const u32x4 v =
                *reinterpret_cast<const u32x4*>(lds + (is_w ? W0 : 0) + at + piece_at(row, chunk + 4 * half));
            if constexpr (is_w) o.b[t][frag] = v;
            else o.a[t][frag] = v;
        }
    };
    auto mfma_op = [&](auto parity, auto idx, const UnitOps& o, const PairScales& s) {
        constexpr int q = decltype(idx)::value;
        constexpr int t = q / (FM * FN), i = (q / FN) % FM, j = q % FN;
        constexpr int byte = 2 * decltype(parity)::value + t;
        acc[i][j] = mfma_mx4<byte, byte>(o.b[t][j], s.b[j], o.a[t][i], s.a[i], acc[i][j]);
    };

    const int last_pair = (ksteps - 1) / 2, last_chunk = (ksteps - 1) / kChunkUnits;
    auto all = [&](auto count, auto&& f) {
        [&]<int... Q>(std::integer_sequence<int, Q...>) {
            (f(std::integral_constant<int, Q>{}), ...);
        }(std::make_integer_sequence<int, decltype(count)::value>{});
    };
    constexpr std::integral_constant<int, INSTR> kPieces{};
    constexpr std::integral_constant<int, SCALE_INSTR> kScalePieces{};
    all(kScalePieces, [&](auto q) { issue_scales(0, q); });
    all(kPieces, [&](auto q) { issue_x(0, 0, q); });
    all(kPieces, [&](auto q) { issue_w(0, 0, q); });
    all(kPieces, [&](auto q) { issue_x(min(1, last_pair), SLOT, q); });
    all(kPieces, [&](auto q) { issue_w(min(1, last_pair), SLOT, q); });
    all(kScalePieces, [&](auto q) { issue_scales(1, q); });   // past the row's end: zeros or other scales, unused

    UnitOps ops[2];
    wait_vmcnt_and_barrier<kWaits.prologue>();
    PairScales scales[2];
    all(std::integral_constant<int, 3 * (FM + FN)>{},
        [&](auto r) { read_op(std::integral_constant<int, 0>{}, r, ops[0], scales[0]); });

    auto step = [&](auto idx, int kt) {
        constexpr int I = decltype(idx)::value;               // kt % 8
        constexpr int DATA_LOADS = I % 2 ? 2 * INSTR : 0, LOADS = DATA_LOADS + (I == 7 ? SCALE_INSTR : 0);
        constexpr int N_READS = (I % 2 ? 3 : 2) * (FM + FN), N_MEM = N_READS + LOADS;
        constexpr int PRE = N_MFMA >= 16 ? kPreBarrierMfma : 0;
        // The step's memory instructions, spread evenly over the MFMAs behind the barrier, and the loads evenly among
        // the reads. Two of either behind an MFMA for as long as they lasted took 8192 x 8192 x 16384 to 462 us (this:
        // 435): an MFMA waited behind the LDS pipe in the first half of a step, and nothing used it in the second.
        constexpr auto kSlotOf = [](int m) { return PRE + m * (N_MFMA - PRE) / N_MEM; };
        constexpr auto kLoadsBefore = [](int m) { return m * LOADS / N_MEM; };
        const UnitOps& cur = ops[I % 2];
        UnitOps& nxt = ops[(I + 1) % 2];
        PairScales& cur_scales = scales[I / 2 % 2];
        PairScales& nxt_scales = scales[(I + 1) / 2 % 2];
        const int pair = min((kt - 1) / 2 + 2, last_pair);    // into the slot of the pair that unit kt ends
        const int chunk = min((kt - 7) / kChunkUnits + 2, last_chunk + 1);
        if constexpr (I % 2 == 0) {
            if (kt / 2 == half_pair) {   // no unit there: 2^-127 for whatever lies behind the row's scales
#pragma unroll
                for (int i = 0; i < FM; ++i) cur_scales.a[i] = half ? 0u : cur_scales.a[i];
#pragma unroll
                for (int j = 0; j < FN; ++j) cur_scales.b[j] = half ? 0u : cur_scales.b[j];
            }
        }
        [&]<int... Q>(std::integer_sequence<int, Q...>) {
            ([&] {
                if constexpr (Q == PRE) {
                    wait_vmcnt_and_barrier<kWaits.step[I]>();
                    __builtin_amdgcn_sched_barrier(0);
                }
                mfma_op(std::integral_constant<int, I % 2>{}, std::integral_constant<int, Q>{}, cur, cur_scales);
                constexpr int here = Q;
                [&]<int... R>(std::integer_sequence<int, R...>) {
                    ([&] {
                        constexpr int m = R;
                        if constexpr (kSlotOf(m) == here) {
                            constexpr int l = kLoadsBefore(m), at = (I / 2) % 2 * SLOT;
                            if constexpr (kLoadsBefore(m + 1) > l) {
                                if constexpr (l >= DATA_LOADS)
                                    issue_scales(chunk, std::integral_constant<int, l - DATA_LOADS>{});
                                else if constexpr (l < INSTR) issue_x(pair, at, std::integral_constant<int, l>{});
                                else issue_w(pair, at, std::integral_constant<int, l - INSTR>{});
                            } else {
                                read_op(std::integral_constant<int, I + 1>{}, std::integral_constant<int, m - l>{}, nxt,
                                        nxt_scales);
                            }
                        }
                    }(), ...);
                }(std::make_integer_sequence<int, N_MEM>{});
                __builtin_amdgcn_sched_barrier(0);
            }(), ...);
        }(std::make_integer_sequence<int, N_MFMA>{});
    };
    for (int kt = 0; kt < ksteps; kt += kChunkUnits) {
        [&]<int... I>(std::integer_sequence<int, I...>) {
            ((kt + I < ksteps ? step(std::integral_constant<int, I>{}, kt + I) : void()), ...);
        }(std::make_integer_sequence<int, kChunkUnits>{});
        slot_flip ^= SCALE_SLOT;
    }
    wait_vmcnt_and_barrier<0>();

    // Register 4g + q of lane l holds out(32i + l % 32, 32j + 8g + 4 (l / 32) + q).
    if constexpr (BM < 256) {
        if (args.planes != nullptr) {
            float* part = args.planes + ((int64_t)split * args.total + ex.first) * args.ldp;
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const int m = m0 + wm * WTM + 32 * i + r32;
                if (m >= M) continue;
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int n = n0 + wn * WTN + 32 * j + 8 * g + 4 * half;   // ldp is a multiple of 4
                        const f32x16& v = acc[i][j];
                        if (n < args.ldp)
                            *reinterpret_cast<f32x4*>(part + m * (int64_t)args.ldp + n) =
                                f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
                    }
            }
            return;
        }
    }

    // 16-bit rows through LDS, stored as whole row segments.
    unsigned char* ob = args.out + (int64_t)ex.first * args.ldo;
    constexpr int ROW_BYTES = WTN * 2, ROW_CHUNKS = ROW_BYTES / 16;
    static_assert(4 * WTM * ROW_BYTES <= LDS_BYTES, "the waves' tiles must fit the LDS rings");
    unsigned char* stage = lds + wave * WTM * ROW_BYTES;
    constexpr int GROUP = WTM >= 128 ? 32 : WTM;   // rows per staged group
    constexpr int ROWS_PER_STORE = 64 / ROW_CHUNKS;
    constexpr int STORES = GROUP / ROWS_PER_STORE;
    constexpr int BATCH = STORES < 8 ? STORES : 8;
    const int oc = lane % ROW_CHUNKS, orow = lane / ROW_CHUNKS;
    const int col = n0 + wn * WTN + 8 * oc, left = args.N - col;
#pragma unroll
    for (int grp = 0; grp < WTM / GROUP; ++grp) {
#pragma unroll
        for (int i = grp * (GROUP / 32); i < (grp + 1) * (GROUP / 32); ++i) {
            const int r = 32 * i + r32;
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x16& v = acc[i][j];
                    const int chunk = (4 * j + g) ^ (r % ROW_CHUNKS);
                    *reinterpret_cast<u32x2*>(stage + r * ROW_BYTES + chunk * 16 + 8 * half) =
                        pack4<DT>(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
                }
        }
        const unsigned char* from = stage + grp * GROUP * ROW_BYTES;
#pragma unroll
        for (int p0 = 0; p0 < STORES; p0 += BATCH) {
            u32x4 v[BATCH];
#pragma unroll
            for (int p = 0; p < BATCH; ++p) {
                const int r = ROWS_PER_STORE * (p0 + p) + orow;
                v[p] = *reinterpret_cast<const u32x4*>(from + r * ROW_BYTES + ((oc ^ (r % ROW_CHUNKS)) << 4));
            }
#pragma unroll
            for (int p = 0; p < BATCH; ++p) {
                const int m = m0 + wm * WTM + grp * GROUP + ROWS_PER_STORE * (p0 + p) + orow;
                unsigned char* to = ob + m * args.ldo + (int64_t)col * 2;
                if (m >= M) continue;
                if (left >= 8) {
                    // Rows off 16 bytes share cache lines with the neighbouring tiles: ordinary stores.
                    if (args.out_16) __builtin_nontemporal_store(v[p], reinterpret_cast<u32x4*>(to));
                    else *reinterpret_cast<u32x4_2*>(to) = v[p];
                } else {
#pragma unroll
                    for (int e = 0; e < 7; ++e)
                        if (e < left) reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)(v[p][e >> 1] >> 16 * (e & 1));
                }
            }
        }
    }
}

// out = the sum of the splits' planes, in split order; rows of no expert are left alone.
template <int DT>
__global__ void __launch_bounds__(256)
gemm_mx4_sum_kernel(Mx4Args a) {
    const int quads = a.ldp / 4;
    const int64_t i = (int64_t)block_number() * 256 + threadIdx.x;
    const int64_t m = i / quads;
    if (m >= a.total) return;
    if (a.offsets != nullptr && (m < a.offsets[0] || m >= a.offsets[a.experts])) return;
    const int n = 4 * (int)(i - m * quads);
    const float* from = a.planes + m * a.ldp + n;
    f32x4 v = *reinterpret_cast<const f32x4*>(from);
    for (int s = 1; s < a.splits; ++s) v += *reinterpret_cast<const f32x4*>(from + s * (int64_t)a.total * a.ldp);
    const u32x2 p = pack4<DT>(v[0], v[1], v[2], v[3]);
    unsigned char* to = a.out + m * a.ldo + (int64_t)n * 2;
    typedef u32x2 u32x2_2 __attribute__((aligned(2)));
    if (n + 4 <= a.N) {
        *reinterpret_cast<u32x2_2*>(to) = p;
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (n + e < a.N) reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)(p[e >> 1] >> 16 * (e & 1));
    }
}

template <int DT, int CFG>
int launch_mx4(const Mx4Call& c, int splits, void* workspace, hipStream_t stream) {
    constexpr int TILE = kMx4Tiles[CFG];
    const int tiles_n = (int)((c.N + TILE - 1) / TILE);
    const int64_t tiles_m = c.offsets ? c.total_rows / TILE + std::min<int64_t>(c.experts, c.total_rows)
                                      : (c.total_rows + TILE - 1) / TILE;
    const int split_units = (int)((c.units + 2 * splits - 1) / (2 * splits) * 2);   // whole pairs
    splits = (int)((c.units + split_units - 1) / split_units);                      // none is empty
    const bool out_16 = ((reinterpret_cast<uintptr_t>(c.out) | (uintptr_t)(c.ldo * 2)) & 15) == 0;
    const Mx4Args a{static_cast<const unsigned char*>(c.x), static_cast<const unsigned char*>(c.x_scales),
                    static_cast<const unsigned char*>(c.w), static_cast<const unsigned char*>(c.w_scales),
                    static_cast<unsigned char*>(c.out), c.rows, c.offsets, c.ldo * 2, (int)c.units * kMx4UnitBytes,
                    (int)c.units * kMx4UnitScales, (int)c.units, (int)c.x_rows, c.experts, (int)c.total_rows, (int)c.N,
                    splits > 1 ? static_cast<float*>(workspace) : nullptr, splits, split_units,
                    (int)((c.N + 3) / 4 * 4), out_16};
    hipLaunchKernelGGL((gemm_mx4_kernel<DT, TILE>), launch_grid(tiles_m * tiles_n * splits), dim3(256), 0, stream, a,
                       tiles_n, 4);
    MB_HIP_TRY(hipGetLastError());
    if (splits > 1) {
        hipLaunchKernelGGL((gemm_mx4_sum_kernel<DT>), launch_grid((c.total_rows * (a.ldp / 4) + 255) / 256), dim3(256),
                           0, stream, a);
        MB_HIP_TRY(hipGetLastError());
    }
    return MB_OK;
}

template <int DT>
int launch_mx4_config(const Mx4Call& c, const Mx4Plan& plan, void* workspace, hipStream_t stream) {
    if (plan.config == 0) return launch_mx4<DT, 0>(c, plan.splits, workspace, stream);
    if (plan.config == 1) return launch_mx4<DT, 1>(c, plan.splits, workspace, stream);
    return launch_mx4<DT, 2>(c, plan.splits, workspace, stream);
}

}  // namespace
}  // namespace mb

// LDS-DMA pipelined grouped products for gfx950 (bf16 / fp16), 16-byte rows:
// out(m, n) = sum over c of X(m, c) Y(c, n) for each expert, in the forms of
// gemm_grouped.hip.
//
// Each operand comes in one of two layouts, and the pipeline of the dense
// tiled GEMM serves both:
//   along c   rows of the tile run along c (X forward and for the rows'
//             gradient, Y for the rows' gradient): pair slots of two stages,
//             [rows][128 B], read with ds_read_b128
//   across c  rows run along m or n (Y forward, both for the matrices'
//             gradient): stage slots of 32 c, [32][tile width], read with
//             the transposing ds_read_b64_tr_b16
// A step computes one stage (32 c) from registers while every operand of the
// next is read from LDS and later stages are loaded: a pair slot on odd
// steps, a stage slot on every step, into the slot just vacated. One barrier
// per step, behind a vmcnt wait derived at compile time from the issue order
// (step_schedule).
//
// What is ragged: rows of X past the expert's (not there, or `rows` names
// none) and pieces past the end of c get an offset past the buffer, which
// reads as zeros; c past the expert's rows (matrices' gradient) lies past the
// operand's range. Columns past the matrix read whatever follows in range and
// are not stored.
//
// Many rows per expert are bound by the MFMAs at the clock the power limit
// leaves, as the dense kernel is (16384 rows over 8 experts, 4096 -> 14336:
// 1574 to 1654 us on two GPUs, 1.16 to 1.22 PFLOP/s); few rows by the matrices' bytes, which the deep
// rings keep in flight (128 rows over 32 experts, 4096 -> 2048: 88 to 92 us, 5.9 to 6.1 TB/s).
#pragma once

#include "experts_common.hpp"
#include "gemm_tiled_kernels.hpp"

namespace mb {
namespace {

constexpr int kNowhere = (int)0x80000000u;   // past every buffer range used here (below 2^31 bytes)

struct StepWaits {
    int odd, even, prologue;
};

// Loads: operand o is held in pairs (pair[o]) or stages, n[o] slots, instr[o]
// LDS-DMA instructions per wave and slot. Step j issues, X before Y, pair
// (j - 1) / 2 + n of a paired operand when j is odd and stage j + n of a
// staged one; the prologue runs the same rule over the steps before 0. Step j
// reads stage j + 1, so its wait leaves only the loads issued after that
// stage's. (Y first where it has fewer slots: no faster.)
constexpr StepWaits step_schedule(bool px, int nx, int ix, bool py, int ny, int iy) {
    constexpr int kSteps = 64;
    const bool pair[2] = {px, py};
    const int n[2] = {nx, ny}, instr[2] = {ix, iy};
    int end[2][2 * kSteps] = {}, before[kSteps] = {};
    int total = 0;
    for (int v = -2 * kSteps / 4; v < kSteps; ++v) {
        if (v >= 0) before[v] = total;
        for (int o = 0; o < 2; ++o) {
            if (pair[o] && (v & 1) == 0) continue;
            const int i = pair[o] ? (v - 1) / 2 + n[o] : v + n[o];   // v - 1 is even
            if (i >= 0 && i < 2 * kSteps) end[o][i] = (total += instr[o]);
        }
    }
    StepWaits r{1 << 20, 1 << 20, 0};
    r.prologue = before[0] - (end[0][0] > end[1][0] ? end[0][0] : end[1][0]);
    for (int j = 0; j + 1 < kSteps; ++j) {
        int need = 0;
        for (int o = 0; o < 2; ++o) {
            const int e = end[o][pair[o] ? (j + 1) / 2 : j + 1];
            need = e > need ? e : need;
        }
        const int w = before[j] - need;
        if (j & 1) r.odd = w < r.odd ? w : r.odd;
        else r.even = w < r.even ? w : r.even;
    }
    return r;
}

struct GroupedArgs {
    const unsigned char *x, *y;
    unsigned char* out;
    const int32_t *rows, *offsets;
    int ldx, ldy;          // bytes per row
    int64_t ldo;           // bytes per row
    int x_rows, experts, total, N, K;
    // Splits of the contraction: split s of a tile writes its fp32 sums to plane s of `planes` ([rows of out][ldp]).
    // c_len: c per split (forward, rows' gradient), whole pairs of stages.
    float* planes;
    int splits, c_len, ldp;
};

// One operand of one tile: its LDS ring, DMA offsets and operand reads. ALONG: rows along c.
template <bool ALONG, int T, int W, int N_SLOTS>
struct Ring {
    static constexpr int kSlot = ALONG ? 2 * T * kStageK : 32 * T * 2;   // bytes per slot
    static constexpr int kInstr = kSlot / 1024 / W;                       // DMA instructions per wave and slot
    static constexpr int kBytes = N_SLOTS * kSlot;
    static_assert(kSlot % (1024 * W) == 0, "a slot must split over the waves");
};

// Sorted row p of expert `ex` -> row of x, -1 for none.
__device__ __forceinline__ int sorted_row(const GroupedArgs& a, const ExpertRows& ex, int p) {
    if (p >= ex.count) return -1;
    const int r = a.rows[ex.first + p];
    return r < a.x_rows ? r : -1;
}

// GATHER: x is read through `rows`.
template <int DT, int OP, int BM, int BN, int NX, int NY, bool RAGGED_C, bool GATHER>
__global__ void __launch_bounds__(256)
gemm_grouped_kernel(GroupedArgs args, int tiles_m_max, int tiles_n, int group_m) {
    typedef Traits<DT> Tr;
    typedef typename Tr::Frag Frag;
    constexpr bool WEIGHTS = OP == MB_GROUPED_GRAD_WEIGHTS;
    constexpr bool XA = !WEIGHTS, YA = OP == MB_GROUPED_GRAD_ROWS;   // along c
    constexpr int W = 4;
    constexpr int WTM = BM / 2, WTN = BN / 2;
    constexpr int FM = WTM / 32, FN = WTN / 32;
    typedef Ring<XA, BM, W, NX> RX;
    typedef Ring<YA, BN, W, NY> RY;
    constexpr int LDS_BYTES = RX::kBytes + RY::kBytes;
    static_assert(LDS_BYTES <= 160 * 1024, "LDS rings do not fit");
    constexpr StepWaits kWaits = step_schedule(XA, NX, RX::kInstr, YA, NY, RY::kInstr);
    static_assert(kWaits.prologue >= 0 && kWaits.odd >= 0 && kWaits.even >= 0 && kWaits.prologue < 64 &&
                  kWaits.odd < 64 && kWaits.even < 64, "a needed stage is unissued, or vmcnt overflows");
    __shared__ __attribute__((aligned(1024))) unsigned char lds[LDS_BYTES];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int half = lane >> 5;

    // Tile of this block.
    ExpertRows ex;
    const int block = (int)block_number();
    int tm, tn, split;
    if constexpr (WEIGHTS) {
        // An expert's tiles are dealt to the 8 XCDs (block b runs on XCD b % 8)
        // in runs, so every XCD gets its share of every expert, however uneven
        // the experts' rows; within it, a compact patch.
        const int tiles = tiles_m_max * tiles_n * args.splits, e = block / tiles;
        if (e >= args.experts) return;
        block_coords(block - e * tiles, tiles_m_max, tiles_n, args.splits, group_m, &tm, &tn, &split);
        ex = expert_rows(args.offsets, e, args.total);
        if (args.splits > 1) {   // this split's share of the expert's rows; none for the last splits of a short one
            const int share = (ex.count + 32 * args.splits - 1) / (32 * args.splits) * 32;
            const int from = min(split * share, ex.count);
            ex.first += from;
            ex.count = min(share, ex.count - from);
        }
        ex.first = __builtin_amdgcn_readfirstlane(ex.first);
        ex.count = __builtin_amdgcn_readfirstlane(ex.count);
    } else {
        const int tiles_m = count_row_tiles(args.offsets, args.experts, args.total, BM);
        if (block >= tiles_m * tiles_n * args.splits) return;
        block_coords(block, tiles_m, tiles_n, args.splits, group_m, &tm, &tn, &split);
        if (!find_row_tile(args.offsets, args.experts, args.total, tm, BM, &ex, &tm)) return;
    }
    const int M = WEIGHTS ? args.K : ex.count;
    const int NN = YA ? args.K : args.N;
    const int C = WEIGHTS ? ex.count : YA ? args.N : args.K;
    const int m0 = tm * BM, n0 = tn * BN;
    const int ldx = args.ldx, ldy = args.ldy;
    const int c0 = WEIGHTS ? 0 : split * args.c_len;   // first c of this block

    // Buffer resources. Along c: the tile's rows (gathered: all of x). Across c: the expert's rows from the
    // tile's first column on.
    const unsigned char* xb = args.x;
    const unsigned char* yb = args.y;
    int x_range, y_range;
    if constexpr (XA) {
        if constexpr (!GATHER) xb += ((int64_t)ex.first + m0) * ldx;
        x_range = ((GATHER ? args.x_rows : min(M - m0, BM)) - 1) * ldx + C * 2;
    } else {
        if constexpr (!GATHER) xb += (int64_t)ex.first * ldx;
        xb += m0 * 2;
        x_range = ((GATHER ? args.x_rows : C) - 1) * ldx + (M - m0) * 2;
    }
    if constexpr (YA) {
        yb += (int64_t)ex.expert * args.K * ldy + (int64_t)n0 * ldy;
        y_range = (min(NN - n0, BN) - 1) * ldy + C * 2;
    } else {
        yb += (WEIGHTS ? (int64_t)ex.first : (int64_t)ex.expert * args.K) * ldy + n0 * 2;
        y_range = (C - 1) * ldy + (NN - n0) * 2;
    }
    const __amdgpu_buffer_rsrc_t rx =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(xb), (short)0, max(x_range, 0), kBufferFlags);
    const __amdgpu_buffer_rsrc_t ry =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(yb), (short)0, max(y_range, 0), kBufferFlags);

    // This lane's byte offsets of its pieces in slot 0. Along c: instruction q
    // of a wave fills rows 8 (wave kInstr + q) .. + 7 of a pair, 128 bytes
    // each. Across c: 1024 / (2 T) rows of c per instruction.
    int x_off[RX::kInstr], y_off[RY::kInstr], kbyte[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int row = q * 8 + (lane >> 3);   // the swizzle repeats every 16 rows and kInstr is even
        kbyte[q] = ((lane & 7) ^ swz_a2(row)) << 4;
    }
    constexpr int X_ROW = BM * 2, Y_ROW = BN * 2;   // bytes per LDS row, across c
#pragma unroll
    for (int q = 0; q < RX::kInstr; ++q) {
        const int lin = (wave * RX::kInstr + q) * 1024 + lane * 16;
        if constexpr (XA) {
            static_assert(RX::kInstr % 2 == 0 || !XA, "two swizzles serve an even number of instructions");
            const int r = lin >> 7;
            const int row = GATHER ? sorted_row(args, ex, m0 + r) : m0 + r < M ? r : -1;
            x_off[q] = row < 0 ? kNowhere : row * ldx + kbyte[q & 1];
        } else {
            const int r = lin / X_ROW;
            const int col = (((lin % X_ROW) >> 4) ^ b_swizzle<2, X_ROW>(r)) << 4;
            x_off[q] = GATHER ? col : r * ldx + col;
        }
    }
#pragma unroll
    for (int q = 0; q < RY::kInstr; ++q) {
        const int lin = (wave * RY::kInstr + q) * 1024 + lane * 16;
        if constexpr (YA) {
            static_assert(RY::kInstr % 2 == 0 || !YA, "two swizzles serve an even number of instructions");
            y_off[q] = (lin >> 7) * ldy + kbyte[q & 1];
        } else {
            const int r = lin / Y_ROW;
            y_off[q] = r * ldy + ((((lin % Y_ROW) >> 4) ^ b_swizzle<2, Y_ROW>(r)) << 4);
        }
    }

    auto lds_of = [&](int at) { return (unsigned)(uintptr_t)(MB_LDS unsigned char*)(lds + at); };
    auto along = [&](int off, int kb, int q) -> int {   // zeros for pieces past the end of c
        if constexpr (RAGGED_C) return kb + kbyte[q & 1] < C * 2 ? off : kNowhere;
        return off;
    };
    // Gathered rows of c (matrices' gradient): the row numbers of a wave's 8 rows of stage `kt`, by scalar
    // loads (lgkmcnt, so the vmcnt waits stay exact).
    constexpr int kShare = 8;
    auto gather = [&](int kt, int (&listed)[kShare]) {
        if constexpr (WEIGHTS && GATHER) {
            typedef int i32x8_4 __attribute__((ext_vector_type(8), aligned(4)));
            typedef const __attribute__((address_space(4))) int32_t* ConstRows;
            typedef const __attribute__((address_space(4))) i32x8_4* ConstRows8;
            const ConstRows list = (ConstRows)(uintptr_t)args.rows;
            const int first = ex.first + kt * 32 + wave * kShare;
            if (first + kShare <= args.total) {
                const i32x8 v = *(ConstRows8)(list + first);
#pragma unroll
                for (int i = 0; i < kShare; ++i) listed[i] = v[i];
            } else {
#pragma unroll
                for (int i = 0; i < kShare; ++i) listed[i] = list[min(first + i, args.total - 1)];
            }
        }
    };
    // DMA instruction q of X into slot byte `at`: pair (along) or stage (across) number i.
    auto issue_x = [&](int i, int at, auto idx, const int (&listed)[kShare]) {
        constexpr int q = decltype(idx)::value;
        const unsigned to = lds_of(at) + (wave * RX::kInstr + q) * 1024;
        if constexpr (XA) {
            const int kb = c0 * 2 + i * 2 * kStageK;
            lds_dma16(rx, to, along(x_off[q], kb, q), kb);
        } else if constexpr (GATHER) {
            constexpr int per = 1024 / X_ROW;   // rows of c per instruction
            int base = 0;
#pragma unroll
            for (int s = 0; s < per; ++s) {
                // Scalars: a select among array elements would become an indexed load.
                const unsigned r = (unsigned)__builtin_amdgcn_readfirstlane(listed[q * per + s]);
                const int off = r < (unsigned)args.x_rows ? (int)r * ldx : kNowhere;
                base = s == 0 || lane / (64 / per) == s ? off : base;
            }
            // Past the expert's rows of c: nowhere, whichever row the list names there.
            const int p = i * 32 + wave * kShare + q * per + lane / (64 / per);
            const int off = base + x_off[q];
            lds_dma16(rx, to, ((base < 0) | (p >= ex.count)) ? kNowhere : off, 0);
        } else {
            lds_dma16(rx, to, x_off[q], i * 32 * ldx);
        }
    };
    auto issue_y = [&](int i, int at, auto idx) {
        constexpr int q = decltype(idx)::value;
        const unsigned to = lds_of(at) + (wave * RY::kInstr + q) * 1024;
        if constexpr (YA) {
            const int kb = c0 * 2 + i * 2 * kStageK;
            lds_dma16(ry, to, along(y_off[q], kb, q), kb);
        } else {
            lds_dma16(ry, to, y_off[q], (c0 + i * 32) * ldy);
        }
    };
    constexpr int Y0 = RX::kBytes;   // the Y ring follows the X ring

    f32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    // Operands of a stage: two substeps of 16 c, one fragment per 32 rows (columns).
    struct StageOps {
        Frag a[2][FM];
        Frag b[2][FN];
    };
    constexpr int XP = XA ? 1 : 2, YP = YA ? 1 : 2;   // LDS reads per fragment
    constexpr int PER_SUB = FM * XP + FN * YP;
    constexpr int N_READS = 2 * PER_SUB;
    constexpr int N_MFMA = 2 * FM * FN;
    auto read_frag = [&](auto is_along, auto tile, const unsigned char* slot, int row, auto par, int s, int t,
                         Frag& f) {
        if constexpr (decltype(is_along)::value) {
            f = read_a_piece(slot, row + (lane & 31), 4 * decltype(par)::value + 2 * s + half);
        } else {
            const u32x2 v = read_b_piece<DT, decltype(tile)::value>(slot, row, s, t, lane);
            f[2 * t] = v[0];
            f[2 * t + 1] = v[1];
        }
    };
    // Read number r of a stage, in the order the MFMAs consume operands: per
    // substep X fragment 0, the Y fragments, then X fragments 1 ...
    auto read_op = [&](const unsigned char* xs, const unsigned char* ys, auto par, auto idx, StageOps& o) {
        constexpr int r = decltype(idx)::value;
        constexpr int s = r / PER_SUB, u = r % PER_SUB;
        if constexpr (u >= XP && u < XP + FN * YP) {
            constexpr int j = (u - XP) / YP, t = (u - XP) % YP;
            read_frag(std::bool_constant<YA>{}, std::integral_constant<int, BN>{}, ys, wn * WTN + 32 * j, par, s, t,
                      o.b[s][j]);
        } else {
            constexpr int v = u < XP ? u : u - FN * YP;
            constexpr int i = v / XP, t = v % XP;
            read_frag(std::bool_constant<XA>{}, std::integral_constant<int, BM>{}, xs, wm * WTM + 32 * i, par, s, t,
                      o.a[s][i]);
        }
    };
    auto mfma_op = [&](auto idx, const StageOps& o) {
        constexpr int q = decltype(idx)::value;
        constexpr int s = q / (FM * FN), i = (q / FN) % FM, j = q % FN;
        acc[i][j] = Tr::mfma(o.b[s][j], o.a[s][i], acc[i][j]);
    };

    const int ksteps = max(((WEIGHTS ? C : min(C - c0, args.c_len)) + 31) >> 5, 1);
    const int last = ksteps - 1, last_pair = last / 2;
    // Every load of one operand's pair or stage that step v issues, as N_SLOTS of them exist.
    constexpr int VX = XA ? 2 * NX - 1 : NX, VY = YA ? 2 * NY - 1 : NY;
    constexpr int V = VX > VY ? VX : VY;
    [&]<int... U>(std::integer_sequence<int, U...>) {
        ([&] {
            constexpr int v = U - V;
            constexpr int ix = XA ? (v - 1) / 2 + NX : v + NX, iy = YA ? (v - 1) / 2 + NY : v + NY;
            if constexpr ((!XA || (v & 1) != 0) && ix >= 0) {
                const int i = min(ix, XA ? last_pair : last);
                int listed[kShare] = {};
                gather(i, listed);
                [&]<int... Q>(std::integer_sequence<int, Q...>) {
                    (issue_x(i, ix * RX::kSlot, std::integral_constant<int, Q>{}, listed), ...);
                }(std::make_integer_sequence<int, RX::kInstr>{});
            }
            if constexpr ((!YA || (v & 1) != 0) && iy >= 0) {
                const int i = min(iy, YA ? last_pair : last);
                [&]<int... Q>(std::integer_sequence<int, Q...>) {
                    (issue_y(i, Y0 + iy * RY::kSlot, std::integral_constant<int, Q>{}), ...);
                }(std::make_integer_sequence<int, RY::kInstr>{});
            }
        }(), ...);
    }(std::make_integer_sequence<int, V>{});

    StageOps ops[2];
    int list_sets[2][kShare] = {};   // row numbers for this step's loads and the next's
    gather(min(NX, last), list_sets[0]);
    wait_vmcnt_and_barrier<kWaits.prologue>();
    [&]<int... R>(std::integer_sequence<int, R...>) {
        (read_op(lds, lds + Y0, std::integral_constant<int, 0>{}, std::integral_constant<int, R>{}, ops[0]), ...);
    }(std::make_integer_sequence<int, N_READS>{});

    // Slot of stage (or of the pair that holds stage) I in a ring.
    auto slot = [](bool is_along, int n, int stage) constexpr { return is_along ? (stage / 2) % n : stage % n; };
    auto step = [&](auto idx, int kt) {
        constexpr int I = decltype(idx)::value;
        constexpr bool ODD = (I & 1) != 0;
        constexpr int X_LOADS = !XA || ODD ? RX::kInstr : 0, Y_LOADS = !YA || ODD ? RY::kInstr : 0;
        constexpr int LOADS = X_LOADS + Y_LOADS;
        constexpr int N_MEM = N_READS + LOADS;
        constexpr int PRE = N_MFMA >= 16 ? kPreBarrierMfma : 0;
        constexpr int PER = (N_MEM + N_MFMA - PRE - 1) / (N_MFMA - PRE);
        constexpr int kStride = LOADS > 0 ? N_MEM / LOADS : N_MEM + 1;   // loads sit evenly among the reads
        constexpr auto kIsLoad = [](int m) { return (m + 1) % kStride == 0 && (m + 1) / kStride <= LOADS; };
        const unsigned char* next_x = lds + slot(XA, NX, I + 1) * RX::kSlot;
        const unsigned char* next_y = lds + Y0 + slot(YA, NY, I + 1) * RY::kSlot;
        constexpr int LX = XA ? ((I + 2 * NX - 1) / 2) % NX : I % NX;    // the slot this step's load fills
        constexpr int LY = YA ? ((I + 2 * NY - 1) / 2) % NY : I % NY;
        const StageOps& cur = ops[I % 2];
        StageOps& nxt = ops[(I + 1) % 2];
        const int x_load = XA ? min((kt - 1) / 2 + NX, last_pair) : min(kt + NX, last);
        const int y_load = YA ? min((kt - 1) / 2 + NY, last_pair) : min(kt + NY, last);
        [&]<int... Q>(std::integer_sequence<int, Q...>) {
            ([&] {
                if constexpr (Q == PRE) {
                    wait_vmcnt_and_barrier<ODD ? kWaits.odd : kWaits.even>();
                    __builtin_amdgcn_sched_barrier(0);
                    gather(min(kt + 1 + NX, last), list_sets[(I + 1) % 2]);   // for the next step's loads
                    __builtin_amdgcn_sched_barrier(0);
                }
                mfma_op(std::integral_constant<int, Q>{}, cur);
                constexpr int S = Q < PRE ? 0 : (Q - PRE) * PER;
                constexpr int lo = Q < PRE ? 0 : S < N_MEM ? S : N_MEM;
                constexpr int hi = Q < PRE ? 0 : S + PER < N_MEM ? S + PER : N_MEM;
                [&]<int... R>(std::integer_sequence<int, R...>) {
                    ([&] {
                        constexpr int m = lo + R;
                        if constexpr (kIsLoad(m)) {
                            constexpr int l = (m + 1) / kStride - 1;
                            if constexpr (l < X_LOADS)
                                issue_x(x_load, LX * RX::kSlot, std::integral_constant<int, l>{}, list_sets[I % 2]);
                            else
                                issue_y(y_load, Y0 + LY * RY::kSlot, std::integral_constant<int, l - X_LOADS>{});
                        } else {
                            constexpr int loads_before = m / kStride < LOADS ? m / kStride : LOADS;
                            read_op(next_x, next_y, std::integral_constant<int, (I + 1) & 1>{},
                                    std::integral_constant<int, m - loads_before>{}, nxt);
                        }
                    }(), ...);
                }(std::make_integer_sequence<int, hi - lo>{});
                __builtin_amdgcn_sched_barrier(0);
            }(), ...);
        }(std::make_integer_sequence<int, N_MFMA>{});
    };
    constexpr int UNROLL = std::lcm(2, std::lcm(XA ? 2 * NX : NX, YA ? 2 * NY : NY));
    for (int kt = 0; kt < ksteps; kt += UNROLL) {
        [&]<int... I>(std::integer_sequence<int, I...>) {
            ((kt + I < ksteps ? step(std::integral_constant<int, I>{}, kt + I) : void()), ...);
        }(std::make_integer_sequence<int, UNROLL>{});
    }
    wait_vmcnt_and_barrier<0>();

    if constexpr (BM < 256) {
        if (args.planes != nullptr) {
            const int64_t rows = WEIGHTS ? (int64_t)args.experts * args.K : args.total;
            float* part = args.planes + (split * rows + (WEIGHTS ? (int64_t)ex.expert * args.K : ex.first)) * args.ldp;
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const int m = m0 + wm * WTM + 32 * i + (lane & 31);
                if (m >= M) continue;
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int n = n0 + wn * WTN + 32 * j + 8 * g + 4 * half;   // ldp is a multiple of 8
                        const f32x16& v = acc[i][j];
                        if (n < args.ldp)
                            *reinterpret_cast<f32x4*>(part + m * (int64_t)args.ldp + n) =
                                f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
                    }
            }
            return;
        }
    }

    // Epilogue: 16-bit rows through LDS, stored as whole row segments; register 4g + q of lane l holds
    // out(32i + l % 32, 32j + 8g + 4 (l / 32) + q).
    unsigned char* ob = args.out + (WEIGHTS ? (int64_t)ex.expert * args.K : (int64_t)ex.first) * args.ldo;
    constexpr int ROW_BYTES = WTN * 2, ROW_CHUNKS = ROW_BYTES / 16;
    static_assert(W * WTM * ROW_BYTES <= LDS_BYTES, "the waves' tiles must fit the LDS rings");
    unsigned char* stage = lds + wave * WTM * ROW_BYTES;
    constexpr int GROUP = WTM >= 128 ? 32 : WTM;   // rows per staged group
    constexpr int ROWS_PER_STORE = 64 / ROW_CHUNKS;
    constexpr int STORES = GROUP / ROWS_PER_STORE;
    constexpr int BATCH = STORES < 8 ? STORES : 8;
    const int oc = lane % ROW_CHUNKS, orow = lane / ROW_CHUNKS;
    const int col = n0 + wn * WTN + 8 * oc;
#pragma unroll
    for (int grp = 0; grp < WTM / GROUP; ++grp) {
#pragma unroll
        for (int i = grp * (GROUP / 32); i < (grp + 1) * (GROUP / 32); ++i) {
            const int r = 32 * i + (lane & 31);
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
                if (m < M && col < NN)
                    __builtin_nontemporal_store(v[p], reinterpret_cast<u32x4*>(ob + m * args.ldo + col * 2));
            }
        }
    }
}

// out = the sum of the splits' planes, in split order; rows of no expert are left alone.
template <int DT>
__global__ void __launch_bounds__(256)
gemm_grouped_sum_kernel(GroupedArgs a, int64_t rows, int columns, bool sorted) {
    const int quads = a.ldp / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t m = i / quads;
    if (m >= rows) return;
    if (sorted && (m < a.offsets[0] || m >= a.offsets[a.experts])) return;
    const int n = 4 * (int)(i - m * quads);
    const float* from = a.planes + m * a.ldp + n;
    f32x4 v = *reinterpret_cast<const f32x4*>(from);
    for (int s = 1; s < a.splits; ++s) v += *reinterpret_cast<const f32x4*>(from + s * rows * a.ldp);
    if (n < columns) *reinterpret_cast<u32x2*>(a.out + m * a.ldo + n * 2) = pack4<DT>(v[0], v[1], v[2], v[3]);
}

struct GroupedConfig {
    int group_m;
    int nx[3], ny[3];   // ring slots by op
};

// Tiles of kGroupedTiles; 256 x 256 fills the LDS of a CU, 128 x 128 half of it, 64 x 64 a third.
constexpr GroupedConfig kGroupedConfigs[kGroupedTileCount] = {
    {4, {3, 3, 5}, {4, 2, 5}},
    {4, {2, 2, 5}, {6, 3, 5}},
    {4, {3, 2, 5}, {6, 3, 5}},
};

template <int DT, int OP, int CFG>
int launch_grouped(const GroupedCall& c, int splits, float* planes, hipStream_t stream) {
    constexpr GroupedConfig cfg = kGroupedConfigs[CFG];
    constexpr int TILE = kGroupedTiles[CFG];
    const int64_t NN = OP == MB_GROUPED_GRAD_ROWS ? c.K : c.N;
    const int tiles_n = (int)((NN + TILE - 1) / TILE);
    const bool weights = OP == MB_GROUPED_GRAD_WEIGHTS;
    const int64_t tiles_m = weights ? (c.K + TILE - 1) / TILE
                                    : c.total_rows / TILE + std::min<int64_t>(c.experts, c.total_rows);
    const int64_t contraction = OP == MB_GROUPED_FORWARD ? c.K : c.N;
    const int c_len = (int)((contraction + 64 * splits - 1) / (64 * splits) * 64);
    if (!weights) splits = (int)((contraction + c_len - 1) / c_len);   // none is empty
    if (splits == 1) planes = nullptr;
    const int64_t blocks = tiles_m * tiles_n * (weights ? c.experts : 1) * splits;
    GroupedArgs a{static_cast<const unsigned char*>(c.x), static_cast<const unsigned char*>(c.y),
                  static_cast<unsigned char*>(c.out), c.rows, c.offsets, (int)c.ldx * 2, (int)c.ldy * 2, c.ldo * 2,
                  (int)c.x_rows, c.experts, (int)c.total_rows, (int)c.N, (int)c.K, planes, splits, c_len, (int)NN};
    // c past the expert's rows needs no check of its own: the matrices' gradient never takes the ragged form.
    auto pick = [&](auto gathered) {
        constexpr bool G = decltype(gathered)::value;
        constexpr int NX = cfg.nx[OP], NY = cfg.ny[OP];
        if constexpr (OP != MB_GROUPED_GRAD_WEIGHTS) {
            if (contraction % 32 != 0) return gemm_grouped_kernel<DT, OP, TILE, TILE, NX, NY, true, G>;
        }
        return gemm_grouped_kernel<DT, OP, TILE, TILE, NX, NY, false, G>;
    };
    auto kernel = c.rows ? pick(std::true_type{}) : pick(std::false_type{});
    hipLaunchKernelGGL(kernel, launch_grid(blocks), dim3(256), 0, stream, a, (int)tiles_m, tiles_n, cfg.group_m);
    MB_HIP_TRY(hipGetLastError());
    if (splits > 1) {
        const int64_t rows = weights ? c.experts * c.K : c.total_rows;
        hipLaunchKernelGGL((gemm_grouped_sum_kernel<DT>), dim3((unsigned)((rows * (NN / 4) + 255) / 256)), dim3(256), 0,
                           stream, a, rows, (int)NN, !weights);
        MB_HIP_TRY(hipGetLastError());
    }
    return MB_OK;
}

template <int DT>
int launch_grouped_dtype(const GroupedCall& c, const GroupedPlan& plan, void* workspace, hipStream_t stream) {
    const int config = plan.config;
    auto* planes = static_cast<float*>(workspace);
    auto by_op = [&](auto cfg) {
        constexpr int CFG = decltype(cfg)::value;
        if (c.op == MB_GROUPED_FORWARD)
            return launch_grouped<DT, MB_GROUPED_FORWARD, CFG>(c, plan.splits, planes, stream);
        if (c.op == MB_GROUPED_GRAD_ROWS)
            return launch_grouped<DT, MB_GROUPED_GRAD_ROWS, CFG>(c, plan.splits, planes, stream);
        return launch_grouped<DT, MB_GROUPED_GRAD_WEIGHTS, CFG>(c, plan.splits, planes, stream);
    };
    if (config == 0) return by_op(std::integral_constant<int, 0>{});
    if (config == 1) return by_op(std::integral_constant<int, 1>{});
    return by_op(std::integral_constant<int, 2>{});
}

}  // namespace
}  // namespace mb

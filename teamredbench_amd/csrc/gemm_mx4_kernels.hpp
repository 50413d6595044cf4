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
struct Mx4Tile {
    int bm, bn;
    bool x_pairs;   // a ring slot holds a pair of units (whole 128-byte lines of every row), or one
    int nx;
    bool w_pairs;
    int nw;
};
#ifndef MX4_BIG
#define MX4_BIG {256, 256, true, 3, false, 3}
#endif
constexpr Mx4Tile kMx4Tiles[kMx4TileCount] = {MX4_BIG, {128, 128, true, 2, true, 2}, {64, 64, true, 2, true, 2}};

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

// One operand's LDS ring: slots of T rows, one unit (64 bytes) or a pair (128) each, then their scales.
template <bool PAIR, int T, int N_SLOTS>
struct Mx4Ring {
    static constexpr int kRow = PAIR ? 128 : 64;
    static constexpr int kScaleRow = PAIR ? 8 : 4;
    static constexpr int kData = T * kRow;
    static constexpr int kDwords = T * kScaleRow / 4 / 4;              // scale dwords per wave and slot
    static constexpr int kScaleInstr = (kDwords + 63) / 64;
    // A wave with half an instruction's dwords loads its neighbour's too; the last wave's go to the slack behind.
    static constexpr int kSlot = kData + T * kScaleRow + (kScaleInstr * 64 - kDwords) * 4;
    static constexpr int kDataInstr = kData / 1024 / 4;
    static constexpr int kInstr = kDataInstr + kScaleInstr;
    static constexpr int kBytes = N_SLOTS * kSlot;
    static_assert(kData % 4096 == 0 && kSlot % 16 == 0, "a slot must split over the waves");
};

template <bool PAIR>
__device__ __forceinline__ int mx4_swizzle(int row) {
    return PAIR ? swz_a2(row) : swz_a(row);
}

template <int DT, int CFG>
__global__ void __launch_bounds__(256)
gemm_mx4_kernel(Mx4Args args, int tiles_n, int group_m) {
    constexpr Mx4Tile kTile = kMx4Tiles[CFG];
    constexpr int BM = kTile.bm, BN = kTile.bn, NX = kTile.nx, NW = kTile.nw;
    constexpr bool XP = kTile.x_pairs, WP = kTile.w_pairs;
    constexpr int WTM = BM / 2, WTN = BN / 2;
    constexpr int FM = WTM / 32, FN = WTN / 32;
    typedef Mx4Ring<XP, BM, NX> RX;
    typedef Mx4Ring<WP, BN, NW> RW;
    constexpr int LDS_BYTES = RX::kBytes + RW::kBytes;
    static_assert(LDS_BYTES <= 160 * 1024, "LDS rings do not fit");
    constexpr StepWaits kWaits = step_schedule(XP, NX, RX::kInstr, WP, NW, RW::kInstr);
    static_assert(kWaits.prologue >= 0 && kWaits.odd >= 0 && kWaits.even >= 0 && kWaits.prologue < 64 &&
                  kWaits.odd < 64 && kWaits.even < 64, "a needed stage is unissued, or vmcnt overflows");
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
    const int u0 = split * args.split_units;

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
    const __amdgpu_buffer_rsrc_t rxs = resource(args.xs, x_first, args.lds, x_count);
    const __amdgpu_buffer_rsrc_t rws = resource(args.ws, w_first, args.lds, w_count);

    // This lane's byte offsets of its pieces in slot 0: 16 bytes of elements (an instruction fills 8 rows of a
    // pair, or 16 of a unit) and scale dwords.
    int x_off[RX::kDataInstr], xs_off[RX::kScaleInstr], w_off[RW::kDataInstr], ws_off[RW::kScaleInstr];
    auto offsets = [&](auto ring, auto pair, auto row_of, int (&off)[decltype(ring)::kDataInstr],
                       int (&s_off)[decltype(ring)::kScaleInstr], int rows) {
        typedef decltype(ring) R;
        constexpr int kChunks = R::kRow / 16, kScales = R::kScaleRow / 4;
#pragma unroll
        for (int q = 0; q < R::kDataInstr; ++q) {
            const int lin = (wave * R::kDataInstr + q) * 64 + lane;
            const int row = row_of(lin / kChunks);
            const int chunk = (lin % kChunks) ^ mx4_swizzle<decltype(pair)::value>(lin / kChunks);
            off[q] = row < 0 ? kNowhere : row * args.ld + 16 * chunk;
        }
#pragma unroll
        for (int q = 0; q < R::kScaleInstr; ++q) {
            const int lin = wave * R::kDwords + q * 64 + lane;
            const int row = lin / kScales < rows ? row_of(lin / kScales) : -1;
            s_off[q] = row < 0 ? kNowhere : row * args.lds + 4 * (lin % kScales);
        }
    };
    offsets(RX{}, std::bool_constant<XP>{}, [&](int r) {
        if (m0 + r >= M) return -1;
        if (!gather) return r;
        const int listed = args.rows[ex.first + m0 + r];
        return listed < args.x_rows ? listed : -1;
    }, x_off, xs_off, BM);
    offsets(RW{}, std::bool_constant<WP>{}, [&](int r) { return n0 + r < args.N ? r : -1; }, w_off, ws_off, BN);

    auto lds_of = [&](int at) { return (unsigned)(uintptr_t)(MB_LDS unsigned char*)(lds + at); };
    // DMA instruction q of unit (pair) i into the slot at byte `at`.
    auto issue = [&](auto ring, const __amdgpu_buffer_rsrc_t& r, const __amdgpu_buffer_rsrc_t& rs, const int* off,
                     const int* s_off, int i, int at, auto idx) {
        typedef decltype(ring) R;
        constexpr int q = decltype(idx)::value;
        if constexpr (q < R::kDataInstr) {
            lds_dma16(r, lds_of(at) + (wave * R::kDataInstr + q) * 1024, off[q], u0 * 64 + i * R::kRow);
        } else {
            constexpr int s = q - R::kDataInstr;
            lds_dma4(rs, lds_of(at + R::kData) + (wave * R::kDwords + s * 64) * 4, s_off[s],
                     u0 * 4 + i * R::kScaleRow);
        }
    };
    auto issue_x = [&](int i, int at, auto idx) { issue(RX{}, rx, rxs, x_off, xs_off, i, at, idx); };
    auto issue_w = [&](int i, int at, auto idx) { issue(RW{}, rw, rws, w_off, ws_off, i, at, idx); };
    constexpr int W0 = RX::kBytes;   // w's ring follows x's

    f32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    // Operands of a unit: two substeps of 64 k. Lane half h takes blocks 2h and 2h + 1 of a row's four, so one
    // 16-bit read brings both of its scales, the first MFMA takes byte 0 and the second byte 1.
    struct UnitOps {
        u32x4 a[2][FM], b[2][FN];
        unsigned sa[FM], sb[FN];
    };
    constexpr int N_READS = 3 * (FM + FN);
    constexpr int N_MFMA = 2 * FM * FN;
    auto read_piece = [&](auto ring, auto pair, const unsigned char* slot, int row, auto par, int t) {
        typedef decltype(ring) R;
        constexpr int first = R::kRow == 128 ? 4 * decltype(par)::value : 0;
        const int chunk = (first + 2 * half + t) ^ mx4_swizzle<decltype(pair)::value>(row);
        return *reinterpret_cast<const u32x4*>(slot + row * R::kRow + 16 * chunk);
    };
    auto read_scales = [&](auto ring, const unsigned char* slot, int row, auto par) -> unsigned {
        typedef decltype(ring) R;
        constexpr int first = R::kRow == 128 ? 4 * decltype(par)::value : 0;
        return *reinterpret_cast<const uint16_t*>(slot + R::kData + row * R::kScaleRow + first + 2 * half);
    };
    // Read number r of a unit, in the order the MFMAs consume operands: x fragment 0, w's, x's others; with substep
    // 0's elements their scales.
    auto read_op = [&](const unsigned char* xslot, const unsigned char* wslot, auto par, auto idx, UnitOps& o) {
        constexpr int r = decltype(idx)::value;
        constexpr int t = r < 2 * (FM + FN) ? 0 : 1;
        constexpr int f = t == 0 ? r / 2 : r - 2 * (FM + FN);
        constexpr bool scales = t == 0 && r % 2 == 1;
        if constexpr (f >= 1 && f <= FN) {
            constexpr int j = f - 1;
            const int row = wn * WTN + 32 * j + r32;
            if constexpr (scales) o.sb[j] = read_scales(RW{}, wslot, row, par);
            else o.b[t][j] = read_piece(RW{}, std::bool_constant<WP>{}, wslot, row, par, t);
        } else {
            constexpr int i = f == 0 ? 0 : f - FN;
            const int row = wm * WTM + 32 * i + r32;
            if constexpr (scales) o.sa[i] = read_scales(RX{}, xslot, row, par);
            else o.a[t][i] = read_piece(RX{}, std::bool_constant<XP>{}, xslot, row, par, t);
        }
    };
    auto mfma_op = [&](auto idx, const UnitOps& o) {
        constexpr int q = decltype(idx)::value;
        constexpr int t = q / (FM * FN), i = (q / FN) % FM, j = q % FN;
        acc[i][j] = mfma_mx4<t, t>(o.b[t][j], o.sb[j], o.a[t][i], o.sa[i], acc[i][j]);
    };

    const int ksteps = min(args.units - u0, args.split_units);
    const int last = ksteps - 1, last_pair = last / 2;
    constexpr int VX = XP ? 2 * NX - 1 : NX, VW = WP ? 2 * NW - 1 : NW;
    constexpr int V = VX > VW ? VX : VW;
    [&]<int... U>(std::integer_sequence<int, U...>) {
        ([&] {
            constexpr int v = U - V;
            constexpr int ix = XP ? (v - 1) / 2 + NX : v + NX, iw = WP ? (v - 1) / 2 + NW : v + NW;
            if constexpr ((!XP || (v & 1) != 0) && ix >= 0) {
                [&]<int... Q>(std::integer_sequence<int, Q...>) {
                    (issue_x(min(ix, XP ? last_pair : last), ix * RX::kSlot, std::integral_constant<int, Q>{}), ...);
                }(std::make_integer_sequence<int, RX::kInstr>{});
            }
            if constexpr ((!WP || (v & 1) != 0) && iw >= 0) {
                [&]<int... Q>(std::integer_sequence<int, Q...>) {
                    (issue_w(min(iw, WP ? last_pair : last), W0 + iw * RW::kSlot, std::integral_constant<int, Q>{}),
                     ...);
                }(std::make_integer_sequence<int, RW::kInstr>{});
            }
        }(), ...);
    }(std::make_integer_sequence<int, V>{});

    UnitOps ops[2];
    wait_vmcnt_and_barrier<kWaits.prologue>();
    [&]<int... R>(std::integer_sequence<int, R...>) {
        (read_op(lds, lds + W0, std::integral_constant<int, 0>{}, std::integral_constant<int, R>{}, ops[0]), ...);
    }(std::make_integer_sequence<int, N_READS>{});

    auto slot = [](bool pairs, int n, int unit) constexpr { return pairs ? (unit / 2) % n : unit % n; };
    auto step = [&](auto idx, int kt) {
        constexpr int I = decltype(idx)::value;
        constexpr bool ODD = (I & 1) != 0;
        constexpr int X_LOADS = !XP || ODD ? RX::kInstr : 0, W_LOADS = !WP || ODD ? RW::kInstr : 0;
        constexpr int LOADS = X_LOADS + W_LOADS;
        constexpr int N_MEM = N_READS + LOADS;
        constexpr int PRE = N_MFMA >= 16 ? kPreBarrierMfma : 0;
        constexpr int PER = (N_MEM + N_MFMA - PRE - 1) / (N_MFMA - PRE);
        constexpr int kStride = LOADS > 0 ? N_MEM / LOADS : N_MEM + 1;   // loads sit evenly among the reads
        constexpr auto kIsLoad = [](int m) { return (m + 1) % kStride == 0 && (m + 1) / kStride <= LOADS; };
        const unsigned char* next_x = lds + slot(XP, NX, I + 1) * RX::kSlot;
        const unsigned char* next_w = lds + W0 + slot(WP, NW, I + 1) * RW::kSlot;
        constexpr int LX = XP ? ((I + 2 * NX - 1) / 2) % NX : I % NX;    // the slot this step's load fills
        constexpr int LW = WP ? ((I + 2 * NW - 1) / 2) % NW : I % NW;
        const UnitOps& cur = ops[I % 2];
        UnitOps& nxt = ops[(I + 1) % 2];
        const int x_load = XP ? min((kt - 1) / 2 + NX, last_pair) : min(kt + NX, last);
        const int w_load = WP ? min((kt - 1) / 2 + NW, last_pair) : min(kt + NW, last);
        [&]<int... Q>(std::integer_sequence<int, Q...>) {
            ([&] {
                if constexpr (Q == PRE) {
                    wait_vmcnt_and_barrier<ODD ? kWaits.odd : kWaits.even>();
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
                                issue_x(x_load, LX * RX::kSlot, std::integral_constant<int, l>{});
                            else
                                issue_w(w_load, W0 + LW * RW::kSlot, std::integral_constant<int, l - X_LOADS>{});
                        } else {
                            constexpr int loads_before = m / kStride < LOADS ? m / kStride : LOADS;
                            read_op(next_x, next_w, std::integral_constant<int, (I + 1) & 1>{},
                                    std::integral_constant<int, m - loads_before>{}, nxt);
                        }
                    }(), ...);
                }(std::make_integer_sequence<int, hi - lo>{});
                __builtin_amdgcn_sched_barrier(0);
            }(), ...);
        }(std::make_integer_sequence<int, N_MFMA>{});
    };
    constexpr int UNROLL = std::lcm(2, std::lcm(XP ? 2 * NX : NX, WP ? 2 * NW : NW));
    for (int kt = 0; kt < ksteps; kt += UNROLL) {
        [&]<int... I>(std::integer_sequence<int, I...>) {
            ((kt + I < ksteps ? step(std::integral_constant<int, I>{}, kt + I) : void()), ...);
        }(std::make_integer_sequence<int, UNROLL>{});
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
    constexpr Mx4Tile kTile = kMx4Tiles[CFG];
    const int tiles_n = (int)((c.N + kTile.bn - 1) / kTile.bn);
    const int64_t tiles_m = c.offsets ? c.total_rows / kTile.bm + std::min<int64_t>(c.experts, c.total_rows)
                                      : (c.total_rows + kTile.bm - 1) / kTile.bm;
    const int split_units = (int)((c.units + 2 * splits - 1) / (2 * splits) * 2);   // whole pairs
    splits = (int)((c.units + split_units - 1) / split_units);                      // none is empty
    const bool out_16 = ((reinterpret_cast<uintptr_t>(c.out) | (uintptr_t)(c.ldo * 2)) & 15) == 0;
    const Mx4Args a{static_cast<const unsigned char*>(c.x), static_cast<const unsigned char*>(c.x_scales),
                    static_cast<const unsigned char*>(c.w), static_cast<const unsigned char*>(c.w_scales),
                    static_cast<unsigned char*>(c.out), c.rows, c.offsets, c.ldo * 2, (int)c.units * kMx4UnitBytes,
                    (int)c.units * kMx4UnitScales, (int)c.units, (int)c.x_rows, c.experts, (int)c.total_rows, (int)c.N,
                    splits > 1 ? static_cast<float*>(workspace) : nullptr, splits, split_units,
                    (int)((c.N + 3) / 4 * 4), out_16};
    hipLaunchKernelGGL((gemm_mx4_kernel<DT, CFG>), launch_grid(tiles_m * tiles_n * splits), dim3(256), 0, stream, a,
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

// LDS-DMA pipelined products of MX4 matrices for gfx950: out(m, n) = sum over k of
// X(m, k) W(n, k), both operands in rows along k (layout: mx4_common.hpp), dense
// or by expert, on v_mfma_scale_f32_32x32x64_f8f6f4.
//
// A block of four waves makes a tile of rows x columns (kMx4Tiles), a wave a quarter of it in accumulators of 32 x 32.
// What feeds them: LDS-DMA of 16 bytes a lane into rings of slots, elements a pair of units (256 of K: a 128-byte
// line of every row) at a time, scales eight units (32 bytes of every row: a dword a row and unit cost as many lines
// of L1 as the elements did). A step is one unit: the MFMAs of unit j, the LDS reads of unit j + 1 spread evenly among
// them, and the loads of a pair or of scales some slots ahead; one barrier and one vmcnt wait a step, derived from the
// order of the loads at compile time (mx4_schedule). 16-byte chunk c of a row lies at chunk c ^ swz_a2(row) of its
// slot, so that the 64 lanes of a read of elements meet every bank evenly (4 LDS cycles, no conflicts). Lane half h takes
// blocks 4h .. 4h + 3 of a pair: K may come in any order that both operands share, and so one dword brings a lane its
// four scales. Those dwords, of rows 32 bytes apart, take 8 LDS cycles where 2 would do, and are most of the 26% of its LDS
// cycles that 8192^3 spends in bank conflicts; LDS is busy for 29% of that product's cycles.
//
// 256 x 256 tiles, persistent blocks of one a CU: 8192^3 232-245 us on the GPUs seen, 4.5-4.7 PFLOP/s, 69-71% of what
// these MFMAs sustain alone there (6.5-6.7). 8192 x 8192 x K, four tiles a block, on one GPU: K = 2048 88.2 us at 1.69
// GHz, 4096 139 (1.67), 8192 245 (1.55), 16384 457 (1.51). So a tile takes 37200, 58000, 95100 and 172600 cycles: about
// 1190 for a unit of K, 1024 of them MFMAs, and 18000 to 20000 around the K loop (first loads, stores, its part of the
// launch; the next tile's first loads run among the stores). The clock is what the power limit leaves; the MFMAs
// alone run at 1.56 GHz there, no slower than 8192^3 with its idle cycles. The last half round of tiles of 4096 x 14336 x
// 4096 costs 23 us, a whole one 34.
#pragma once

#include "gemm_grouped_kernels.hpp"
#include "gemm_mx4_plan.hpp"
#include "mx4_common.hpp"

namespace mb {

int gemm_mx4_tiled_bf16(const Mx4Call& c, const Mx4Plan& plan, int cus, void* workspace,
                        hipStream_t stream);
int gemm_mx4_tiled_f16(const Mx4Call& c, const Mx4Plan& plan, int cus, void* workspace,
                        hipStream_t stream);

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
    bool out_lines;                       // out's rows start on lines of 128 bytes
};

// Ring slots: elements two or four slots of a pair of units (whole 128-byte lines of every row), scales two slots of
// 8 units (32 bytes of every row).
constexpr int kPairBytes = 128, kChunkUnits = 8, kChunkBytes = 32;

// Loads of step j: pair (j - 1) / 2 + slots of x and w on odd j, then scale chunk (j - 7) / 8 + 2 where j % 8 == 7,
// `pair` and `chunk` instructions per wave. Before step 0: chunk 0, pairs 0 .. slots - 1, chunk 1. Step j reads unit
// j + 1, so its wait leaves only what was issued after that unit's loads (a wave's vector memory operations complete in
// the order of their issue). By j % 8, the least of all steps.
//
// A tile whose block stored the one before with `groups` of `pieces` stores has them among its first loads: group g's
// go out behind the loads of group g + 1, those of the first kLoadGroups. `behind_prologue` and `behind` are the waits
// of the prologue and of the first three steps then.
constexpr int kLoadGroups = 4;
struct Mx4Waits {
    int step[kChunkUnits], prologue, behind_prologue, behind[3];
};
constexpr Mx4Waits mx4_schedule(int slots, int pair, int chunk, int groups, int pieces) {
    constexpr int kSteps = 64;
    int pair_end[kSteps] = {}, chunk_end[kSteps] = {}, before[kSteps] = {};
    Mx4Waits r{};
    for (int stores = 0; stores < 2; ++stores) {
        int total = 0;
        const int first = chunk + slots * pair;   // chunk 0, pair 0, pair 1 ...
        chunk_end[0] = chunk;
        for (int p = 0; p < slots; ++p) pair_end[p] = chunk + (p + 1) * pair;
        if (stores) {
            for (int g = 0; g < groups; ++g) {
                for (int l = 0; g < kLoadGroups && l < first; ++l) {
                    if (l * kLoadGroups / first != g) continue;
                    ++total;
                    for (int p = 0; p < slots; ++p)
                        if (l + 1 == chunk + (p + 1) * pair) pair_end[p] = total;
                }
                if (g > 0) total += pieces;
            }
            total += pieces;
        } else {
            total = first;
        }
        chunk_end[1] = (total += chunk);
        (stores ? r.behind_prologue : r.prologue) = total - pair_end[0];
        for (int j = 0; j < kSteps; ++j) {
            before[j] = total;
            if ((j & 1) != 0) pair_end[(j - 1) / 2 + slots] = (total += pair);
            if ((j & 7) == 7) chunk_end[(j + 1) / kChunkUnits + 1] = (total += chunk);
        }
        for (int i = 0; !stores && i < kChunkUnits; ++i) r.step[i] = 63;
        for (int j = 0; j + 1 < kSteps; ++j) {
            const int p = pair_end[(j + 1) / 2], c = chunk_end[(j + 1) / kChunkUnits];
            const int wait = before[j] - (p > c ? p : c);
            if (stores && j < 3) r.behind[j] = wait;   // these three need nothing that the steps loaded
            if (!stores && wait < r.step[j % kChunkUnits]) r.step[j % kChunkUnits] = wait;
        }
    }
    return r;
}

// Row tile and column of tile b of a persistent launch of `stride` blocks: in groups of kGroupM row tiles, as in
// block_coords, and round by round, each XCD (block b runs on XCD b % 8) taking an eighth of a round's tiles, one patch of
// them. So the XCDs share a group's rows, and one expert's w at a time (each XCD its own eighth of all tiles: 16384 rows
// over 8 experts, 4096 -> 14336, 519 us for 502; 2048 x 50257 x 4096 244 for 229). Divides by a multiplication:
// `magic` is 2^40 / (kGroupM tiles_n), rounded up.
constexpr int kGroupM = 4;
__host__ __device__ __forceinline__ void tile_coords(int b, int stride, int tiles, int tiles_m, int tiles_n,
                                                     uint64_t magic, int* tm, int* tn) {
    const int c = (int)((unsigned)b % (unsigned)stride), n = min(tiles - (b - c), stride);
    const int t = b - c + (c & 7) * (n >> 3) + min(c & 7, n & 7) + (c >> 3);
    const int per_group = kGroupM * tiles_n;
    int g = (int)(((uint64_t)(unsigned)t * magic) >> 40);
    if ((int64_t)g * per_group > t) --g;
    const int first_m = g * kGroupM, rows = min(tiles_m - first_m, kGroupM), r = t - g * per_group;
    const int column = rows == kGroupM ? r / kGroupM : rows == 3 ? r / 3 : r >> (rows - 1);
    *tm = first_m + r - column * rows;
    *tn = column;
}

// lds_dma16 of what is read once.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void lds_dma16_once(__amdgpu_buffer_rsrc_t rsrc, unsigned lds_addr, int voff, int soff) {
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen nt lds"
                 :
                 : "s"(lds_addr), "v"(voff), "s"(rsrc), "s"(soff)
                 : "memory", "m0");
}
#pragma clang diagnostic pop

// An accumulator's value, from where the matrix instructions keep it: left to itself the compiler copies all 256
// into vector registers at once, and spills. The caller keeps the wait states behind the last matrix instruction.
__device__ __forceinline__ float read_acc(float v) {
    float f;
    asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(f) : "a"(v));
    return f;
}

template <int DT, int CFG, bool STREAM>
__global__ void __launch_bounds__(256)
gemm_mx4_kernel(Mx4Args all_args, int tiles_n, uint64_t magic) {
    constexpr int BM = kMx4Tiles[CFG].rows, BN = kMx4Tiles[CFG].columns, SLOTS = kMx4Tiles[CFG].slots;
    constexpr int WTM = BM / 2, WTN = BN / 2;
    constexpr int FM = WTM / 32, FN = WTN / 32;
    // A wave loads as many scales as any other: of both operands those of the longer side's rows.
    constexpr int SIDE = BM > BN ? BM : BN;
    constexpr int X_SLOT = BM * kPairBytes, W_SLOT = BN * kPairBytes, SCALE_SLOT = SIDE * kChunkBytes;
    // LDS: x's elements, w's (SLOTS slots each); slot 0 of x's scales and of w's, slot 1 of both.
    constexpr int W0 = SLOTS * X_SLOT, XS0 = W0 + SLOTS * W_SLOT, WS0 = XS0 + SCALE_SLOT, NEXT_SCALES = 2 * SCALE_SLOT;
    constexpr int LDS_BYTES = XS0 + 2 * NEXT_SCALES;
    // DMA instructions per wave: of x and of w a pair, of both operands' scales a chunk.
    constexpr int X_INSTR = X_SLOT / 1024 / 4, W_INSTR = W_SLOT / 1024 / 4, PAIR_INSTR = X_INSTR + W_INSTR;
    constexpr int SCALE_INSTR = 2 * SCALE_SLOT / 1024 / 4;
    static_assert(LDS_BYTES <= 160 * 1024 && X_SLOT % 8192 == 0 && W_SLOT % 8192 == 0 && SCALE_INSTR >= 1, "LDS rings");
    // Stores: groups of 32 rows and up to 64 columns of a wave's tile go through LDS and out as whole lines. A
    // persistent block (one per CU) stages them in the second scale slot, while the next tile's loads fill the rest.
    constexpr bool PERSISTENT = BM == 256;
    constexpr int GC = WTN < 64 ? WTN : 64, STAGE = 32 * GC * 2, PIECES = STAGE / 1024;
    constexpr int STAGE0 = PERSISTENT ? XS0 + NEXT_SCALES : 0;
    constexpr int GROUPS = FM * (WTN / GC);                  // of a wave's tile
    static_assert(!PERSISTENT || (4 * STAGE == NEXT_SCALES && STAGE == SCALE_INSTR * 1024),
                  "a wave stages its stores in what its own loads of the second scale slot fill");
    constexpr Mx4Waits kWaits = mx4_schedule(SLOTS, PAIR_INSTR, SCALE_INSTR, GROUPS, PIECES);
    static_assert([&] {
        for (int w : kWaits.step)
            if (w < 0 || w >= 64) return false;
        for (int w : kWaits.behind)
            if (PERSISTENT && (w < 0 || w >= 64)) return false;
        return kWaits.prologue >= 0 && kWaits.prologue < 64 && (!PERSISTENT || kWaits.behind_prologue < 64);
    }(), "a needed unit is unissued, or vmcnt overflows");
    __shared__ __attribute__((aligned(1024))) unsigned char lds[LDS_BYTES];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int half = lane >> 5, r32 = lane & 31;

    // The arguments, read again for each tile: kept in registers they would crowd the K loop's out.
    auto arguments = [&]() -> Mx4Args {
#if defined(__HIP_DEVICE_COMPILE__)
        if constexpr (PERSISTENT) {
            auto p = (const __attribute__((address_space(4))) Mx4Args*)__builtin_amdgcn_kernarg_segment_ptr();
            asm volatile("" : "+s"(p));
            return *p;
        }
#endif
        return all_args;
    };

    struct Tile {
        ExpertRows ex;
        int m0, n0, split;
    };
    int tm, tn, tiles_before = 0;   // row tiles before the tile's expert
    int t = (int)block_number(), tiles, tiles_m;
    const int stride = (int)(gridDim.x * gridDim.y);   // tiles of this block: t, t + stride ...
    Tile cur{{0, 0, 0}, 0, 0, 0};
    {
        const Mx4Args args = arguments();
        const bool by_expert = args.offsets != nullptr;
        // Offsets out of order may count any number of tiles.
        tiles_m = by_expert ? min(count_row_tiles(args.offsets, args.experts, args.total, BM),
                                  args.total / BM + min(args.experts, args.total))
                            : (args.total + BM - 1) / BM;
        tiles = tiles_m * tiles_n * args.splits;
        if (t >= tiles) return;
        if (PERSISTENT) tile_coords(t, stride, tiles, tiles_m, tiles_n, magic, &tm, &tn);
        else block_coords(t, tiles_m, tiles_n, args.splits, kGroupM, &tm, &tn, &cur.split);
        cur.ex.count = args.total;
        if (by_expert) {
            int in_expert;
            if (!find_row_tile(args.offsets, args.experts, args.total, tm, BM, &cur.ex, &in_expert)) return;
            tiles_before = tm - in_expert;
        }
        cur.m0 = (tm - tiles_before) * BM;
        cur.n0 = tn * BN;
    }
    // Another tile: its expert is near the last one's. Scalar loads, which the vmcnt waits do not see.
    const bool by_expert = all_args.offsets != nullptr;
    auto locate = [&](Tile& tile) {
        tile_coords(t + stride, stride, tiles, tiles_m, tiles_n, magic, &tm, &tn);
        if (by_expert) {
            const Mx4Args args = arguments();
            typedef const __attribute__((address_space(4))) int32_t* ConstRows;
            const ConstRows list = (ConstRows)(uintptr_t)args.offsets;
            auto rows_of = [&](int i) {
                const int lo = min(max(list[i], 0), args.total), hi = min(max(list[i + 1], 0), args.total);
                return ExpertRows{i, lo, max(hi - lo, 0)};
            };
            int e = __builtin_amdgcn_readfirstlane(tile.ex.expert);
            ExpertRows ex = rows_of(e);
            while (tm < tiles_before && e > 0) {
                ex = rows_of(--e);
                tiles_before -= (ex.count + BM - 1) / BM;
            }
            while (tm >= tiles_before + (ex.count + BM - 1) / BM && e + 1 < args.experts) {
                tiles_before += (ex.count + BM - 1) / BM;
                ex = rows_of(++e);
            }
            tile.ex = ex;
        }
        tile.m0 = __builtin_amdgcn_readfirstlane((tm - tiles_before) * BM);
        tile.n0 = __builtin_amdgcn_readfirstlane(tn * BN);
    };

    // The rows of x that this lane's loads go through (-1: none): of the wave's quarter of the tile, and of the half
    // whose scales it loads (waves 0 and 1 load x's scales, 2 and 3 w's).
    const bool scales_of_x = wave < 2;
    constexpr int X_ROWS = BM / 4, W_ROWS = BN / 4, SCALE_ROWS = SIDE / 2;
    struct XRows {
        int data, scales[2];
    };
    auto x_rows = [&](const Mx4Args& args, const Tile& tile) {
        auto row = [&](int r) {
            if (tile.m0 + r >= tile.ex.count) return -1;
            return args.rows != nullptr ? args.rows[tile.ex.first + tile.m0 + r] : r;
        };
        XRows x{row(wave * X_ROWS + lane % X_ROWS), {-1, -1}};
        if (scales_of_x) {
            x.scales[0] = row(wave * SCALE_ROWS + lane % SCALE_ROWS);
            if constexpr (SCALE_ROWS > 64) x.scales[1] = row(wave * SCALE_ROWS + 64 + lane);
        }
        return x;
    };

    // A tile's loads: buffer resources over its rows (gathered: all of x), past which rows and units read as zeros,
    // and this lane's byte offsets of its 16-byte pieces. An instruction fills 8 rows of a pair, or the scales of 32.
    struct Loads {
        __amdgpu_buffer_rsrc_t x, w, scales;
        int x_off[X_INSTR], w_off[2], s_off[SCALE_INSTR];
        int ld16, at, scales_at;               // 16 rows of w; bytes to the first unit of K
        int ksteps, k_bytes, half_pair;        // units of K, in whole pairs; the pair whose second unit is not there
    };
    int k_byte[2];   // of this lane's pieces within their pair (the swizzle repeats every 16 rows)
#pragma unroll
    for (int q = 0; q < 2; ++q) k_byte[q] = ((lane & 7) ^ swz_a2(q * 8 + (lane >> 3))) << 4;
    auto loads_of = [&](const Mx4Args& args, const Tile& tile, const XRows& rows) {
        auto resource = [](const unsigned char* p, int64_t first, int ld, int count) {
            const uint64_t at = (uint64_t)(uintptr_t)p + first * ld;   // the same in every lane, and held so
            const uint64_t lo = (unsigned)__builtin_amdgcn_readfirstlane((int)at);
            const uint64_t hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(at >> 32));
            return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(hi << 32 | lo), (short)0,
                                                     __builtin_amdgcn_readfirstlane(count * ld), kBufferFlags);
        };
        const bool gather = args.rows != nullptr;
        const int64_t x_first = gather ? 0 : (int64_t)tile.ex.first + tile.m0;
        const int64_t w_first = (int64_t)tile.ex.expert * args.N + tile.n0;
        const int x_count = gather ? args.x_rows : max(min(tile.ex.count - tile.m0, BM), 0);
        const int w_count = min(args.N - tile.n0, BN);
        Loads l;
        l.x = resource(args.x, x_first, args.ld, x_count);
        l.w = resource(args.w, w_first, args.ld, w_count);
        l.scales = resource(scales_of_x ? args.xs : args.ws, scales_of_x ? x_first : w_first, args.lds,
                            scales_of_x ? x_count : w_count);
#pragma unroll
        for (int q = 0; q < X_INSTR; ++q) {
            const int r = q * 8 + (lane >> 3), row = __shfl(rows.data, r);
            l.x_off[q] = row < 0 || row >= x_count ? kNowhere : row * args.ld + k_byte[q & 1];
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) l.w_off[q] = (wave * W_ROWS + q * 8 + (lane >> 3)) * args.ld + k_byte[q];
#pragma unroll
        for (int q = 0; q < SCALE_INSTR; ++q) {
            const int r = q * 32 + (lane >> 1), byte = ((lane & 1) ^ ((r >> 3) & 1)) << 4;
            const int listed = __shfl(rows.scales[q / 2], r % 64);
            const int row = scales_of_x ? (listed < x_count ? listed : -1) : (wave & 1) * SCALE_ROWS + r;
            l.s_off[q] = row < 0 ? kNowhere : row * args.lds + byte;
        }
        const int u0 = tile.split * args.split_units, units = min(args.units - u0, args.split_units);
        l.ld16 = 16 * args.ld;
        l.at = u0 * kMx4UnitBytes;
        l.scales_at = u0 * kMx4UnitScales;
        l.ksteps = (units + 1) & ~1;
        l.k_bytes = units * kMx4UnitBytes;
        l.half_pair = units & 1 ? units / 2 : -1;
        return l;
    };
    XRows rows;
    Loads from;
    {
        const Mx4Args args = arguments();
        rows = x_rows(args, cur);
        from = loads_of(args, cur, rows);
    }

    const unsigned lds0 = (unsigned)(uintptr_t)(MB_LDS unsigned char*)lds;
    // Pieces past the end of K are zeros, and not fetched.
    auto issue_x = [&](int pair, int at, auto idx) {
        constexpr int q = decltype(idx)::value;
        const int off = k_byte[q & 1] < from.k_bytes - pair * kPairBytes ? from.x_off[q] : kNowhere;
        lds_dma16(from.x, lds0 + at + (wave * X_INSTR + q) * 1024, off, from.at + pair * kPairBytes);
    };
    auto issue_w = [&](int pair, int at, auto idx) {
        constexpr int q = decltype(idx)::value;
        const int off = k_byte[q & 1] < from.k_bytes - pair * kPairBytes ? from.w_off[q & 1] : kNowhere;
        constexpr auto load = STREAM ? lds_dma16_once : lds_dma16;
        load(from.w, lds0 + W0 + at + (wave * W_INSTR + q) * 1024, off,
             from.at + pair * kPairBytes + (q >> 1) * from.ld16);
    };
    auto issue_scales = [&](int chunk, auto idx) {
        constexpr int q = decltype(idx)::value;
        const unsigned to = lds0 + (scales_of_x ? XS0 : WS0) + (chunk & 1) * NEXT_SCALES;
        lds_dma16(from.scales, to + ((wave & 1) * SCALE_INSTR + q) * 1024, from.s_off[q],
                  from.scales_at + chunk * kChunkBytes);
    };
    auto all = [&](auto count, auto&& f) {
        [&]<int... Q>(std::integer_sequence<int, Q...>) {
            (f(std::integral_constant<int, Q>{}), ...);
        }(std::make_integer_sequence<int, decltype(count)::value>{});
    };
    // Load l of a tile's first: scale chunk 0, a pair for every slot.
    constexpr int FIRST_LOADS = SCALE_INSTR + SLOTS * PAIR_INSTR;
    auto first_load = [&](auto idx) {
        constexpr int l = decltype(idx)::value, d = l - SCALE_INSTR, pair = d / PAIR_INSTR, q = d % PAIR_INSTR;
        if constexpr (d < 0) issue_scales(0, idx);
        else if constexpr (q < X_INSTR) issue_x(pair, pair * X_SLOT, std::integral_constant<int, q>{});
        else issue_w(pair, pair * W_SLOT, std::integral_constant<int, q - X_INSTR>{});
    };
    constexpr std::integral_constant<int, FIRST_LOADS> kFirstLoads{};
    constexpr std::integral_constant<int, SCALE_INSTR> kScalePieces{};
    // Chunk 1, where a persistent block's stores are staged: a wave's loads fill what the wave itself staged. Past the
    // row's end: zeros or other scales, unused.
    auto second_chunk = [&] { all(kScalePieces, [&](auto q) { issue_scales(1, q); }); };

    f32x16 acc[FM][FN];
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
    int slot_flip = 0;   // byte offset of the current chunk's slot
    // Read number r of unit u (its number modulo 8, 8 for the next chunk's first), in the order the MFMAs consume
    // operands: x fragment 0, w's, x's others; a pair's first unit brings the pair's scales too.
    auto read_op = [&](auto unit, auto idx, UnitOps& o, PairScales& s) {
        constexpr int u = decltype(unit)::value, r = decltype(idx)::value;
        constexpr int FIRST = (u % 2 ? 1 : 2) * (FM + FN);   // reads of substep 0
        constexpr int t = r < FIRST ? 0 : 1;
        constexpr int f = t == 1 ? r - FIRST : u % 2 ? r : r / 2;
        constexpr bool scales = u % 2 == 0 && t == 0 && r % 2 == 1;
        constexpr int slot = (u / 2) % SLOTS, chunk = 2 * (u % 2) + t;
        constexpr bool is_w = f >= 1 && f <= FN;
        constexpr int frag = is_w ? f - 1 : f == 0 ? 0 : f - FN;
        const int row = (is_w ? w_lane : x_lane) + 32 * frag;
        if constexpr (scales) {
            const int flip = u == kChunkUnits ? slot_flip ^ NEXT_SCALES : slot_flip;
            const unsigned v =
                *reinterpret_cast<const unsigned*>(lds + (is_w ? WS0 : XS0) + flip + scales_at(row, u % kChunkUnits));
            if constexpr (is_w) s.b[frag] = v;
            else s.a[frag] = v;
        } else {
            constexpr int at = is_w ? W0 + slot * W_SLOT : slot * X_SLOT;
            const u32x4 v = *reinterpret_cast<const u32x4*>(lds + at + piece_at(row, chunk + 4 * half));
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

    UnitOps ops[2];
    PairScales scales[2];
    bool behind_stores = false;   // the first loads went out among the stores of a whole tile
    auto step = [&](auto idx, int kt) {
        constexpr int I = decltype(idx)::value;               // kt % 8
        constexpr int DATA_LOADS = I % 2 ? PAIR_INSTR : 0, LOADS = DATA_LOADS + (I == 7 ? SCALE_INSTR : 0);
        constexpr int N_READS = (I % 2 ? 3 : 2) * (FM + FN), N_MEM = N_READS + LOADS;
        constexpr int PRE = N_MFMA >= 16 ? kPreBarrierMfma : 0;
        // The step's memory instructions, spread evenly over the MFMAs behind the barrier, and the loads evenly among
        // the reads. Two of either behind an MFMA for as long as they lasted took 8192 x 8192 x 16384 to 462 us (this:
        // 435): an MFMA waited behind the LDS pipe in the first half of a step, and nothing used it in the second.
        constexpr auto kSlotOf = [](int m) { return PRE + m * (N_MFMA - PRE) / N_MEM; };
        constexpr auto kLoadsBefore = [](int m) { return m * LOADS / N_MEM; };
        const UnitOps& cur_ops = ops[I % 2];
        UnitOps& nxt = ops[(I + 1) % 2];
        PairScales& cur_scales = scales[I / 2 % 2];
        PairScales& nxt_scales = scales[(I + 1) / 2 % 2];
        const int pair = (kt - 1) / 2 + SLOTS;                // into the slot of the pair that unit kt ends
        const int chunk = (kt - 7) / kChunkUnits + 2;         // past the row's end: zeros or other scales, unused
        if constexpr (I % 2 == 0) {
            if (kt / 2 == from.half_pair) {   // no unit there: 2^-127 for whatever lies behind the row's scales
#pragma unroll
                for (int i = 0; i < FM; ++i) cur_scales.a[i] = half ? 0u : cur_scales.a[i];
#pragma unroll
                for (int j = 0; j < FN; ++j) cur_scales.b[j] = half ? 0u : cur_scales.b[j];
            }
        }
        [&]<int... Q>(std::integer_sequence<int, Q...>) {
            ([&] {
                if constexpr (Q == PRE) {
                    if constexpr (I < 3 && PERSISTENT) {
                        if (behind_stores && kt == I) wait_vmcnt_and_barrier<kWaits.behind[I < 3 ? I : 0]>();
                        else wait_vmcnt_and_barrier<kWaits.step[I]>();
                    } else {
                        wait_vmcnt_and_barrier<kWaits.step[I]>();
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                mfma_op(std::integral_constant<int, I % 2>{}, std::integral_constant<int, Q>{}, cur_ops, cur_scales);
                constexpr int here = Q;
                [&]<int... R>(std::integer_sequence<int, R...>) {
                    ([&] {
                        constexpr int m = R;
                        if constexpr (kSlotOf(m) == here) {
                            constexpr int l = kLoadsBefore(m), slot = (I / 2) % SLOTS;
                            if constexpr (kLoadsBefore(m + 1) > l) {
                                if constexpr (l >= DATA_LOADS)
                                    issue_scales(chunk, std::integral_constant<int, l - DATA_LOADS>{});
                                else if constexpr (l < X_INSTR)
                                    issue_x(pair, slot * X_SLOT, std::integral_constant<int, l>{});
                                else
                                    issue_w(pair, slot * W_SLOT, std::integral_constant<int, l - X_INSTR>{});
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

    all(kFirstLoads, first_load);
    second_chunk();
    while (true) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
        if (PERSISTENT && behind_stores) wait_vmcnt_and_barrier<PERSISTENT ? kWaits.behind_prologue : 0>();
        else wait_vmcnt_and_barrier<kWaits.prologue>();
        all(std::integral_constant<int, 3 * (FM + FN)>{},
            [&](auto r) { read_op(std::integral_constant<int, 0>{}, r, ops[0], scales[0]); });
        Tile next = cur;
        const bool more = PERSISTENT && t + stride < tiles;
        for (int kt = 0; kt < from.ksteps; kt += kChunkUnits) {
            if (more && kt + kChunkUnits >= from.ksteps) {   // the next tile's rows arrive during the last steps
                locate(next);
                rows = x_rows(arguments(), next);
            }
            [&]<int... I>(std::integer_sequence<int, I...>) {
                ((kt + I < from.ksteps ? step(std::integral_constant<int, I>{}, kt + I) : void()), ...);
            }(std::make_integer_sequence<int, kChunkUnits>{});
            slot_flip ^= NEXT_SCALES;
        }
        wait_vmcnt_and_barrier<0>();
        asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");   // what the last MFMAs wrote is read behind these
        slot_flip = 0;
        const Mx4Args args = arguments();
        if (more) from = loads_of(args, next, rows);   // the next tile's first loads run while this one is stored

        // Register 4g + q of lane l holds out(32i + l % 32, 32j + 8g + 4 (l / 32) + q).
        const int M = cur.ex.count;
        if (!PERSISTENT && args.planes != nullptr) {
            float* part = args.planes + ((int64_t)cur.split * args.total + cur.ex.first) * args.ldp;
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const int m = cur.m0 + wm * WTM + 32 * i + r32;
                if (m >= M) continue;
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int n = cur.n0 + wn * WTN + 32 * j + 8 * g + 4 * half;   // ldp is a multiple of 4
                        const f32x16& v = acc[i][j];
                        if (n < args.ldp)
                            *reinterpret_cast<f32x4*>(part + m * (int64_t)args.ldp + n) =
                                f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
                    }
            }
            return;
        }
        // Group by group through LDS. A wave's LDS accesses take effect in their order, so a group's reads need no wait
        // behind its writes, nor the next group's writes behind those reads.
        const bool whole = cur.m0 + BM <= M && cur.n0 + BN <= args.N, out_lines = args.out_lines;
        constexpr int CHUNKS = GC / 8, ROWS = 64 / CHUNKS;   // rows per store
        unsigned char* stage = lds + STAGE0 + wave * STAGE;
        const int oc = lane % CHUNKS, orow = lane / CHUNKS;
        const int m0 = cur.m0 + wm * WTM + orow, n0 = cur.n0 + wn * WTN + 8 * oc;
        unsigned char* to = args.out + (int64_t)(cur.ex.first + m0) * args.ldo + (int64_t)n0 * 2;
        const int64_t row_step = ROWS * args.ldo;
        auto write_group = [&](auto idx) {
            constexpr int i = decltype(idx)::value / (WTN / GC), j0 = decltype(idx)::value % (WTN / GC) * (GC / 32);
            asm volatile("" ::: "memory");
#pragma unroll
            for (int j = j0; j < j0 + GC / 32; ++j)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = read_acc(acc[i][j][4 * g + e]);
                    const int chunk = (4 * (j - j0) + g) ^ (r32 % CHUNKS);
                    *reinterpret_cast<u32x2*>(stage + r32 * GC * 2 + chunk * 16 + 8 * half) =
                        pack4<DT>(v[0], v[1], v[2], v[3]);
                }
            asm volatile("" ::: "memory");
        };
        auto read_piece = [&](int p) {
            const int r = p * ROWS + orow;
            return *reinterpret_cast<const u32x4*>(stage + r * GC * 2 + ((oc ^ (r % CHUNKS)) << 4));
        };
        auto to_group = [&](auto idx) {
            constexpr int i = decltype(idx)::value / (WTN / GC), j0 = decltype(idx)::value % (WTN / GC) * (GC / 32);
            return to + i * (32 / ROWS) * row_step + j0 * 64;
        };
        if (whole) {
            u32x4 v[2][PIECES];
            auto store_group = [&](auto idx) {
                constexpr int g = decltype(idx)::value;
                unsigned char* at = to_group(idx);
                if (out_lines) {
#pragma unroll
                    for (int p = 0; p < PIECES; ++p, at += row_step)
                        __builtin_nontemporal_store(v[g % 2][p], reinterpret_cast<u32x4*>(at));
                } else {   // parts of lines, which L2 joins: 8192 x 8200 x 4096 153 us, past it 181
#pragma unroll
                    for (int p = 0; p < PIECES; ++p, at += row_step) *reinterpret_cast<u32x4_2*>(at) = v[g % 2][p];
                }
            };
            all(std::integral_constant<int, GROUPS>{}, [&](auto idx) {
                constexpr int g = decltype(idx)::value;
                if constexpr (PERSISTENT && g < kLoadGroups) {
                    if (more) all(kFirstLoads, [&](auto l) {
                        if constexpr (decltype(l)::value * kLoadGroups / FIRST_LOADS == g) first_load(l);
                    });
                }
                write_group(idx);
                if constexpr (g > 0) store_group(std::integral_constant<int, g - 1>{});
                asm volatile("" ::: "memory");
#pragma unroll
                for (int p = 0; p < PIECES; ++p) v[g % 2][p] = read_piece(p);
            });
            store_group(std::integral_constant<int, GROUPS - 1>{});
        } else {
            if (more) all(kFirstLoads, first_load);
            all(std::integral_constant<int, GROUPS>{}, [&](auto idx) {
                constexpr int i = decltype(idx)::value / (WTN / GC), j0 = decltype(idx)::value % (WTN / GC) * (GC / 32);
                write_group(idx);
                unsigned char* at = to_group(idx);
                const int left = args.N - (n0 + 32 * j0), rows_left = M - (m0 + 32 * i);
                u32x4 v[PIECES];
#pragma unroll
                for (int p = 0; p < PIECES; ++p) v[p] = read_piece(p);
                if (left >= 8) {
#pragma unroll
                    for (int p = 0; p < PIECES; ++p, at += row_step)
                        if (p * ROWS < rows_left) *reinterpret_cast<u32x4_2*>(at) = v[p];
                } else if (left > 0) {   // the last columns
#pragma unroll
                    for (int p = 0; p < PIECES; ++p, at += row_step)
#pragma unroll
                        for (int e = 0; e < 7; ++e)
                            if (p * ROWS < rows_left && e < left)
                                reinterpret_cast<uint16_t*>(at)[e] = (uint16_t)(v[p][e >> 1] >> 16 * (e & 1));
                }
            });
        }
        behind_stores = whole;
        if (!more) return;
        if (!behind_stores) __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): the waits count none of these stores
        second_chunk();
        cur = next;
        t += stride;
    }
}

// Four columns of a row, `left` of them in it.
template <int DT>
__device__ __forceinline__ void store4(unsigned char* to, const f32x4& v, int left) {
    typedef u32x2 u32x2_2 __attribute__((aligned(2)));
    const u32x2 p = pack4<DT>(v[0], v[1], v[2], v[3]);
    if (left >= 4) {
        *reinterpret_cast<u32x2_2*>(to) = p;
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < left) reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)(p[e >> 1] >> 16 * (e & 1));
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
    store4<DT>(a.out + m * a.ldo + (int64_t)n * 2, v, a.N - n);
}

template <int DT>
int mx4_sum(const Mx4Args& a, hipStream_t stream) {
    hipLaunchKernelGGL((gemm_mx4_sum_kernel<DT>), launch_grid(((int64_t)a.total * (a.ldp / 4) + 255) / 256), dim3(256),
                       0, stream, a);
    MB_HIP_TRY(hipGetLastError());
    return MB_OK;
}

// The kernels' arguments; `planes` where K is split.
inline Mx4Args mx4_args(const Mx4Call& c, int splits, void* planes) {
    const int split_units = (int)((c.units + 2 * splits - 1) / (2 * splits) * 2);   // whole pairs
    const bool out_lines = ((reinterpret_cast<uintptr_t>(c.out) | (uintptr_t)(c.ldo * 2)) & 127) == 0;
    return Mx4Args{static_cast<const unsigned char*>(c.x), static_cast<const unsigned char*>(c.x_scales),
                   static_cast<const unsigned char*>(c.w), static_cast<const unsigned char*>(c.w_scales),
                   static_cast<unsigned char*>(c.out), c.rows, c.offsets, c.ldo * 2, (int)c.units * kMx4UnitBytes,
                   (int)c.units * kMx4UnitScales, (int)c.units, (int)c.x_rows, c.experts, (int)c.total_rows, (int)c.N,
                   static_cast<float*>(planes), splits, split_units, (int)((c.N + 3) / 4 * 4), out_lines};
}

template <int DT, int CFG>
int launch_mx4(const Mx4Call& c, int splits, bool stream_w, int cus, void* workspace, hipStream_t stream) {
    constexpr int BM = kMx4Tiles[CFG].rows, BN = kMx4Tiles[CFG].columns;
    const int tiles_n = (int)((c.N + BN - 1) / BN);
    const int64_t tiles_m = c.offsets ? c.total_rows / BM + std::min<int64_t>(c.experts, c.total_rows)
                                      : (c.total_rows + BM - 1) / BM;
    const int64_t pairs = (c.units + 1) / 2, split_pairs = (pairs + splits - 1) / splits;
    splits = (int)((pairs + split_pairs - 1) / split_pairs);   // none is empty
    const Mx4Args a = mx4_args(c, splits, splits > 1 ? workspace : nullptr);
    // Tiles of 256: a block per CU, which loads its next tile while it stores one.
    const int64_t blocks = tiles_m * tiles_n * splits;
    const uint64_t per_group = (uint64_t)kGroupM * tiles_n, magic = ((1ull << 40) + per_group - 1) / per_group;
    auto kernel = stream_w ? gemm_mx4_kernel<DT, CFG, true> : gemm_mx4_kernel<DT, CFG, false>;
    hipLaunchKernelGGL(kernel, launch_grid(BM == 256 ? std::min<int64_t>(blocks, cus) : blocks),
                       dim3(256), 0, stream, a, tiles_n, magic);
    MB_HIP_TRY(hipGetLastError());
    return splits > 1 ? mx4_sum<DT>(a, stream) : MB_OK;
}

template <int DT>
int launch_mx4_config(const Mx4Call& c, const Mx4Plan& plan, int cus, void* workspace, hipStream_t stream) {
    switch (plan.config) {
        case 0: return launch_mx4<DT, 0>(c, plan.splits, plan.stream, cus, workspace, stream);
        case 1: return launch_mx4<DT, 1>(c, plan.splits, plan.stream, cus, workspace, stream);
        case 2: return launch_mx4<DT, 2>(c, plan.splits, plan.stream, cus, workspace, stream);
        case 3: return launch_mx4<DT, 3>(c, plan.splits, plan.stream, cus, workspace, stream);
        default: return launch_mx4<DT, 4>(c, plan.splits, plan.stream, cus, workspace, stream);
    }
}

}  // namespace
}  // namespace mb

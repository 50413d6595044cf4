// Products of MX4 matrices: out[p][n] = sum over k of x[rows[p]][k] w[e][n][k],
// both operands in rows along k (layout: mx4_common.hpp), dense or by expert.
//
// gemm_mx4_any_kernel: a wave makes 32 rows x 32 columns from operands that go
// from global memory straight into the matrix cores' registers. 64-bit addresses, any size; for lists of rows over more
// than 2^31 bytes, which buffer offsets do not span. 8192^3 takes it 2.9 ms (tiles: 0.24), each load bringing 32 of
// a line's 128 bytes.
//
// gemm_mx4_rows_kernel: few rows, bound by the bytes of w. 1 x 14336 x 4096 7.3 us (31 MB: 6.2 at the rate of a copy,
// launch included in neither), 64 tokens x 4 of 64 experts, 4096 -> 2048, 47.5 us (6.0 TB/s of w's, x's and out's bytes).
//
// gemm_mx4_launch: which kernel (gemm_mx4_plan.hpp).
#include "gemm_mx4_kernels.hpp"

namespace mb {
namespace {

constexpr int kTile = 32;

__global__ void __launch_bounds__(64)
gemm_mx4_any_kernel(Mx4Call c, int tiles_n) {
    const int lane = threadIdx.x, half = lane >> 5, r32 = lane & 31;
    const int64_t block = block_number();
    int tm = (int)(block / tiles_n);
    const int64_t n0 = (block - (int64_t)tm * tiles_n) * kTile;
    ExpertRows ex{0, 0, (int)c.total_rows};
    if (c.offsets != nullptr && !find_row_tile(c.offsets, c.experts, (int)c.total_rows, tm, kTile, &ex, &tm)) return;
    const int m = tm * kTile + r32;   // this lane's row of the expert
    if (tm * kTile >= ex.count) return;
    int64_t row = m < ex.count ? (int64_t)ex.first + m : -1;
    if (row >= 0 && c.rows != nullptr) {
        row = c.rows[row];
        if (row >= c.x_rows) row = -1;
    }
    const int64_t n = min(n0 + r32, c.N - 1);   // columns past N are not stored
    const int64_t wrow = (int64_t)ex.expert * c.N + n;
    const auto* xp = static_cast<const u32x4*>(c.x) + max(row, (int64_t)0) * c.units * 4 + 2 * half;
    const auto* wp = static_cast<const u32x4*>(c.w) + wrow * c.units * 4 + 2 * half;
    const auto* xs = static_cast<const uint16_t*>(c.x_scales) + max(row, (int64_t)0) * c.units * 2 + half;
    const auto* ws = static_cast<const uint16_t*>(c.w_scales) + wrow * c.units * 2 + half;
    f32x16 acc;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    for (int64_t u = 0; u < c.units; ++u) {   // lane half h takes blocks 2h and 2h + 1 of the unit
        u32x4 a0 = {0, 0, 0, 0}, a1 = {0, 0, 0, 0};
        unsigned sa = 0;
        if (row >= 0) {
            a0 = xp[4 * u];
            a1 = xp[4 * u + 1];
            sa = xs[2 * u];
        }
        const unsigned sb = ws[2 * u];
        acc = mfma_mx4<0, 0>(wp[4 * u], sb, a0, sa, acc);
        acc = mfma_mx4<1, 1>(wp[4 * u + 1], sb, a1, sa, acc);
    }
    // Register 4g + q of lane l: row l % 32, column 8g + 4 (l / 32) + q.
    if (m >= ex.count) return;
    auto* out = static_cast<uint16_t*>(c.out) + (int64_t)(ex.first + m) * c.ldo + n0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int col = 8 * (i >> 2) + 4 * half + (i & 3);
        if (n0 + col < c.N)
            out[col] = c.dtype == MB_DT_FLOAT16 ? to_bits<MB_DT_FLOAT16>(acc[i]) : to_bits<MB_DT_BFLOAT16>(acc[i]);
    }
}

// Few rows: a wave makes XR rows x 32 columns over its share of K, on a ring of its own in LDS (no barriers: only the
// wave reads what it loads), and the waves of a block add their sums in wave order.
constexpr int kRowsDepth = 4;   // pairs of units in flight per wave
constexpr int kRowsWaves = 2;   // per block: more leave fewer blocks to a CU (1 x 14336 x 4096: 7.6 us, 6 waves 9.6)
template <int XR>
struct RowsRing {
    static constexpr int kX = XR * kPairBytes, kW = 32 * kPairBytes, kSlot = kW + kX;
    static constexpr int kInstr = kSlot / 1024;                   // DMA instructions of a pair
    static constexpr int kScales = 2 * 1024;                      // of 8 units: w's 32 rows, x's
    static constexpr int kBytes = kRowsDepth * kSlot + 2 * kScales;
};

template <int DT, int XR, bool STREAM>
__global__ void __launch_bounds__(64 * kRowsWaves)
gemm_mx4_rows_kernel(Mx4Args args, int tiles_m, int tiles_n) {
    typedef RowsRing<XR> R;
    constexpr int W = kRowsWaves;
    static_assert(XR == 8 || XR == 32, "rows of x of a tile");
    __shared__ __attribute__((aligned(1024))) unsigned char lds[W * R::kBytes];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, r32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int block = (int)block_number();
    ExpertRows ex{0, 0, args.total};
    int tm, tn;
    if (args.offsets != nullptr) {
        tm = block / tiles_n;
        tn = block - tm * tiles_n;
        if (!find_row_tile(args.offsets, args.experts, args.total, tm, XR, &ex, &tm)) return;
    } else {   // the row tiles of one column tile 8 blocks apart, on one XCD: its L2 has w for the others
        tn = block / (8 * tiles_m) * 8 + block % 8;
        tm = block / 8 % tiles_m;
        if (tn >= tiles_n) return;
    }
    const int n0 = tn * 32, m0 = tm * XR, M = ex.count - m0;   // rows of this tile: the first M

    const bool gather = args.rows != nullptr;
    auto resource = [](const unsigned char* p, int64_t first, int ld, int count) {
        const uint64_t at = (uint64_t)(uintptr_t)p + first * ld;   // the same in every lane, and held so
        const uint64_t lo = (unsigned)__builtin_amdgcn_readfirstlane((int)at);
        const uint64_t hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(at >> 32));
        return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(hi << 32 | lo), (short)0,
                                                 __builtin_amdgcn_readfirstlane(count * ld), kBufferFlags);
    };
    const int64_t x_first = gather ? 0 : (int64_t)ex.first + m0, w_first = (int64_t)ex.expert * args.N + n0;
    const int x_count = gather ? args.x_rows : min(M, XR), w_count = min(args.N - n0, 32);
    const __amdgpu_buffer_rsrc_t rx = resource(args.x, x_first, args.ld, x_count);
    const __amdgpu_buffer_rsrc_t rw = resource(args.w, w_first, args.ld, w_count);
    const __amdgpu_buffer_rsrc_t rxs = resource(args.xs, x_first, args.lds, x_count);
    const __amdgpu_buffer_rsrc_t rws = resource(args.ws, w_first, args.lds, w_count);
    auto x_row = [&](int r) {
        if (r >= M) return -1;
        const int row = gather ? args.rows[ex.first + m0 + r] : r;
        return row < x_count ? row : -1;
    };

    // This lane's 16-byte pieces: an instruction brings 8 rows of a pair, or 8 units' scales of 32 rows.
    int x_off[XR / 8], w_off[4], k_byte[2];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int r = q * 8 + (lane >> 3);
        if (q < 2) k_byte[q] = ((lane & 7) ^ swz_a2(r)) << 4;
        w_off[q] = r * args.ld + k_byte[q & 1];
        if (q < XR / 8) {
            const int row = x_row(r);
            x_off[q] = row < 0 ? kNowhere : row * args.ld + k_byte[q & 1];
        }
    }
    const int s_row = lane >> 1, s_byte = ((lane & 1) ^ ((s_row >> 3) & 1)) << 4;
    const int xs_row = s_row < XR ? x_row(s_row) : -1;
    const int xs_off = xs_row < 0 ? kNowhere : xs_row * args.lds + s_byte, ws_off = s_row * args.lds + s_byte;

    // This wave's pairs.
    const int pairs = (args.units + 1) / 2;
    const int first = pairs * wave / W, count = pairs * (wave + 1) / W - first;
    const int k_bytes = args.units * kMx4UnitBytes - first * kPairBytes;           // from its first on
    const int half_pair = args.units & 1 ? pairs - 1 - first : -1;
    const unsigned ring = (unsigned)(uintptr_t)(MB_LDS unsigned char*)lds + wave * R::kBytes;
    unsigned char* mine = lds + wave * R::kBytes;
    constexpr int SCALES0 = kRowsDepth * R::kSlot;
    constexpr auto load_w = STREAM ? lds_dma16_once : lds_dma16;
    auto issue = [&](int pair, int slot) {   // pairs past the wave's: nothing is fetched
        const int left = pair < count ? k_bytes - pair * kPairBytes : 0, at = (first + pair) * kPairBytes;
        if (slot == 0) {
            const unsigned to = ring + SCALES0 + (pair / kRowsDepth & 1) * R::kScales;
            const int from = (first + pair) * 2 * kMx4UnitScales;
            lds_dma16(rws, to, left > 0 ? ws_off : kNowhere, from);
            lds_dma16(rxs, to + 1024, left > 0 ? xs_off : kNowhere, from);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
            load_w(rw, ring + slot * R::kSlot + q * 1024, k_byte[q & 1] < left ? w_off[q] : kNowhere, at);
#pragma unroll
        for (int q = 0; q < XR / 8; ++q)
            lds_dma16(rx, ring + slot * R::kSlot + R::kW + q * 1024, k_byte[q & 1] < left ? x_off[q] : kNowhere, at);
    };
    f32x16 acc;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
#pragma unroll
    for (int s = 0; s < kRowsDepth; ++s) issue(s, s);
    const int xr = XR == 8 ? r32 & 7 : r32;   // 8 rows: the others repeat them, and are not stored
    auto scales_at = [&](int row, int pair) {   // as in gemm_mx4_kernel
        return row * kChunkBytes + ((((pair >> 1) & 1) ^ ((row >> 3) & 1)) << 4) + 8 * (pair & 1) + 4 * half;
    };
    for (int p0 = 0; p0 < count; p0 += kRowsDepth) {
        [&]<int... S>(std::integer_sequence<int, S...>) {
            ([&] {
                constexpr int s = S;
                const int p = p0 + s;
                if (p >= count) return;
                // Behind this pair's loads: those of the next three, and of a chunk of scales among them.
                constexpr int kWait = (kRowsDepth - 1) * R::kInstr + (s == 0 ? 0 : 2);
                static_assert(kWait < 64, "vmcnt overflows");
                __builtin_amdgcn_s_waitcnt((kWait & 0xF) | ((kWait >> 4) << 14) | 0x0F70);
                asm volatile("" ::: "memory");
                const unsigned char* slot = mine + s * R::kSlot;
                const unsigned char* sc = mine + SCALES0 + (p0 / kRowsDepth & 1) * R::kScales;
                unsigned sb = *reinterpret_cast<const unsigned*>(sc + scales_at(r32, s));
                unsigned sa = *reinterpret_cast<const unsigned*>(sc + 1024 + scales_at(xr, s));
                u32x4 a[4], b[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int bk = ((4 * half + i) ^ swz_a2(r32)) << 4, ak = ((4 * half + i) ^ swz_a2(xr)) << 4;
                    b[i] = *reinterpret_cast<const u32x4*>(slot + r32 * kPairBytes + bk);
                    a[i] = *reinterpret_cast<const u32x4*>(slot + R::kW + xr * kPairBytes + ak);
                }
                if (p == half_pair) {   // no unit there: 2^-127 for whatever lies behind the row's scales
                    sa = half ? 0u : sa;
                    sb = half ? 0u : sb;
                }
                acc = mfma_mx4<0, 0>(b[0], sb, a[0], sa, acc);
                acc = mfma_mx4<1, 1>(b[1], sb, a[1], sa, acc);
                acc = mfma_mx4<2, 2>(b[2], sb, a[2], sa, acc);
                acc = mfma_mx4<3, 3>(b[3], sb, a[3], sa, acc);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the slot has been read
                issue(p + kRowsDepth, s);
            }(), ...);
        }(std::make_integer_sequence<int, kRowsDepth>{});
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the ring takes the sums

    constexpr int ROW = 36;   // floats of a row of sums
    float* sums = reinterpret_cast<float*>(mine);
    if (r32 < XR) {
#pragma unroll
        for (int g = 0; g < 4; ++g)   // register 4g + q of lane l: row l % 32, column 8g + 4 (l / 32) + q
            *reinterpret_cast<f32x4*>(sums + r32 * ROW + 8 * g + 4 * half) =
                f32x4{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
    }
    __syncthreads();
    for (int i = tid; i < XR * 8; i += 64 * W) {
        const int r = i / 8, col = 4 * (i % 8), n = n0 + col;
        if (r >= M || n >= args.N) continue;
        f32x4 v = *reinterpret_cast<const f32x4*>(lds + (r * ROW + col) * 4);
#pragma unroll
        for (int w = 1; w < W; ++w) v += *reinterpret_cast<const f32x4*>(lds + w * R::kBytes + (r * ROW + col) * 4);
        const int64_t m = ex.first + m0 + r;
        store4<DT>(args.out + m * args.ldo + (int64_t)n * 2, v, args.N - n);
    }
}

template <int DT, int XR>
int launch_rows(const Mx4Call& c, bool stream_w, hipStream_t stream) {
    const int64_t tiles_m = c.offsets ? c.total_rows / XR + std::min<int64_t>(c.experts, c.total_rows)
                                      : (c.total_rows + XR - 1) / XR;
    const int64_t tiles_n = (c.N + 31) / 32, columns = c.offsets ? tiles_n : (tiles_n + 7) / 8 * 8;
    auto kernel = stream_w ? gemm_mx4_rows_kernel<DT, XR, true> : gemm_mx4_rows_kernel<DT, XR, false>;
    hipLaunchKernelGGL(kernel, launch_grid(tiles_m * columns), dim3(64 * kRowsWaves), 0, stream,
                       mx4_args(c, 1, nullptr), (int)tiles_m, (int)tiles_n);
    MB_HIP_TRY(hipGetLastError());
    return MB_OK;
}

template <int DT>
int launch_rows_config(const Mx4Call& c, const Mx4Plan& plan, hipStream_t stream) {
    return plan.config == kMx4Rows8 ? launch_rows<DT, 8>(c, plan.stream, stream)
                                    : launch_rows<DT, 32>(c, plan.stream, stream);
}

int launch_any(const Mx4Call& c, hipStream_t stream) {
    const int64_t tiles_m = c.offsets ? c.total_rows / kTile + std::min<int64_t>(c.experts, c.total_rows)
                                      : (c.total_rows + kTile - 1) / kTile;
    const int64_t tiles_n = (c.N + kTile - 1) / kTile;
    hipLaunchKernelGGL(gemm_mx4_any_kernel, launch_grid(tiles_m * tiles_n), dim3(64), 0, stream, c, (int)tiles_n);
    MB_HIP_TRY(hipGetLastError());
    return MB_OK;
}

}  // namespace

int gemm_mx4_launch(const Mx4Call& c, void* workspace, size_t workspace_bytes, const DeviceProps& props,
                    hipStream_t stream) {
    // The workspace only makes small calls faster: one off 16 bytes is left alone.
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) workspace_bytes = 0;
    const Mx4Shape shape{c.total_rows, c.N, c.units, c.x_rows, c.experts, c.offsets != nullptr, c.rows != nullptr};
    const Mx4Plan plan = mx4_plan(shape, workspace_bytes, props.cu_count, tuning(MB_TUNE_MX4_CONFIG),
                                  tuning(MB_TUNE_MX4_SPLITS));
    const bool half = c.dtype == MB_DT_FLOAT16;
    if (plan.config == kMx4Any) return launch_any(c, stream);
    if (plan.config >= kMx4TileCount)
        return half ? launch_rows_config<MB_DT_FLOAT16>(c, plan, stream)
                    : launch_rows_config<MB_DT_BFLOAT16>(c, plan, stream);
    return half ? gemm_mx4_tiled_f16(c, plan, props.cu_count, workspace, stream)
                : gemm_mx4_tiled_bf16(c, plan, props.cu_count, workspace, stream);
}

}  // namespace mb

// Pieces shared by the expert layer's kernels: element conversion, the search
// for a tile's expert, and the plan/launch entry points.
#pragma once

#include "mb_common.hpp"

#include <algorithm>

namespace mb {

typedef u32x4 u32x4_any __attribute__((aligned(2)));   // 16 bytes on any 16-bit element

int route_launch(int dtype, const void* logits, int64_t ld, int64_t tokens, int experts, int top_k, bool normalize,
                 float* weights, int32_t* expert_ids, int32_t* offsets, int32_t* rows, int32_t* slots,
                 void* workspace, hipStream_t stream);
size_t route_workspace(int64_t tokens, int experts);
int route_grad_launch(int dtype, const void* logits, int64_t ld, const int32_t* expert_ids, const float* grad_weights,
                      int64_t tokens, int experts, int top_k, bool normalize, void* grad_logits, int64_t ld_grad,
                      hipStream_t stream);

int combine_launch(int dtype, const void* y, int64_t ldy, int64_t y_rows, const float* weights, const int32_t* slots,
                   int64_t tokens, int top_k, int64_t N, void* out, int64_t ldo, hipStream_t stream);
int combine_grad_launch(int dtype, const void* grad_out, int64_t ldg, const void* y, int64_t ldy, int64_t y_rows,
                        const float* weights, const int32_t* slots, int64_t tokens, int top_k, int64_t N, void* grad_y,
                        int64_t ld_grad_y, float* grad_weights, hipStream_t stream);

// One call of mb_gemm_grouped, checked. Leading dimensions are filled in.
struct GroupedCall {
    int op, dtype, experts;
    const void *x, *y;
    void* out;
    const int32_t *rows, *offsets;
    int64_t ldx, ldy, ldo, x_rows, total_rows, N, K;
};
// Tile heights and widths of the pipelined grouped kernels.
constexpr int kGroupedTileCount = 3;
constexpr int kGroupedTiles[kGroupedTileCount] = {256, 128, 64};
struct GroupedPlan {
    int config;   // tiles of kGroupedTiles[config] on the pipelined kernels; -1: the kernel for any rows
    int splits;   // of the contraction, over fp32 planes in the workspace (tiles of 128 and 64)
};
// The pipelined kernels (rows on 16 bytes), one per input type.
int gemm_grouped_tiled_bf16(const GroupedCall& c, const GroupedPlan& plan, void* workspace, hipStream_t stream);
int gemm_grouped_tiled_f16(const GroupedCall& c, const GroupedPlan& plan, void* workspace, hipStream_t stream);
int gemm_grouped_launch(const GroupedCall& c, void* workspace, size_t workspace_bytes, const DeviceProps& props,
                        hipStream_t stream);

// One call of mb_gemm_w4, checked. offsets NULL: one expert with total_rows rows.
struct W4Call {
    int dtype, experts, group;
    const void *x, *q, *scales, *zeros;
    void* out;
    const int32_t *rows, *offsets;
    int64_t ldx, ldo, x_rows, total_rows, N, K;
};
int gemm_w4_launch(const W4Call& c, void* workspace, size_t workspace_bytes, const DeviceProps& props,
                   hipStream_t stream);

namespace {

// A grid of at least `blocks` blocks. One dimension of a grid spans below 2^32
// threads and more are not refused but lost: blocks past kGridX go along y, and
// those past the last (fewer than kGridX) return at once.
constexpr int kGridX = 1 << 21;   // 2^31 threads in blocks of 1024
inline dim3 launch_grid(int64_t blocks) {
    return dim3((unsigned)std::min<int64_t>(blocks, kGridX), (unsigned)((blocks + kGridX - 1) / kGridX));
}
__device__ __forceinline__ unsigned block_number() { return blockIdx.y * (unsigned)kGridX + blockIdx.x; }

// 16-bit element <-> fp32.
template <int DT>
__device__ __forceinline__ float from_bits(uint16_t v) {
    if constexpr (DT == MB_DT_FLOAT16) return (float)__builtin_bit_cast(_Float16, v);
    else return __builtin_bit_cast(float, (unsigned)v << 16);
}
template <int DT>
__device__ __forceinline__ uint16_t to_bits(float v) {
    if constexpr (DT == MB_DT_FLOAT16) return __builtin_bit_cast(uint16_t, (_Float16)v);
    else return __builtin_bit_cast(uint16_t, (__bf16)v);
}
template <int DT>
__device__ __forceinline__ void unpack8(const u32x4& p, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = from_bits<DT>((uint16_t)(p[i] & 0xFFFFu));
        v[2 * i + 1] = from_bits<DT>((uint16_t)(p[i] >> 16));
    }
}
template <int DT>
__device__ __forceinline__ u32x4 pack8(const float* v) {
    u32x4 p;
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = (unsigned)to_bits<DT>(v[2 * i]) | ((unsigned)to_bits<DT>(v[2 * i + 1]) << 16);
    return p;
}

// An expert's sorted rows: [first, first + count).
struct ExpertRows {
    int expert, first, count;
};

// Expert e's rows as `offsets` gives them, held to 0 .. total whatever it holds.
__device__ __forceinline__ ExpertRows expert_rows(const int32_t* offsets, int e, int total) {
    const int lo = min(max(offsets[e], 0), total), hi = min(max(offsets[e + 1], 0), total);
    return {e, lo, max(hi - lo, 0)};
}

// Tiles of BM rows that all experts' rows make. Called by whole waves.
__device__ __forceinline__ int count_row_tiles(const int32_t* offsets, int experts, int total, int BM) {
    int tiles = 0;
    for (int e = __lane_id(); e < experts; e += 64) tiles += (expert_rows(offsets, e, total).count + BM - 1) / BM;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) tiles += __shfl_xor(tiles, d);
    return __builtin_amdgcn_readfirstlane(tiles);
}

// Row tile `tile` of all experts' tiles of BM rows, in expert order: its
// expert's rows and the tile's number among them; false past the last. Called by
// whole waves with a uniform `tile`; 64 experts a step, one a lane.
__device__ __forceinline__ bool find_row_tile(const int32_t* offsets, int experts, int total, int tile, int BM,
                                              ExpertRows* found, int* tile_in_expert) {
    const int lane = __lane_id();
    int before = 0;
    for (int e0 = 0; e0 < experts; e0 += 64) {
        const int e = e0 + lane;
        const ExpertRows r = e < experts ? expert_rows(offsets, e, total) : ExpertRows{0, 0, 0};
        const int tiles = (r.count + BM - 1) / BM;
        int upto = tiles;   // tiles of this step's experts up to and including this lane's
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(upto, d);
            if (lane >= d) upto += v;
        }
        const uint64_t past = __ballot(before + upto > tile);
        if (past != 0) {
            const int src = __builtin_ctzll(past);
            found->expert = e0 + src;
            found->first = __builtin_amdgcn_readlane(r.first, src);
            found->count = __builtin_amdgcn_readlane(r.count, src);
            *tile_in_expert = tile - before - __builtin_amdgcn_readlane(upto - tiles, src);
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

}  // namespace
}  // namespace mb

// Router: the top_k logits of each token, their softmax weights, and all
// assignments sorted by expert (stable in token order), plus the gradient.
//
// Choice. One wave per token; lane l holds logits l PER .. l PER + PER - 1,
// -inf for what cannot be chosen. Each of top_k rounds takes the wave's maximum
// (six DPP steps on the vector unit, no LDS), finds the first lane that holds it and that
// lane's first logit equal to it -- the lowest expert among equals -- and
// clears it. The weights are exp(l - m) / Z in fp32, m the largest logit.
//
// Order. Within an expert, assignments stand in token order (a token has an
// expert once), so the place of token t's assignment to expert e is the number
// of assignments to experts below e plus the number of tokens before t that
// chose e. Tokens go in groups of 64: one 64-bit mask per expert in LDS says
// which tokens of the group chose it, its population count is the group's
// count, and the count below bit t is t's rank. Masks are built with LDS
// ORs, whose result does not depend on their order. At most kMaxBlocks
// blocks, each over a run of groups, write their counts per expert ([expert][block]);
// a second kernel adds up the counts of earlier blocks and of lower experts
// (a wave per expert, a block's count a lane) and places. One block (up to 64 tokens) does both in
// one launch.
#include "experts_common.hpp"

#include <algorithm>
#include <type_traits>

namespace mb {
namespace {

constexpr int kGroup = 64;        // tokens per mask
constexpr int kMaxBlocks = 256;
constexpr int kWaves = 16;        // waves per block of the choosing kernel
constexpr float kLargest = 3.4028234663852886e38f;   // stands for +inf

template <int DT>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
    if constexpr (DT == MB_DT_FLOAT32) return static_cast<const float*>(p)[i];
    else return from_bits<DT>(static_cast<const uint16_t*>(p)[i]);
}

// Whether a logit can be chosen; +inf counts as the largest finite value.
__device__ __forceinline__ bool usable(float v) { return v > -__builtin_inff(); }   // false for NaN

// Lane 63's value of a reduction over the wave, by DPP: shifts by 1, 2, 4 and 8
// within rows of 16 lanes, then each row's last lane to the next row(s). Lanes without a source take `none`.
template <class Op>
__device__ __forceinline__ float wave_reduce(float v, float none, Op op) {
    const auto moved = [&](auto ctrl, float x) {
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none),
                                                                     __builtin_bit_cast(int, x),
                                                                     decltype(ctrl)::value, 0xF, 0xF, false));
    };
    v = op(v, moved(std::integral_constant<int, 0x111>{}, v));   // row_shr:1
    v = op(v, moved(std::integral_constant<int, 0x112>{}, v));
    v = op(v, moved(std::integral_constant<int, 0x114>{}, v));
    v = op(v, moved(std::integral_constant<int, 0x118>{}, v));   // row_shr:8
    v = op(v, moved(std::integral_constant<int, 0x142>{}, v));   // row_bcast:15
    v = op(v, moved(std::integral_constant<int, 0x143>{}, v));   // row_bcast:31
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ float wave_max(float v) {
    return wave_reduce(v, -__builtin_inff(), [](float a, float b) { return fmaxf(a, b); });
}
// The row_bcast steps add a row's total into every lane of the next row(s): in lane 63, each lane's value once.
__device__ __forceinline__ float wave_sum(float v) {
    return wave_reduce(v, 0.f, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// Logits l PER .. of a token as this lane holds them: -inf for what cannot be chosen.
template <int DT, int PER>
__device__ __forceinline__ void load_logits(const void* logits, int64_t base, int experts, int lane, float* v) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane * PER + i;
        v[i] = e < experts ? load_logit<DT>(logits, base + e) : -__builtin_inff();
        if (v[i] > kLargest) v[i] = kLargest;
        if (!usable(v[i])) v[i] = -__builtin_inff();
    }
}

// One token's choices by one wave: ids and weights of its top_k, written by lane j. Returns lane
// j's id (j < top_k), -1 for an empty choice.
template <int DT, int PER>
__device__ __forceinline__ int choose(const void* logits, int64_t base, int experts, int top_k, bool normalize,
                                      float* weights, int32_t* ids, int lane) {
    float v[PER], left[PER];
    load_logits<DT, PER>(logits, base, experts, lane, v);
#pragma unroll
    for (int i = 0; i < PER; ++i) left[i] = v[i];
    float mine = -__builtin_inff(), m = 0.f;   // choice `lane` of the token; the largest logit
    int id = -1;
    for (int j = 0; j < top_k; ++j) {
        float best = left[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) best = fmaxf(best, left[i]);
        const float top = wave_max(best);
        if (!usable(top)) break;   // uniform: no logit left
        if (j == 0) m = top;
        const int owner = __builtin_ctzll(__ballot(best == top));
        int at = 0;
#pragma unroll
        for (int i = PER - 1; i >= 0; --i) at = left[i] == top ? i : at;
        const int e = owner * PER + __builtin_amdgcn_readlane(at, owner);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (lane * PER + i == e) left[i] = -__builtin_inff();
        if (lane == j) {
            mine = top;
            id = e;
        }
    }
    const float e_mine = id >= 0 ? expf(mine - m) : 0.f;
    float z = e_mine;
    if (!normalize) {
        z = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) z += usable(v[i]) ? expf(v[i] - m) : 0.f;
    }
    z = wave_sum(z);
    if (lane < top_k) {
        weights[lane] = id >= 0 ? e_mine / z : 0.f;
        ids[lane] = id;
    }
    return id;
}

// Places one group's assignments from its masks; `start[e]` is where expert
// e's rows of this group begin.
__device__ __forceinline__ void place(const uint64_t* masks, const int* start, int64_t group, int64_t tokens,
                                      int top_k, const int32_t* ids, int32_t* rows, int32_t* slots) {
    const int64_t first = group * kGroup;
    const int here = (int)std::min<int64_t>(kGroup, tokens - first) * top_k;
    for (int a = threadIdx.x; a < here; a += blockDim.x) {
        const int t = a / top_k, e = ids[first * top_k + a];
        int slot = -1;
        if (e >= 0) {
            slot = start[e] + __popcll(masks[e] & ((1ull << t) - 1));
            rows[slot] = (int32_t)(first + t);
        }
        slots[first * top_k + a] = slot;
    }
}

// The exclusive prefix of counts[0 .. experts) into start[], and the total
// into start[experts], by the whole block (experts <= 1024 <= 64 * 16).
__device__ __forceinline__ void prefix(const int* counts, int* start, int experts) {
    const int lane = threadIdx.x & 63;
    if (threadIdx.x < 64) {
        int before = 0;
        for (int e0 = 0; e0 < experts; e0 += 64) {
            const int c = e0 + lane < experts ? counts[e0 + lane] : 0;
            int upto = c;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int v = __shfl_up(upto, d);
                if (lane >= d) upto += v;
            }
            if (e0 + lane < experts) start[e0 + lane] = before + upto - c;
            before += __shfl(upto, 63);
        }
        if (lane == 0) start[experts] = before;
    }
    __syncthreads();
}

// Choices of every token, and each block's count per expert. ONE: the only block, which also places.
template <int DT, int PER, bool ONE>
__global__ void __launch_bounds__(64 * kWaves)
route_choose_kernel(const void* __restrict__ logits, int64_t ld, int64_t tokens, int experts, int top_k,
                    int normalize, int groups_per_block, float* __restrict__ weights, int32_t* ids,
                    int32_t* __restrict__ counts, int32_t* __restrict__ offsets, int32_t* __restrict__ rows,
                    int32_t* __restrict__ slots) {
    __shared__ uint64_t masks[64 * PER];
    __shared__ int count[64 * PER], start[64 * PER + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t groups = (tokens + kGroup - 1) / kGroup;
    for (int e = threadIdx.x; e < experts; e += blockDim.x) count[e] = 0;
    for (int i = 0; i < groups_per_block; ++i) {
        const int64_t group = (int64_t)blockIdx.x * groups_per_block + i;
        if (group >= groups) break;
        for (int e = threadIdx.x; e < experts; e += blockDim.x) masks[e] = 0;
        __syncthreads();
        for (int t = wave; t < kGroup; t += kWaves) {
            const int64_t token = group * kGroup + t;
            if (token >= tokens) break;
            const int id = choose<DT, PER>(logits, token * ld, experts, top_k, normalize != 0,
                                           weights + token * top_k, ids + token * top_k, lane);
            if (lane < top_k && id >= 0)
                atomicOr(reinterpret_cast<unsigned long long*>(&masks[id]), 1ull << t);
        }
        __syncthreads();
        for (int e = threadIdx.x; e < experts; e += blockDim.x) count[e] += __popcll(masks[e]);
        if constexpr (!ONE) __syncthreads();
    }
    if constexpr (ONE) {
        __syncthreads();
        prefix(count, start, experts);
        for (int e = threadIdx.x; e <= experts; e += blockDim.x) offsets[e] = start[e];
        for (int p = start[experts] + threadIdx.x; p < (int)tokens * top_k; p += blockDim.x) rows[p] = -1;
        place(masks, start, 0, tokens, top_k, ids, rows, slots);
    } else {
        for (int e = threadIdx.x; e < experts; e += blockDim.x) counts[(int64_t)e * gridDim.x + blockIdx.x] = count[e];
    }
}

// Places every block's assignments: the counts of all blocks give offsets,
// those of earlier blocks this block's start in each expert.
__global__ void __launch_bounds__(64 * kWaves)
route_place_kernel(const int32_t* __restrict__ counts, int blocks, int64_t tokens, int experts, int top_k,
                   int groups_per_block, const int32_t* __restrict__ ids, int32_t* __restrict__ offsets,
                   int32_t* __restrict__ rows, int32_t* __restrict__ slots) {
    __shared__ uint64_t masks[MB_ROUTE_MAX_EXPERTS];
    __shared__ int total[MB_ROUTE_MAX_EXPERTS], start[MB_ROUTE_MAX_EXPERTS + 1], earlier[MB_ROUTE_MAX_EXPERTS];
    const int64_t groups = (tokens + kGroup - 1) / kGroup;
    const int lane = threadIdx.x & 63;
    for (int e = threadIdx.x >> 6; e < experts; e += kWaves) {
        int before = 0, all = 0;
#pragma unroll
        for (int b0 = 0; b0 < kMaxBlocks; b0 += 64) {
            const int b = b0 + lane, c = b < blocks ? counts[(int64_t)e * blocks + b] : 0;
            before += b < (int)blockIdx.x ? c : 0;
            all += c;
        }
        before = wave_sum(before);
        all = wave_sum(all);
        if (lane == 0) {
            earlier[e] = before;
            total[e] = all;
        }
    }
    __syncthreads();
    prefix(total, start, experts);
    if (blockIdx.x == 0) {
        for (int e = threadIdx.x; e <= experts; e += blockDim.x) offsets[e] = start[e];
    }
    const int64_t assignments = tokens * top_k;
    for (int64_t p = start[experts] + (int64_t)blockIdx.x * blockDim.x + threadIdx.x; p < assignments;
         p += (int64_t)blocks * blockDim.x)
        rows[p] = -1;
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += blockDim.x) start[e] += earlier[e];
    for (int i = 0; i < groups_per_block; ++i) {
        const int64_t group = (int64_t)blockIdx.x * groups_per_block + i;
        if (group >= groups) break;
        for (int e = threadIdx.x; e < experts; e += blockDim.x) masks[e] = 0;
        __syncthreads();
        const int64_t first = group * kGroup;
        const int here = (int)std::min<int64_t>(kGroup, tokens - first) * top_k;
        for (int a = threadIdx.x; a < here; a += blockDim.x) {
            const int id = ids[first * top_k + a];
            if (id >= 0) atomicOr(reinterpret_cast<unsigned long long*>(&masks[id]), 1ull << (a / top_k));
        }
        __syncthreads();
        place(masks, start, group, tokens, top_k, ids, rows, slots);
        __syncthreads();
        for (int e = threadIdx.x; e < experts; e += blockDim.x) start[e] += __popcll(masks[e]);
    }
}

// The logits' gradient, one wave per token: w (g - sum w g) on the chosen
// logits (normalize), or p (g - sum p g), p over all and g zero off the chosen.
template <int DT, int PER>
__global__ void __launch_bounds__(256)
route_grad_kernel(const void* __restrict__ logits, int64_t ld, const int32_t* __restrict__ ids,
                  const float* __restrict__ grad_weights, int64_t tokens, int experts, int top_k, int normalize,
                  void* __restrict__ grad_logits, int64_t ld_grad) {
    const int lane = threadIdx.x & 63;
    const int64_t token = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (token >= tokens) return;
    int id = -1;
    float g = 0.f;
    if (lane < top_k) {
        id = ids[token * top_k + lane];
        g = grad_weights[token * top_k + lane];
        if (id < 0 || id >= experts) id = -1;
    }
    float v[PER], gv[PER];
    bool chosen[PER];
    load_logits<DT, PER>(logits, token * ld, experts, lane, v);
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        chosen[i] = false;
        gv[i] = 0.f;
        m = fmaxf(m, v[i]);
    }
    for (int j = 0; j < top_k; ++j) {
        const int c = __builtin_amdgcn_readlane(id, j);
        const float gj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, g), j));
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (c == lane * PER + i) {
                chosen[i] = true;
                gv[i] = gj;
            }
    }
    m = wave_max(m);
    float p[PER], z = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        p[i] = usable(v[i]) && (chosen[i] || !normalize) ? expf(v[i] - m) : 0.f;
        z += p[i];
        dot += p[i] * gv[i];
    }
    z = wave_sum(z);
    dot = wave_sum(dot);
    const float inv = z > 0.f ? 1.f / z : 0.f;
    dot *= inv;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane * PER + i;
        if (e >= experts) continue;
        const float out = p[i] * inv * (gv[i] - dot);
        if constexpr (DT == MB_DT_FLOAT32) static_cast<float*>(grad_logits)[token * ld_grad + e] = out;
        else static_cast<uint16_t*>(grad_logits)[token * ld_grad + e] = to_bits<DT>(out);
    }
}

// f(integral_constant logits per lane): the experts held by one lane, a power of two up to 16.
template <class F>
int with_per_lane(int experts, F f) {
    if (experts <= 64) return f(std::integral_constant<int, 1>{});
    if (experts <= 128) return f(std::integral_constant<int, 2>{});
    if (experts <= 256) return f(std::integral_constant<int, 4>{});
    return f(std::integral_constant<int, 16>{});
}
template <class F>
int with_logit_type(int dtype, F f) {
    if (dtype == MB_DT_FLOAT32) return f(std::integral_constant<int, MB_DT_FLOAT32>{});
    if (dtype == MB_DT_BFLOAT16) return f(std::integral_constant<int, MB_DT_BFLOAT16>{});
    return f(std::integral_constant<int, MB_DT_FLOAT16>{});
}

int route_blocks(int64_t tokens) {
    return (int)std::min<int64_t>(kMaxBlocks, (tokens + kGroup - 1) / kGroup);
}

}  // namespace

size_t route_workspace(int64_t tokens, int experts) {
    const int blocks = route_blocks(tokens);
    return blocks <= 1 ? 0 : (size_t)blocks * experts * sizeof(int32_t);
}

int route_launch(int dtype, const void* logits, int64_t ld, int64_t tokens, int experts, int top_k, bool normalize,
                 float* weights, int32_t* expert_ids, int32_t* offsets, int32_t* rows, int32_t* slots,
                 void* workspace, hipStream_t stream) {
    int blocks = std::max(1, route_blocks(tokens));
    const int64_t groups = (tokens + kGroup - 1) / kGroup;
    const int per_block = (int)((groups + blocks - 1) / blocks);
    auto* counts = static_cast<int32_t*>(workspace);
    return with_logit_type(dtype, [&](auto dt) {
        return with_per_lane(experts, [&](auto per) {
            constexpr int DT = decltype(dt)::value, PER = decltype(per)::value;
            if (blocks == 1) {
                hipLaunchKernelGGL((route_choose_kernel<DT, PER, true>), dim3(1), dim3(64 * kWaves), 0, stream, logits,
                                   ld, tokens, experts, top_k, (int)normalize, per_block, weights, expert_ids, counts,
                                   offsets, rows, slots);
                MB_HIP_TRY(hipGetLastError());
                return (int)MB_OK;
            }
            hipLaunchKernelGGL((route_choose_kernel<DT, PER, false>), dim3(blocks), dim3(64 * kWaves), 0, stream,
                               logits, ld, tokens, experts, top_k, (int)normalize, per_block, weights, expert_ids,
                               counts, offsets, rows, slots);
            MB_HIP_TRY(hipGetLastError());
            hipLaunchKernelGGL(route_place_kernel, dim3(blocks), dim3(64 * kWaves), 0, stream, counts, blocks, tokens, experts,
                               top_k, per_block, expert_ids, offsets, rows, slots);
            MB_HIP_TRY(hipGetLastError());
            return (int)MB_OK;
        });
    });
}

int route_grad_launch(int dtype, const void* logits, int64_t ld, const int32_t* expert_ids, const float* grad_weights,
                      int64_t tokens, int experts, int top_k, bool normalize, void* grad_logits, int64_t ld_grad,
                      hipStream_t stream) {
    return with_logit_type(dtype, [&](auto dt) {
        return with_per_lane(experts, [&](auto per) {
            constexpr int DT = decltype(dt)::value, PER = decltype(per)::value;
            hipLaunchKernelGGL((route_grad_kernel<DT, PER>), dim3((unsigned)((tokens + 3) / 4)), dim3(256), 0, stream,
                               logits, ld, expert_ids, grad_weights, tokens, experts, top_k, (int)normalize,
                               grad_logits, ld_grad);
            MB_HIP_TRY(hipGetLastError());
            return (int)MB_OK;
        });
    });
}

}  // namespace mb

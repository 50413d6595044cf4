// Router: the top_k logits of each token, their softmax weights, and all
// assignments sorted by expert (stable in token order), plus the gradient.
//
// Choice. One wave per token; lane l holds logits l, l + 64, ... as 64-bit keys
// whose order is the wanted one: the logit's bits mapped so that unsigned
// order is float order, then the complement of the expert's number, so equal logits
// go to the lower expert and every key is distinct. -inf and NaN have key 0. Each of top_k
// rounds takes the wave's maximum and clears it. The weights are
// exp(l - m) / Z in fp32, m the largest logit.
//
// Order. Within an expert, assignments stand in token order (a token has an
// expert once), so the place of token t's assignment to expert e is the number
// of assignments to experts below e plus the number of tokens before t that
// chose e. Tokens go in groups of 64: one 64-bit mask per expert in LDS says
// which tokens of the group chose it, its population count is the group's
// count, and the count below bit t is t's rank. Masks are built with LDS
// ORs, whose result does not depend on their order. At most kMaxBlocks
// blocks, each over a run of groups, write their counts per expert;
// a second kernel adds up the counts of earlier blocks and of lower experts and places.
// One block (up to 64 tokens) does both in one launch.
#include "experts_common.hpp"

#include <algorithm>

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

// Float order as unsigned order; every usable logit maps above 0.
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __builtin_bit_cast(unsigned, v == 0.f ? 0.f : v);   // -0 and +0 tie
    return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(unsigned u) {
    return __builtin_bit_cast(float, (u >> 31) ? u & 0x7FFFFFFFu : ~u);
}

__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const uint64_t o = __shfl_xor(v, d);
        v = o > v ? o : v;
    }
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// One token's choices by one wave: ids and weights of its top_k, written by lane j. Returns lane
// j's id (j < top_k), -1 for an empty choice.
template <int DT, int PER>
__device__ __forceinline__ int choose(const void* logits, int64_t base, int experts, int top_k, bool normalize,
                                      float* weights, int32_t* ids, int lane) {
    uint64_t key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane + 64 * i;
        float v = e < experts ? load_logit<DT>(logits, base + e) : -__builtin_inff();
        if (v > kLargest) v = kLargest;
        key[i] = usable(v) ? ((uint64_t)ordered(v) << 32) | (unsigned)~e : 0;
    }
    uint64_t local[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) local[i] = key[i];
    uint64_t mine = 0;   // choice `lane` of the token
    float m = 0.f;
    for (int j = 0; j < top_k; ++j) {
        uint64_t best = local[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) best = local[i] > best ? local[i] : best;
        best = wave_max(best);
        if (j == 0) m = unordered((unsigned)(best >> 32));
        if (best == 0) break;   // uniform: no logit left
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (local[i] == best) local[i] = 0;
        if (lane == j) mine = best;
    }
    const float e_mine = mine ? expf(unordered((unsigned)(mine >> 32)) - m) : 0.f;
    float z = e_mine;
    if (!normalize) {
        z = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (key[i]) z += expf(unordered((unsigned)(key[i] >> 32)) - m);
    }
    z = wave_sum(z);
    const int id = mine ? (int)~(unsigned)mine : -1;
    if (lane < top_k) {
        weights[lane] = mine ? e_mine / z : 0.f;
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
        for (int e = threadIdx.x; e < experts; e += blockDim.x) counts[(int64_t)blockIdx.x * experts + e] = count[e];
    }
}

// Places every block's assignments: the counts of all blocks give offsets,
// those of earlier blocks this block's start in each expert.
__global__ void __launch_bounds__(256)
route_place_kernel(const int32_t* __restrict__ counts, int blocks, int64_t tokens, int experts, int top_k,
                   int groups_per_block, const int32_t* __restrict__ ids, int32_t* __restrict__ offsets,
                   int32_t* __restrict__ rows, int32_t* __restrict__ slots) {
    __shared__ uint64_t masks[MB_ROUTE_MAX_EXPERTS];
    __shared__ int total[MB_ROUTE_MAX_EXPERTS], start[MB_ROUTE_MAX_EXPERTS + 1], earlier[MB_ROUTE_MAX_EXPERTS];
    const int64_t groups = (tokens + kGroup - 1) / kGroup;
    for (int e = threadIdx.x; e < experts; e += blockDim.x) {
        int before = 0, all = 0;
        for (int b = 0; b < blocks; ++b) {
            const int c = counts[(int64_t)b * experts + e];
            if (b < (int)blockIdx.x) before += c;
            all += c;
        }
        earlier[e] = before;
        total[e] = all;
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
    bool live[PER], chosen[PER];
    float m = -kLargest;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane + 64 * i;
        v[i] = e < experts ? load_logit<DT>(logits, token * ld + e) : -__builtin_inff();
        if (v[i] > kLargest) v[i] = kLargest;
        live[i] = usable(v[i]);
        chosen[i] = false;
        gv[i] = 0.f;
        if (live[i]) m = fmaxf(m, v[i]);
    }
    for (int j = 0; j < top_k; ++j) {
        const int c = __shfl(id, j);
        const float gj = __shfl(g, j);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (c == lane + 64 * i) {
                chosen[i] = true;
                gv[i] = gj;
            }
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    float p[PER], z = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        p[i] = live[i] && (chosen[i] || !normalize) ? expf(v[i] - m) : 0.f;
        z += p[i];
        dot += p[i] * gv[i];
    }
    z = wave_sum(z);
    dot = wave_sum(dot);
    const float inv = z > 0.f ? 1.f / z : 0.f;
    dot *= inv;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane + 64 * i;
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
            hipLaunchKernelGGL(route_place_kernel, dim3(blocks), dim3(256), 0, stream, counts, blocks, tokens, experts,
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

// Router: the top_k logits of each token, their softmax weights, and all
// assignments sorted by expert (stable in token order), plus the gradient.
//
// Choice. 16 lanes per token (64 past 256 experts or 16 choices); lane l of
// them holds logits l PER .. l PER + PER - 1, -inf for what cannot be chosen.
// Each of top_k rounds takes the token's maximum and then the lowest expert
// that has it, by rotations within the 16 lanes (DPP: no LDS), and clears it.
// The weights are exp(l - m) / Z in fp32, m the largest logit. The rounds' two
// reductions, one after the other, are its time, and four tokens share each
// instruction: 8.2 us at 16384 x 128 top 8, against 17.5 us with a whole wave per token.
//
// Order. Within an expert, assignments stand in token order (a token has an
// expert once), so the place of token t's assignment to expert e is the number
// of assignments to experts below e plus the number of tokens before t that
// chose e. Tokens go in groups of 64: one 64-bit mask per expert in LDS says
// which tokens of the group chose it, its population count is the group's
// count, and the count below bit t is t's rank. Masks are built with LDS
// ORs, whose result does not depend on their order. At most kMaxBlocks blocks,
// each over a run of groups, write their counts per expert ([expert][block]); a
// second kernel adds up the counts of earlier blocks and of lower experts (a
// wave per expert, a block's count a lane: 8 us where a thread per expert took
// 64) and places. One block (up to 64 tokens) does both in one launch, 3.4 us.
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

template <int CTRL, class T>
__device__ __forceinline__ T dpp(T x, T none) {   // `none` for lanes without a source
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, x),
                                                             CTRL, 0xF, 0xF, false));
}

// A reduction over a token's lanes, in all of them. 16: rotations within the
// row. 64: shifts by 1, 2, 4 and 8 within rows, then each row's last lane into
// the next row(s), which leaves in lane 63 each lane's value once.
template <int LANES, class T, class Op>
__device__ __forceinline__ T reduce(T v, T none, Op op) {
    if constexpr (LANES == 16) {
        v = op(v, dpp<0x128>(v, none));   // row_ror:8
        v = op(v, dpp<0x124>(v, none));
        v = op(v, dpp<0x122>(v, none));
        return op(v, dpp<0x121>(v, none));
    } else {
        v = op(v, dpp<0x111>(v, none));   // row_shr:1
        v = op(v, dpp<0x112>(v, none));
        v = op(v, dpp<0x114>(v, none));
        v = op(v, dpp<0x118>(v, none));
        v = op(v, dpp<0x142>(v, none));   // row_bcast:15
        v = op(v, dpp<0x143>(v, none));   // row_bcast:31
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
    }
}
template <int LANES>
__device__ __forceinline__ float max_of(float v) {
    return reduce<LANES>(v, -__builtin_inff(), [](float a, float b) { return fmaxf(a, b); });
}
template <int LANES>
__device__ __forceinline__ int min_of(int v) {
    return reduce<LANES>(v, 0x7FFFFFFF, [](int a, int b) { return min(a, b); });
}
template <int LANES, class T>
__device__ __forceinline__ T sum_of(T v) {
    return reduce<LANES>(v, T(0), [](T a, T b) { return a + b; });
}

// Logits l PER .. of a token as this lane holds them: -inf for what cannot be chosen.
template <int DT, int PER>
__device__ __forceinline__ void load_logits(const void* logits, int64_t base, int experts, int lane, float* v) {
    if (lane * PER + PER <= experts) {   // one load of PER elements, on any element
        if constexpr (DT == MB_DT_FLOAT32) {
            typedef float vec __attribute__((ext_vector_type(PER), aligned(4)));
            const vec p = *reinterpret_cast<const vec*>(static_cast<const float*>(logits) + base + lane * PER);
#pragma unroll
            for (int i = 0; i < PER; ++i) v[i] = p[i];
        } else {
            typedef uint16_t vec __attribute__((ext_vector_type(PER), aligned(2)));
            const vec p = *reinterpret_cast<const vec*>(static_cast<const uint16_t*>(logits) + base + lane * PER);
#pragma unroll
            for (int i = 0; i < PER; ++i) v[i] = from_bits<DT>(p[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane * PER + i;
            v[i] = e < experts ? load_logit<DT>(logits, base + e) : -__builtin_inff();
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (v[i] > kLargest) v[i] = kLargest;
        if (!usable(v[i])) v[i] = -__builtin_inff();
    }
}

// One token's choices by LANES lanes: ids and weights of its top_k, written by lane j. Returns lane
// j's id (j < top_k), -1 for an empty choice.
template <int DT, int LANES, int PER>
__device__ __forceinline__ int choose(const void* logits, int64_t base, int experts, int top_k, bool normalize,
                                      float* weights, int32_t* ids, int lane) {
    float v[PER], left[PER];
    load_logits<DT, PER>(logits, base, experts, lane, v);
#pragma unroll
    for (int i = 0; i < PER; ++i) left[i] = v[i];
    float mine = 0.f, m = 0.f;   // choice `lane` of the token; the largest logit
    int id = -1;
    for (int j = 0; j < top_k; ++j) {
        float best = left[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) best = fmaxf(best, left[i]);
        const float top = max_of<LANES>(best);
        int at = 0x7FFFFFFF;
#pragma unroll
        for (int i = PER - 1; i >= 0; --i) at = left[i] == top ? lane * PER + i : at;
        const int e = min_of<LANES>(at);
#pragma unroll
        for (int i = 0; i < PER; ++i) left[i] = lane * PER + i == e ? -__builtin_inff() : left[i];
        if (j == 0) m = usable(top) ? top : 0.f;
        if (lane == j && usable(top)) {
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
    z = sum_of<LANES>(z);
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
template <int DT, int LANES, int PER, bool ONE>
__global__ void __launch_bounds__(64 * kWaves)
route_choose_kernel(const void* __restrict__ logits, int64_t ld, int64_t tokens, int experts, int top_k,
                    int normalize, int groups_per_block, float* __restrict__ weights, int32_t* ids,
                    int32_t* __restrict__ counts, int32_t* __restrict__ offsets, int32_t* __restrict__ rows,
                    int32_t* __restrict__ slots) {
    __shared__ uint64_t masks[LANES * PER];
    __shared__ int count[LANES * PER], start[LANES * PER + 1];
    const int lane = threadIdx.x & (LANES - 1), own = threadIdx.x / LANES;   // lane, and which token's lanes
    const int64_t groups = (tokens + kGroup - 1) / kGroup;
    for (int e = threadIdx.x; e < experts; e += blockDim.x) count[e] = 0;
    for (int i = 0; i < groups_per_block; ++i) {
        const int64_t group = (int64_t)blockIdx.x * groups_per_block + i;
        if (group >= groups) break;
        for (int e = threadIdx.x; e < experts; e += blockDim.x) masks[e] = 0;
        __syncthreads();
        for (int t = own; t < kGroup; t += 64 * kWaves / LANES) {
            const int64_t token = group * kGroup + t;
            if (token >= tokens) break;
            const int id = choose<DT, LANES, PER>(logits, token * ld, experts, top_k, normalize != 0,
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
        before = sum_of<64>(before);
        all = sum_of<64>(all);
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

// The logits' gradient, LANES lanes per token: w (g - sum w g) on the chosen
// logits (normalize), or p (g - sum p g), p over all and g zero off the chosen.
template <int DT, int LANES, int PER>
__global__ void __launch_bounds__(256)
route_grad_kernel(const void* __restrict__ logits, int64_t ld, const int32_t* __restrict__ ids,
                  const float* __restrict__ grad_weights, int64_t tokens, int experts, int top_k, int normalize,
                  void* __restrict__ grad_logits, int64_t ld_grad) {
    const int lane = threadIdx.x & (LANES - 1);
    const int64_t token = (int64_t)block_number() * (256 / LANES) + threadIdx.x / LANES;
    if (token >= tokens) return;   // all of a token's lanes: no reduction misses any
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
        const int c = __shfl(id, j, LANES);
        const float gj = __shfl(g, j, LANES);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (c == lane * PER + i) {
                chosen[i] = true;
                gv[i] = gj;
            }
    }
    m = max_of<LANES>(m);
    float p[PER], z = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        p[i] = usable(v[i]) && (chosen[i] || !normalize) ? expf(v[i] - m) : 0.f;
        z += p[i];
        dot += p[i] * gv[i];
    }
    z = sum_of<LANES>(z);
    dot = sum_of<LANES>(dot);
    const float inv = z > 0.f ? 1.f / z : 0.f;
    dot *= inv;
    float out[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) out[i] = p[i] * inv * (gv[i] - dot);
    const auto store = [&](auto* to, auto round) {
        typedef std::remove_pointer_t<decltype(to)> T;
        typedef T vec __attribute__((ext_vector_type(PER), aligned(sizeof(T))));
        to += token * ld_grad + lane * PER;
        if (lane * PER + PER <= experts) {
            vec whole;
#pragma unroll
            for (int i = 0; i < PER; ++i) whole[i] = round(out[i]);
            *reinterpret_cast<vec*>(to) = whole;
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (lane * PER + i < experts) to[i] = round(out[i]);
        }
    };
    if constexpr (DT == MB_DT_FLOAT32) store(static_cast<float*>(grad_logits), [](float f) { return f; });
    else store(static_cast<uint16_t*>(grad_logits), [](float f) { return to_bits<DT>(f); });
}

// f(lanes per token, logits per lane).
template <class F>
int with_lanes(int experts, int top_k, F f) {
    const auto call = [&](auto lanes, auto per) { return f(lanes, per); };
    constexpr std::integral_constant<int, 16> row;
    constexpr std::integral_constant<int, 64> wave;
    if (experts > 256) return call(wave, std::integral_constant<int, 16>{});
    if (top_k > 16) return call(wave, std::integral_constant<int, 4>{});
    if (experts <= 32) return call(row, std::integral_constant<int, 2>{});
    if (experts <= 64) return call(row, std::integral_constant<int, 4>{});
    if (experts <= 128) return call(row, std::integral_constant<int, 8>{});
    return call(row, std::integral_constant<int, 16>{});
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
        return with_lanes(experts, top_k, [&](auto lanes, auto per) {
            constexpr int DT = decltype(dt)::value, LANES = decltype(lanes)::value, PER = decltype(per)::value;
            if (blocks == 1) {
                hipLaunchKernelGGL((route_choose_kernel<DT, LANES, PER, true>), dim3(1), dim3(64 * kWaves), 0, stream,
                                   logits, ld, tokens, experts, top_k, (int)normalize, per_block, weights, expert_ids, counts,
                                   offsets, rows, slots);
                MB_HIP_TRY(hipGetLastError());
                return (int)MB_OK;
            }
            hipLaunchKernelGGL((route_choose_kernel<DT, LANES, PER, false>), dim3(blocks), dim3(64 * kWaves), 0, stream,
                               logits, ld, tokens, experts, top_k, (int)normalize, per_block, weights, expert_ids,
                               counts, offsets, rows, slots);
            MB_HIP_TRY(hipGetLastError());
            hipLaunchKernelGGL(route_place_kernel, dim3(blocks), dim3(64 * kWaves), 0, stream, counts, blocks, tokens,
                               experts, top_k, per_block, expert_ids, offsets, rows, slots);
            MB_HIP_TRY(hipGetLastError());
            return (int)MB_OK;
        });
    });
}

int route_grad_launch(int dtype, const void* logits, int64_t ld, const int32_t* expert_ids, const float* grad_weights,
                      int64_t tokens, int experts, int top_k, bool normalize, void* grad_logits, int64_t ld_grad,
                      hipStream_t stream) {
    return with_logit_type(dtype, [&](auto dt) {
        return with_lanes(experts, top_k, [&](auto lanes, auto per) {
            constexpr int DT = decltype(dt)::value, LANES = decltype(lanes)::value, PER = decltype(per)::value;
            constexpr int kTokens = 256 / LANES;   // per block
            hipLaunchKernelGGL((route_grad_kernel<DT, LANES, PER>), launch_grid((tokens + kTokens - 1) / kTokens),
                               dim3(256), 0, stream, logits, ld, expert_ids, grad_weights, tokens, experts, top_k,
                               (int)normalize,
                               grad_logits, ld_grad);
            MB_HIP_TRY(hipGetLastError());
            return (int)MB_OK;
        });
    });
}

}  // namespace mb

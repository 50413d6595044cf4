// The way back from sorted rows to tokens, and its gradient.
//
//   out[t] = sum over j of w[t][j] y[slots[t][j]]            (combine)
//   grad_y[slots[t][j]] = w[t][j] g[t]                        (gradient)
//   grad_w[t][j] = <g[t], y[slots[t][j]]>
//
// Memory-bound: each row is read once and each output row written once, 16
// bytes a lane, all of a token's rows in flight together. Sums are fp32, in
// order of j. Rows off 16 bytes take the same loads (the hardware
// takes 16 bytes at any address); the columns past the last whole 8 go one by one.
#include "experts_common.hpp"

#include <type_traits>

namespace mb {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 8;      // rows of a token in flight together

// 8 columns from column c of a row, zeros past N. STREAM: nontemporal, for
// rows read or written once that together pass the caches (8192 tokens of
// 4 x 4096: 66 us with it, 85 without; the gradient, 114 without and 122 with).
template <int DT, bool STREAM>
__device__ __forceinline__ void load_columns(const uint16_t* row, int64_t c, int64_t N, float* v) {
    if (c + 8 <= N) {
        const auto* from = reinterpret_cast<const u32x4_any*>(row + c);
        const u32x4 p = STREAM ? __builtin_nontemporal_load(from) : *from;
        unpack8<DT>(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < N ? from_bits<DT>(row[c + i]) : 0.f;
    }
}
template <int DT, bool STREAM>
__device__ __forceinline__ void store_columns(uint16_t* row, int64_t c, int64_t N, const float* v) {
    if (c + 8 <= N) {
        auto* to = reinterpret_cast<u32x4_any*>(row + c);
        if constexpr (STREAM) __builtin_nontemporal_store(pack8<DT>(v), to);
        else *to = pack8<DT>(v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < N) row[c + i] = to_bits<DT>(v[i]);
    }
}

// One thread per 8 columns of a token: 2^lanes_log2 threads side by side on
// one token's columns, `parts` such runs per token. K: rows in flight together.
template <int DT, int K>
__global__ void __launch_bounds__(kThreads)
combine_kernel(const uint16_t* __restrict__ y, int64_t ldy, int64_t y_rows, const float* __restrict__ weights,
               const int32_t* __restrict__ slots, int64_t tokens, int top_k, int64_t N, uint16_t* __restrict__ out,
               int64_t ldo, int lanes_log2, unsigned parts) {
    const unsigned run = (unsigned)(((uint64_t)block_number() * kThreads + threadIdx.x) >> lanes_log2);
    const unsigned token = parts == 1 ? run : run / parts;
    const int64_t t = token;
    const int64_t c = ((int64_t)((run - token * parts) << lanes_log2) + (threadIdx.x & ((1u << lanes_log2) - 1))) * 8;
    if (t >= tokens || c >= N) return;
    float sum[8] = {};
    for (int j0 = 0; j0 < top_k; j0 += K) {
        float v[K][8], w[K];
#pragma unroll
        for (int u = 0; u < K; ++u) {
            w[u] = 0.f;
            const int64_t a = t * top_k + j0 + u;
            const int64_t slot = j0 + u < top_k ? slots[a] : -1;
            if (slot >= 0 && slot < y_rows) {
                load_columns<DT, true>(y + slot * ldy, c, N, v[u]);
                w[u] = weights ? weights[a] : 1.f;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[u][e] = 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < K; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] = fmaf(w[u], v[u][e], sum[e]);
    }
    store_columns<DT, true>(out + t * ldo, c, N, sum);
}

// One block per token: its grad_y rows, and the dot products over its columns.
template <int DT>
__global__ void __launch_bounds__(kThreads)
combine_grad_kernel(const uint16_t* __restrict__ g, int64_t ldg, const uint16_t* __restrict__ y, int64_t ldy,
                    int64_t y_rows, const float* __restrict__ weights, const int32_t* __restrict__ slots,
                    int64_t tokens, int top_k, int64_t N, uint16_t* __restrict__ grad_y, int64_t ld_grad_y,
                    float* __restrict__ grad_weights) {
    __shared__ float part[kThreads / 64][kBatch];
    const int64_t t = block_number();
    if (t >= tokens) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int j0 = 0; j0 < top_k; j0 += kBatch) {
        int64_t slot[kBatch];
        float w[kBatch], dot[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int64_t a = t * top_k + j0 + u;
            slot[u] = j0 + u < top_k ? slots[a] : -1;
            if (slot[u] >= y_rows) slot[u] = -1;
            w[u] = slot[u] >= 0 && weights ? weights[a] : 1.f;
            dot[u] = 0.f;
        }
        for (int64_t c = (int64_t)threadIdx.x * 8; c < N; c += kThreads * 8) {
            float gv[8];
            load_columns<DT, false>(g + t * ldg, c, N, gv);
            if (grad_weights != nullptr) {
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    if (slot[u] < 0) continue;
                    float yv[8];
                    load_columns<DT, false>(y + slot[u] * ldy, c, N, yv);
#pragma unroll
                    for (int e = 0; e < 8; ++e) dot[u] = fmaf(gv[e], yv[e], dot[u]);
                }
            }
            if (grad_y != nullptr) {
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    if (slot[u] < 0) continue;
                    float dv[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) dv[e] = w[u] * gv[e];
                    store_columns<DT, false>(grad_y + slot[u] * ld_grad_y, c, N, dv);
                }
            }
        }
        if (grad_weights != nullptr) {
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
#pragma unroll
                for (int d = 32; d > 0; d >>= 1) dot[u] += __shfl_xor(dot[u], d);
                if (lane == 0) part[wave][u] = dot[u];
            }
            __syncthreads();
            if (threadIdx.x < kBatch && j0 + (int)threadIdx.x < top_k) {
                float sum = 0.f;
#pragma unroll
                for (int v = 0; v < kThreads / 64; ++v) sum += part[v][threadIdx.x];
                grad_weights[t * top_k + j0 + threadIdx.x] = sum;
            }
            __syncthreads();
        }
    }
}

}  // namespace

int combine_launch(int dtype, const void* y, int64_t ldy, int64_t y_rows, const float* weights, const int32_t* slots,
                   int64_t tokens, int top_k, int64_t N, void* out, int64_t ldo, hipStream_t stream) {
    const int64_t chunks = (N + 7) / 8;
    int lanes_log2 = 0;
    while (lanes_log2 < 8 && (1 << lanes_log2) < chunks) ++lanes_log2;
    const int64_t parts = (chunks + (1 << lanes_log2) - 1) >> lanes_log2;
    const int64_t blocks = (((tokens * parts) << lanes_log2) + kThreads - 1) / kThreads;
    const auto* yp = static_cast<const uint16_t*>(y);
    auto* op = static_cast<uint16_t*>(out);
    auto pick = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        return top_k == 1 ? combine_kernel<DT, 1> : top_k == 2 ? combine_kernel<DT, 2>
             : top_k <= 4 ? combine_kernel<DT, 4> : combine_kernel<DT, kBatch>;
    };
    auto kernel = dtype == MB_DT_FLOAT16 ? pick(std::integral_constant<int, MB_DT_FLOAT16>{})
                                         : pick(std::integral_constant<int, MB_DT_BFLOAT16>{});
    hipLaunchKernelGGL(kernel, launch_grid(blocks), dim3(kThreads), 0, stream, yp, ldy, y_rows, weights, slots,
                       tokens, top_k, N, op, ldo, lanes_log2, (unsigned)parts);
    MB_HIP_TRY(hipGetLastError());
    return MB_OK;
}

int combine_grad_launch(int dtype, const void* grad_out, int64_t ldg, const void* y, int64_t ldy, int64_t y_rows,
                        const float* weights, const int32_t* slots, int64_t tokens, int top_k, int64_t N, void* grad_y,
                        int64_t ld_grad_y, float* grad_weights, hipStream_t stream) {
    const auto* gp = static_cast<const uint16_t*>(grad_out);
    const auto* yp = static_cast<const uint16_t*>(y);
    auto* gy = static_cast<uint16_t*>(grad_y);
    auto kernel = dtype == MB_DT_FLOAT16 ? combine_grad_kernel<MB_DT_FLOAT16> : combine_grad_kernel<MB_DT_BFLOAT16>;
    hipLaunchKernelGGL(kernel, launch_grid(tokens), dim3(kThreads), 0, stream, gp, ldg, yp, ldy, y_rows, weights,
                       slots, tokens, top_k, N, gy, ld_grad_y, grad_weights);
    MB_HIP_TRY(hipGetLastError());
    return MB_OK;
}

}  // namespace mb

// The balance loss of a mixture-of-experts router for gfx950: how many of the
// tokens' slots each expert has, the mean of the tokens' probabilities for it, the
// loss that their products give, and the logits' gradient.  No counterpart in the
// reference, whose feed-forward layer is dense.
//
//   p_t = softmax(l_t) over all experts;  c_e = slots with id e;  n valid tokens
//   loss = coef E / (k n) sum_e c_e P_e,  P_e = sum_t p_te / n
//   dl_te = dloss coef E / (k n^2) p_te (c_e - sum_f p_tf c_f)
//
// A row's logits lie in the registers of L lanes as in the router's kernels.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "mi_common.hpp"
#include "mi_logits.hpp"
#include "mi_rowtype.hpp"

namespace mi {

namespace {

constexpr int kFwdThreads = 512;
constexpr int kFwdBlocks = 256;
constexpr int kOneTokens = 256;  // tokens of a call that one workgroup does alone
constexpr int kFinThreads = 1024;
constexpr int kBwdThreads = 256;
constexpr int kMaxGrid = 1 << 20;

// e^(v - max) of a row's logits, and 1 over their sum: 0 for a row of -inf alone; a
// NaN or +inf makes all of them NaN.
template <int L, int P>
__device__ __forceinline__ float softmax_terms(float (&v)[P]) {
    float top = v[0];
#pragma unroll
    for (int p = 1; p < P; ++p) top = fmaxf(top, v[p]);
    top = group_max<L>(top);
    if (top == -__builtin_inff()) top = 0.0f;
    float s = 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        v[p] = __builtin_amdgcn_exp2f((v[p] - top) * kLog2e);
        s += v[p];
    }
    s = group_sum<L>(s);
    return s == 0.0f ? 0.0f : 1.0f / s;
}

// The loss from all experts' counts and mean probabilities, by a whole workgroup of NT
// threads, in 64 bits.  Thread 0 has it.
template <int NT>
__device__ __forceinline__ float loss_of(const int* count, const float* prob, int experts, int k,
                                         float coef, double* red) {
    double s = 0.0;
    for (int e = threadIdx.x; e < experts; e += NT)
        s += static_cast<double>(count[e]) * static_cast<double>(prob[e]);
    red[threadIdx.x] = s;
    __syncthreads();
#pragma unroll
    for (int h = NT / 2; h >= 1; h /= 2) {
        if (static_cast<int>(threadIdx.x) < h) red[threadIdx.x] += red[threadIdx.x + h];
        __syncthreads();
    }
    const int n = count[experts];
    return n == 0 ? 0.0f
                  : static_cast<float>(red[0] * static_cast<double>(coef) * experts /
                                       (static_cast<double>(k) * n));
}

// Sums of the probabilities and counts over a workgroup's tokens: a lane adds its experts'
// over its rows in registers, the waves' sums meet in LDS, in order.  ONE: the only
// workgroup, which writes the results; else a partial row of both.
template <int T, int L, int P, bool ONE>
__global__ __launch_bounds__(kFwdThreads) void balance_fwd_kernel(
    const void* __restrict__ logits, const int* __restrict__ ids, int tokens, int experts, int k,
    const unsigned char* __restrict__ valid, float* __restrict__ part, int* __restrict__ part_n,
    int* __restrict__ counts, float* __restrict__ probs, float* __restrict__ loss, float coef) {
    constexpr int PER = kFwdThreads / L, WAVES = kFwdThreads / kWave;
    constexpr int N = kPiece<T, P>;
    __shared__ __align__(16) float sums[WAVES][L * P];
    __shared__ int count[kMaxExperts + 1];
    [[maybe_unused]] __shared__ double red[ONE ? kFwdThreads : 1];
    const int gl = threadIdx.x & (L - 1);
    const int wave = threadIdx.x / kWave;
    for (int e = threadIdx.x; e <= experts; e += kFwdThreads) count[e] = 0;
    __syncthreads();
    float acc[P];
#pragma unroll
    for (int p = 0; p < P; ++p) acc[p] = 0.0f;
    for (long long base = static_cast<long long>(blockIdx.x) * PER; base < tokens;
         base += static_cast<long long>(gridDim.x) * PER) {
        const long long want = base + threadIdx.x / L;
        const size_t row = want < tokens ? static_cast<size_t>(want)
                                         : static_cast<size_t>(tokens) - 1;
        const bool live = want < tokens && (!valid || valid[row] != 0);
        const int id = live && gl < k ? ids[row * k + gl] : -1;
        float v[P];
        load_logits<T, L, P>(logits, row, tokens, gl, experts, v);
        const float inv = softmax_terms<L, P>(v);
#pragma unroll
        for (int p = 0; p < P; ++p) acc[p] += live ? v[p] * inv : 0.0f;
        if (id >= 0 && id < experts) atomicAdd(&count[id], 1);
        if (live && gl == 0) atomicAdd(&count[experts], 1);
    }
    // the wave's rows, then the waves
#pragma unroll
    for (int p = 0; p < P; ++p) {
        if constexpr (L == 16) {
            acc[p] += __shfl_xor(acc[p], 16);
            acc[p] += __shfl_xor(acc[p], 32);
        }
        if ((threadIdx.x & (kWave - 1)) < L)
            sums[wave][gl * N + step_expert<T, L, P>(p)] = acc[p];
    }
    __syncthreads();
    [[maybe_unused]] const float n = static_cast<float>(max(count[experts], 1));
    for (int e = threadIdx.x; e < experts; e += kFwdThreads) {
        float s = sums[0][e];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += sums[w][e];
        if constexpr (ONE) {
            sums[0][e] = s / n;
            probs[e] = s / n;
            counts[e] = count[e];
        } else {
            part[static_cast<size_t>(blockIdx.x) * experts + e] = s;
            part_n[static_cast<size_t>(blockIdx.x) * (experts + 1) + e] = count[e];
        }
    }
    if constexpr (ONE) {
        __syncthreads();
        const float l = loss_of<kFwdThreads>(count, sums[0], experts, k, coef, red);
        if (threadIdx.x == 0) {
            *loss = l;
            counts[experts] = count[experts];
        }
    } else if (threadIdx.x == 0) {
        part_n[static_cast<size_t>(blockIdx.x) * (experts + 1) + experts] = count[experts];
    }
}

// Adds the partial rows, in slices of them side by side, each in order.
__global__ __launch_bounds__(kFinThreads) void balance_finish_kernel(
    const float* __restrict__ part, const int* __restrict__ part_n, int blocks, int experts, int k,
    float coef, int* __restrict__ counts, float* __restrict__ probs, float* __restrict__ loss) {
    __shared__ float prob[kFinThreads];
    __shared__ int count[kFinThreads + 1];
    __shared__ int total;
    __shared__ double red[kFinThreads];
    int width = 1;
    while (width < experts) width *= 2;
    const int slices = kFinThreads / width;
    const int e = threadIdx.x & (width - 1), slice = threadIdx.x / width;
    float s = 0.0f;
    int c = 0;
    if (threadIdx.x == 0) total = 0;
    if (e < experts) {
        for (int b = slice; b < blocks; b += slices) {
            s += part[static_cast<size_t>(b) * experts + e];
            c += part_n[static_cast<size_t>(b) * (experts + 1) + e];
        }
    }
    prob[threadIdx.x] = s;
    count[threadIdx.x] = c;
    __syncthreads();
    int n = 0;
    for (int b = threadIdx.x; b < blocks; b += kFinThreads)
        n += part_n[static_cast<size_t>(b) * (experts + 1) + experts];
    if (n) atomicAdd(&total, n);
    if (slice == 0 && e < experts)
        for (int i = 1; i < slices; ++i) {
            s += prob[i * width + e];
            c += count[i * width + e];
        }
    __syncthreads();
    n = total;
    if (slice == 0 && e < experts) {
        prob[e] = s / static_cast<float>(max(n, 1));
        count[e] = c;
        probs[e] = prob[e];
        counts[e] = c;
    }
    if (threadIdx.x == 0) count[experts] = counts[experts] = n;
    __syncthreads();
    const float l = loss_of<kFinThreads>(count, prob, experts, k, coef, red);
    if (threadIdx.x == 0) *loss = l;
}

// The counts enter less a whole number near their mean, which changes nothing (the p of a row
// add up to 1) and keeps the bits of what is left.
template <int T, int L, int P, bool ADD>
__global__ __launch_bounds__(kBwdThreads) void balance_bwd_kernel(
    const void* __restrict__ logits, void* __restrict__ dlogits, int tokens, int experts, int k,
    float coef, const int* __restrict__ counts, const float* __restrict__ dloss,
    const unsigned char* __restrict__ valid) {
    constexpr int PER = kBwdThreads / L;
    constexpr int N = kPiece<T, P>;
    const int gl = threadIdx.x & (L - 1);
    int c[P];
    float sum = 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int e = gl * N + step_expert<T, L, P>(p);
        c[p] = e < experts ? counts[e] : 0;
        sum += static_cast<float>(c[p]);
    }
    const int mean = static_cast<int>(
        fminf(group_sum<L>(sum) / static_cast<float>(experts), 2147483520.0f));
    float left[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int e = gl * N + step_expert<T, L, P>(p);
        left[p] = e < experts ? static_cast<float>(c[p] - mean) : 0.0f;
    }
    const int n = counts[experts];
    const float per = n > 0 ? 1.0f / static_cast<float>(n) : 0.0f;
    const float scale = (dloss ? *dloss : 1.0f) * coef * static_cast<float>(experts) /
                        static_cast<float>(k) * per * per;
    for (long long base = static_cast<long long>(blockIdx.x) * PER; base < tokens;
         base += static_cast<long long>(gridDim.x) * PER) {
        const long long want = base + threadIdx.x / L;
        const bool inside = want < tokens;
        const size_t row = inside ? static_cast<size_t>(want) : static_cast<size_t>(tokens) - 1;
        const bool live = !valid || valid[row] != 0;
        float v[P];
        [[maybe_unused]] float old[P];
        load_logits<T, L, P>(logits, row, tokens, gl, experts, v);
        if constexpr (ADD) load_logits<T, L, P>(dlogits, row, tokens, gl, experts, old);
        const float inv = softmax_terms<L, P>(v);
        float d = 0.0f;
#pragma unroll
        for (int p = 0; p < P; ++p) d += v[p] * left[p];
        d = group_sum<L>(d) * inv;
        const float factor = inv * scale;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const float g = live ? v[p] * factor * (left[p] - d) : 0.0f;
            v[p] = ADD ? old[p] + g : g;
        }
        if (!inside || (ADD && !live)) continue;
#pragma unroll
        for (int p0 = 0; p0 < P; p0 += N) {
            const int e0 = gl * N + step_expert<T, L, P>(p0);
            float part[N];
#pragma unroll
            for (int e = 0; e < N; ++e) part[e] = v[p0 + e];
            if (e0 + N <= experts) {
                row_put_n<T, N>(dlogits, row * experts + e0, part);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (e0 + e < experts) row_put<T>(dlogits, row * experts + e0 + e, part[e]);
            }
        }
    }
}

int fwd_blocks(int tokens, int experts) {
    if (tokens <= kOneTokens) return 1;
    const int per = kFwdThreads / (experts <= 256 ? 16 : 64);
    return static_cast<int>(
        std::min<long long>((static_cast<long long>(tokens) + per - 1) / per, kFwdBlocks));
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

size_t mi_moe_balance_workspace(int tokens, int experts) {
    if (tokens <= kOneTokens || experts <= 0) return 0;
    return colsum_part_offset() + static_cast<size_t>(fwd_blocks(tokens, experts)) *
                                      (2 * static_cast<size_t>(experts) + 1) * sizeof(float);
}

int mi_moe_balance_forward(const void* logits, const int* ids, const unsigned char* valid,
                           int* counts, float* probs, float* loss, int tokens, int experts, int k,
                           float coef, int type, void* stream) {
    const char* name = "mi_moe_balance_forward";
    if (int rc = check_gate_args(name, tokens, experts, k, type)) return rc;
    if (!counts || !probs || !loss || (tokens > 0 && (!logits || !ids)))
        return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    hipStream_t st = to_stream(stream);
    const int blocks = fwd_blocks(tokens, experts);
    float* part = nullptr;
    int* part_n = nullptr;
    if (blocks > 1) {
        int err = MI_OK;
        char* ws = static_cast<char*>(
            workspace_get(mi_moe_balance_workspace(tokens, experts), st, &err));
        if (!ws) return err;
        part = reinterpret_cast<float*>(ws + colsum_part_offset());
        part_n = reinterpret_cast<int*>(part + static_cast<size_t>(blocks) * experts);
    }
    with_row_type(type, [&](auto t) {
        with_gate_shape<false>(experts, false, [&](auto l, auto p) {
            constexpr int T = decltype(t)::value, L = decltype(l)::value, P = decltype(p)::value;
            with_flag(blocks == 1, [&](auto one) {
                hipLaunchKernelGGL((balance_fwd_kernel<T, L, P, decltype(one)::value>),
                                   dim3(blocks), dim3(kFwdThreads), 0, st, logits, ids, tokens,
                                   experts, k, valid, part, part_n, counts, probs, loss, coef);
            });
        });
    });
    if (int rc = check_launch(name)) return rc;
    if (blocks == 1) return MI_OK;
    hipLaunchKernelGGL(balance_finish_kernel, dim3(1), dim3(kFinThreads), 0, st, part, part_n,
                       blocks, experts, k, coef, counts, probs, loss);
    return check_launch(name);
}

int mi_moe_balance_backward(const void* logits, const unsigned char* valid, const int* counts,
                            const float* dloss, void* dlogits, int tokens, int experts, int k,
                            float coef, int accumulate, int type, void* stream) {
    const char* name = "mi_moe_balance_backward";
    if (int rc = check_gate_args(name, tokens, experts, k, type)) return rc;
    if (tokens == 0) return MI_OK;
    if (!logits || !counts || !dlogits)
        return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    with_row_type(type, [&](auto t) {
        with_gate_shape<false>(experts, false, [&](auto l, auto p) {
            constexpr int T = decltype(t)::value, L = decltype(l)::value, P = decltype(p)::value;
            constexpr int PER = kBwdThreads / L;
            const unsigned grid = static_cast<unsigned>(
                std::min<long long>((static_cast<long long>(tokens) + PER - 1) / PER, kMaxGrid));
            with_flag(accumulate != 0, [&](auto add) {
                hipLaunchKernelGGL((balance_bwd_kernel<T, L, P, decltype(add)::value>), dim3(grid),
                                   dim3(kBwdThreads), 0, to_stream(stream), logits, dlogits,
                                   tokens, experts, k, coef, counts, dloss, valid);
            });
        });
    });
    return check_launch(name);
}

}  // extern "C"

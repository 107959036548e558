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

constexpr int kFwdThreads = 1024;
constexpr int kFwdBlocks = 256;
constexpr int kOneTrips = 4;  // rows of a lane group in a call that one workgroup does alone
constexpr int kFinThreads = 1024;
constexpr int kFinExperts = 16;  // experts of a workgroup that adds partial rows
constexpr int kFinSlices = kFinThreads / kFinExperts;
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

// sum c_e P_e to the loss.
__device__ __forceinline__ float loss_of(double sum, int experts, int k, int n, float coef) {
    return n == 0 ? 0.0f
                  : static_cast<float>(sum * static_cast<double>(coef) * experts /
                                       (static_cast<double>(k) * n));
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) v += __shfl_xor(v, m);
    return v;
}

// What the workgroups that add partial rows leave for the last of them.
struct Finish {
    double sum[kMaxExperts / kFinExperts];
    unsigned done;
};

// Sums of the probabilities and counts over a workgroup's tokens: a lane adds its experts'
// over its rows in registers, the waves' sums meet in LDS, in order.  ONE: the only
// workgroup, which writes the results; else a partial row of both.
template <int T, int L, int P, bool ONE>
__global__ __launch_bounds__(kFwdThreads) void balance_fwd_kernel(
    const void* __restrict__ logits, const int* __restrict__ ids, int tokens, int experts, int k,
    const unsigned char* __restrict__ valid, float* __restrict__ part, int* __restrict__ part_n,
    Finish* __restrict__ finish, int* __restrict__ counts, float* __restrict__ probs,
    float* __restrict__ loss, float coef) {
    constexpr int PER = kFwdThreads / L, WAVES = kFwdThreads / kWave;
    constexpr int N = kPiece<T, P>;
    constexpr int SLOTS = L * P > 512 ? WAVES / 2 : WAVES;  // 32 KB of sums at most
    __shared__ __align__(16) float sums[SLOTS][L * P];
    __shared__ int count[kMaxExperts + 1];
    const int gl = threadIdx.x & (L - 1), lane = threadIdx.x & (kWave - 1);
    const int wave = threadIdx.x / kWave;
    for (int e = threadIdx.x; e <= experts; e += kFwdThreads) count[e] = 0;
    if (!ONE && blockIdx.x == 0 && threadIdx.x == 0) finish->done = 0;
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
        const int id = want < tokens && gl < k ? ids[row * k + gl] : -1;
        float v[P];
        load_logits<T, L, P>(logits, row, tokens, gl, experts, v);
        const float inv = softmax_terms<L, P>(v);
#pragma unroll
        for (int p = 0; p < P; ++p) acc[p] += live ? v[p] * inv : 0.0f;
        if (live && id >= 0 && id < experts) atomicAdd(&count[id], 1);
        const unsigned long long rows = __ballot(live && gl == 0);
        if (lane == 0 && rows) atomicAdd(&count[experts], __popcll(rows));
    }
    // the wave's rows, then the waves
    if constexpr (L == 16) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            acc[p] += __shfl_xor(acc[p], 16);
            acc[p] += __shfl_xor(acc[p], 32);
        }
    }
    auto put = [&](int slot) {
        if (lane < L) {
#pragma unroll
            for (int p = 0; p < P; ++p) sums[slot][gl * N + step_expert<T, L, P>(p)] = acc[p];
        }
    };
    if constexpr (SLOTS < WAVES) {
        if (wave >= SLOTS) put(wave - SLOTS);
        __syncthreads();
        if (wave < SLOTS) {
#pragma unroll
            for (int p = 0; p < P; ++p)
                acc[p] += sums[wave][gl * N + step_expert<T, L, P>(p)];
        }
        if (wave < SLOTS) put(wave);
    } else {
        put(wave);
    }
    __syncthreads();
    if constexpr (ONE) {
        __shared__ double red[WAVES];
        const int n = count[experts];
        double s = 0.0;
        for (int e = threadIdx.x; e < experts; e += kFwdThreads) {
            float p = sums[0][e];
#pragma unroll
            for (int w = 1; w < SLOTS; ++w) p += sums[w][e];
            p /= static_cast<float>(max(n, 1));
            probs[e] = p;
            counts[e] = count[e];
            s += static_cast<double>(count[e]) * static_cast<double>(p);
        }
        s = wave_sum_d(s);
        if (lane == 0) red[wave] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
#pragma unroll
            for (int w = 1; w < WAVES; ++w) s += red[w];
            *loss = loss_of(s, experts, k, n, coef);
            counts[experts] = n;
        }
    } else {
        for (int e = threadIdx.x; e < experts; e += kFwdThreads) {
            float s = sums[0][e];
#pragma unroll
            for (int w = 1; w < SLOTS; ++w) s += sums[w][e];
            part[static_cast<size_t>(blockIdx.x) * experts + e] = s;
        }
        for (int e = threadIdx.x; e <= experts; e += kFwdThreads)
            part_n[static_cast<size_t>(blockIdx.x) * (experts + 1) + e] = count[e];
    }
}

// Adds the partial rows: a workgroup has 16 experts, 64 slices of the rows side by side, each in
// order, then added pairwise.  The workgroup that ends last adds all workgroups' sums of c_e P_e,
// in order, whichever it is.
__global__ __launch_bounds__(kFinThreads) void balance_finish_kernel(
    const float* __restrict__ part, const int* __restrict__ part_n, int blocks, int experts, int k,
    float coef, int* __restrict__ counts, float* __restrict__ probs, float* __restrict__ loss,
    Finish* finish) {
    constexpr int TRIPS = kFwdBlocks / kFinSlices;
    __shared__ float sum[kFinSlices][kFinExperts];
    __shared__ int count[kFinSlices][kFinExperts];
    __shared__ int total;
    const int col = threadIdx.x & (kFinExperts - 1), slice = threadIdx.x / kFinExperts;
    const int e = blockIdx.x * kFinExperts + col;
    if (threadIdx.x == 0) total = 0;
    const int rows = static_cast<int>(threadIdx.x) < blocks
                         ? part_n[static_cast<size_t>(threadIdx.x) * (experts + 1) + experts]
                         : 0;
    float p[TRIPS];
    int c[TRIPS];
#pragma unroll
    for (int i = 0; i < TRIPS; ++i) {
        const int b = slice + i * kFinSlices;
        const bool there = b < blocks && e < experts;
        p[i] = there ? part[static_cast<size_t>(b) * experts + e] : 0.0f;
        c[i] = there ? part_n[static_cast<size_t>(b) * (experts + 1) + e] : 0;
    }
#pragma unroll
    for (int i = 1; i < TRIPS; ++i) {
        p[0] += p[i];
        c[0] += c[i];
    }
    sum[slice][col] = p[0];
    count[slice][col] = c[0];
    __syncthreads();
    if (rows) atomicAdd(&total, rows);
#pragma unroll
    for (int h = kFinSlices / 2; h >= 1; h /= 2) {
        if (slice < h) {
            sum[slice][col] += sum[slice + h][col];
            count[slice][col] += count[slice + h][col];
        }
        __syncthreads();
    }
    if (threadIdx.x >= kWave) return;
    const int n = total;
    double s = 0.0;
    if (threadIdx.x < kFinExperts && e < experts) {
        const float mean = sum[0][col] / static_cast<float>(max(n, 1));
        probs[e] = mean;
        counts[e] = count[0][col];
        s = static_cast<double>(count[0][col]) * static_cast<double>(mean);
    }
    s = wave_sum_d(s);
    if (gridDim.x > 1) {
        unsigned before = 0;
        if (threadIdx.x == 0) {
            __hip_atomic_store(&finish->sum[blockIdx.x], s, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
            before = __hip_atomic_fetch_add(&finish->done, 1u, __ATOMIC_ACQ_REL,
                                            __HIP_MEMORY_SCOPE_AGENT);
        }
        if (static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(before))) !=
            gridDim.x - 1)
            return;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
        s = threadIdx.x < gridDim.x
                ? __hip_atomic_load(&finish->sum[threadIdx.x], __ATOMIC_RELAXED,
                                    __HIP_MEMORY_SCOPE_AGENT)
                : 0.0;
        s = wave_sum_d(s);
    }
    if (threadIdx.x == 0) {
        *loss = loss_of(s, experts, k, n, coef);
        counts[experts] = n;
    }
}
static_assert(kMaxExperts / kFinExperts <= kWave && kFwdBlocks <= kFinThreads,
              "a lane for each workgroup's sum, a thread for each partial row");

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
    const int per = kFwdThreads / (experts <= 256 ? 16 : 64);
    if (tokens <= kOneTrips * per) return 1;
    return static_cast<int>(
        std::min<long long>((static_cast<long long>(tokens) + per - 1) / per, kFwdBlocks));
}

size_t partial_bytes(int blocks, int experts) {
    return static_cast<size_t>(blocks) * (2 * static_cast<size_t>(experts) + 1) * sizeof(float);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

size_t mi_moe_balance_workspace(int tokens, int experts) {
    if (tokens <= 0 || experts <= 0) return 0;
    const int blocks = fwd_blocks(tokens, experts);
    return blocks == 1 ? 0
                       : colsum_part_offset() + round_up(sizeof(Finish), 256) +
                             partial_bytes(blocks, experts);
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
    Finish* finish = nullptr;
    float* part = nullptr;
    int* part_n = nullptr;
    if (blocks > 1) {
        int err = MI_OK;
        char* ws = static_cast<char*>(
            workspace_get(mi_moe_balance_workspace(tokens, experts), st, &err));
        if (!ws) return err;
        finish = reinterpret_cast<Finish*>(ws + colsum_part_offset());
        part = reinterpret_cast<float*>(ws + colsum_part_offset() + round_up(sizeof(Finish), 256));
        part_n = reinterpret_cast<int*>(part + static_cast<size_t>(blocks) * experts);
    }
    with_row_type(type, [&](auto t) {
        with_gate_shape<false>(experts, false, [&](auto l, auto p) {
            constexpr int T = decltype(t)::value, L = decltype(l)::value, P = decltype(p)::value;
            with_flag(blocks == 1, [&](auto one) {
                hipLaunchKernelGGL((balance_fwd_kernel<T, L, P, decltype(one)::value>),
                                   dim3(blocks), dim3(kFwdThreads), 0, st, logits, ids, tokens,
                                   experts, k, valid, part, part_n, finish, counts, probs, loss,
                                   coef);
            });
        });
    });
    if (int rc = check_launch(name)) return rc;
    if (blocks == 1) return MI_OK;
    hipLaunchKernelGGL(balance_finish_kernel, dim3((experts + kFinExperts - 1) / kFinExperts),
                       dim3(kFinThreads), 0, st, part, part_n, blocks, experts, k, coef, counts,
                       probs, loss, finish);
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

// The balance loss of a mixture-of-experts router for gfx950: how many of the
// tokens' slots each expert has, the mean of the tokens' probabilities for it, the
// loss that their products give, and the logits' gradient.  No counterpart in the
// reference, whose feed-forward layer is dense.
//
//   p_t = softmax(l_t) over all experts;  c_e = slots with id e;  n valid tokens
//   loss = coef E / (k n) sum_e c_e P_e,  P_e = sum_t p_te / n
//   dl_te = dloss coef E / (k n^2) p_te (c_e - sum_f p_tf c_f)
//
// A row's logits lie in the registers of L lanes as in the router's kernels, and are read once.
// Backward: bound by memory, [65536, 256] fp32 added to what is there 37.3 us, 5.4 TB/s, [32768,
// 256] bf16 7.7 us, 4.4 TB/s.  Forward: [32768, 256] bf16, 8 slots, 10.7 us for 18 MB.  Its first
// launch (7.6) takes 5.0 for 300 tokens and 5.3 for 4096: a workgroup's start, the exchange of its
// waves' sums and its end.  What more tokens add is bound by memory (131072 17.5 us, 262144 29.3: 90
// ps and 544 bytes each, 6.0 TB/s).  The second (3) is bound by the round trips to the partial rows
// and to the word.
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
constexpr int kFinThreads = 256;
constexpr int kFinExperts = 16;  // experts of a workgroup that adds partial rows
constexpr int kFinSlices = kFinThreads / kFinExperts;
constexpr int kBwdThreads = 256;
constexpr int kMaxGrid = 1 << 20;

// A lane's pieces of a row: where piece p begins, and how many of its first elements another
// lane has.  A row that is no whole number of pieces ends with one that begins early (there are
// no fewer experts than a piece has, for the number of experts decides P); what is shared counts
// once in sums, and is written twice with the same bits.  So every load is whole and inside the
// row, and a row's loads go out together: with the cut ones behind branches each waited for the
// one before (gradient of [32768, 256] bf16 19.4 us, 7.7 so, of [8192, 512] 12.0, 6.6).
template <int T, int L, int P>
struct Pieces {
    static constexpr int N = kPiece<T, P>;
    int begin[P / N], skip[P / N];
    __device__ __forceinline__ Pieces(int gl, int experts) {
#pragma unroll
        for (int i = 0; i < P / N; ++i) {
            const int e0 = gl * N + i * N * L, last = experts - N;
            begin[i] = min(e0, last);
            skip[i] = min(max(e0 - last, 0), N);
        }
    }
    // More than half of the lanes' places have an expert.
    static constexpr bool whole(int i) { return L * P > 16 && (i + 1) * N * L <= L * P / 2; }
    __device__ __forceinline__ bool own(int i, int e) const { return whole(i) || e >= skip[i]; }
};

// A row's pieces as they are in memory: converted only where they are used, so that nothing waits
// for them before.
template <int T, int P>
struct RawPieces {
    static constexpr int N = kPiece<T, P>;
    typedef row_elem<T> small __attribute__((ext_vector_type(N < row_vec<T>() ? N : 1)));
    typedef typename std::conditional<N == row_vec<T>(), u32x4, small>::type piece;
    piece raw[P / N];
    __device__ __forceinline__ void values(float (&v)[P]) const {
#pragma unroll
        for (int i = 0; i < P / N; ++i) {
            float part[N];
            if constexpr (N == row_vec<T>()) {
                row_unpack<T>(raw[i], part);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) part[e] = static_cast<float>(raw[i][e]);
            }
#pragma unroll
            for (int e = 0; e < N; ++e) v[i * N + e] = part[e];
        }
    }
};

template <int T, int L, int P, bool NT>
__device__ __forceinline__ void load_pieces(const void* logits, size_t row, int experts,
                                            const Pieces<T, L, P>& at, RawPieces<T, P>& r) {
    constexpr int N = Pieces<T, L, P>::N;
    const row_elem<T>* p = static_cast<const row_elem<T>*>(logits) + row * experts;
#pragma unroll
    for (int i = 0; i < P / N; ++i) {
        if constexpr (N == row_vec<T>())
            r.raw[i] = load16b<NT>(p + at.begin[i]);
        else
            r.raw[i] = load_piece<typename RawPieces<T, P>::piece>(
                reinterpret_cast<const char*>(p + at.begin[i]));
    }
}

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

// The sum of lanes l, l + 16, l + 32 and l + 48, in all four: a swap exchanges odd rows of 16 lanes
// of the first operand with even rows of the second, or the halves.
__device__ __forceinline__ float add_rows_of_16(float v) {
    auto both = [](auto pair) { return __uint_as_float(pair[0]) + __uint_as_float(pair[1]); };
    unsigned u = __float_as_uint(v);
    v = both(__builtin_amdgcn_permlane16_swap(u, u, false, false));
    u = __float_as_uint(v);
    return both(__builtin_amdgcn_permlane32_swap(u, u, false, false));
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

// sum c_e P_e over the workgroups that add partial rows.  Each adds its share of n k, the largest
// such sum, in units of 2^-49 of it, to bits 7 to 56 of one word, 1 to the bits below, so that the
// last one knows that it is, and 1 to those above where its share is no number: as whole numbers
// they add up the same in any order, and the word says all, so nothing has to be ordered by it.
// A share loses less than a unit: a sum of less than kEnough of them (the chosen experts have hardly
// any probability, 1 / E where the router is balanced) is added again from the shares themselves,
// in 64 bits, which every workgroup writes when it has counted itself.
constexpr int kMaxFin = kMaxExperts / kFinExperts;
constexpr double kShare = 0x1p49;
constexpr unsigned long long kEnough = 1ull << 32;  // 64 units lost are 2^-26 of it
constexpr unsigned long long kNone = ~0ull;         // a share not written yet: NaN bits that none has

struct Finish {
    unsigned long long word;
    unsigned long long share[kMaxFin];
};

// Sums of the probabilities and counts over a workgroup's tokens: a lane adds its experts'
// over its rows in registers, the waves' sums meet in LDS, in order.  ONE: the only
// workgroup, which writes the results; else a partial row of both.  One workgroup of 16 waves a CU:
// two of them, or twice as many of 8 waves, start and end more (13.0, 15.3 us at [32768, 256]
// bf16, 11.9 so, in a build between).
template <int T, int L, int P, bool ONE, bool NT>
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
    const Pieces<T, L, P> at(gl, experts);
    const unsigned char* flags = valid ? valid : reinterpret_cast<const unsigned char*>(ids);
    struct Row {
        RawPieces<T, P> raw;
        int id;
        unsigned char flag;
        bool inside;
    };
    auto load = [&](long long base, Row& r) {
        const long long want = base + threadIdx.x / L;
        const bool inside = want < tokens;
        const size_t row = inside ? static_cast<size_t>(want) : static_cast<size_t>(tokens) - 1;
        load_pieces<T, L, P, NT>(logits, row, experts, at, r.raw);
        r.id = ids[row * k + min(gl, k - 1)];
        r.flag = flags[row];
        r.inside = inside;
    };
    const long long stride = static_cast<long long>(gridDim.x) * PER;
    long long base = static_cast<long long>(blockIdx.x) * PER;
    float acc[P];
#pragma unroll
    for (int p = 0; p < P; ++p) acc[p] = 0.0f;
    auto add = [&](const Row& r) {
        const bool live_row = r.inside & ((r.flag != 0) | !valid);
        float v[P];
        r.raw.values(v);
#pragma unroll
        for (int p = 0; p < P; ++p)
            if (!at.own(p / N, p % N)) v[p] = -__builtin_inff();
        const float inv = softmax_terms<L, P>(v);
        const unsigned long long live = __ballot(live_row);
        if (live == ~0ull) {
#pragma unroll
            for (int p = 0; p < P; ++p) acc[p] += v[p] * inv;
        } else {
#pragma unroll
            for (int p = 0; p < P; ++p) acc[p] += live_row ? v[p] * inv : 0.0f;
        }
        if (live_row & (gl < k) & (r.id >= 0) & (r.id < experts)) atomicAdd(&count[r.id], 1);
        if (lane == 0 && live) atomicAdd(&count[experts], __popcll(live) / L);
    };
    // the next rows' loads go out before rows are worked on: two sets of registers in turn, for
    // copies from one to the other would wait for the loads
    Row r0, r1;
    if (tokens > 0) load(base, r0);
    for (int e = threadIdx.x; e <= experts; e += kFwdThreads) count[e] = 0;
    __syncthreads();
    while (base < tokens) {
        load(base + stride, r1);
        add(r0);
        if (base + stride >= tokens) break;
        load(base + 2 * stride, r0);
        add(r1);
        base += 2 * stride;
    }
    // the wave's rows, then the waves
    if constexpr (L == 16) {
#pragma unroll
        for (int p = 0; p < P; ++p) acc[p] = add_rows_of_16(acc[p]);
    }
    auto put = [&](int slot) {
        if (lane < L) {
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (at.own(p / N, p % N)) sums[slot][at.begin[p / N] + p % N] = acc[p];
        }
    };
    if constexpr (SLOTS < WAVES) {
        if (wave >= SLOTS) put(wave - SLOTS);
        __syncthreads();
        if (wave < SLOTS) {
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (at.own(p / N, p % N)) acc[p] += sums[wave][at.begin[p / N] + p % N];
            put(wave);
        }
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
        if (blockIdx.x == 0) {
            if (threadIdx.x == 0) finish->word = 0;
            if (threadIdx.x < kMaxFin) finish->share[threadIdx.x] = kNone;
        }
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

// Adds the partial rows: a workgroup has 16 experts, and 16 slices of the rows side by side, each
// in order, which the first wave then adds.  ([32768, 256], 256 rows: 3.9 us; one workgroup for all
// experts 10.5, workgroups that hand their sums to the last one through memory, with the caches
// written back for it, 7.)
__global__ __launch_bounds__(kFinThreads) void balance_finish_kernel(
    const float* __restrict__ part, const int* __restrict__ part_n, int blocks, int experts, int k,
    float coef, int* __restrict__ counts, float* __restrict__ probs, float* __restrict__ loss,
    Finish* finish) {
    constexpr int TRIPS = kFwdBlocks / kFinSlices;
    __shared__ float sum[kFinSlices][kFinExperts];
    __shared__ int count[kFinSlices][kFinExperts], tokens[kFinThreads / kWave];
    const int col = threadIdx.x & (kFinExperts - 1), slice = threadIdx.x / kFinExperts;
    const int e = blockIdx.x * kFinExperts + col, at = min(e, experts - 1);
    // every load goes out, from a place that is there, and counts where its place is
    const int mine = min(static_cast<int>(threadIdx.x), blocks - 1);
    int rows = part_n[static_cast<size_t>(mine) * (experts + 1) + experts];
    float p[TRIPS];
    int c[TRIPS];
#pragma unroll
    for (int i = 0; i < TRIPS; ++i) {
        const int b = min(slice + i * kFinSlices, blocks - 1);
        p[i] = part[static_cast<size_t>(b) * experts + at];
        c[i] = part_n[static_cast<size_t>(b) * (experts + 1) + at];
    }
    rows = static_cast<int>(threadIdx.x) < blocks ? rows : 0;
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) rows += __shfl_xor(rows, m);
    if ((threadIdx.x & (kWave - 1)) == 0) tokens[threadIdx.x / kWave] = rows;
#pragma unroll
    for (int i = 0; i < TRIPS; ++i) {
        const bool there = slice + i * kFinSlices < blocks;
        p[i] = there ? p[i] : 0.0f;
        c[i] = there ? c[i] : 0;
        if (i > 0) {
            p[0] += p[i];
            c[0] += c[i];
        }
    }
    sum[slice][col] = p[0];
    count[slice][col] = c[0];
    __syncthreads();
    if (threadIdx.x >= kWave) return;
    // the first wave: lanes of the same expert 16 apart
    float s = 0.0f;
    int m = 0;
#pragma unroll
    for (int i = 0; i < kFinSlices / 4; ++i) {
        s += sum[slice * (kFinSlices / 4) + i][col];
        m += count[slice * (kFinSlices / 4) + i][col];
    }
    s = add_rows_of_16(s);
    m += __shfl_xor(m, 16);
    m += __shfl_xor(m, 32);
    int n = tokens[0];
#pragma unroll
    for (int w = 1; w < kFinThreads / kWave; ++w) n += tokens[w];
    const float mean = s / static_cast<float>(max(n, 1));
    double share = 0.0;
    if (threadIdx.x < kFinExperts && e < experts) {
        probs[e] = mean;
        counts[e] = m;
        share = static_cast<double>(m) * static_cast<double>(mean);
    }
    share = wave_sum_d(share);
    const double most = static_cast<double>(k) * max(n, 1);
    const bool number = share - share == 0.0;
    unsigned long long word = 0;
    if (threadIdx.x == 0) {
        const unsigned long long own =
            (number ? static_cast<unsigned long long>(share / most * kShare) << 7 : 1ull << 57) + 1;
        word = own + __hip_atomic_fetch_add(&finish->word, own, __ATOMIC_RELAXED,
                                            __HIP_MEMORY_SCOPE_AGENT);
        // behind it, for what comes before it is waited for together with it
        __hip_atomic_store(&finish->share[blockIdx.x],
                           static_cast<unsigned long long>(__double_as_longlong(number ? share : 0.0)),
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    word = __shfl(word, 0);
    if ((word & 127) != gridDim.x) return;
    const unsigned long long units = word >> 7 & ((1ull << 50) - 1);
    double all = static_cast<double>(units) / kShare * most;
    if (units < kEnough) {
        // Every workgroup has counted itself, and its share comes right behind: the wait for it ends.
        unsigned long long bits = 0;
        if (threadIdx.x < gridDim.x) {
            do {
                bits = __hip_atomic_load(&finish->share[threadIdx.x], __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);
            } while (bits == kNone);
        }
        all = wave_sum_d(__longlong_as_double(static_cast<long long>(bits)));
    }
    if (threadIdx.x != 0) return;
    *loss = word >> 57 ? __builtin_nanf("") : loss_of(all, experts, k, n, coef);
    counts[experts] = n;
}
static_assert(kMaxFin <= kWave && kFwdBlocks <= kFinThreads,
              "a lane for each workgroup's share, of which 7 bits count; a thread for each partial row");

// The counts enter less a whole number near their mean, which changes nothing (the p of a row
// add up to 1) and keeps the bits of what is left.
template <int T, int L, int P, bool ADD, bool NT>
__global__ __launch_bounds__(kBwdThreads) void balance_bwd_kernel(
    const void* __restrict__ logits, void* dlogits, int tokens, int experts, int k,
    float coef, const int* __restrict__ counts, const float* __restrict__ dloss,
    const unsigned char* __restrict__ valid) {
    constexpr int PER = kBwdThreads / L;
    constexpr int N = kPiece<T, P>;
    const int gl = threadIdx.x & (L - 1);
    const Pieces<T, L, P> at(gl, experts);
    // read in any case: a branch would wait for what is on its way
    const unsigned char* flags = valid ? valid : static_cast<const unsigned char*>(logits);
    int c[P];
    float sum = 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        c[p] = counts[at.begin[p / N] + p % N];
        sum += at.own(p / N, p % N) ? static_cast<float>(c[p]) : 0.0f;
    }
    const int mean = static_cast<int>(
        fminf(group_sum<L>(sum) / static_cast<float>(experts), 2147483520.0f));
    float left[P];
#pragma unroll
    for (int p = 0; p < P; ++p) left[p] = static_cast<float>(c[p] - mean);
    const int n = counts[experts];
    const float per = n > 0 ? 1.0f / static_cast<float>(n) : 0.0f;
    const float scale = (dloss ? *dloss : 1.0f) * coef * static_cast<float>(experts) /
                        static_cast<float>(k) * per * per;
    for (long long base = static_cast<long long>(blockIdx.x) * PER; base < tokens;
         base += static_cast<long long>(gridDim.x) * PER) {
        const long long want = base + threadIdx.x / L;
        const bool inside = want < tokens;
        const size_t row = inside ? static_cast<size_t>(want) : static_cast<size_t>(tokens) - 1;
        RawPieces<T, P> raw;
        [[maybe_unused]] RawPieces<T, P> raw_old;
        load_pieces<T, L, P, NT>(logits, row, experts, at, raw);
        if constexpr (ADD) load_pieces<T, L, P, NT>(dlogits, row, experts, at, raw_old);
        const bool live = (flags[row] != 0) | !valid;
        float v[P];
        [[maybe_unused]] float old[P];
        raw.values(v);
        if constexpr (ADD) raw_old.values(old);
        // e^(v - max) of shared elements is needed for what is written, not for the sum
        float top = -__builtin_inff();
#pragma unroll
        for (int p = 0; p < P; ++p) top = at.own(p / N, p % N) ? fmaxf(top, v[p]) : top;
        top = group_max<L>(top);
        if (top == -__builtin_inff()) top = 0.0f;
        float s = 0.0f, d = 0.0f;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            v[p] = __builtin_amdgcn_exp2f((v[p] - top) * kLog2e);
            const float own = at.own(p / N, p % N) ? v[p] : 0.0f;
            s += own;
            d += own * left[p];
        }
        s = group_sum<L>(s);
        const float inv = s == 0.0f ? 0.0f : 1.0f / s;
        d = group_sum<L>(d) * inv;
        const float factor = inv * scale;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const float g = live ? v[p] * factor * (left[p] - d) : 0.0f;
            v[p] = rounded(ADD ? old[p] + g : g);
        }
        wave_order();  // the loads of what is written twice come before the stores
        if (!inside || (ADD && !live)) continue;
        row_elem<T>* out = static_cast<row_elem<T>*>(dlogits) + row * experts;
#pragma unroll
        for (int i = 0; i < P / N; ++i) {
            if (!Pieces<T, L, P>::whole(i) && at.skip[i] == N) continue;
            float part[N];
#pragma unroll
            for (int e = 0; e < N; ++e) part[e] = v[i * N + e];
            if constexpr (N == row_vec<T>())
                store16b(out + at.begin[i], row_pack<T>(part));
            else
                row_put_n<T, N>(out, at.begin[i], part);
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
            auto launch = [&](auto one, auto nt) {
                hipLaunchKernelGGL(
                    (balance_fwd_kernel<T, L, P, decltype(one)::value, decltype(nt)::value>),
                    dim3(blocks), dim3(kFwdThreads), 0, st, logits, ids, tokens, experts, k, valid,
                    part, part_n, finish, counts, probs, loss, coef);
            };
            if (blocks == 1)
                launch(std::true_type(), std::false_type());
            else
                with_flag(stream_loads(static_cast<double>(tokens) * experts * row_type_size(type)),
                          [&](auto nt) { launch(std::false_type(), nt); });
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
    hipStream_t st = to_stream(stream);
    with_row_type(type, [&](auto t) {
        with_gate_shape<false>(experts, false, [&](auto l, auto p) {
            constexpr int T = decltype(t)::value, L = decltype(l)::value, P = decltype(p)::value;
            constexpr int PER = kBwdThreads / L;
            const unsigned grid = static_cast<unsigned>(
                std::min<long long>((static_cast<long long>(tokens) + PER - 1) / PER, kMaxGrid));
            const bool nt = stream_loads(static_cast<double>(tokens) * experts *
                                         row_type_size(type) * (accumulate ? 2 : 1));
            with_flag(accumulate != 0, [&](auto add) {
                with_flag(nt, [&](auto stream) {
                    hipLaunchKernelGGL(
                        (balance_bwd_kernel<T, L, P, decltype(add)::value, decltype(stream)::value>),
                        dim3(grid), dim3(kBwdThreads), 0, st, logits, dlogits, tokens, experts, k,
                        coef, counts, dloss, valid);
                });
            });
        });
    });
    return check_launch(name);
}

}  // extern "C"

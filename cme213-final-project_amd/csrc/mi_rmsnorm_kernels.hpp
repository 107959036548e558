// Root-mean-square norm forward / backward for gfx950, with the residual's
// addition and with an output in 8 bits.  Beside the LayerNorm of
// FINAL_CLEAN_CODE/src/kernels/layernorm.cu:10-308 (its fused residual form and
// its backward into the residual stream's gradient); the reference has no RMS
// norm.  Rows are fp32, fp16 or bf16; gamma, statistics and sums fp32 (64 bits where a thread adds
// thousands of numbers one after another).
//
//   h = a + b (or x);  r = 1 / sqrt(mean(h^2) + eps);  y = h r gamma
//   dx = r (g - n mean(g n)),  n = h r,  g = dy gamma;  dgamma += sum_rows dy n
//
// A group of GT threads (a part of a wave, a wave, or several) holds a row in
// registers, in units of 16 bytes that its threads take in turn, so a row is
// read once.  The last unit of a row that is no whole number of them begins
// early, at the row's last 16 bytes: the elements that it shares with the unit
// before it count once in the sums, and are written twice with the same bits.
// Rows of less than one unit, and rows too long for registers, are walked twice.
//
// y is computed from the unrounded sum a + b; the rounded one is what is kept
// for the backward pass, with r as it was.  An output is rounded to its type from
// its fp32 value (`rounded`: or the compiler may join the last product with its
// conversion to fp16 in one of two threads that write the same element).
#pragma once

#include <algorithm>
#include <type_traits>

#include "mi_rmsnorm.hpp"
#include "mi_rowtype.hpp"

namespace mi {
namespace rms {

constexpr int kThreads = 256;
constexpr int kMaxGrid = 1 << 20;  // workgroups over the rows, which are taken in strides
// What reads one row and writes 8 bits moves so little that starting a workgroup for each counts:
// [32768, 4096] bf16 to e4m3 81 -> 75 us, [20000, 8192] 100 -> 91; but with the residual, or a row
// out, they are the faster ones ([32768, 4096] with both 157 -> 161, [100000, 768] fp32 96 -> 101).
constexpr int kRow8Grid = 8192;
constexpr int kFewRows = 1024;
constexpr int kLine = 128;  // bytes of a cache line
constexpr float kLeast = 0x1p-100f;  // a row or block counts as at least this large

template <int GT>
constexpr int kGroupThreads = GT > kThreads ? GT : kThreads;

// The unit that thread t of a row's group has in step k: where it begins, and how many of its
// first elements belong to another unit (all of them behind the row's end).
template <int V>
struct UnitAt {
    int col, skip;
};

template <int V>
__device__ __forceinline__ UnitAt<V> unit_at(int j, int units, int cols) {
    const int shared = units * V - cols;
    return {min(j * V, cols - V), j < units - 1 ? 0 : j == units - 1 ? shared : V};
}

template <int T>
__device__ __forceinline__ const char* element_ptr(const void* p, size_t i) {
    return static_cast<const char*>(p) + i * sizeof(row_elem<T>);
}
template <int T>
__device__ __forceinline__ char* element_ptr(void* p, size_t i) {
    return static_cast<char*>(p) + i * sizeof(row_elem<T>);
}

template <int V>
__device__ __forceinline__ void load_gamma(const float* gamma, int col, float (&g)[V]) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        const u32x4 w = load16b<false>(gamma + col + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) g[i + e] = __uint_as_float(w[e]);
    }
}

__device__ __forceinline__ unsigned larger(unsigned v, unsigned w) { return v > w ? v : w; }

// Largest of the L lanes (16, 32 or 64) around a lane, as unsigned integers:
// the order of magnitudes, with infinities and NaN above all.
template <int L>
__device__ __forceinline__ unsigned lanes_max(unsigned v) {
    auto step = [&](auto ctrl) {
        v = larger(v, static_cast<unsigned>(dpp_move_i<decltype(ctrl)::value>(static_cast<int>(v))));
    };
    step(std::integral_constant<int, 0xB1>());
    step(std::integral_constant<int, 0x4E>());
    step(std::integral_constant<int, 0x141>());
    step(std::integral_constant<int, 0x140>());
    if constexpr (L >= 32) v = larger(v, static_cast<unsigned>(__shfl_xor(static_cast<int>(v), 16)));
    if constexpr (L >= 64) v = larger(v, static_cast<unsigned>(__shfl_xor(static_cast<int>(v), 32)));
    return v;
}

__device__ __forceinline__ unsigned magnitude(float v) {
    return __float_as_uint(v) & 0x7fffffffu;
}

template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (L == 32) {
        v = group_sum<16>(v);
        return v + __shfl_xor(v, 16);
    } else {
        return group_sum<L>(v);
    }
}

struct SumTop {
    float sum;
    unsigned top;
};

// Sum and largest over the GT threads of a row's group, in every one of them.  Groups of
// several waves exchange through LDS; `turn` alternates between two places, so that the next
// exchange's writes cannot meet this one's reads (a barrier lies between any two of the same
// place).
template <int GT>
struct GroupRed {
    static constexpr int kWavesOf = kGroupThreads<GT> / kWave;
    SumTop (*red)[kWavesOf];
    int turn = 0;

    template <bool TOP>
    __device__ __forceinline__ SumTop both(float sum, unsigned top) {
        if constexpr (GT <= kWave) {
            return {lanes_sum<GT>(sum), TOP ? lanes_max<GT>(top) : 0u};
        } else {
            sum = wave_sum(sum);
            if constexpr (TOP) top = lanes_max<kWave>(top);
            SumTop* r = red[turn];
            turn ^= 1;
            if ((threadIdx.x & (kWave - 1)) == 0) r[threadIdx.x / kWave] = {sum, top};
            __syncthreads();
            const int w0 = static_cast<int>(threadIdx.x) / GT * (GT / kWave);
            SumTop t = r[w0];
#pragma unroll
            for (int i = 1; i < GT / kWave; ++i) {
                t.sum += r[w0 + i].sum;
                if constexpr (TOP) t.top = larger(t.top, r[w0 + i].top);
            }
            return t;
        }
    }
    __device__ __forceinline__ float sum(float v) { return both<false>(v, 0u).sum; }
    __device__ __forceinline__ unsigned max(unsigned v) { return both<true>(0.0f, v).top; }
};

// The scale of values v r (v = h gamma) whose largest magnitude of v has the bits `top`, and
// what v is multiplied by (0 where one of them is no number: their codes are 0, the scale NaN).
// r, the same for all of them, cancels in the codes and adds no rounding to them.  The factor of
// the smallest v passes fp32's range (where r is large, as eps far below its usual sizes allows):
// they are first multiplied by kUp, exactly.  Others need no factor above 2^119.
struct Scale {
    float scale, mul;
    bool up;
};
constexpr float kUp = 0x1p64f, kSmall = 0x1p-110f;

__device__ __forceinline__ Scale scale_of(unsigned top, float r, int format) {
    const float largest = format == MI_ROW8_INT8 ? 127.0f : 448.0f;
    const float v = __uint_as_float(top), m = v * r;
    if (!(m < __builtin_inff())) return {__builtin_nanf(""), 0.0f, false};
    const bool up = v < kSmall;
    if (m >= kLeast) return {m / largest, largest / (up ? v * kUp : v), up};
    return {kLeast / largest, (up ? r / kUp : r) * (largest / kLeast), up};
}

// The codes of N values (4 or 8), the first in the lowest byte.  int8: adding 1.5 2^23
// leaves rint(v mul) in the low bits of the sum, two's complement.
template <int N>
__device__ __forceinline__ uint64_t codes_of(const float (&values)[N], const Scale& s, int format) {
    uint32_t q[2] = {0, 0};
    float v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = values[e];
    if (__ballot(s.up)) {  // hardly ever: no lane pays for it otherwise
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] *= s.up ? kUp : 1.0f;
    }
    if (s.mul != 0.0f) {
#pragma unroll
        for (int h = 0; h < N / 4; ++h) {
            if (format == MI_ROW8_INT8) {
                uint32_t b[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    b[e] = __float_as_uint(fmaf(v[4 * h + e], s.mul, 12582912.0f));
                const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u);
                const uint32_t hi = __builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u);
                q[h] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
            } else {
                int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] * s.mul, v[4 * h + 1] * s.mul, 0,
                                                        false);
                w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] * s.mul, v[4 * h + 3] * s.mul, w,
                                                    true);
                q[h] = static_cast<uint32_t>(w);
            }
        }
    }
    return static_cast<uint64_t>(q[1]) << 32 | q[0];
}

// A unit's codes without the `skip` first ones, to the place of the others.
template <int V>
__device__ __forceinline__ void store_codes(char* p, uint64_t q, int skip) {
    if (skip == 0) {
        // not kept in the caches, like all rows that are written (32768 x 4096 bf16: 163 -> 159 us)
        typedef uint64_t u64_at1 __attribute__((aligned(1)));
        typedef uint32_t u32_at1 __attribute__((aligned(1)));
        if constexpr (V == 8)
            __builtin_nontemporal_store(q, reinterpret_cast<u64_at1*>(p));
        else
            __builtin_nontemporal_store(static_cast<uint32_t>(q), reinterpret_cast<u32_at1*>(p));
        return;
    }
    const int n = V - skip;
    p += skip;
    q >>= 8 * skip;
    if (n & 4) {
        store_piece(p, static_cast<uint32_t>(q));
        p += 4;
        q >>= 32;
    }
    if (n & 2) {
        store_piece(p, static_cast<uint16_t>(q));
        p += 2;
        q >>= 16;
    }
    if (n & 1) store_piece(p, static_cast<uint8_t>(q));
}

// The workgroup's turn among the rows.  Consecutive workgroups run on different XCDs, each with its
// own L2: of every 128 those on one XCD take consecutive rows, which share cache lines where rows
// end inside them ([40000, 2143] fp16 with the residual to e4m3 155 -> 142 us, [12000, 8111] bf16
// 166 -> 162, [32768, 4096] to e4m3 157 -> 156; the backward kernel, whose workgroups take many
// rows, gains nothing by it, and takes longer with consecutive rows each, 171 -> 187).
__device__ __forceinline__ unsigned rows_turn() {
    constexpr unsigned XCDS = 8, EACH = 16, ALL = XCDS * EACH;
    const unsigned b = blockIdx.x;
    if (b >= gridDim.x / ALL * ALL) return b;
    return b / ALL * ALL + b % XCDS * EACH + b / XCDS % EACH;
}

// ---------------------------------------------------------------------------
// Forward: one row a group at a time.  out may be a (without RESID), residual_out
// a or b: a row's loads all end before its first store.
//
// Bound by memory: [8192, 1600] bf16 with the residual 16.3 us (105 MB, 6.4 TB/s, partly the
// last-level cache), [32768, 4096] to e4m3 with a scale for 128 columns 157 us (944 MB, 6.0 TB/s); 16
// rows of 1600 by the launch (4.4 us, the kernel 2.9).  The squares' sum and a row's largest
// |h gamma| are exchanged together: the codes need no second exchange, for r cancels in them.
// ---------------------------------------------------------------------------
enum class Out { Rows, Row8, Block8 };  // rows; 8 bits with a scale a row, or 128 columns

template <int T, int GT, int N, bool RESID, Out OUT, bool NT>
__global__ __launch_bounds__(kGroupThreads<GT>) void rms_fwd_kernel(
    int rows, int cols, const void* a, const void* b, const float* __restrict__ gamma,
    void* residual_out, void* out, float eps, float* __restrict__ inv_rms, char* __restrict__ q,
    float* __restrict__ scales, int format) {
    constexpr bool Q8 = OUT != Out::Rows;
    constexpr int V = row_vec<T>();
    constexpr int PER = kGroupThreads<GT> / GT;
    __shared__ SumTop red[2][GroupRed<GT>::kWavesOf];
    GroupRed<GT> group{red};
    const int t = threadIdx.x & (GT - 1);
    const int units = (cols + V - 1) / V;
    for (long long row0 = static_cast<long long>(rows_turn()) * PER; row0 < rows;
         row0 += static_cast<long long>(gridDim.x) * PER) {
        const long long want = row0 + threadIdx.x / GT;
        const bool valid = want < rows;  // the others repeat the last row and store nothing
        const size_t row = valid ? static_cast<size_t>(want) : static_cast<size_t>(rows) - 1;
        const size_t base = row * cols;
        UnitAt<V> at[N];
#pragma unroll
        for (int k = 0; k < N; ++k) at[k] = unit_at<V>(t + k * GT, units, cols);

        u32x4 x[N];
        [[maybe_unused]] u32x4 y[N];
        float v[N][V];  // gamma, then h gamma
#pragma unroll
        for (int k = 0; k < N; ++k) {
            x[k] = load16b<NT>(element_ptr<T>(a, base + at[k].col));
            if constexpr (RESID) y[k] = load16b<NT>(element_ptr<T>(b, base + at[k].col));
        }
#pragma unroll
        for (int k = 0; k < N; ++k) load_gamma<V>(gamma, at[k].col, v[k]);
        // Only the last step's units can be partial or behind the row's end.
        float s = 0.0f;
        unsigned row_top = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int skip = k == N - 1 ? at[k].skip : 0;
            float h[V];
            row_unpack<T>(x[k], h);
            if constexpr (RESID) {
                float other[V];
                row_unpack<T>(y[k], other);
#pragma unroll
                for (int e = 0; e < V; ++e) h[e] = rounded(h[e] + other[e]);
                x[k] = row_pack<T>(h);  // as it is kept
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[k][e] *= h[e];
                s += e < skip ? 0.0f : h[e] * h[e];
                if constexpr (OUT == Out::Row8)
                    row_top = larger(row_top, e < skip ? 0u : magnitude(v[k][e]));
            }
        }
        const SumTop all = group.template both<OUT == Out::Row8>(s, row_top);
        const float r = 1.0f / sqrtf(all.sum / static_cast<float>(cols) + eps);
        wave_order();
        if (valid && t == 0 && inv_rms) inv_rms[row] = r;

        [[maybe_unused]] Scale sc{};
        if constexpr (OUT == Out::Row8) {
            sc = scale_of(all.top, r, format);
            if (valid && t == 0) scales[row] = sc.scale;
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const bool stored = valid && (k < N - 1 || at[k].skip < V);
            if constexpr (RESID) {
                if (stored) store16b(element_ptr<T>(residual_out, base + at[k].col), x[k]);
            }
            if (!Q8 || out) {
                float o[V];
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] = rounded(v[k][e] * r);
                if (stored) store16b(element_ptr<T>(out, base + at[k].col), row_pack<T>(o));
            }
            if constexpr (Q8) {
                if constexpr (OUT == Out::Block8) {
                    constexpr int L = MI_ROW8_BLOCK / V;         // units of a block,
                    constexpr int STEPS = L > GT ? L / GT : 1;   // in how many steps of the group
                    const int j = t + k * GT;
                    if (k % STEPS == 0) {
                        unsigned top = 0;
#pragma unroll
                        for (int i = k; i < k + STEPS && i < N; ++i)
#pragma unroll
                            for (int e = 0; e < V; ++e)
                                top = larger(top, i == N - 1 && e < at[i].skip
                                                      ? 0u
                                                      : magnitude(v[i][e]));
                        sc = scale_of(lanes_max<(L < GT ? L : GT)>(top), r, format);
                    }
                    const int blocks = (cols + MI_ROW8_BLOCK - 1) / MI_ROW8_BLOCK;
                    if (stored && j % L == 0) scales[row * blocks + j / L] = sc.scale;
                }
                const uint64_t codes = codes_of<V>(v[k], sc, format);
                if (stored) store_codes<V>(q + base + at[k].col, codes, at[k].skip);
            }
        }
    }
}

// Forward, rows of less than a unit or more than the registers hold: a workgroup a row,
// which it walks twice.  A wave takes 128 columns at a time, the columns of a scale.  A thread adds
// up to 65536 columns one after another, in 64 bits: in 32 the roundings of equal values go the
// same way, and the sum is off by 9e-4.  Bound by single-element loads and, where rows are few, by
// one workgroup's walk: [2048, 16384] fp32 with the residual 160 us (537 MB, 3.4 TB/s), [64, 131072]
// bf16 328 us (67 MB).
template <int T, bool RESID, Out OUT>
__global__ __launch_bounds__(kThreads) void rms_fwd_walk_kernel(
    int rows, int cols, const void* a, const void* b, const float* __restrict__ gamma,
    void* residual_out, void* out, float eps, float* __restrict__ inv_rms, char* __restrict__ q,
    float* __restrict__ scales, int format) {
    constexpr bool Q8 = OUT != Out::Rows;
    __shared__ SumTop red[2][kThreads / kWave];
    GroupRed<kThreads> group{red};
    const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
    const int blocks = (cols + MI_ROW8_BLOCK - 1) / MI_ROW8_BLOCK;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const size_t base = static_cast<size_t>(row) * cols;
        auto value = [&](int c) {
            float h = row_get<T>(a, base + c);
            if constexpr (RESID) h = rounded(h + row_get<T>(b, base + c));
            return h;
        };
        double s = 0.0;
        for (int c = threadIdx.x; c < cols; c += kThreads) {
            const float h = value(c);
            s += static_cast<double>(h) * static_cast<double>(h);
        }
        const float mean = group.sum(static_cast<float>(s)) / static_cast<float>(cols);
        const float r = 1.0f / sqrtf(mean + eps);
        Scale sc{};
        if constexpr (OUT == Out::Row8) {
            unsigned top = 0;
            for (int c = threadIdx.x; c < cols; c += kThreads)
                top = larger(top, magnitude(value(c) * gamma[c]));
            sc = scale_of(group.max(top), r, format);
            if (threadIdx.x == 0) scales[row] = sc.scale;
        }
        for (int i = wave; i < blocks; i += kThreads / kWave) {
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // the first two are the lane's columns
            unsigned top = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = i * MI_ROW8_BLOCK + e * kWave + lane;
                if (c >= cols) continue;
                const float h = value(c);
                v[e] = h * gamma[c];
                top = larger(top, magnitude(v[e]));
                if constexpr (RESID) row_put<T>(residual_out, base + c, h);
                if (!Q8 || out) row_put<T>(out, base + c, rounded(v[e] * r));
            }
            if constexpr (Q8) {
                if constexpr (OUT == Out::Block8) {
                    sc = scale_of(lanes_max<kWave>(top), r, format);
                    if (lane == 0) scales[static_cast<size_t>(row) * blocks + i] = sc.scale;
                }
                const uint64_t codes = codes_of<4>(v, sc, format);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int c = i * MI_ROW8_BLOCK + e * kWave + lane;
                    if (c < cols) q[base + c] = static_cast<char>(codes >> (8 * e));
                }
            }
        }
        if (threadIdx.x == 0 && inv_rms) inv_rms[row] = r;
    }
}

// ---------------------------------------------------------------------------
// Backward.  A group walks its rows, holding gamma and its columns' sums of
// dgamma in registers; a workgroup's groups add theirs through LDS, in order, into
// one partial row, and colsum_finalize adds the partial rows.
//
// Bound by memory, and the second launch: [8192, 768] fp32 into the residual stream's gradient 18.5
// us (101 MB), [16384, 4096] bf16 92.7 us (537 MB, 5.8 TB/s; with loads that are kept in the caches
// 100), [4095, 769] fp16, rows off any alignment, 8.3 (19 MB).
// ---------------------------------------------------------------------------
template <int GT>
constexpr int kBwdGroupThreads = GT > kBwdThreads ? GT : kBwdThreads;

template <int T, int GT, int N, bool ADD, bool NT>
__global__ __launch_bounds__(kBwdGroupThreads<GT>) void rms_bwd_kernel(
    int rows, int cols, const void* dy, const void* __restrict__ x,
    const float* __restrict__ inv_rms, const float* __restrict__ gamma, void* dx,
    float* __restrict__ part) {
    constexpr int V = row_vec<T>();
    constexpr int WG = kBwdGroupThreads<GT>;
    constexpr int PER = WG / GT;
    extern __shared__ __align__(16) float sums[];  // [PER][cols]
    __shared__ float red[2][WG / kWave];
    const int t = threadIdx.x & (GT - 1), grp = threadIdx.x / GT;
    const int units = (cols + V - 1) / V;
    UnitAt<V> at[N];
    float gm[N][V], acc[N][V];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        at[k] = unit_at<V>(t + k * GT, units, cols);
        load_gamma<V>(gamma, at[k].col, gm[k]);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[k][e] = 0.0f;
    }
    struct Row {
        u32x4 d[N], x[N], o[ADD ? N : 1];
        float r;
    };
    auto load = [&](long long want, Row& w) {
        const size_t row = want < rows ? static_cast<size_t>(want) : static_cast<size_t>(rows) - 1;
        const size_t base = row * cols;
        w.r = inv_rms[row];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            w.d[k] = load16b<NT>(element_ptr<T>(dy, base + at[k].col));
            w.x[k] = load16b<NT>(element_ptr<T>(x, base + at[k].col));
            if constexpr (ADD)
                w.o[k] =
                    load16b<NT>(element_ptr<T>(static_cast<const void*>(dx), base + at[k].col));
        }
    };
    int turn = 0;
    auto process = [&](long long want, const Row& w) {
        const bool valid = want < rows;
        const size_t base = (valid ? static_cast<size_t>(want) : 0) * cols;
        const float r = w.r;
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float d[V], n[V];
            row_unpack<T>(w.d[k], d);
            row_unpack<T>(w.x[k], n);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const bool counts = valid && !(k == N - 1 && e < at[k].skip);
                const float dn = counts ? d[e] * (n[e] * r) : 0.0f;
                acc[k][e] += dn;
                s += dn * gm[k][e];
            }
        }
        float total;
        if constexpr (GT <= kWave) {
            total = lanes_sum<GT>(s);
        } else {
            s = wave_sum(s);
            if ((threadIdx.x & (kWave - 1)) == 0) red[turn][threadIdx.x / kWave] = s;
            __syncthreads();
            const int w0 = grp * (GT / kWave);
            total = red[turn][w0];
#pragma unroll
            for (int i = 1; i < GT / kWave; ++i) total += red[turn][w0 + i];
            turn ^= 1;
        }
        wave_order();
        const float m = total / static_cast<float>(cols);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float d[V], n[V], o[V];
            row_unpack<T>(w.d[k], d);
            row_unpack<T>(w.x[k], n);
            if constexpr (ADD) row_unpack<T>(w.o[k], o);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float v = r * (d[e] * gm[k][e] - n[e] * r * m);
                o[e] = rounded(ADD ? o[e] + v : v);
            }
            if (valid && (k < N - 1 || at[k].skip < V))
                store16b(element_ptr<T>(dx, base + at[k].col), row_pack<T>(o));
        }
    };
    const long long stride = static_cast<long long>(gridDim.x) * PER;
    long long row0 = static_cast<long long>(blockIdx.x) * PER;
    if constexpr (GT <= kWave) {
        // The next row's loads go out before a row is worked on: two sets of registers in turn,
        // for copies from one to the other would wait for the loads.
        Row w0, w1;
        load(row0 + grp, w0);
        while (row0 < rows) {
            load(row0 + stride + grp, w1);
            process(row0 + grp, w0);
            if (row0 + stride >= rows) break;
            load(row0 + 2 * stride + grp, w0);
            process(row0 + stride + grp, w1);
            row0 += 2 * stride;
        }
    } else {
        for (; row0 < rows; row0 += stride) {
            Row w;
            load(row0 + grp, w);
            process(row0 + grp, w);
        }
    }
    float* prow = part + static_cast<size_t>(blockIdx.x) * cols;
    float* own = PER > 1 ? sums + static_cast<size_t>(grp) * cols : prow;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e >= at[k].skip) own[at[k].col + e] = acc[k][e];
    if constexpr (PER > 1) {
        __syncthreads();
        for (int c = threadIdx.x; c < cols; c += WG) {
            float v = sums[c];
            for (int g = 1; g < PER; ++g) v += sums[static_cast<size_t>(g) * cols + c];
            prow[c] = v;
        }
    }
}

// Backward, rows of less than a unit or too long for registers: a workgroup walks a row twice
// and keeps its columns' sums in its partial row, each column with one thread.  A row's products
// are added in 64 bits, as the forward kernel's squares are.  Rows of less than a unit can be
// hundreds of millions: their columns' sums stay in a register, in 64 bits too.  Bound as the
// forward kernel, and by the partial row's read and write beside each element: [2048, 16384] fp32
// onto the residual stream's gradient 491 us (537 MB), [64, 131072] bf16 353 us.
template <int T, bool ADD>
__global__ __launch_bounds__(kThreads) void rms_bwd_walk_kernel(
    int rows, int cols, const void* dy, const void* __restrict__ x,
    const float* __restrict__ inv_rms, const float* __restrict__ gamma, void* dx,
    float* __restrict__ part) {
    __shared__ SumTop red[2][kThreads / kWave];
    GroupRed<kThreads> group{red};
    float* prow = part + static_cast<size_t>(blockIdx.x) * cols;
    const bool narrow = cols < row_vec<T>();
    double own = 0.0;  // the thread's column's, where narrow
    for (int c = threadIdx.x; c < cols; c += kThreads) prow[c] = 0.0f;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const size_t base = static_cast<size_t>(row) * cols;
        const float r = inv_rms[row];
        double s = 0.0;
        for (int c = threadIdx.x; c < cols; c += kThreads)
            s += static_cast<double>(row_get<T>(dy, base + c) * (row_get<T>(x, base + c) * r)) *
                 static_cast<double>(gamma[c]);
        const float m = group.sum(static_cast<float>(s)) / static_cast<float>(cols);
        auto put = [&](int c) {  // the row's gradient in column c; gives gamma's
            const float d = row_get<T>(dy, base + c), n = row_get<T>(x, base + c) * r;
            float v = r * (d * gamma[c] - n * m);
            if constexpr (ADD) v += row_get<T>(dx, base + c);
            row_put<T>(dx, base + c, rounded(v));
            return d * n;
        };
        if (narrow) {
            if (static_cast<int>(threadIdx.x) < cols) own += static_cast<double>(put(threadIdx.x));
        } else {
            for (int c = threadIdx.x; c < cols; c += kThreads) prow[c] += put(c);
        }
    }
    if (narrow && static_cast<int>(threadIdx.x) < cols) prow[threadIdx.x] = static_cast<float>(own);
}

// ---------------------------------------------------------------------------
// Host dispatch.
// ---------------------------------------------------------------------------

// Calls f(GT, N): threads of a row's group and units of a thread.
template <int GT, int FROM, int TO, class F>
void with_steps(int units, F f) {
    if constexpr (FROM < TO) {
        if (units > GT * FROM) return with_steps<GT, FROM + 1, TO>(units, f);
    }
    f(std::integral_constant<int, GT>(), std::integral_constant<int, FROM>());
}

// A wave holds a row of up to 2048 columns; a few rows, and longer ones, take more waves each.  Many
// rows that do not fill one take 16 or 32 lanes: [34973, 339] fp16, 43 units, to e4m3 14.1 -> 9.9 us,
// [44187, 576] bf16, 72 units, 20.6 -> 14.5, [100000, 256] fp32, 64 units, which a wave has one of a
// lane, 31.8 -> 25.4; but [65536, 1024] bf16, 128 units, 75.1 -> 76.5.
// 16-bit rows of up to 4096 columns, without the residual, that are too long for a wave take two:
// [39009, 2688] bf16 to e4m3 75 -> 65, as rows 74 -> 71; but with the residual [30227, 3469] 150 ->
// 154, and fp32 [11872, 4000] 45 -> 50.
//
// Streamed rows that end inside cache lines take a wave where one unit a lane is enough, with the
// residual, or for nine tenths of its lanes: a part of a wave's access to each of several rows
// splits a line at either end ([120000, 500] bf16 with the residual 108 -> 81, without 80 -> 67,
// [148883, 403] with it 112 -> 86; but [302114, 331] without 83 -> 89, and whole lines, [157108,
// 384] with it, 67 -> 75).
template <int T, bool RESID, class F>
void with_fwd_shape(int rows, int cols, bool streamed, F f) {
    constexpr int STEPS = fwd_steps(T), NARROW = kFwdNarrowSteps;
    constexpr bool PAIRS = T != MI_TYPE_F32 && !RESID;
    const int units = units_of(cols, T);
    const bool split = streamed && cols * row_type_size(T) % kLine != 0;
    const bool narrow =
        rows >= kManyRows && (units > 64 ? !fills_wave(units) : !split || !(RESID || fills_wave(units)));
    if (units <= 16 || (narrow && units <= 16 * NARROW))
        with_steps<16, 1, NARROW>(units, f);
    else if (units <= 32)
        with_steps<32, 1, 1>(units, f);
    else if (narrow && units <= 32 * NARROW)
        with_steps<32, NARROW / 2 + 1, NARROW>(units, f);
    else if (units <= 64 || (units <= 64 * STEPS && rows > kFewRows))
        with_steps<64, 1, STEPS>(units, f);
    else if (PAIRS && units <= 128 * STEPS && rows > kFewRows)
        with_steps<PAIRS ? 128 : 256, STEPS / 2 + 1, STEPS>(units, f);
    else if (units <= 256 * STEPS)
        with_steps<256, 1, STEPS>(units, f);
    else
        with_steps<1024, STEPS / 4 + 1, wide_steps(T)>(units, f);
}

inline unsigned row_grid(int rows, int per, int most) {
    return static_cast<unsigned>(
        std::min<long long>((static_cast<long long>(rows) + per - 1) / per, most));
}

template <int T, bool RESID, Out OUT>
void launch_forward(const Forward& c, hipStream_t st) {
    char* q = static_cast<char*>(c.q);
    if (walked(c.cols, T, 1024 * wide_steps(T))) {
        hipLaunchKernelGGL((rms_fwd_walk_kernel<T, RESID, OUT>), dim3(row_grid(c.rows, 1, kMaxGrid)),
                           dim3(kThreads), 0, st, c.rows, c.cols, c.a, c.b, c.gamma,
                           c.residual_out, c.out, c.eps, c.inv_rms, q, c.scales, c.format);
        return;
    }
    const bool nt = stream_loads(static_cast<double>(c.rows) * c.cols * row_type_size(T) *
                                 (RESID ? 2 : 1));
    const int most = !RESID && !c.out ? kRow8Grid : kMaxGrid;
    with_fwd_shape<T, RESID>(c.rows, c.cols, nt, [&](auto gt, auto n) {
        constexpr int GT = decltype(gt)::value, N = decltype(n)::value;
        // a few rows alone have four waves for what one holds: they are never streamed
        constexpr bool FEW = GT == 256 && N <= fwd_steps(T) / 4;
        with_flag(nt && !FEW, [&](auto stream) {
            constexpr bool NT = decltype(stream)::value && !FEW;
            hipLaunchKernelGGL((rms_fwd_kernel<T, GT, N, RESID, OUT, NT>),
                               dim3(row_grid(c.rows, kGroupThreads<GT> / GT, most)),
                               dim3(kGroupThreads<GT>), 0, st, c.rows, c.cols, c.a, c.b, c.gamma,
                               c.residual_out, c.out, c.eps, c.inv_rms, q, c.scales, c.format);
        });
    });
}

template <int T>
void forward(const Forward& c, hipStream_t st) {
    with_flag(c.b != nullptr, [&](auto resid) {
        constexpr bool RESID = decltype(resid)::value;
        if (!c.q)
            launch_forward<T, RESID, Out::Rows>(c, st);
        else if (c.block)
            launch_forward<T, RESID, Out::Block8>(c, st);
        else
            launch_forward<T, RESID, Out::Row8>(c, st);
    });
}

template <int T, class F>
void with_bwd_shape(int rows, int units, F f) {
    constexpr int STEPS = bwd_steps(T);
    switch (bwd_threads(rows, units, T)) {
        case 16: return with_steps<16, 1, bwd_narrow_steps(T)>(units, f);
        case 32: return with_steps<32, 1, bwd_narrow_steps(T)>(units, f);
        case 64: return with_steps<64, 1, STEPS>(units, f);
        case 256: return with_steps<256, 1, STEPS>(units, f);
        default: return with_steps<1024, STEPS / 4 + 1, wide_steps(T)>(units, f);
    }
}

template <int T>
void backward(const Backward& c, hipStream_t st) {
    const int blocks = backward_blocks(c.rows, c.cols, T);
    const bool nt = stream_loads(static_cast<double>(c.rows) * c.cols * row_type_size(T) *
                                 (c.add ? 3 : 2));
    with_flag(c.add, [&](auto add) {
        constexpr bool ADD = decltype(add)::value;
        if (walked(c.cols, T, 1024 * wide_steps(T))) {
            hipLaunchKernelGGL((rms_bwd_walk_kernel<T, ADD>), dim3(blocks), dim3(kThreads), 0, st,
                               c.rows, c.cols, c.grad_out, c.x, c.inv_rms, c.gamma, c.dx, c.part);
            return;
        }
        with_bwd_shape<T>(c.rows, units_of(c.cols, T), [&](auto gt, auto n) {
            constexpr int GT = decltype(gt)::value, N = decltype(n)::value;
            constexpr int WG = kBwdGroupThreads<GT>, PER = WG / GT;
            with_flag(nt, [&](auto stream) {
                hipLaunchKernelGGL((rms_bwd_kernel<T, GT, N, ADD, decltype(stream)::value>),
                                   dim3(blocks), dim3(WG),
                                   PER > 1 ? static_cast<size_t>(PER) * c.cols * sizeof(float) : 0,
                                   st, c.rows, c.cols, c.grad_out, c.x, c.inv_rms, c.gamma, c.dx,
                                   c.part);
            });
        });
    });
}

}  // namespace rms
}  // namespace mi

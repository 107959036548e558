// What a mixture-of-experts feed-forward layer does around its matrix
// products, for gfx950: the router's choice of experts and its gradient, the
// slots sorted by expert, token rows copied to their experts' rows and back.
// No counterpart in the reference, whose feed-forward layer is dense; the rows
// move as in its embedding gather and scatter-add
// (FINAL_CLEAN_CODE/src/kernels/embedding.cu:4-79), without atomics.
//
// Notation: N tokens, k choices each; slot t * k + j is choice j of token t.
// The sorted buffer has `rows` rows; position[slot] is the slot's row, and any
// value outside [0, rows) means the slot was dropped.
#include <algorithm>
#include <climits>
#include <type_traits>
#include <utility>

#include "mi_common.hpp"
#include "mi_rowtype.hpp"

namespace mi {

namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxChoices = 16;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxGrid = 1 << 20;  // workgroups over the tokens, which are taken in strides
constexpr int kMaxCols = 1 << 22;  // keeps a row's segments in the grid's second dimension

// ---------------------------------------------------------------------------
// Router.  A row's E logits lie in the registers of L lanes, P in each.  A logit
// becomes an integer key of the same order: the bits, the lower 31 inverted for
// negative numbers, -0 made +0; NaN ranks above all and -inf is the lowest key,
// which is never chosen.  Key and expert make one double, key * 1024 - expert:
// exact, all different, and in the order wanted, equal logits by rising expert.
// Each lane sorts its P doubles once, by a network of minima and maxima; a round
// takes the largest of the lanes' first ones (DPP) and the lane that held it
// moves up.  Lane j of the group keeps the double of round j.
//
// Bound by these instructions, not by memory (32768 x 256 fp32, 8 chosen: 12.2 us, its
// 36 MB take 7; bf16 12.4, for half the bytes): comparisons are of 64 bits, and the
// network sorts all of a lane's logits however few are chosen (2 chosen 9.4 us, 1 7.6).
// 16 lanes a row (four rows a wave) share the steps between lanes among four rows.
// Rounds that search each lane's logits for the largest key instead took 17.6 us
// there, and 6.9 instead of 4.3 for 1024 rows.
// ---------------------------------------------------------------------------
constexpr int kNoKey = static_cast<int>(0xff800000u ^ 0x7fffffffu);  // of -inf
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ int order_key(float f) {
    const int b = __float_as_int(f + 0.0f);
    const int key = b ^ ((b >> 31) & 0x7fffffff);
    return f != f ? INT_MAX : key;
}

// The logit of a key (NaN for NaN's key).
__device__ __forceinline__ float key_value(int key) {
    return __int_as_float(key ^ ((key >> 31) & 0x7fffffff));
}

// A lane's logits of a row: P, in pieces of one access that it takes in turn with the row's
// other lanes.  Their experts are gl * N, N = kPiece, and the steps that step_expert gives.
template <int T, int P>
constexpr int kPiece = P < row_vec<T>() ? P : row_vec<T>();

template <int T, int L, int P>
constexpr int step_expert(int p) {
    constexpr int N = kPiece<T, P>;
    return p / N * (N * L) + p % N;
}

// Loads them, -inf behind the last expert.  Accesses may run into the next row, and are
// cut to single elements only at the tensor's end.
template <int T, int L, int P>
__device__ __forceinline__ void load_logits(const void* logits, size_t row, size_t rows, int gl,
                                            int experts, float (&v)[P]) {
    constexpr int N = kPiece<T, P>;
    const size_t base = row * experts, total = rows * experts;
#pragma unroll
    for (int c = 0; c < P; c += N) {
        const int e0 = gl * N + step_expert<T, L, P>(c);
        float part[N];
#pragma unroll
        for (int e = 0; e < N; ++e) part[e] = 0.0f;
        if (e0 < experts) {
            if (base + e0 + N <= total) {
                row_get_n<T, N>(logits, base + e0, part);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (e0 + e < experts) part[e] = row_get<T>(logits, base + e0 + e);
            }
        }
#pragma unroll
        for (int e = 0; e < N; ++e) v[c + e] = e0 + e < experts ? part[e] : -__builtin_inff();
    }
}

template <int CTRL>
__device__ __forceinline__ double dpp_move_d(double v) {
    const u32x2 b = __builtin_bit_cast(u32x2, v);
    const u32x2 r = {static_cast<uint32_t>(dpp_move_i<CTRL>(static_cast<int>(b.x))),
                     static_cast<uint32_t>(dpp_move_i<CTRL>(static_cast<int>(b.y)))};
    return __builtin_bit_cast(double, r);
}

// The last lane of a row of 16 (CTRL 0x142) or of 32 (0x143) to the rows behind it that
// ROWS names; the others keep v.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_bcast_d(double v) {
    const u32x2 b = __builtin_bit_cast(u32x2, v);
    const int x = static_cast<int>(b.x), y = static_cast<int>(b.y);
    const u32x2 r = {
        static_cast<uint32_t>(__builtin_amdgcn_update_dpp(x, x, CTRL, ROWS, 0xF, false)),
        static_cast<uint32_t>(__builtin_amdgcn_update_dpp(y, y, CTRL, ROWS, 0xF, false))};
    return __builtin_bit_cast(double, r);
}

__device__ __forceinline__ double readlane_d(double v, int lane) {
    const u32x2 b = __builtin_bit_cast(u32x2, v);
    const u32x2 r = {
        static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b.x), lane)),
        static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b.y), lane))};
    return __builtin_bit_cast(double, r);
}

template <int L>
__device__ __forceinline__ double group_max_d(double v) {
    v = fmax(v, dpp_move_d<0xB1>(v));
    v = fmax(v, dpp_move_d<0x4E>(v));
    v = fmax(v, dpp_move_d<0x141>(v));
    v = fmax(v, dpp_move_d<0x140>(v));
    if constexpr (L == 64) {
        v = fmax(v, dpp_bcast_d<0x142, 0xA>(v));
        v = fmax(v, dpp_bcast_d<0x143, 0xC>(v));
        v = readlane_d(v, 63);
    }
    return v;
}

__device__ __forceinline__ double rank_of(int key, double expert) {
    return fma(static_cast<double>(key), 1024.0, -expert);
}

__device__ __forceinline__ int rank_key(double rank) {
    return static_cast<int>(ceil(rank * (1.0 / 1024.0)));
}

__device__ __forceinline__ int rank_expert(double rank, int key) {
    return static_cast<int>(fma(static_cast<double>(key), 1024.0, -rank));
}

// Batcher's odd-even merge sort of P values (a power of two): its comparisons, in
// order, as pairs of places.
template <int P>
struct SortNet {
    int lo[P * 8] = {}, hi[P * 8] = {};
    int n = 0;
    constexpr SortNet() {
        for (int p = 1; p < P; p *= 2)
            for (int k = p; k >= 1; k /= 2)
                for (int i = k % p; i + k < P; ++i)
                    if ((i - k % p) / k % 2 == 0 && i / (2 * p) == (i + k) / (2 * p)) {
                        lo[n] = i;
                        hi[n++] = i + k;
                    }
    }
};

template <int P, int... I>
__device__ __forceinline__ void sort_falling(double (&d)[P], std::integer_sequence<int, I...>) {
    constexpr SortNet<P> net;
    auto place = [&](auto at) {
        constexpr int a = net.lo[decltype(at)::value], b = net.hi[decltype(at)::value];
        const double big = fmax(d[a], d[b]), small = fmin(d[a], d[b]);
        d[a] = big;
        d[b] = small;
    };
    (place(std::integral_constant<int, I>()), ...);
}

template <int P>
__device__ __forceinline__ void sort_falling(double (&d)[P]) {
    sort_falling(d, std::make_integer_sequence<int, SortNet<P>().n>());
}

// Where `won`, each of the first D values takes the next one's place.  (With the
// places written out: a loop's select becomes a search for place p + won.)
template <int D, int P, int... I>
__device__ __forceinline__ void move_up(double (&d)[P], bool won, double last,
                                        std::integer_sequence<int, I...>) {
    ((d[I] = won ? d[I + 1] : d[I]), ...);
    d[D - 1] = won ? last : d[D - 1];
}

// D: how many of a lane's logits may be chosen, at most.
template <int T, int L, int P, int D, bool RENORM>
__global__ __launch_bounds__(kThreads) void gate_fwd_kernel(const void* __restrict__ logits,
                                                            int* __restrict__ ids,
                                                            float* __restrict__ weights,
                                                            int tokens, int experts, int k) {
    constexpr int PER = kThreads / L;  // rows per workgroup
    const int gl = threadIdx.x & (L - 1);
    for (long long base = static_cast<long long>(blockIdx.x) * PER; base < tokens;
         base += static_cast<long long>(gridDim.x) * PER) {
        const long long want = base + threadIdx.x / L;
        const bool valid = want < tokens;  // the others repeat the last row and store nothing
        const size_t row = valid ? static_cast<size_t>(want) : static_cast<size_t>(tokens) - 1;
        float v[P];
        load_logits<T, L, P>(logits, row, tokens, gl, experts, v);
        double rank[P];
        const double own = gl * kPiece<T, P>;  // the lane's first expert
#pragma unroll
        for (int p = 0; p < P; ++p)
            rank[p] = rank_of(order_key(v[p]), own) - step_expert<T, L, P>(p);
        sort_falling(rank);

        double first = 0.0, mine = rank_of(kNoKey, 0.0);
        for (int j = 0; j < k; ++j) {
            const double m = group_max_d<L>(rank[0]);
            const bool won = rank[0] == m;
            move_up<D>(rank, won, rank_of(kNoKey, 1023.0),
                       std::make_integer_sequence<int, D - 1>());
            first = j == 0 ? m : first;
            mine = gl == j ? m : mine;
        }
        const int top_key = rank_key(first), key = rank_key(mine);
        const float top = top_key == kNoKey ? 0.0f : key_value(top_key);
        const float e = key == kNoKey ? 0.0f : expf(key_value(key) - top);
        float s = e;
        if constexpr (!RENORM) {
            s = 0.0f;
#pragma unroll
            for (int p = 0; p < P; ++p) s += __builtin_amdgcn_exp2f((v[p] - top) * kLog2e);
        }
        const float total = group_sum<L>(s);
        if (valid && gl < k) {
            ids[row * k + gl] = key == kNoKey ? -1 : rank_expert(mine, key);
            weights[row * k + gl] = key == kNoKey ? 0.0f : e / total;
        }
    }
}

// dl_e = sum over the slots j with id_j = e of w_j (dw_j [- d]) - p_e d, with
// d = sum_j w_j dw_j; the term in p_e only where the weights are not
// renormalised, [- d] only where they are.  The slots' terms are added into a
// row of zeros in LDS, slot after slot (a wave's LDS operations run in order),
// which costs less than comparing every element's number with every slot's (32768 x
// 256 fp32, 8 slots: 51.0 -> 18.4 us).  A row's lanes take its pieces in turn, so that
// their accesses, of LDS too, are consecutive: with 16 numbers of a lane side by side it
// took 18.0 us, 11.7 so (6.0 TB/s), bf16 14.7, 10.5, renormalised 13.8, 8.7.  16-bit rows
// (3.5 TB/s) are bound by instructions: every element passes through the row in LDS.
template <int T, int L, int P, bool RENORM>
__global__ __launch_bounds__(kThreads) void gate_bwd_kernel(
    const void* __restrict__ logits, const int* __restrict__ ids,
    const float* __restrict__ weights, const float* __restrict__ dweights,
    void* __restrict__ dlogits, int tokens, int experts, int k) {
    constexpr int PER = kThreads / L;
    constexpr int N = kPiece<T, P>;
    __shared__ __align__(16) float terms[PER][L * P];
    const int gl = threadIdx.x & (L - 1);
    float* own = terms[threadIdx.x / L];
#pragma unroll
    for (int p = 0; p < P; ++p) own[gl * N + step_expert<T, L, P>(p)] = 0.0f;
    for (long long base = static_cast<long long>(blockIdx.x) * PER; base < tokens;
         base += static_cast<long long>(gridDim.x) * PER) {
        const long long want = base + threadIdx.x / L;
        const bool valid = want < tokens;
        const size_t row = valid ? static_cast<size_t>(want) : static_cast<size_t>(tokens) - 1;

        int id = -1;
        float w = 0.0f, dw = 0.0f;
        if (gl < k) {
            id = ids[row * k + gl];
            w = weights[row * k + gl];
            dw = dweights[row * k + gl];
        }
        float v[P];
        if constexpr (!RENORM) load_logits<T, L, P>(logits, row, tokens, gl, experts, v);
        const bool live = id >= 0 && id < experts;
        const float wd = live ? w * dw : 0.0f;
        const float d = group_sum<L>(wd);
        const float term = RENORM ? w * (dw - d) : wd;
        wave_order();
        for (int j = 0; j < k; ++j)
            if (gl == j && live) atomicAdd(&own[id], term);
        if constexpr (!RENORM) {
            float top = v[0];
#pragma unroll
            for (int p = 1; p < P; ++p) top = fmaxf(top, v[p]);
            top = group_max<L>(top);
            if (top == -__builtin_inff()) top = 0.0f;  // every e below is 0, or NaN
            float s = 0.0f;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                v[p] = __builtin_amdgcn_exp2f((v[p] - top) * kLog2e);
                s += v[p];
            }
            s = group_sum<L>(s);
            const float scale = -d / (s == 0.0f ? 1.0f : s);
#pragma unroll
            for (int p = 0; p < P; ++p) v[p] *= scale;
        }
        wave_order();
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const float t = own[gl * N + step_expert<T, L, P>(p)];
            v[p] = RENORM ? t : v[p] + t;
        }
#pragma unroll
        for (int p = 0; p < P; ++p) own[gl * N + step_expert<T, L, P>(p)] = 0.0f;
#pragma unroll
        for (int c = 0; c < P; c += N) {
            const int e0 = gl * N + step_expert<T, L, P>(c);
            float part[N];
#pragma unroll
            for (int e = 0; e < N; ++e) part[e] = v[c + e];
            if (valid && e0 + N <= experts) {
                row_put_n<T, N>(dlogits, row * experts + e0, part);
            } else if (valid) {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (e0 + e < experts) row_put<T>(dlogits, row * experts + e0 + e, part[e]);
            }
        }
    }
}

// f(L, P): 16 lanes a row up to 256 experts, 64 lanes above; where `wide`, 16 up to 512.
template <bool MAY_BE_WIDE, class F>
void with_gate_shape(int experts, bool wide, F f) {
    using std::integral_constant;
    if constexpr (MAY_BE_WIDE) {
        if (wide && experts > 256 && experts <= 512)
            return f(integral_constant<int, 16>(), integral_constant<int, 32>());
    }
    if (experts <= 16)
        f(integral_constant<int, 16>(), integral_constant<int, 1>());
    else if (experts <= 32)
        f(integral_constant<int, 16>(), integral_constant<int, 2>());
    else if (experts <= 64)
        f(integral_constant<int, 16>(), integral_constant<int, 4>());
    else if (experts <= 128)
        f(integral_constant<int, 16>(), integral_constant<int, 8>());
    else if (experts <= 256)
        f(integral_constant<int, 16>(), integral_constant<int, 16>());
    else if (experts <= 512)
        f(integral_constant<int, 64>(), integral_constant<int, 8>());
    else
        f(integral_constant<int, 64>(), integral_constant<int, 16>());
}

unsigned gate_grid(int tokens, int lanes) {
    const int per = kThreads / lanes;
    return static_cast<unsigned>(
        std::min<long long>((static_cast<long long>(tokens) + per - 1) / per, kMaxGrid));
}

// ---------------------------------------------------------------------------
// Stable sort of the slots by expert (a counting sort).  A workgroup takes a
// chunk of consecutive slots, each of its 16 waves a consecutive part of it.
// A wave takes 64 slots at a time: the lanes with the same expert are found by
// one ballot per bit of the id, a slot's rank among them is the number of such
// lanes before it, and the first of them advances the wave's count of that
// expert.  Counts are whole numbers, so the result does not depend on timing.
//
// Latency-bound: a handful of memory and LDS round trips one after the other.
// One chunk is one launch; more take a first launch that counts each chunk's
// experts.  Slots a lane in a sort of several chunks, both launches: 262144 slots
// of 256 experts one 17.0 us, two 12.5, four 12.0; 32768 of 64 6.9, 7.2, 8.8;
// 65536 of 8 6.2, 6.7, 8.6.
// ---------------------------------------------------------------------------
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kSortOneTrips = 4;  // slots of a lane in a sort of one chunk, at most
constexpr int kSortTrips = 2;     // slots of a lane in one of several, at least
constexpr int kSortMaxChunks = 256;

struct SortPlan {
    int trips;   // slots of a lane
    int chunks;
    long long chunk() const { return static_cast<long long>(trips) * kSortThreads; }
};

SortPlan plan_sort(int slots) {
    auto parts = [&](long long of) {
        return static_cast<int>((static_cast<long long>(slots) + of - 1) / of);
    };
    SortPlan p;
    p.trips = std::max(1, parts(kSortThreads));
    if (p.trips > kSortOneTrips)
        p.trips =
            std::max(kSortTrips, parts(static_cast<long long>(kSortMaxChunks) * kSortThreads));
    p.chunks = std::max(1, parts(p.chunk()));
    return p;
}

// hist[c][e]: slots of expert e in chunk c.
__global__ __launch_bounds__(kSortThreads) void sort_hist_kernel(const int* __restrict__ ids,
                                                                 int* __restrict__ hist,
                                                                 int slots, int experts,
                                                                 int trips) {
    extern __shared__ int count[];
    for (int e = threadIdx.x; e < experts; e += kSortThreads) count[e] = 0;
    __syncthreads();
    const long long begin = static_cast<long long>(blockIdx.x) * trips * kSortThreads;
    for (int i = 0; i < trips; ++i) {
        const long long s = begin + i * kSortThreads + threadIdx.x;
        const int id = s < slots ? ids[s] : -1;
        if (id >= 0 && id < experts) atomicAdd(&count[id], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += kSortThreads)
        hist[static_cast<size_t>(blockIdx.x) * experts + e] = count[e];
}

// The lanes whose id equals this lane's, among the lanes with an id.
__device__ __forceinline__ unsigned long long same_id(int id, bool has, int bits) {
    unsigned long long m = __ballot(has);
    for (int b = 0; b < bits; ++b) {
        const bool one = (id >> b) & 1;
        const unsigned long long ones = __ballot(one);
        m &= one ? ones : ~ones;
    }
    return m;
}

// hist == nullptr: there is one chunk.  NR: the lane's ids, up to NR of them,
// stay in registers from the counting to the placing (0: they are read again).
template <int NR>
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(
    const int* __restrict__ ids, const int* __restrict__ hist, int* __restrict__ offsets,
    int* __restrict__ order, int* __restrict__ position, int slots, int experts, int trips,
    int chunks, int bits) {
    extern __shared__ int count[];  // [kSortWaves][experts], then [2][experts] of the chunks
    __shared__ int wave_total[kSortWaves];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = threadIdx.x / kWave;
    const long long begin =
        static_cast<long long>(blockIdx.x) * trips * kSortThreads +
        static_cast<long long>(wave) * trips * kWave + lane;
    auto slot_id = [&](int i) {
        const long long s = begin + i * kWave;
        const int id = s < slots ? ids[s] : -1;
        return id < experts ? id : -1;
    };
    int held[NR ? NR : 1];
#pragma unroll
    for (int i = 0; i < NR; ++i) held[i] = i < trips ? slot_id(i) : -1;

    int* totals = count + kSortWaves * experts;  // slots of each expert in all chunks
    int* befores = totals + experts;             // and in the chunks before this one
    const int cells = (kSortWaves + (hist == nullptr ? 0 : 2)) * experts;
    for (int i = threadIdx.x; i < cells; i += kSortThreads) count[i] = 0;
    __syncthreads();
    int* mine = count + wave * experts;
    if constexpr (NR > 0) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
            if (held[i] >= 0) atomicAdd(&mine[held[i]], 1);
    } else {
        for (int i = 0; i < trips; ++i) {
            const int id = slot_id(i);
            if (id >= 0) atomicAdd(&mine[id], 1);
        }
    }
    if (hist != nullptr) {
        // as many threads an expert as there are, each some of the chunks
        const int per = kSortThreads / experts;
        const int part = threadIdx.x / experts, x = threadIdx.x % experts;
        if (part < per) {
            int total = 0, before = 0;
#pragma unroll 4
            for (int c = part; c < chunks; c += per) {
                const int h = hist[static_cast<size_t>(c) * experts + x];
                before += c < static_cast<int>(blockIdx.x) ? h : 0;
                total += h;
            }
            atomicAdd(&totals[x], total);
            atomicAdd(&befores[x], before);
        }
    }
    __syncthreads();

    // Thread e owns expert e (experts <= kSortThreads).
    const int e = threadIdx.x;
    int n[kSortWaves], total = 0, before = 0;
    if (e < experts) {
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) n[w] = count[w * experts + e];
        if (hist != nullptr) {
            total = totals[e];
            before = befores[e];
        } else {
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) total += n[w];
        }
    }
    // exclusive sum of the totals over the experts
    int incl = total;
    for (int d = 1; d < kWave; d <<= 1) {
        const int up = __shfl_up(incl, d);
        if (lane >= d) incl += up;
    }
    if (lane == kWave - 1) wave_total[wave] = incl;
    __syncthreads();
    if (e < experts) {
        int first = incl - total;
        for (int w = 0; w < wave; ++w) first += wave_total[w];
        if (blockIdx.x == 0) {
            offsets[e] = first;
            if (e == experts - 1) offsets[experts] = first + total;
        }
        int at = first + before;
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            count[w * experts + e] = at;
            at += n[w];
        }
    }
    __syncthreads();

    auto place = [&](int i, int id) {
        const long long s = begin + i * kWave;
        const bool has = id >= 0;
        const unsigned long long same = same_id(id, has, bits);
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const int at = has ? mine[id] : 0;
        wave_order();
        if (has && rank == 0) mine[id] = at + __popcll(same);
        wave_order();
        if (s < slots) position[s] = has ? at + rank : -1;
        if (has && order != nullptr) order[at + rank] = static_cast<int>(s);
    };
    if constexpr (NR > 0) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
            if (i < trips) place(i, held[i]);
    } else {
        for (int i = 0; i < trips; ++i) place(i, slot_id(i));
    }
}

// ---------------------------------------------------------------------------
// Rows moved between token order and expert order.  A wave takes one token
// and a segment of U * 64 16-byte chunks of its row, so the token's positions
// are wave-uniform; of rows of at most 16 or 32 chunks it takes as many tokens as
// fit, LT = 16 or 32 lanes each.  Where the row is no multiple of 16 bytes the
// last chunk is moved back to end with the row: the elements that it shares with
// the one before are computed twice, with the same result.
//
// Memory-bound: 4.6 to 6.1 TB/s on tensors past the last-level cache.
// ---------------------------------------------------------------------------
struct Chunk {
    bool on;
    size_t at;  // byte offset in the row
};

__device__ __forceinline__ Chunk row_chunk(int c, int chunks, size_t row_bytes) {
    const size_t at = static_cast<size_t>(c) * 16;
    return {c < chunks, at < row_bytes - 16 ? at : row_bytes - 16};
}

// The first token of this lane, and the tokens of a workgroup.
template <int LT>
constexpr int workgroup_tokens() {
    return kThreads / LT;
}

template <int LT>
__device__ __forceinline__ long long first_token(unsigned workgroup) {
    const int in = LT == kWave ? __builtin_amdgcn_readfirstlane(threadIdx.x / LT)
                               : static_cast<int>(threadIdx.x / LT);
    return static_cast<long long>(workgroup) * workgroup_tokens<LT>() + in;
}

// Segments of a row are taken by eight workgroups' tokens side by side: consecutive
// workgroups run on different XCDs, so all of a row goes through one L2 at about one time
// (fp32 [9460 tokens, 3 choices] of 3686 columns 135.9 us with all first segments before
// all second ones, 128.3 so; of 3712 120.0, 115.1; bf16 [8192, 4] of 2049 48.2, 45.5).
// The sums' reads gain nothing from it (bf16 [8192, 8] of 2050 57.6 -> 68.0).
template <int U, int LT>
__global__ __launch_bounds__(kThreads) void scatter_rows_kernel(
    const char* __restrict__ x, const int* __restrict__ position, char* __restrict__ out,
    int tokens, int k, int rows, int chunks, size_t row_bytes) {
    const int lane = threadIdx.x & (LT - 1);
    const unsigned segs = LT < kWave ? 1u : (chunks + U * LT - 1u) / (U * LT);
    const unsigned groups = gridDim.x / segs;
    unsigned seg = 0, group = blockIdx.x;
    if (segs > 1) {
        const unsigned first = blockIdx.x / (8 * segs) * 8;
        const unsigned side = min(8u, groups - first), i = blockIdx.x - first * segs;
        seg = i / side;
        group = first + i % side;
    }
    for (long long token = first_token<LT>(group); token < tokens;
         token += static_cast<long long>(groups) * workgroup_tokens<LT>()) {
        const char* src = x + static_cast<size_t>(token) * row_bytes;
        u32x4 v[U];
        Chunk ch[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            ch[u] = row_chunk(static_cast<int>(seg) * U * LT + u * LT + lane, chunks, row_bytes);
            if (ch[u].on) v[u] = load16b<false>(src + ch[u].at);
        }
        const int* pos = position + static_cast<size_t>(token) * k;
        for (int j = 0; j < k; ++j) {
            const int p = pos[j];
            if (p < 0 || p >= rows) continue;
            char* dst = out + static_cast<size_t>(p) * row_bytes;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (ch[u].on) store16b(dst + ch[u].at, v[u]);
        }
    }
}

// out[t] = sum over j, in order, of [w[t, j]] rows[position[t, j]].  A choice's position,
// then its chunks one by one are waited for before the next is loaded, so that nothing
// of a dropped slot is read; many waves hide this ([8192 tokens, 8 choices] of 4096 bf16
// 99 us, 6.1 TB/s), few do not (16 tokens of it 3.8 us; the shortest kernel here 1.4).
template <int T, int U, int LT, bool WEIGHTED, bool NT>
__global__ __launch_bounds__(kThreads) void gather_sum_kernel(
    const char* __restrict__ src, const int* __restrict__ position,
    const float* __restrict__ weights, char* __restrict__ out, int tokens, int k, int rows,
    int chunks, size_t row_bytes) {
    constexpr int V = row_vec<T>();
    const int lane = threadIdx.x & (LT - 1);
    for (long long token = first_token<LT>(blockIdx.x); token < tokens;
         token += static_cast<long long>(gridDim.x) * workgroup_tokens<LT>()) {
        Chunk ch[U];
        float acc[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            ch[u] = row_chunk(static_cast<int>(blockIdx.y) * U * LT + u * LT + lane, chunks,
                              row_bytes);
#pragma unroll
            for (int e = 0; e < V; ++e) acc[u][e] = 0.0f;
        }
        const size_t slot = static_cast<size_t>(token) * k;
        for (int j = 0; j < k; ++j) {
            const int p = position[slot + j];
            if (p < 0 || p >= rows) continue;
            const float w = WEIGHTED ? weights[slot + j] : 1.0f;
            const char* r = src + static_cast<size_t>(p) * row_bytes;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (ch[u].on) {
                    float y[V];
                    row_unpack<T>(load16b<NT>(r + ch[u].at), y);
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        acc[u][e] = WEIGHTED ? fmaf(w, y[e], acc[u][e]) : acc[u][e] + y[e];
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (ch[u].on)
                store16b(out + static_cast<size_t>(token) * row_bytes + ch[u].at,
                         row_pack<T>(acc[u]));
    }
}

// dy[position[t, j]] = w[t, j] dout[t]; dw[t, j] = dout[t] . y[position[t, j]].
// G waves, or LT lanes of one, per token; KB is k rounded up to a power of two, so that
// the k sums stay in registers: a slot that does not exist costs a cached load and FMAs
// (bf16 [8192 tokens] of 1024 columns, 4 choices 29.5 us, 5.1 TB/s, 5 38.2, 4.8, 8 56.9,
// 5.0, 9 67.4, 4.7, 16 115.6, 4.8).  All loads of a step (UC chunks of dout, KB of y for each)
// are issued before its first store; a dropped slot reads dout's chunk in the
// place of y's, and what the moved-back last chunk shares with its neighbour is
// left out of its sums.  dy may be y: a chunk of dy is written after the same chunk
// of y was read, by the same lane; a moved-back chunk also writes into its
// neighbour's, so the two must not lie in different waves (see combine_waves): in
// one wave, its loads of both come before its stores of the later one.
template <int T, int KB, int G, int LT, bool NT>
__global__ __launch_bounds__(G > kWaves ? G * kWave : kThreads) void combine_bwd_kernel(
    int tokens, int k, int rows, int chunks, size_t row_bytes, const int* __restrict__ position,
    const float* __restrict__ weights, const char* __restrict__ dout, const char* y, char* dy,
    float* __restrict__ dweights) {
    constexpr int V = row_vec<T>();
    constexpr int S = 16 / V;
    constexpr int UC = KB >= 4 ? 1 : 4 / KB;
    static_assert(G == 1 || (G >= kWaves && LT == kWave), "several waves: one token a workgroup");
    constexpr int TOKENS = G > 1 ? 1 : workgroup_tokens<LT>();
    __shared__ float sums[G][KB];  // used where G > 1
    const int lane = threadIdx.x & (LT - 1);
    const int part = G > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) : 0;
    for (long long token =
             G > 1 ? static_cast<long long>(blockIdx.x) : first_token<LT>(blockIdx.x);
         token < tokens; token += static_cast<long long>(gridDim.x) * TOKENS) {
        const size_t slot = static_cast<size_t>(token) * k;
        const char* g_row = dout + static_cast<size_t>(token) * row_bytes;
        int pos[KB];
        float w[KB], dot[KB];
#pragma unroll
        for (int j = 0; j < KB; ++j) {
            const int p = j < k ? position[slot + j] : -1;
            pos[j] = p < rows ? p : -1;
            w[j] = j < k ? weights[slot + j] : 0.0f;
            dot[j] = 0.0f;
        }
        for (int c = part * LT + lane; c < chunks; c += UC * G * LT) {
            size_t at[UC];
            u32x4 graw[UC], yraw[UC][KB];
#pragma unroll
            for (int u = 0; u < UC; ++u) {
                at[u] = row_chunk(min(c + u * G * LT, chunks - 1), chunks, row_bytes).at;
                graw[u] = load16b<NT>(g_row + at[u]);
#pragma unroll
                for (int j = 0; j < KB; ++j) {
                    const char* r =
                        pos[j] < 0 ? g_row : y + static_cast<size_t>(pos[j]) * row_bytes;
                    yraw[u][j] = load16b<NT>(r + at[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < UC; ++u) {
                const bool on = c + u * G * LT < chunks;
                const int first =
                    on ? static_cast<int>((static_cast<size_t>(c + u * G * LT) * 16 - at[u]) / S)
                       : V;
                float g[V];
                row_unpack<T>(graw[u], g);
#pragma unroll
                for (int j = 0; j < KB; ++j) {
                    float v[V];
                    row_unpack<T>(yraw[u][j], v);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        dot[j] = e < first ? dot[j] : fmaf(g[e], v[e], dot[j]);
                        v[e] = w[j] * g[e];
                    }
                    if (on && pos[j] >= 0)
                        store16b(dy + static_cast<size_t>(pos[j]) * row_bytes + at[u],
                                 row_pack<T>(v));
                }
            }
        }
#pragma unroll
        for (int j = 0; j < KB; ++j) {
            float s = group_sum<LT == 32 ? 16 : LT>(dot[j]);
            if constexpr (LT == 32) s += __shfl_xor(s, 16);
            if constexpr (G > 1) {
                if (lane == 0) sums[part][j] = s;
            } else if (lane == 0 && j < k) {
                dweights[slot + j] = pos[j] < 0 ? 0.0f : s;
            }
        }
        if constexpr (G > 1) {
            // one token a workgroup: its waves are here together
            __syncthreads();
            if (static_cast<int>(threadIdx.x) < k) {
                const int j = threadIdx.x;
                const int p = position[slot + j];
                float s = sums[0][j];
#pragma unroll
                for (int g = 1; g < G; ++g) s += sums[g][j];
                dweights[slot + j] = p >= 0 && p < rows ? s : 0.0f;
            }
            __syncthreads();
        }
    }
}

// Rows of less than 16 bytes: one thread per token.
enum class Narrow { Scatter, Sum, WeightedSum, Backward };

template <int T, Narrow OP>
__global__ __launch_bounds__(kThreads) void narrow_kernel(
    const void* a, const void* y, const int* __restrict__ position,
    const float* __restrict__ weights, void* out, float* __restrict__ dweights, int tokens, int k,
    int rows, int cols) {
    const long long t = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
    if (t >= tokens) return;
    const size_t slot = static_cast<size_t>(t) * k, row = static_cast<size_t>(t) * cols;
    if constexpr (OP == Narrow::Sum || OP == Narrow::WeightedSum) {
        for (int c = 0; c < cols; ++c) {
            float s = 0.0f;
            for (int j = 0; j < k; ++j) {
                const int p = position[slot + j];
                if (p < 0 || p >= rows) continue;
                const float v = row_get<T>(a, static_cast<size_t>(p) * cols + c);
                s = OP == Narrow::Sum ? s + v : fmaf(weights[slot + j], v, s);
            }
            row_put<T>(out, row + c, s);
        }
    } else {
        for (int j = 0; j < k; ++j) {
            const int p = position[slot + j];
            const bool there = p >= 0 && p < rows;
            float dot = 0.0f;
            if (there)
                for (int c = 0; c < cols; ++c) {
                    const size_t r = static_cast<size_t>(p) * cols + c;
                    const float v = row_get<T>(a, row + c);
                    if constexpr (OP == Narrow::Backward) {
                        dot += v * row_get<T>(y, r);
                        row_put<T>(out, r, weights[slot + j] * v);
                    } else {
                        row_put<T>(out, r, v);
                    }
                }
            if constexpr (OP == Narrow::Backward) dweights[slot + j] = dot;
        }
    }
}

template <Narrow OP>
int launch_narrow(const char* name, const void* a, const void* y, const int* position,
                  const float* weights, void* out, float* dweights, int tokens, int k, int rows,
                  int cols, int type, hipStream_t st) {
    const dim3 grid(
        static_cast<unsigned>((static_cast<long long>(tokens) + kThreads - 1) / kThreads));
    with_row_type(type, [&](auto t) {
        hipLaunchKernelGGL((narrow_kernel<decltype(t)::value, OP>), grid, dim3(kThreads), 0, st, a,
                           y, position, weights, out, dweights, tokens, k, rows, cols);
    });
    return check_launch(name);
}

unsigned token_grid(int tokens, int per_workgroup) {
    return static_cast<unsigned>(std::min<long long>(
        (static_cast<long long>(tokens) + per_workgroup - 1) / per_workgroup, kMaxGrid));
}

// Lanes of a token, and its chunks a lane takes.
struct RowShape {
    int lanes, u;
};

// f(lanes, u) and the launch's grid for rows of `chunks` chunks.
template <class F>
void with_row_shape(RowShape shape, int tokens, int chunks, F f) {
    using std::integral_constant;
    const dim3 grid(token_grid(tokens, kThreads / shape.lanes),
                    (chunks + shape.u * shape.lanes - 1) / (shape.u * shape.lanes));
    if (shape.lanes == 16)
        f(integral_constant<int, 16>(), integral_constant<int, 1>(), grid);
    else if (shape.lanes == 32)
        f(integral_constant<int, 32>(), integral_constant<int, 1>(), grid);
    else if (shape.u == 1)
        f(integral_constant<int, 64>(), integral_constant<int, 1>(), grid);
    else if (shape.u == 2)
        f(integral_constant<int, 64>(), integral_constant<int, 2>(), grid);
    else
        f(integral_constant<int, 64>(), integral_constant<int, 4>(), grid);
}

int row_lanes(int chunks) { return chunks <= 16 ? 16 : chunks <= 32 ? 32 : 64; }

// Segments of the copies' rows: short ones while there are few waves.
RowShape scatter_shape(int tokens, int chunks) {
    const long long waves = static_cast<long long>(tokens) * ((chunks + kWave - 1) / kWave);
    if (waves >= 8192 && chunks > 2 * kWave) return {64, 4};
    if (waves >= 4096 && chunks > kWave) return {64, 2};
    return {row_lanes(chunks), 1};
}

// Of the sums' rows, whose chunks a lane takes one after another for every choice: bf16
// [1024 tokens, 4 choices] of 4096 columns in segments of one, two, four chunks a lane
// 6.9, 7.1, 8.9 us, [4096, 8] of 2048 33.7, 24.9, 28.8, fp32 [8192, 6] of 1600 72.3, 67.7,
// 62.1.
RowShape gather_shape(int tokens, int chunks) {
    const long long waves = static_cast<long long>(tokens) * ((chunks + kWave - 1) / kWave);
    if (waves >= 32768 && chunks > 2 * kWave) return {64, 4};
    if (waves >= 4096 && chunks > kWave) return {64, 2};
    return {row_lanes(chunks), 1};
}

int check_rows_args(const char* name, int tokens, int k, int rows, int cols, int type) {
    if (tokens < 0 || k < 1 || k > kMaxChoices || rows < 0 || cols < 1 || cols > kMaxCols)
        return set_error(MI_ERR_INVALID_ARG,
                         "%s: invalid shape tokens=%d k=%d rows=%d cols=%d (k is 1 to %d, cols 1 "
                         "to %d)",
                         name, tokens, k, rows, cols, kMaxChoices, kMaxCols);
    if (static_cast<long long>(tokens) * k > INT_MAX)
        return set_error(MI_ERR_INVALID_ARG, "%s: tokens * k = %lld slots exceed an int", name,
                         static_cast<long long>(tokens) * k);
    if (!row_type_ok(type))
        return set_error(MI_ERR_INVALID_ARG, "%s: unknown type %d", name, type);
    return MI_OK;
}

// Bytes of the token rows and of `times` the slots' rows.
double moved_bytes(int tokens, int k, int rows, size_t row_bytes, int times) {
    const double slots = std::min(static_cast<double>(tokens) * k, static_cast<double>(rows));
    return (tokens + times * slots) * static_cast<double>(row_bytes);
}

template <bool WEIGHTED>
int gather_sum(const char* name, const void* src, const int* position, const float* weights,
               void* out, int tokens, int k, int rows, int cols, int type, hipStream_t st) {
    const size_t row_bytes = static_cast<size_t>(cols) * row_type_size(type);
    if (row_bytes < 16)
        return launch_narrow<WEIGHTED ? Narrow::WeightedSum : Narrow::Sum>(
            name, src, nullptr, position, weights, out, nullptr, tokens, k, rows, cols, type, st);
    const int chunks = static_cast<int>((row_bytes + 15) / 16);
    const bool stream = stream_loads(moved_bytes(tokens, k, rows, row_bytes, 1));
    with_row_type(type, [&](auto t) {
        with_row_shape(gather_shape(tokens, chunks), tokens, chunks,
                       [&](auto lanes, auto u, dim3 grid) {
            constexpr int T = decltype(t)::value, LT = decltype(lanes)::value;
            constexpr int U = decltype(u)::value;
            with_flag(stream, [&](auto nt) {
                hipLaunchKernelGGL((gather_sum_kernel<T, U, LT, WEIGHTED, decltype(nt)::value>),
                                   grid, dim3(kThreads), 0, st, static_cast<const char*>(src),
                                   position, weights, static_cast<char*>(out), tokens, k, rows,
                                   chunks, row_bytes);
            });
        });
    });
    return check_launch(name);
}

// Waves a token in combine's gradient: one where a wave has the row in few
// steps, more where rows are long (bf16 [8192 tokens, 4 choices] of 2048 columns 63.4
// -> 54.4 us, of 4096 125 -> 110; 1600 columns 21.6 -> 22.3, 16384 tokens of 1024 28.8
// -> 40.7) or tokens few (8 tokens of 6152 fp32 32.2 us by one, 11.4 by four, 6.5 by
// 16; 67 of 896, 8 choices, 8.9 -> 4.8).  Past 8 choices 16 waves lack registers.
// In place, a moved-back last chunk that would fall to another wave than its
// neighbour takes one wave.
int combine_waves(int tokens, int k, int chunks, bool in_place, bool ragged) {
    if (in_place && ragged && (chunks - 1) % kWave == 0) return 1;
    if (tokens < 512 && chunks > 4 * kWave && k <= 8) return 16;
    return chunks >= 4 * kWave || (tokens < 512 && chunks > kWave) ? 4 : 1;
}

int check_gate_args(const char* name, int tokens, int experts, int k, int type) {
    if (tokens < 0 || experts < 1 || experts > kMaxExperts || k < 1 || k > kMaxChoices ||
        k > experts)
        return set_error(MI_ERR_INVALID_ARG,
                         "%s: invalid shape tokens=%d experts=%d k=%d (experts is 1 to %d, k 1 to "
                         "%d and at most experts)",
                         name, tokens, experts, k, kMaxExperts, kMaxChoices);
    if (static_cast<long long>(tokens) * k > INT_MAX)
        return set_error(MI_ERR_INVALID_ARG, "%s: tokens * k = %lld slots exceed an int", name,
                         static_cast<long long>(tokens) * k);
    if (!row_type_ok(type))
        return set_error(MI_ERR_INVALID_ARG, "%s: unknown type %d", name, type);
    return MI_OK;
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

int mi_moe_gate_forward(const void* logits, int* ids, float* weights, int tokens, int experts,
                        int k, int renormalise, int type, void* stream) {
    const char* name = "mi_moe_gate_forward";
    if (int rc = check_gate_args(name, tokens, experts, k, type)) return rc;
    if (tokens == 0) return MI_OK;
    if (!logits || !ids || !weights)
        return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    with_row_type(type, [&](auto t) {
        // 512 experts, 8 chosen: 32768 tokens 30.5 us by 64 lanes a row, 23.7 by 16, 8192
        // 9.8, 6.9, 3000 5.3, 5.2, but 1024 4.1, 5.0; 2 chosen, 32768 tokens 17.9, 20.0
        with_gate_shape<true>(experts, tokens >= 4096 && k > 2, [&](auto l, auto p) {
            constexpr int T = decltype(t)::value, L = decltype(l)::value, P = decltype(p)::value;
            auto launch = [&](auto d, auto renorm) {
                hipLaunchKernelGGL((gate_fwd_kernel<T, L, P, decltype(d)::value,
                                                    decltype(renorm)::value>),
                                   dim3(gate_grid(tokens, L)), dim3(kThreads), 0,
                                   to_stream(stream), logits, ids, weights, tokens, experts, k);
            };
            with_flag(renormalise != 0, [&](auto renorm) {
                if constexpr (P > 8) {
                    if (k <= 8) return launch(std::integral_constant<int, 8>(), renorm);
                }
                launch(std::integral_constant<int, std::min(P, kMaxChoices)>(), renorm);
            });
        });
    });
    return check_launch(name);
}

int mi_moe_gate_backward(const void* logits, const int* ids, const float* weights,
                         const float* dweights, void* dlogits, int tokens, int experts, int k,
                         int renormalise, int type, void* stream) {
    const char* name = "mi_moe_gate_backward";
    if (int rc = check_gate_args(name, tokens, experts, k, type)) return rc;
    if (tokens == 0) return MI_OK;
    if ((!logits && !renormalise) || !ids || !weights || !dweights || !dlogits)
        return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    with_row_type(type, [&](auto t) {
        with_gate_shape<false>(experts, false, [&](auto l, auto p) {
            constexpr int T = decltype(t)::value, L = decltype(l)::value, P = decltype(p)::value;
            if (renormalise)
                hipLaunchKernelGGL((gate_bwd_kernel<T, L, P, true>), dim3(gate_grid(tokens, L)),
                                   dim3(kThreads), 0, to_stream(stream), logits, ids, weights,
                                   dweights, dlogits, tokens, experts, k);
            else
                hipLaunchKernelGGL((gate_bwd_kernel<T, L, P, false>), dim3(gate_grid(tokens, L)),
                                   dim3(kThreads), 0, to_stream(stream), logits, ids, weights,
                                   dweights, dlogits, tokens, experts, k);
        });
    });
    return check_launch(name);
}

size_t mi_moe_sort_workspace(int slots, int experts) {
    if (slots <= 0 || experts <= 0) return 0;
    const SortPlan p = plan_sort(slots);
    return p.chunks > 1
               ? colsum_part_offset() + static_cast<size_t>(p.chunks) * experts * sizeof(int)
               : 0;
}

int mi_moe_sort(const int* ids, int* offsets, int* order, int* position, int slots, int experts,
                void* stream) {
    const char* name = "mi_moe_sort";
    if (slots < 0 || experts < 1 || experts > kMaxExperts)
        return set_error(MI_ERR_INVALID_ARG,
                         "%s: invalid shape slots=%d experts=%d (experts is 1 to %d)", name, slots,
                         experts, kMaxExperts);
    if (!offsets || (slots > 0 && (!ids || !position)))
        return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    hipStream_t st = to_stream(stream);
    const SortPlan p = plan_sort(slots);
    int* hist = nullptr;
    if (p.chunks > 1) {
        int err = MI_OK;
        char* ws =
            static_cast<char*>(workspace_get(mi_moe_sort_workspace(slots, experts), st, &err));
        if (!ws) return err;
        hist = reinterpret_cast<int*>(ws + colsum_part_offset());
        hipLaunchKernelGGL(sort_hist_kernel, dim3(p.chunks), dim3(kSortThreads),
                           experts * sizeof(int), st, ids, hist, slots, experts, p.trips);
        if (int rc = check_launch(name)) return rc;
    }
    int bits = 0;
    while ((1 << bits) < experts) ++bits;
    const size_t lds = (kSortWaves + (hist ? 2 : 0)) * experts * sizeof(int);
    auto place = [&](auto nr) {
        hipLaunchKernelGGL((sort_place_kernel<decltype(nr)::value>), dim3(p.chunks),
                           dim3(kSortThreads), lds, st, ids, hist, offsets, order, position, slots,
                           experts, p.trips, p.chunks, bits);
    };
    if (p.trips == 1)
        place(std::integral_constant<int, 1>());
    else if (p.trips == 2)
        place(std::integral_constant<int, 2>());
    else if (p.trips <= 4)
        place(std::integral_constant<int, 4>());
    else
        place(std::integral_constant<int, 0>());
    return check_launch(name);
}

int mi_moe_dispatch_forward(const void* x, const int* position, void* out, int tokens, int k,
                            int rows, int cols, int type, void* stream) {
    const char* name = "mi_moe_dispatch_forward";
    if (int rc = check_rows_args(name, tokens, k, rows, cols, type)) return rc;
    if (tokens == 0 || rows == 0) return MI_OK;
    if (!x || !position || !out) return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    hipStream_t st = to_stream(stream);
    const size_t row_bytes = static_cast<size_t>(cols) * row_type_size(type);
    if (row_bytes < 16)
        return launch_narrow<Narrow::Scatter>(name, x, nullptr, position, nullptr, out, nullptr,
                                              tokens, k, rows, cols, type, st);
    const int chunks = static_cast<int>((row_bytes + 15) / 16);
    with_row_shape(scatter_shape(tokens, chunks), tokens, chunks,
                   [&](auto lanes, auto u, dim3 grid) {
        const unsigned groups = std::min(grid.x, std::max(1u, 2u * kMaxGrid / grid.y));
        hipLaunchKernelGGL((scatter_rows_kernel<decltype(u)::value, decltype(lanes)::value>),
                           dim3(groups * grid.y), dim3(kThreads), 0, st,
                           static_cast<const char*>(x), position, static_cast<char*>(out), tokens,
                           k, rows, chunks, row_bytes);
    });
    return check_launch(name);
}

int mi_moe_dispatch_backward(const void* dout, const int* position, void* dx, int tokens, int k,
                             int rows, int cols, int type, void* stream) {
    const char* name = "mi_moe_dispatch_backward";
    if (int rc = check_rows_args(name, tokens, k, rows, cols, type)) return rc;
    if (tokens == 0) return MI_OK;
    if ((!dout && rows > 0) || !position || !dx)
        return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    return gather_sum<false>(name, dout, position, nullptr, dx, tokens, k, rows, cols, type,
                             to_stream(stream));
}

int mi_moe_combine_forward(const void* y, const int* position, const float* weights, void* out,
                           int tokens, int k, int rows, int cols, int type, void* stream) {
    const char* name = "mi_moe_combine_forward";
    if (int rc = check_rows_args(name, tokens, k, rows, cols, type)) return rc;
    if (tokens == 0) return MI_OK;
    if ((!y && rows > 0) || !position || !weights || !out)
        return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    return gather_sum<true>(name, y, position, weights, out, tokens, k, rows, cols, type,
                            to_stream(stream));
}

int mi_moe_combine_backward(const void* dout, const void* y, const int* position,
                            const float* weights, void* dy, float* dweights, int tokens, int k,
                            int rows, int cols, int type, void* stream) {
    const char* name = "mi_moe_combine_backward";
    if (int rc = check_rows_args(name, tokens, k, rows, cols, type)) return rc;
    if (tokens == 0) return MI_OK;
    if (!dout || (rows > 0 && (!y || !dy)) || !position || !weights || !dweights)
        return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    hipStream_t st = to_stream(stream);
    const size_t row_bytes = static_cast<size_t>(cols) * row_type_size(type);
    if (row_bytes < 16)
        return launch_narrow<Narrow::Backward>(name, dout, y, position, weights, dy, dweights,
                                               tokens, k, rows, cols, type, st);
    const int chunks = static_cast<int>((row_bytes + 15) / 16);
    with_row_type(type, [&](auto t) {
        constexpr int T = decltype(t)::value;
        auto launch = [&](auto kb) {
            constexpr int KB = decltype(kb)::value;
            auto with_waves = [&](auto g, auto lanes, auto nt) {
                constexpr int G = decltype(g)::value, LT = decltype(lanes)::value;
                const dim3 grid(token_grid(tokens, G > 1 ? 1 : kThreads / LT));
                hipLaunchKernelGGL((combine_bwd_kernel<T, KB, G, LT, decltype(nt)::value>), grid,
                                   dim3(G > kWaves ? G * kWave : kThreads), 0, st, tokens, k,
                                   rows, chunks, row_bytes, position, weights,
                                   static_cast<const char*>(dout), static_cast<const char*>(y),
                                   static_cast<char*>(dy), dweights);
            };
            using std::integral_constant;
            const int g = combine_waves(tokens, k, chunks, dy == y, row_bytes % 16 != 0);
            const bool stream = stream_loads(moved_bytes(tokens, k, rows, row_bytes, 2));
            if constexpr (KB <= 8)
                if (g == 16)
                    return with_waves(integral_constant<int, 16>(), integral_constant<int, 64>(),
                                      std::false_type());
            if (g == 4)
                with_flag(stream, [&](auto nt) {
                    with_waves(integral_constant<int, 4>(), integral_constant<int, 64>(), nt);
                });
            else if (row_lanes(chunks) == 16)
                with_waves(integral_constant<int, 1>(), integral_constant<int, 16>(),
                           std::false_type());
            else if (row_lanes(chunks) == 32)
                with_waves(integral_constant<int, 1>(), integral_constant<int, 32>(),
                           std::false_type());
            else
                with_flag(stream, [&](auto nt) {
                    with_waves(integral_constant<int, 1>(), integral_constant<int, 64>(), nt);
                });
        };
        if (k <= 1)
            launch(std::integral_constant<int, 1>());
        else if (k <= 2)
            launch(std::integral_constant<int, 2>());
        else if (k <= 4)
            launch(std::integral_constant<int, 4>());
        else if (k <= 8)
            launch(std::integral_constant<int, 8>());
        else
            launch(std::integral_constant<int, 16>());
    });
    return check_launch(name);
}

}  // extern "C"

// A model's gradients in many tensors, for gfx950: the global norm, and every
// tensor times the clip scale.  The reference has them in one flat fp32 buffer
// (buffer_norm_sq_acc, compute_clip_scale and scale_buffer,
// FINAL_CLEAN_CODE/src/kernels/activations.cu:349-392); these calls take them where
// they are, fp32, fp16 and bf16 mixed.
//
// A launch takes up to kBatch tensors, described in its arguments: no table in device
// memory has to be kept or copied, and a captured graph holds what it needs.  Where there are
// more, the norm's launches leave their descriptions in the workspace, and one launch scales all.
// A launch with such arguments costs 4.3 us of the host's time, of however many tensors, so that
// small lists take as long as their launches: tensors are described in few bytes.
// Tensors are cut into units, numbered through the whole list; a workgroup takes consecutive
// units, whichever tensors they are in.
//
// Bound by memory: 434 tensors of 1.55 billion bf16 elements into fp32 2131 us, the norm 495 (6.3
// TB/s), the scaling 1660 (9.3 GB, 5.6 TB/s; with 16 bytes read and 32 written a lane, whose stores
// are not side by side, 1750).  In place the norm alone is read where nothing is clipped.  Small
// lists are bound by their two launches (41 tensors of 3.7 MB 8.7 us).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "mi_common.hpp"
#include "mi_rowtype.hpp"

namespace mi {

namespace {

constexpr int kThreads = 256;
// Tensors of a launch, in at most 3.9 KB of arguments: in place, or with outs.
template <bool WIDE>
constexpr int kBatch = WIDE ? 192 : 320;
constexpr int kShift = 13;            // a unit has 2^kShift elements,
constexpr int kFewShift = 11;         // or 2^kFewShift where all tensors have less than
constexpr long long kFew = 1ll << 23; // so many together
constexpr int kNormBlocks = 2048;     // workgroups of a norm launch
// Elements up to which every workgroup of the scaling launch adds the norm's partial sums itself,
// at most so many of them, which saves a launch: 20 tensors of 24.7 MB in place 12.4 -> 9.2 us.
constexpr long long kFused = 1ll << 24;
constexpr int kFusedParts = 1024;
// Workgroups of the scaling launch, at most: short ones are faster (a billion fp32 elements in
// place 1423 us with 131072, 1537 with 8192), but in place they mostly only read the scale and end
// (434 tensors of 790 MB below the limit 151 us with 131072, 141 with 8192).
constexpr int kScaleBlocks = 131072;
constexpr int kInPlaceBlocks = 32768;
constexpr int kFinThreads = 1024;
constexpr long long kMaxUnits = 1ll << 30;

// A tensor's address, above it (13 bits) the elements of its last unit less one, and its type.
using Packed = unsigned long long;
constexpr int kAddressBits = 48;
constexpr int kTypeShift = 61;
static_assert(kAddressBits + kShift == kTypeShift, "the last unit's elements fit between");

Packed pack(const void* data, long long elements, int type, int shift) {
    const unsigned long long last = static_cast<unsigned long long>(elements - 1) & ((1ull << shift) - 1);
    return reinterpret_cast<Packed>(data) | last << kAddressBits |
           static_cast<Packed>(type) << kTypeShift;
}

struct Tensor {
    const void* data;
    void* out;
    long long elements;
    int type;
};

// The tensors of a launch, in its arguments.
template <bool WIDE>
struct Batch;
template <>
struct Batch<false> {
    Packed tensor[kBatch<false>];
    unsigned end[kBatch<false>];  // units up to the tensor's last; the largest number behind the last one
    unsigned first;               // units before the first tensor
    int count;
    int shift;
};
template <>
struct Batch<true> {
    Packed tensor[kBatch<true>];
    void* out[kBatch<true>];
    unsigned end[kBatch<true>];
    unsigned first;
    int count;
    int shift;
};

static_assert(sizeof(Batch<false>) <= 3936 && sizeof(Batch<true>) <= 3936,
              "a launch's arguments are 4 KB at most");

// All of a list's tensors, in device memory.  out: NULL in place.
struct Table {
    Packed* tensor;
    void** out;
    unsigned* end;
    int count;
    int shift;
};

// The first tensor that ends behind unit u: the number of ends up to u, which the lanes count.
// One round trip: the arguments may lie in host memory.
template <bool WIDE>
__device__ __forceinline__ int tensor_of(const Batch<WIDE>& b, unsigned u) {
    const int lane = threadIdx.x & (kWave - 1);
    constexpr int ENDS = kBatch<WIDE> / kWave;  // a lane
    static_assert(kBatch<WIDE> % kWave == 0, "every lane has as many");
    unsigned end[ENDS];
    int before = 0;
#pragma unroll
    for (int i = 0; i < ENDS; ++i) end[i] = b.end[lane + i * kWave];
#pragma unroll
    for (int i = 0; i < ENDS; ++i) before += __popcll(__ballot(end[i] <= u));
    return before;
}

// A 64th of the range at a time.
__device__ __forceinline__ int tensor_of(const Table& b, unsigned u) {
    const int lane = threadIdx.x & (kWave - 1);
    int from = 0, n = b.count;
    while (n > 0) {
        const int step = (n + kWave - 1) / kWave;
        const int last = (lane + 1) * step - 1;  // of the lane's part
        const bool before = last < n && b.end[from + last] <= u;
        from += __popcll(__ballot(before)) * step;
        n = step > 1 ? min(step, b.count - from) : 0;
    }
    return from;
}

template <bool WIDE>
__device__ __forceinline__ unsigned first_unit(const Batch<WIDE>& b, int i) {
    return i ? b.end[i - 1] : b.first;
}
__device__ __forceinline__ unsigned first_unit(const Table& b, int i) {
    return i ? b.end[i - 1] : 0u;
}

// Calls f(tensor, first element, end element) for the pieces of units [u, end).
template <bool WIDE, class List, class F>
__device__ __forceinline__ void for_pieces(const List& b, unsigned u, unsigned end, F f) {
    if (u >= end) return;
    const int shift = b.shift;
    for (int i = __builtin_amdgcn_readfirstlane(tensor_of(b, u)); u < end; ++i) {
        const unsigned from = first_unit(b, i), all = b.end[i], to = min(end, all);
        const Packed p = b.tensor[i];
        Tensor t;
        t.data = reinterpret_cast<const void*>(p & ((1ull << kAddressBits) - 1));
        if constexpr (WIDE)
            t.out = b.out[i];
        else
            t.out = const_cast<void*>(t.data);
        t.elements = (static_cast<long long>(all - from - 1u) << shift) +
                     static_cast<int>(p >> kAddressBits & ((1u << kShift) - 1u)) + 1;
        t.type = static_cast<int>(p >> kTypeShift);
        f(t, static_cast<long long>(u - from) << shift,
          min(t.elements, static_cast<long long>(to - from) << shift));
        u = to;
    }
}

// A workgroup's share of `units` units from `first` on.
struct Share {
    unsigned begin, end;
};

__device__ __forceinline__ Share share_of(unsigned first, unsigned units) {
    const unsigned long long n = units;
    return {first + static_cast<unsigned>(n * blockIdx.x / gridDim.x),
            first + static_cast<unsigned>(n * (blockIdx.x + 1ull) / gridDim.x)};
}

template <int T, bool NT>
__device__ __forceinline__ void add_squares(const void* data, long long first, long long end,
                                            float (&acc)[8]) {
    constexpr int V = row_vec<T>(), U = 4;
    const char* p = static_cast<const char*>(data);
    const long long whole = first + (end - first) / V * V;
    constexpr long long kStep = static_cast<long long>(kThreads) * V;
    long long at = first + static_cast<long long>(threadIdx.x) * V;
    auto add = [&](const u32x4& raw) {
        float v[V];
        row_unpack<T>(raw, v);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += v[e] * v[e];
    };
    for (; at + (U - 1) * kStep < whole; at += U * kStep) {
        u32x4 raw[U];
#pragma unroll
        for (int i = 0; i < U; ++i)
            raw[i] = load16b<NT>(p + (at + i * kStep) * sizeof(row_elem<T>));
#pragma unroll
        for (int i = 0; i < U; ++i) add(raw[i]);
    }
    for (; at < whole; at += kStep) add(load16b<NT>(p + at * sizeof(row_elem<T>)));
    if (whole + threadIdx.x < end) {
        const float v = row_get<T>(data, static_cast<size_t>(whole) + threadIdx.x);
        acc[0] += v * v;
    }
}

// table: where the descriptions go (tensor NULL: nowhere).
template <bool WIDE>
__global__ __launch_bounds__(kThreads) void tensors_sumsq_kernel(float* __restrict__ part,
                                                                 unsigned units, bool nt,
                                                                 const Table table,
                                                                 const Batch<WIDE> b) {
    __shared__ float red[kThreads / kWave];
    if (table.tensor && blockIdx.x == 0) {
        for (int i = threadIdx.x; i < b.count; i += kThreads) {
            table.tensor[i] = b.tensor[i];
            table.end[i] = b.end[i];
            if constexpr (WIDE) table.out[i] = b.out[i];
        }
    }
    const Share u = share_of(b.first, units);
    float acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
    for_pieces<false>(b, u.begin, u.end, [&](const Tensor& t, long long first, long long end) {
        auto add = [&](auto stream) {
            constexpr bool NT = decltype(stream)::value;
            if (t.type == MI_TYPE_F32)
                add_squares<MI_TYPE_F32, NT>(t.data, first, end, acc);
            else if (t.type == MI_TYPE_F16)
                add_squares<MI_TYPE_F16, NT>(t.data, first, end, acc);
            else
                add_squares<MI_TYPE_BF16, NT>(t.data, first, end, acc);
        };
        if (nt)
            add(std::true_type());
        else
            add(std::false_type());
    });
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s += acc[e];
    s = wave_sum(s);
    if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        float t = red[0];
#pragma unroll
        for (int w = 1; w < kThreads / kWave; ++w) t += red[w];
        part[blockIdx.x] = t;
    }
}

// The partial sums in 64 bits, in a fixed order; every thread gets the total.
template <int NT>
__device__ __forceinline__ double add_parts(const float* part, int parts, double* red) {
    constexpr int AT_ONCE = 4;
    double s = 0.0;
    for (int i0 = threadIdx.x; i0 < parts; i0 += AT_ONCE * NT) {
        float p[AT_ONCE];  // every load goes out, from a place that is there
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) p[i] = part[min(i0 + i * NT, parts - 1)];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
            s += i0 + i * NT < parts ? static_cast<double>(p[i]) : 0.0;
    }
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) s += __shfl_xor(s, m);
    if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = s;
    __syncthreads();
    s = red[0];
#pragma unroll
    for (int w = 1; w < NT / kWave; ++w) s += red[w];
    return s;
}

__device__ __forceinline__ float clip_scale(float norm_sq, float max_norm) {
    const float norm = sqrtf(norm_sq);
    return norm > max_norm ? max_norm / norm : 1.0f;
}

__global__ __launch_bounds__(kFinThreads) void tensors_finish_kernel(
    const float* __restrict__ part, int parts, float* __restrict__ result, bool accumulate,
    float* __restrict__ clip, float max_norm) {
    __shared__ double red[kFinThreads / kWave];
    const double s = add_parts<kFinThreads>(part, parts, red);
    if (threadIdx.x == 0) {
        const float total = static_cast<float>(accumulate ? *result + s : s);
        *result = total;
        if (clip) *clip = clip_scale(total, max_norm);
    }
}

// The elements of a load: 16 bytes, or as many as make 16 bytes of fp32, so that the lanes' stores
// are side by side too.
template <int T, bool WIDE>
constexpr int kScaleVec = WIDE ? 4 : row_vec<T>();

template <int T, int V, bool NT>
__device__ __forceinline__ void load_values(const char* p, float (&v)[V]) {
    if constexpr (V == row_vec<T>()) {
        row_unpack<T>(load16b<NT>(p), v);
    } else {
        typedef u32x2 u32x2_at2 __attribute__((aligned(2)));
        u32x2 half;
        if constexpr (NT)
            half = __builtin_nontemporal_load(reinterpret_cast<const u32x2_at2*>(p));
        else
            half = *reinterpret_cast<const u32x2_at2*>(p);
        float w[2 * V];
        row_unpack<T>(u32x4{half.x, half.y, 0u, 0u}, w);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = w[e];
    }
}

// A product is rounded to fp32 and then to the type, wherever it stands (rounded: a multiplication
// may otherwise be joined with its conversion to fp16, or not).
template <int T, bool WIDE, bool NT>
__device__ __forceinline__ void scale_piece(const Tensor& t, long long first, long long end,
                                            float c) {
    constexpr int V = kScaleVec<T, WIDE>, O = WIDE ? MI_TYPE_F32 : T;
    constexpr int U = 64 / (V * static_cast<int>(sizeof(row_elem<T>)));
    constexpr long long kStep = static_cast<long long>(kThreads) * V;
    const char* p = static_cast<const char*>(t.data);
    char* o = static_cast<char*>(t.out);
    const long long whole = first + (end - first) / V * V;
    long long at = first + static_cast<long long>(threadIdx.x) * V;
    auto put = [&](long long i, float (&v)[V]) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = rounded(v[e] * c);
        store16b(o + i * sizeof(row_elem<O>), row_pack<O>(v));
    };
    for (; at + (U - 1) * kStep < whole; at += U * kStep) {
        float v[U][V];
#pragma unroll
        for (int i = 0; i < U; ++i)
            load_values<T, V, NT>(p + (at + i * kStep) * sizeof(row_elem<T>), v[i]);
#pragma unroll
        for (int i = 0; i < U; ++i) put(at + i * kStep, v[i]);
    }
    for (; at < whole; at += kStep) {
        float v[V];
        load_values<T, V, NT>(p + at * sizeof(row_elem<T>), v);
        put(at, v);
    }
    if (whole + threadIdx.x < end) {
        const size_t i = static_cast<size_t>(whole) + threadIdx.x;
        row_put<O>(t.out, i, rounded(row_get<T>(t.data, i) * c));
    }
}

// The norm's partial sums, which every workgroup adds (the same way) instead of a launch of its
// own: part NULL where the scale is there.
struct Parts {
    const float* part;
    int parts;
    float max_norm;
    float* norm_sq;
    float* clip;
};

template <bool WIDE, bool PARTS, class List>
__global__ __launch_bounds__(kThreads) void tensors_scale_kernel(const float* __restrict__ scale,
                                                                 unsigned first, unsigned units,
                                                                 bool nt, const Parts parts,
                                                                 const List b) {
    float c;
    if constexpr (PARTS) {
        __shared__ double red[kThreads / kWave];
        const float total =
            static_cast<float>(add_parts<kThreads>(parts.part, parts.parts, red));
        c = clip_scale(total, parts.max_norm);
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            *parts.norm_sq = total;
            *parts.clip = c;
        }
    } else {
        c = *scale;
    }
    if (!WIDE && c == 1.0f) return;
    const Share u = share_of(first, units);
    for_pieces<WIDE>(b, u.begin, u.end, [&](const Tensor& t, long long first, long long end) {
        auto put = [&](auto stream) {
            constexpr bool NT = decltype(stream)::value;
            if (t.type == MI_TYPE_F32)
                scale_piece<MI_TYPE_F32, WIDE, NT>(t, first, end, c);
            else if (t.type == MI_TYPE_F16)
                scale_piece<MI_TYPE_F16, WIDE, NT>(t, first, end, c);
            else
                scale_piece<MI_TYPE_BF16, WIDE, NT>(t, first, end, c);
        };
        if (nt)
            put(std::true_type());
        else
            put(std::false_type());
    });
}

struct List {
    const void* const* tensors;
    void* const* outs;
    const long long* sizes;
    const int* types;
    int count;
    int type(int i) const { return types ? types[i] : MI_TYPE_F32; }
};

long long units_of(long long elements, int shift) {
    return (elements + (1ll << shift) - 1) >> shift;
}

struct Totals {
    long long elements = 0, units = 0;
    double bytes = 0.0;
    int shift = kShift, tensors = 0, batches = 0;
};

int batches_of(int tensors, int most) {
    return static_cast<int>((static_cast<long long>(tensors) + most - 1) / most);
}

int check_list(const char* name, const List& l, Totals* total) {
    if (l.count < 0) return set_error(MI_ERR_INVALID_ARG, "%s: count=%d", name, l.count);
    if (l.count > 0 && (!l.tensors || !l.sizes))
        return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    for (int i = 0; i < l.count; ++i) {
        if (l.sizes[i] < 0 || l.sizes[i] > kMaxUnits << kShift)
            return set_error(MI_ERR_INVALID_ARG, "%s: tensor %d has size %lld", name, i,
                             l.sizes[i]);
        if (!row_type_ok(l.type(i)))
            return set_error(MI_ERR_INVALID_ARG, "%s: tensor %d has unknown type %d", name, i,
                             l.type(i));
        if (l.sizes[i] == 0) continue;
        if (!l.tensors[i] || (l.outs && !l.outs[i]))
            return set_error(MI_ERR_INVALID_ARG, "%s: tensor %d: NULL pointer", name, i);
        if (reinterpret_cast<uintptr_t>(l.tensors[i]) >> kAddressBits)
            return set_error(MI_ERR_INVALID_ARG, "%s: tensor %d is at no address", name, i);
        ++total->tensors;
        total->elements += l.sizes[i];
        total->units += units_of(l.sizes[i], kShift);
        total->bytes += static_cast<double>(l.sizes[i]) * row_type_size(l.type(i));
        if (total->units > kMaxUnits)
            return set_error(MI_ERR_INVALID_ARG, "%s: more than %lld elements", name,
                             kMaxUnits << kShift);
    }
    total->batches = batches_of(total->tensors, l.outs ? kBatch<true> : kBatch<false>);
    if (total->elements < kFew) {
        total->shift = kFewShift;
        total->units = 0;
        for (int i = 0; i < l.count; ++i) total->units += units_of(l.sizes[i], kFewShift);
    }
    return MI_OK;
}

// Calls f(batch, its units, tensors before it) for every kBatch tensors that have elements.
template <bool WIDE, class F>
int for_batches(const List& l, int shift, F f) {
    constexpr int MOST = kBatch<WIDE>;
    Batch<WIDE> b;
    b.count = 0;
    b.first = 0;
    b.shift = shift;
    unsigned units = 0;  // up to here
    int before = 0;
    for (int i = 0; i < l.count; ++i) {
        if (l.sizes[i] > 0) {
            const int n = b.count++;
            units += static_cast<unsigned>(units_of(l.sizes[i], shift));
            b.tensor[n] = pack(l.tensors[i], l.sizes[i], l.type(i), shift);
            if constexpr (WIDE) b.out[n] = l.outs[i];
            b.end[n] = units;
        }
        if (b.count > 0 && (b.count == MOST || i == l.count - 1)) {
            for (int n = b.count; n < MOST; ++n) b.end[n] = UINT_MAX;
            if (int rc = f(b, units - b.first, before)) return rc;
            before += b.count;
            b.count = 0;
            b.first = units;
        }
    }
    return MI_OK;
}

// What the library workspace holds: the norm's partial sums, the list's descriptions.
struct Space {
    float* part;
    Table table;
};

size_t parts_bytes(int batches) {
    return round_up(static_cast<size_t>(kNormBlocks) * batches * sizeof(float), 256);
}

// Without tensors the norm is written all the same, through one batch's place.
template <bool WIDE>
size_t space_bytes(int batches) {
    batches = std::max(1, batches);
    const size_t tensors = static_cast<size_t>(kBatch<WIDE>) * batches;
    const size_t each = sizeof(Packed) + (WIDE ? sizeof(void*) : 0) + sizeof(unsigned);
    return colsum_part_offset() + parts_bytes(batches) + (batches > 1 ? tensors * each : 0);
}

// The partial sums of all squares, and where there are several batches the list's descriptions.
template <bool WIDE>
int norm_parts(const char* name, const List& l, const Totals& total, hipStream_t st, Space* space,
               int* parts) {
    int err = MI_OK;
    char* ws = static_cast<char*>(workspace_get(space_bytes<WIDE>(total.batches), st, &err));
    if (!ws) return err;
    space->part = reinterpret_cast<float*>(ws + colsum_part_offset());
    space->table = Table{};
    if (total.batches > 1) {
        const size_t most = static_cast<size_t>(kBatch<WIDE>) * total.batches;
        Packed* tensor =
            reinterpret_cast<Packed*>(ws + colsum_part_offset() + parts_bytes(total.batches));
        void** out = reinterpret_cast<void**>(tensor + most);
        space->table = Table{tensor, WIDE ? out : nullptr,
                             reinterpret_cast<unsigned*>(WIDE ? out + most : out), total.tensors,
                             total.shift};
    }
    *parts = 0;
    const unsigned most =
        total.elements < kFused ? std::max(1, kFusedParts / std::max(1, total.batches)) : kNormBlocks;
    // Streamed where nothing of it is read again soon: where a launch reads all of it next, only
    // past 1 GB (bf16 of 215 MB, into fp32, 115 -> 102 us, of 495 MB 349 -> 318, fp32 of 990 MB 475
    // -> 470, but bf16 of 3.1 GB 2131 -> 2160; the norm alone of 822 MB fp32 153, 171 kept).
    const bool nt = l.outs ? total.bytes > 1073741824.0 : stream_loads(total.bytes);
    return for_batches<WIDE>(l, total.shift, [&](const Batch<WIDE>& b, unsigned units, int before) {
        const int blocks = static_cast<int>(std::min<unsigned>(units, most));
        Table table = space->table;
        if (table.tensor) {
            table.tensor += before;
            table.end += before;
            if (WIDE) table.out += before;
        }
        hipLaunchKernelGGL(tensors_sumsq_kernel<WIDE>, dim3(blocks), dim3(kThreads), 0, st,
                           space->part + *parts, units, nt, table, b);
        *parts += blocks;
        return check_launch(name);
    });
}

int finish_norm(const char* name, const float* part, int parts, float* result, bool accumulate,
                float* clip, float max_norm, hipStream_t st) {
    hipLaunchKernelGGL(tensors_finish_kernel, dim3(1), dim3(kFinThreads), 0, st, part, parts,
                       result, accumulate, clip, max_norm);
    return check_launch(name);
}

template <bool WIDE, class Source>
int launch_scale(const char* name, const Totals& total, unsigned first, unsigned units,
                 const float* scale, const Parts* parts, const Source& source, hipStream_t st) {
    const dim3 grid(std::min<unsigned>(units, WIDE ? kScaleBlocks : kInPlaceBlocks));
    const bool nt = stream_loads(total.bytes);
    with_flag(parts != nullptr, [&](auto add) {
        hipLaunchKernelGGL((tensors_scale_kernel<WIDE, decltype(add)::value, Source>), grid,
                           dim3(kThreads), 0, st, scale, first, units, nt,
                           parts ? *parts : Parts{}, source);
    });
    return check_launch(name);
}

template <bool WIDE>
int scale_batches(const char* name, const List& l, const Totals& total, const float* scale,
                  const Parts* parts, hipStream_t st) {
    return for_batches<WIDE>(l, total.shift, [&](const Batch<WIDE>& b, unsigned units, int) {
        return launch_scale<WIDE>(name, total, b.first, units, scale, parts, b, st);
    });
}

template <bool WIDE>
int clip(const char* name, const List& l, const Totals& total, float max_norm, float* d_norm_sq,
         float* d_clip_scale, hipStream_t st) {
    Space space;
    int parts = 0;
    if (int rc = norm_parts<WIDE>(name, l, total, st, &space, &parts)) return rc;
    const bool fused = total.elements > 0 && total.elements < kFused;
    const Parts p{space.part, parts, max_norm, d_norm_sq, d_clip_scale};
    if (!fused)
        if (int rc =
                finish_norm(name, space.part, parts, d_norm_sq, false, d_clip_scale, max_norm, st))
            return rc;
    const float* scale = fused ? nullptr : d_clip_scale;
    if (total.batches <= 1)
        return scale_batches<WIDE>(name, l, total, scale, fused ? &p : nullptr, st);
    return launch_scale<WIDE>(name, total, 0u, static_cast<unsigned>(total.units), scale,
                              fused ? &p : nullptr, space.table, st);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

size_t mi_tensors_workspace(int count) {
    if (count < 0) return 0;
    // with outs: fewer tensors a launch, in as many bytes, than in place
    return space_bytes<true>(batches_of(count, kBatch<true>));
}

int mi_tensors_norm_sq_acc(const void* const* tensors, const long long* sizes, const int* types,
                           int count, float* d_result, void* stream) {
    const char* name = "mi_tensors_norm_sq_acc";
    const List l{tensors, nullptr, sizes, types, count};
    Totals total;
    if (int rc = check_list(name, l, &total)) return rc;
    if (!d_result) return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    if (total.units == 0) return MI_OK;
    hipStream_t st = to_stream(stream);
    Space space;
    int parts = 0;
    if (int rc = norm_parts<false>(name, l, total, st, &space, &parts)) return rc;
    return finish_norm(name, space.part, parts, d_result, true, nullptr, 0.0f, st);
}

int mi_tensors_scale(const void* const* tensors, void* const* outs, const long long* sizes,
                     const int* types, int count, const float* d_scale, void* stream) {
    const char* name = "mi_tensors_scale";
    const List l{tensors, outs, sizes, types, count};
    Totals total;
    if (int rc = check_list(name, l, &total)) return rc;
    if (!d_scale) return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    hipStream_t st = to_stream(stream);
    return outs ? scale_batches<true>(name, l, total, d_scale, nullptr, st)
                : scale_batches<false>(name, l, total, d_scale, nullptr, st);
}

int mi_tensors_clip(const void* const* tensors, void* const* outs, const long long* sizes,
                    const int* types, int count, float max_norm, float* d_norm_sq,
                    float* d_clip_scale, void* stream) {
    const char* name = "mi_tensors_clip";
    const List l{tensors, outs, sizes, types, count};
    Totals total;
    if (int rc = check_list(name, l, &total)) return rc;
    if (!d_norm_sq || !d_clip_scale) return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    if (!(max_norm >= 0.0f))
        return set_error(MI_ERR_INVALID_ARG, "%s: max_norm=%g", name,
                         static_cast<double>(max_norm));
    hipStream_t st = to_stream(stream);
    return outs ? clip<true>(name, l, total, max_norm, d_norm_sq, d_clip_scale, st)
                : clip<false>(name, l, total, max_norm, d_norm_sq, d_clip_scale, st);
}

}  // extern "C"

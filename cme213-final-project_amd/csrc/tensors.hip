// A model's gradients in many tensors, for gfx950: the global norm, and every
// tensor times the clip scale.  The reference has them in one flat fp32 buffer
// (buffer_norm_sq_acc, compute_clip_scale and scale_buffer,
// FINAL_CLEAN_CODE/src/kernels/activations.cu:349-392); these calls take them where
// they are, fp32, fp16 and bf16 mixed.
//
// A launch takes up to kBatch tensors, described in its arguments: no table in device
// memory has to be kept or copied, and a captured graph holds what it needs.  Where there are
// more, the norm's launches leave their descriptions in the workspace, and one launch scales all.
// Tensors are cut into units, numbered through the whole list; a workgroup takes consecutive
// units, whichever tensors they are in.
//
// Bound by memory: 434 tensors of 1.55 billion bf16 elements into fp32 2131 us, the norm 495 (6.3
// TB/s), the scaling 1630 (9.3 GB, 5.7 TB/s; with 16 bytes read and 32 written a lane, whose stores
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
constexpr int kBatch = 140;           // tensors of a launch: 3.9 KB of arguments
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

struct Tensor {
    const void* data;
    void* out;
    unsigned long long elements;  // and the type in the topmost byte
    __host__ __device__ long long size() const {
        return static_cast<long long>(elements & ((1ull << 56) - 1));
    }
    __host__ __device__ int type() const { return static_cast<int>(elements >> 56); }
};

// The tensors of a launch, in its arguments.
struct Batch {
    Tensor tensor[kBatch];
    unsigned end[kBatch];  // units up to the tensor's last; the largest number behind the last one
    unsigned first;        // units before the first tensor
    int count;
    int shift;
};

static_assert(sizeof(Batch) <= 3936, "a launch's arguments are 4 KB at most");

// All of a list's tensors, in device memory.
struct Table {
    const Tensor* tensor;
    const unsigned* end;
    int count;
    int shift;
};

// The first tensor that ends behind unit u: the number of ends up to u, which the lanes count.
// One round trip: the arguments may lie in host memory.
__device__ __forceinline__ int tensor_of(const Batch& b, unsigned u) {
    const int lane = threadIdx.x & (kWave - 1);
    constexpr int ENDS = (kBatch + kWave - 1) / kWave;  // a lane
    unsigned end[ENDS];
    int before = 0;
#pragma unroll
    for (int i = 0; i < ENDS; ++i) end[i] = b.end[min(lane + i * kWave, kBatch - 1)];
#pragma unroll
    for (int i = 0; i < ENDS; ++i)
        before += __popcll(__ballot(lane + i * kWave < kBatch && end[i] <= u));
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

__device__ __forceinline__ unsigned first_unit(const Batch& b, int i) {
    return i ? b.end[i - 1] : b.first;
}
__device__ __forceinline__ unsigned first_unit(const Table& b, int i) {
    return i ? b.end[i - 1] : 0u;
}

// Calls f(tensor, first element, end element) for the pieces of units [u, end).
template <class List, class F>
__device__ __forceinline__ void for_pieces(const List& b, unsigned u, unsigned end, F f) {
    if (u >= end) return;
    const int shift = b.shift;
    for (int i = __builtin_amdgcn_readfirstlane(tensor_of(b, u)); u < end; ++i) {
        const unsigned from = first_unit(b, i), to = min(end, b.end[i]);
        const Tensor t = b.tensor[i];
        f(t, static_cast<long long>(u - from) << shift,
          min(t.size(), static_cast<long long>(to - from) << shift));
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

// tensor, end: where the descriptions go (NULL: nowhere).
__global__ __launch_bounds__(kThreads) void tensors_sumsq_kernel(float* __restrict__ part,
                                                                 unsigned units, bool nt,
                                                                 Tensor* __restrict__ tensor,
                                                                 unsigned* __restrict__ end,
                                                                 const Batch b) {
    __shared__ float red[kThreads / kWave];
    if (tensor && blockIdx.x == 0 && static_cast<int>(threadIdx.x) < b.count) {
        tensor[threadIdx.x] = b.tensor[threadIdx.x];
        end[threadIdx.x] = b.end[threadIdx.x];
    }
    const Share u = share_of(b.first, units);
    float acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
    for_pieces(b, u.begin, u.end, [&](const Tensor& t, long long first, long long end) {
        auto add = [&](auto stream) {
            constexpr bool NT = decltype(stream)::value;
            if (t.type() == MI_TYPE_F32)
                add_squares<MI_TYPE_F32, NT>(t.data, first, end, acc);
            else if (t.type() == MI_TYPE_F16)
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
    for_pieces(b, u.begin, u.end, [&](const Tensor& t, long long first, long long end) {
        auto put = [&](auto stream) {
            constexpr bool NT = decltype(stream)::value;
            if (t.type() == MI_TYPE_F32)
                scale_piece<MI_TYPE_F32, WIDE, NT>(t, first, end, c);
            else if (t.type() == MI_TYPE_F16)
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
        ++total->tensors;
        total->elements += l.sizes[i];
        total->units += units_of(l.sizes[i], kShift);
        total->bytes += static_cast<double>(l.sizes[i]) * row_type_size(l.type(i));
        if (total->units > kMaxUnits)
            return set_error(MI_ERR_INVALID_ARG, "%s: more than %lld elements", name,
                             kMaxUnits << kShift);
    }
    total->batches = (total->tensors + kBatch - 1) / kBatch;
    if (total->elements < kFew) {
        total->shift = kFewShift;
        total->units = 0;
        for (int i = 0; i < l.count; ++i) total->units += units_of(l.sizes[i], kFewShift);
    }
    return MI_OK;
}

// Calls f(batch, its units, tensors before it) for every kBatch tensors that have elements.
template <class F>
int for_batches(const List& l, int shift, F f) {
    Batch b;
    b.count = 0;
    b.first = 0;
    b.shift = shift;
    unsigned units = 0;  // up to here
    int before = 0;
    for (int i = 0; i < l.count; ++i) {
        if (l.sizes[i] > 0) {
            const int n = b.count++;
            units += static_cast<unsigned>(units_of(l.sizes[i], shift));
            b.tensor[n] = {l.tensors[i], l.outs ? l.outs[i] : const_cast<void*>(l.tensors[i]),
                           static_cast<unsigned long long>(l.sizes[i]) |
                               static_cast<unsigned long long>(l.type(i)) << 56};
            b.end[n] = units;
        }
        if (b.count > 0 && (b.count == kBatch || i == l.count - 1)) {
            for (int n = b.count; n < kBatch; ++n) b.end[n] = UINT_MAX;
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
    Tensor* tensor;
    unsigned* end;
};

size_t parts_bytes(int batches) {
    return round_up(static_cast<size_t>(kNormBlocks) * batches * sizeof(float), 256);
}

size_t space_bytes(int batches) {
    const size_t tensors = static_cast<size_t>(kBatch) * batches;
    return colsum_part_offset() + parts_bytes(batches) +
           (batches > 1 ? tensors * (sizeof(Tensor) + sizeof(unsigned)) : 0);
}

// The partial sums of all squares, and where there are several batches the list's descriptions.
int norm_parts(const char* name, const List& l, const Totals& total, hipStream_t st, Space* space,
               int* parts) {
    int err = MI_OK;
    char* ws = static_cast<char*>(workspace_get(space_bytes(std::max(1, total.batches)), st, &err));
    if (!ws) return err;
    const bool table = total.batches > 1;
    space->part = reinterpret_cast<float*>(ws + colsum_part_offset());
    space->tensor = reinterpret_cast<Tensor*>(ws + colsum_part_offset() + parts_bytes(total.batches));
    space->end = reinterpret_cast<unsigned*>(space->tensor + kBatch * total.batches);
    *parts = 0;
    const unsigned most =
        total.elements < kFused ? std::max(1, kFusedParts / std::max(1, total.batches)) : kNormBlocks;
    // Streamed where nothing of it is read again soon: where a launch reads all of it next, only
    // past 1 GB (bf16 of 215 MB, into fp32, 115 -> 102 us, of 495 MB 349 -> 318, fp32 of 990 MB 475
    // -> 470, but bf16 of 3.1 GB 2131 -> 2160; the norm alone of 822 MB fp32 153, 171 kept).
    const bool nt = l.outs ? total.bytes > 1073741824.0 : stream_loads(total.bytes);
    return for_batches(l, total.shift, [&](const Batch& b, unsigned units, int before) {
        const int blocks = static_cast<int>(std::min<unsigned>(units, most));
        hipLaunchKernelGGL(tensors_sumsq_kernel, dim3(blocks), dim3(kThreads), 0, st,
                           space->part + *parts, units, nt,
                           table ? space->tensor + before : nullptr,
                           table ? space->end + before : nullptr, b);
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

template <class Source>
int launch_scale(const char* name, const List& l, const Totals& total, unsigned first,
                 unsigned units, const float* scale, const Parts* parts, const Source& source,
                 hipStream_t st) {
    const unsigned most = l.outs ? kScaleBlocks : kInPlaceBlocks;
    with_flag(l.outs != nullptr, [&](auto wide) {
        constexpr bool WIDE = decltype(wide)::value;
        const dim3 grid(std::min(units, most));
        const bool nt = stream_loads(total.bytes);
        with_flag(parts != nullptr, [&](auto add) {
            hipLaunchKernelGGL((tensors_scale_kernel<WIDE, decltype(add)::value, Source>), grid,
                               dim3(kThreads), 0, st, scale, first, units, nt,
                               parts ? *parts : Parts{}, source);
        });
    });
    return check_launch(name);
}

int scale_batches(const char* name, const List& l, const Totals& total, const float* scale,
                  const Parts* parts, hipStream_t st) {
    return for_batches(l, total.shift, [&](const Batch& b, unsigned units, int) {
        return launch_scale(name, l, total, b.first, units, scale, parts, b, st);
    });
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

size_t mi_tensors_workspace(int count) {
    if (count < 0) return 0;
    return space_bytes(static_cast<int>((static_cast<long long>(count) + kBatch - 1) / kBatch));
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
    if (int rc = norm_parts(name, l, total, st, &space, &parts)) return rc;
    return finish_norm(name, space.part, parts, d_result, true, nullptr, 0.0f, st);
}

int mi_tensors_scale(const void* const* tensors, void* const* outs, const long long* sizes,
                     const int* types, int count, const float* d_scale, void* stream) {
    const char* name = "mi_tensors_scale";
    const List l{tensors, outs, sizes, types, count};
    Totals total;
    if (int rc = check_list(name, l, &total)) return rc;
    if (!d_scale) return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    return scale_batches(name, l, total, d_scale, nullptr, to_stream(stream));
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
    Space space;
    int parts = 0;
    if (int rc = norm_parts(name, l, total, st, &space, &parts)) return rc;
    const bool fused = total.elements > 0 && total.elements < kFused;
    const Parts p{space.part, parts, max_norm, d_norm_sq, d_clip_scale};
    if (!fused)
        if (int rc =
                finish_norm(name, space.part, parts, d_norm_sq, false, d_clip_scale, max_norm, st))
            return rc;
    const float* scale = fused ? nullptr : d_clip_scale;
    if (total.batches <= 1) return scale_batches(name, l, total, scale, fused ? &p : nullptr, st);
    const Table all{space.tensor, space.end, total.tensors, total.shift};
    return launch_scale(name, l, total, 0u, static_cast<unsigned>(total.units), scale,
                        fused ? &p : nullptr, all, st);
}

}  // extern "C"

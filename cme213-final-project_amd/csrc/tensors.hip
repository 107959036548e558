// A model's gradients in many tensors, for gfx950: the global norm, and every
// tensor times the clip scale.  The reference has them in one flat fp32 buffer
// (buffer_norm_sq_acc, compute_clip_scale and scale_buffer,
// FINAL_CLEAN_CODE/src/kernels/activations.cu:349-392); these calls take them where
// they are, fp32, fp16 and bf16 mixed.
//
// A launch takes up to kBatch tensors, described in its arguments: no table in device
// memory has to be kept or copied, and a captured graph holds what it needs.  Tensors are
// cut into units; a workgroup takes consecutive units, whichever tensors they are in.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "mi_common.hpp"
#include "mi_rowtype.hpp"

namespace mi {

namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 112;           // tensors of a launch: 3.3 KB of arguments
constexpr long long kUnit = 8192;     // elements
constexpr int kNormBlocks = 2048;     // workgroups of the norm's launches, about
constexpr int kScaleBlocks = 131072;
constexpr int kFinThreads = 1024;
constexpr long long kMaxUnits = 1ll << 30;

struct Batch {
    const void* data[kBatch];
    void* out[kBatch];
    long long size[kBatch];
    unsigned end[kBatch];  // units up to the tensor's last
    unsigned char type[kBatch];
    int count;
};

// The first tensor that ends behind unit u.
__device__ __forceinline__ int tensor_of(const Batch& b, unsigned u) {
    int lo = 0, hi = b.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (b.end[mid] > u)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo;
}

// Calls f(tensor, first element, end element) for the pieces of units [u, end).
template <class F>
__device__ __forceinline__ void for_pieces(const Batch& b, unsigned u, unsigned end, F f) {
    for (int i = tensor_of(b, u); u < end; ++i) {
        const unsigned from = i ? b.end[i - 1] : 0u, to = min(end, b.end[i]);
        if (u >= to) continue;
        f(i, static_cast<long long>(u - from) * kUnit,
          min(b.size[i], static_cast<long long>(to - from) * kUnit));
        u = to;
    }
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

__global__ __launch_bounds__(kThreads) void tensors_sumsq_kernel(const Batch b,
                                                                 float* __restrict__ part,
                                                                 unsigned units, bool nt) {
    __shared__ float red[kThreads / kWave];
    const unsigned u0 = static_cast<unsigned>(static_cast<unsigned long long>(units) * blockIdx.x /
                                              gridDim.x);
    const unsigned u1 = static_cast<unsigned>(static_cast<unsigned long long>(units) *
                                              (blockIdx.x + 1ull) / gridDim.x);
    float acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
    for_pieces(b, u0, u1, [&](int i, long long first, long long end) {
        auto add = [&](auto stream) {
            constexpr bool NT = decltype(stream)::value;
            if (b.type[i] == MI_TYPE_F32)
                add_squares<MI_TYPE_F32, NT>(b.data[i], first, end, acc);
            else if (b.type[i] == MI_TYPE_F16)
                add_squares<MI_TYPE_F16, NT>(b.data[i], first, end, acc);
            else
                add_squares<MI_TYPE_BF16, NT>(b.data[i], first, end, acc);
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

// The partial sums in 64 bits, in a fixed order.
__global__ __launch_bounds__(kFinThreads) void tensors_finish_kernel(
    const float* __restrict__ part, int parts, float* __restrict__ result, bool accumulate,
    float* __restrict__ clip, float max_norm) {
    __shared__ double red[kFinThreads];
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += kFinThreads) s += static_cast<double>(part[i]);
    red[threadIdx.x] = s;
    __syncthreads();
#pragma unroll
    for (int h = kFinThreads / 2; h >= 1; h /= 2) {
        if (static_cast<int>(threadIdx.x) < h) red[threadIdx.x] += red[threadIdx.x + h];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const float total = static_cast<float>(accumulate ? *result + red[0] : red[0]);
        *result = total;
        if (clip) {
            const float norm = sqrtf(total);
            *clip = norm > max_norm ? max_norm / norm : 1.0f;
        }
    }
}

// A product is rounded to fp32 and then to the type, wherever it stands (rounded: a multiplication
// may otherwise be joined with its conversion to fp16, or not).
template <int T, bool WIDE, bool NT>
__device__ __forceinline__ void scale_piece(const void* data, void* out, long long first,
                                            long long end, float c) {
    constexpr int V = row_vec<T>(), U = 4;
    constexpr long long kStep = static_cast<long long>(kThreads) * V;
    const char* p = static_cast<const char*>(data);
    const long long whole = first + (end - first) / V * V;
    long long at = first + static_cast<long long>(threadIdx.x) * V;
    auto put = [&](long long i, const u32x4& raw) {
        float v[V];
        row_unpack<T>(raw, v);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = rounded(v[e] * c);
        if constexpr (WIDE) {
#pragma unroll
            for (int e = 0; e < V; e += 4)
                store16b(static_cast<float*>(out) + i + e,
                         u32x4{__float_as_uint(v[e]), __float_as_uint(v[e + 1]),
                               __float_as_uint(v[e + 2]), __float_as_uint(v[e + 3])});
        } else {
            store16b(static_cast<char*>(out) + i * sizeof(row_elem<T>), row_pack<T>(v));
        }
    };
    for (; at + (U - 1) * kStep < whole; at += U * kStep) {
        u32x4 raw[U];
#pragma unroll
        for (int i = 0; i < U; ++i)
            raw[i] = load16b<NT>(p + (at + i * kStep) * sizeof(row_elem<T>));
#pragma unroll
        for (int i = 0; i < U; ++i) put(at + i * kStep, raw[i]);
    }
    for (; at < whole; at += kStep) put(at, load16b<NT>(p + at * sizeof(row_elem<T>)));
    if (whole + threadIdx.x < end) {
        const size_t i = static_cast<size_t>(whole) + threadIdx.x;
        row_put<WIDE ? MI_TYPE_F32 : T>(out, i, rounded(row_get<T>(data, i) * c));
    }
}

template <bool WIDE>
__global__ __launch_bounds__(kThreads) void tensors_scale_kernel(const Batch b,
                                                                 const float* __restrict__ scale,
                                                                 unsigned units, bool nt) {
    const float c = *scale;
    if (!WIDE && c == 1.0f) return;
    const unsigned u0 = static_cast<unsigned>(static_cast<unsigned long long>(units) * blockIdx.x /
                                              gridDim.x);
    const unsigned u1 = static_cast<unsigned>(static_cast<unsigned long long>(units) *
                                              (blockIdx.x + 1ull) / gridDim.x);
    for_pieces(b, u0, u1, [&](int i, long long first, long long end) {
        auto put = [&](auto stream) {
            constexpr bool NT = decltype(stream)::value;
            if (b.type[i] == MI_TYPE_F32)
                scale_piece<MI_TYPE_F32, WIDE, NT>(b.data[i], b.out[i], first, end, c);
            else if (b.type[i] == MI_TYPE_F16)
                scale_piece<MI_TYPE_F16, WIDE, NT>(b.data[i], b.out[i], first, end, c);
            else
                scale_piece<MI_TYPE_BF16, WIDE, NT>(b.data[i], b.out[i], first, end, c);
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
    long long units(int i) const { return (sizes[i] + kUnit - 1) / kUnit; }
};

struct Totals {
    long long units = 0;
    double bytes = 0.0;
};

int check_list(const char* name, const List& l, Totals* total) {
    if (l.count < 0) return set_error(MI_ERR_INVALID_ARG, "%s: count=%d", name, l.count);
    if (l.count > 0 && (!l.tensors || !l.sizes))
        return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    for (int i = 0; i < l.count; ++i) {
        if (l.sizes[i] < 0 || l.sizes[i] > kMaxUnits * kUnit)
            return set_error(MI_ERR_INVALID_ARG, "%s: tensor %d has size %lld", name, i,
                             l.sizes[i]);
        if (!row_type_ok(l.type(i)))
            return set_error(MI_ERR_INVALID_ARG, "%s: tensor %d has unknown type %d", name, i,
                             l.type(i));
        if (l.sizes[i] > 0 && (!l.tensors[i] || (l.outs && !l.outs[i])))
            return set_error(MI_ERR_INVALID_ARG, "%s: tensor %d: NULL pointer", name, i);
        total->units += l.units(i);
        total->bytes += static_cast<double>(l.sizes[i]) * row_type_size(l.type(i));
        if (total->units > kMaxUnits)
            return set_error(MI_ERR_INVALID_ARG, "%s: more than %lld elements", name,
                             kMaxUnits * kUnit);
    }
    return MI_OK;
}

// Calls f(batch, its units) for every kBatch tensors that have elements.
template <class F>
int for_batches(const List& l, F f) {
    Batch b;
    b.count = 0;
    unsigned units = 0;
    for (int i = 0; i < l.count; ++i) {
        if (l.sizes[i] > 0) {
            const int n = b.count++;
            units += static_cast<unsigned>(l.units(i));
            b.data[n] = l.tensors[i];
            b.out[n] = l.outs ? l.outs[i] : const_cast<void*>(l.tensors[i]);
            b.size[n] = l.sizes[i];
            b.end[n] = units;
            b.type[n] = static_cast<unsigned char>(l.type(i));
        }
        if (b.count > 0 && (b.count == kBatch || i == l.count - 1)) {
            if (int rc = f(b, units)) return rc;
            b.count = 0;
            units = 0;
        }
    }
    return MI_OK;
}

// Workgroups of a batch's norm launch: its share of kNormBlocks, at most a unit each.
int norm_blocks(unsigned units, long long all) {
    const long long share = (static_cast<long long>(kNormBlocks) * units + all - 1) / all;
    return static_cast<int>(std::min<long long>(share, units));
}

int norm_sq(const char* name, const List& l, const Totals& total, float* result, bool accumulate,
            float* clip, float max_norm, hipStream_t st) {
    int err = MI_OK;
    char* ws = static_cast<char*>(workspace_get(mi_tensors_workspace(l.count), st, &err));
    if (!ws) return err;
    float* part = reinterpret_cast<float*>(ws + colsum_part_offset());
    int parts = 0;
    const bool nt = stream_loads(total.bytes);
    const int rc = for_batches(l, [&](const Batch& b, unsigned units) {
        const int blocks = norm_blocks(units, total.units);
        hipLaunchKernelGGL(tensors_sumsq_kernel, dim3(blocks), dim3(kThreads), 0, st, b,
                           part + parts, units, nt);
        parts += blocks;
        return check_launch(name);
    });
    if (rc) return rc;
    hipLaunchKernelGGL(tensors_finish_kernel, dim3(1), dim3(kFinThreads), 0, st, part, parts,
                       result, accumulate, clip, max_norm);
    return check_launch(name);
}

int scale_all(const char* name, const List& l, const Totals& total, const float* scale,
              hipStream_t st) {
    const bool nt = stream_loads(total.bytes);
    return for_batches(l, [&](const Batch& b, unsigned units) {
        const dim3 grid(std::min<unsigned>(units, kScaleBlocks));
        with_flag(l.outs != nullptr, [&](auto wide) {
            hipLaunchKernelGGL((tensors_scale_kernel<decltype(wide)::value>), grid,
                               dim3(kThreads), 0, st, b, scale, units, nt);
        });
        return check_launch(name);
    });
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

size_t mi_tensors_workspace(int count) {
    if (count < 0) return 0;
    // a launch's share of kNormBlocks is rounded up
    return colsum_part_offset() +
           (kNormBlocks + static_cast<size_t>(count) / kBatch + 1) * sizeof(float);
}

int mi_tensors_norm_sq_acc(const void* const* tensors, const long long* sizes, const int* types,
                           int count, float* d_result, void* stream) {
    const char* name = "mi_tensors_norm_sq_acc";
    const List l{tensors, nullptr, sizes, types, count};
    Totals total;
    if (int rc = check_list(name, l, &total)) return rc;
    if (!d_result) return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    if (total.units == 0) return MI_OK;
    return norm_sq(name, l, total, d_result, true, nullptr, 0.0f, to_stream(stream));
}

int mi_tensors_scale(const void* const* tensors, void* const* outs, const long long* sizes,
                     const int* types, int count, const float* d_scale, void* stream) {
    const char* name = "mi_tensors_scale";
    const List l{tensors, outs, sizes, types, count};
    Totals total;
    if (int rc = check_list(name, l, &total)) return rc;
    if (!d_scale) return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    return scale_all(name, l, total, d_scale, to_stream(stream));
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
    if (int rc = norm_sq(name, l, total, d_norm_sq, false, d_clip_scale, max_norm, st)) return rc;
    return scale_all(name, l, total, d_clip_scale, st);
}

}  // extern "C"

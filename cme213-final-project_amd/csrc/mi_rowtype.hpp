// Rows of fp32, fp16 or bf16 elements, computed with in fp32: the element
// types of the entry points that take an MI_TYPE_* code, their 16-byte
// accesses and their conversions.
#pragma once

#include <type_traits>

#include "mi_common.hpp"

namespace mi {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// Rows start at any multiple of the element size (an odd width of 2-byte
// elements), so 16-byte accesses state the alignment they can rely on; gfx950
// takes them in one instruction all the same.
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));

template <int T>
struct RowType;
template <>
struct RowType<MI_TYPE_F32> {
    typedef float elem;
};
template <>
struct RowType<MI_TYPE_F16> {
    typedef _Float16 elem;
};
template <>
struct RowType<MI_TYPE_BF16> {
    typedef __bf16 elem;
};

template <int T>
using row_elem = typename RowType<T>::elem;

// Elements of one 16-byte access.
template <int T>
constexpr int row_vec() {
    return 16 / static_cast<int>(sizeof(row_elem<T>));
}

// Every conversion to 16 bits rounds to nearest even (half a step: 2^-11 of
// the value for fp16, 2^-8 for bf16), once, from the fp32 result.
template <int T>
__device__ __forceinline__ float row_get(const void* p, size_t i) {
    return static_cast<float>(static_cast<const row_elem<T>*>(p)[i]);
}

template <int T>
__device__ __forceinline__ void row_put(void* p, size_t i, float v) {
    static_cast<row_elem<T>*>(p)[i] = static_cast<row_elem<T>>(v);
}

// NT: the line is not kept in the caches.  Rows are written so: the last-level cache
// is left to what is read (combine's gradient of 8192 tokens of 768 fp32, 2 choices,
// 27.0 -> 20.3 us).  They are read so where a call's rows are more than half of the 256
// MB cache: combine of [8192 tokens, 4 choices] of 2048 columns bf16 (168 MB) 33.7 ->
// 29.4 us, of 4096 (336 MB) 64.2 -> 58.7, but of [4096, 4] of 1600 (66 MB) 11.1 -> 14.2.
template <bool NT>
__device__ __forceinline__ u32x4 load16b(const void* p) {
    if constexpr (NT) return __builtin_nontemporal_load(static_cast<const u32x4_at2*>(p));
    return *static_cast<const u32x4_at2*>(p);
}

__device__ __forceinline__ void store16b(void* p, const u32x4& v) {
    __builtin_nontemporal_store(v, static_cast<u32x4_at2*>(p));
}

inline bool stream_loads(double bytes) { return bytes > 128.0 * 1048576.0; }

// Calls f with the flag as a compile-time constant.
template <class F>
void with_flag(bool on, F f) {
    if (on)
        f(std::true_type());
    else
        f(std::false_type());
}

template <int T>
__device__ __forceinline__ void row_unpack(const u32x4& raw, float (&v)[row_vec<T>()]) {
    if constexpr (T == MI_TYPE_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(raw[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint16_t h = static_cast<uint16_t>(raw[e / 2] >> (e % 2 * 16));
            if constexpr (T == MI_TYPE_F16)
                v[e] = static_cast<float>(__builtin_bit_cast(_Float16, h));
            else
                v[e] = __uint_as_float(e % 2 ? raw[e / 2] & 0xffff0000u : raw[e / 2] << 16);
        }
    }
}

template <int T>
__device__ __forceinline__ u32x4 row_pack(const float (&v)[row_vec<T>()]) {
    if constexpr (T == MI_TYPE_F32) {
        return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                     __float_as_uint(v[3])};
    } else {
        typedef row_elem<T> pair __attribute__((ext_vector_type(2)));
        u32x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const pair p = {static_cast<row_elem<T>>(v[2 * e]),
                            static_cast<row_elem<T>>(v[2 * e + 1])};
            r[e] = __builtin_bit_cast(uint32_t, p);
        }
        return r;
    }
}

// Unaligned accesses of sizeof(V) bytes.
template <class V>
__device__ __forceinline__ V load_piece(const char* p) {
    V v;
    __builtin_memcpy(&v, p, sizeof(V));
    return v;
}

template <class V>
__device__ __forceinline__ void store_piece(char* p, const V& v) {
    __builtin_memcpy(p, &v, sizeof(V));
}

// N consecutive elements, as one access; N a power of two and at most 16 bytes.
template <int T, int N>
__device__ __forceinline__ void row_get_n(const void* p, size_t i, float (&v)[N]) {
    typedef row_elem<T> vec __attribute__((ext_vector_type(N)));
    const char* at = static_cast<const char*>(p) + i * sizeof(row_elem<T>);
    if constexpr (N == 1) {
        v[0] = row_get<T>(p, i);
    } else {
        const vec x = load_piece<vec>(at);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = static_cast<float>(x[e]);
    }
}

template <int T, int N>
__device__ __forceinline__ void row_put_n(void* p, size_t i, const float (&v)[N]) {
    typedef row_elem<T> vec __attribute__((ext_vector_type(N)));
    char* at = static_cast<char*>(p) + i * sizeof(row_elem<T>);
    if constexpr (N == 1) {
        row_put<T>(p, i, v[0]);
    } else {
        vec x;
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = static_cast<row_elem<T>>(v[e]);
        store_piece(at, x);
    }
}

inline bool row_type_ok(int type) {
    return type == MI_TYPE_F32 || type == MI_TYPE_F16 || type == MI_TYPE_BF16;
}

inline int row_type_size(int type) { return type == MI_TYPE_F32 ? 4 : 2; }

// Calls f with the row type as a compile-time constant.
template <class F>
void with_row_type(int type, F f) {
    if (type == MI_TYPE_F32)
        f(std::integral_constant<int, MI_TYPE_F32>());
    else if (type == MI_TYPE_F16)
        f(std::integral_constant<int, MI_TYPE_F16>());
    else
        f(std::integral_constant<int, MI_TYPE_BF16>());
}

// Sums and maxima over the L lanes (16 or 64) of a row's lane group; every
// lane of the group returns the result, in an order fixed by the code.  All
// lanes of the wave must be active.
template <int L>
__device__ __forceinline__ float group_sum(float v) {
    static_assert(L == 16 || L == 64, "a DPP row or the wave");
    if constexpr (L == 64) {
        return wave_sum(v);
    } else {
        v += dpp_move<0xB1>(v);
        v += dpp_move<0x4E>(v);
        v += dpp_move<0x141>(v);
        v += dpp_move<0x140>(v);
        return v;
    }
}

template <int CTRL>
__device__ __forceinline__ int dpp_move_i(int v) {
    return __builtin_amdgcn_mov_dpp(v, CTRL, 0xF, 0xF, false);
}

template <int L>
__device__ __forceinline__ float group_max(float v) {
    v = fmaxf(v, dpp_move<0xB1>(v));
    v = fmaxf(v, dpp_move<0x4E>(v));
    v = fmaxf(v, dpp_move<0x141>(v));
    v = fmaxf(v, dpp_move<0x140>(v));
    if constexpr (L == 64)
        v = fmaxf(fmaxf(readlane(v, 0), readlane(v, 16)), fmaxf(readlane(v, 32), readlane(v, 48)));
    return v;
}

}  // namespace mi

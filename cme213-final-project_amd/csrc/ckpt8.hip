// Activations kept for the backward pass in 8 bits, for gfx950: rows to a
// checkpoint and back, and bias + tanh-GELU of rows grouped by expert whose
// backward pass reads the checkpoint of its input.  No counterpart in the
// reference, which keeps the activation itself, in fp32 or half
// (FINAL_CLEAN_CODE/src/kernels/activations.cu:199-217,285-323).
//
// Format: 32 consecutive columns of a row share a power of two (the last
// block of a row may be shorter).  With e = max(floor(log2 max |x|), -118) the
// scale byte is e + 127; 255 marks a block that holds a NaN or an infinity, and
// all of it reads as NaN.  An element is
//   int8:  q = rint(x 2^(6-e)), -128 to 127, of value q 2^(e-6) (-128 in the topmost block
//          of a type is -2^(e+1), which rounds to -inf in it);
//   e4m3:  q = e4m3(x 2^(8-e)), at most 448 in magnitude, of value q 2^(e-8).
// The scaling is exact and the rounding (to nearest even) the only one, so a
// value has one code whatever computes it: off by at most 2^(e-7) for int8
// (2^(e-6) where it is cut to 127, in the top 1/256 of the block's range), by
// 2^-4 of itself for normal e4m3 codes (64 2^(e-8) where it is cut to 448).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "mi_common.hpp"
#include "mi_gelu.hpp"
#include "mi_rowtype.hpp"

namespace mi {

namespace {

constexpr int kThreads = 256;
constexpr int kUnit = 8;              // consecutive columns of one lane
constexpr int kTile = kUnit * kWave;  // columns of a full tile
constexpr int kBlock = MI_CKPT8_BLOCK;  // four lanes
constexpr int kLine = 64;  // columns: rows of codes are whole halves of cache lines
constexpr int kMaxGroups = 1024;
constexpr int kMaxRows = 1 << 30;  // keep row and column numbers, one tile or band
constexpr int kMaxCols = 1 << 24;  // further on, inside an int, and the grids legal
static_assert(kBlock == 4 * kUnit, "a block's lanes are one DPP quad");

// ---------------------------------------------------------------------------
// Layout.  A lane takes 8 consecutive columns of a row (a unit), so four
// adjacent lanes hold a block.  A workgroup takes a tile of columns and a band
// of consecutive rows; a tile is 64 units wide (512 columns, one wave a row, four
// rows at a time), and what is left of the width is a narrower tile of its own,
// a power of two of units wide, with more rows at a time, so that few lanes idle.
// Memory-bound.  Workgroups as wide as the row (one row at a time) were slower:
// [16384, 6400] bf16 forward 104 -> 118 us, backward 153 -> 174.
// ---------------------------------------------------------------------------
struct Unit {
    int col;  // first column
    int n;    // columns of it inside the row, 0 to 8
    int from, back;  // of Units::Partial: the eight columns from `from` on, `back` before col
};

// The units of a workgroup's lanes: all whole; whole or empty; one of them partial, in
// rows of at least a unit; the partial unit that is all of a shorter row.
enum class Units { Whole, WholeOrEmpty, Partial, Short };

struct Task {
    int first_col, band;
    int lanes, row_lanes, row_lane;
    Units units;
    Unit un;
};

// The tile beside the full ones, last_lanes units wide (0: there is none), has the
// first last_bands workgroups.  Begun last, its short rows were what the others had
// to be waited for with: step of [16384, 1600] bf16 61.9 -> 57.7 us, of [6007, 2049]
// fp16 37.3 -> 33.1.  The full tiles go along a band; where rows are not whole cache
// lines, along eight bands side by side, since consecutive workgroups are on different
// XCDs: the line that two tiles of a row share is then in one L2 (step of [6007, 2064]
// fp16 35.9 -> 32.5 us, [8192, 6152] bf16 125.6 -> 120.2; but [4096, 4096] bf16 40.0 ->
// 45.9).
__device__ __forceinline__ Task workgroup_task(int cols, int full_tiles, int last_lanes,
                                               int last_bands) {
    Task t;
    int w = static_cast<int>(blockIdx.x) - last_bands;
    if (w >= 0) {
        if (cols % kLine != 0) {
            const int eight = 8 * full_tiles;
            const int begin = w / eight * eight, i = w - begin;
            if (begin + eight <= static_cast<int>(gridDim.x) - last_bands)
                w = begin + i % 8 * full_tiles + i / 8;
        }
        t.band = w / full_tiles;
        t.first_col = (w - t.band * full_tiles) * kTile;
        t.lanes = kWave;
    } else {
        t.band = static_cast<int>(blockIdx.x);
        t.first_col = full_tiles * kTile;
        t.lanes = last_lanes;
    }
    t.row_lanes = kThreads / t.lanes;
    t.row_lane = static_cast<int>(threadIdx.x) / t.lanes;
    t.un.col = t.first_col + static_cast<int>(threadIdx.x & (t.lanes - 1)) * kUnit;
    t.un.n = max(0, min(kUnit, cols - t.un.col));
    t.units = cols - t.first_col >= t.lanes * kUnit ? Units::Whole
              : cols % kUnit == 0                   ? Units::WholeOrEmpty
              : cols > kUnit                        ? Units::Partial
                                                    : Units::Short;
    t.un.from = min(t.un.col, cols - kUnit);
    t.un.back = min(t.un.col - t.un.from, kUnit);
    return t;
}

// A unit of a row, in the row's type.  The row's last unit may be partial: the
// elements behind it read as 0.  It is read with as many elements before it as it lacks
// and moved down, so that its wave's loads all go out together: read as its 4, 2 and 1
// elements, as it is written, step of [30000, 777] bf16 84.2 us, 77.3 so, of [5000, 769]
// fp32 27.7, 25.5, of [6007, 2049] fp16 33.9, 33.4.
template <int N>
__device__ __forceinline__ void move_down(uint32_t (&a)[N], int dwords) {
#pragma unroll
    for (int step = N; step >= 1; step /= 2) {
        const bool on = dwords & step;
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] = on ? (i + step < N ? a[i + step] : 0u) : a[i];
    }
}

template <int T>
struct RawUnit {
    u32x4 a[kUnit / row_vec<T>()];
};

template <int T, Units UN, bool NT>
__device__ __forceinline__ RawUnit<T> load_unit(const char* row, const Unit& un) {
    RawUnit<T> r;
    const char* p = row + static_cast<size_t>(UN == Units::Partial ? un.from : un.col) *
                              sizeof(row_elem<T>);
    const int n = un.n;
    if constexpr (UN == Units::Partial) {
        constexpr int N = 4 * (kUnit / row_vec<T>());
        uint32_t a[N];
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const u32x4 v = load16b<NT>(p + 16 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) a[4 * i + e] = v[e];
        }
        if constexpr (T == MI_TYPE_F32) {
            move_down(a, un.back);
        } else {
            move_down(a, un.back / 2);
#pragma unroll
            for (int i = 0; i < N; ++i)
                a[i] = un.back & 1 ? a[i] >> 16 | (i + 1 < N ? a[i + 1] << 16 : 0u) : a[i];
        }
#pragma unroll
        for (int i = 0; i < N / 4; ++i)
            r.a[i] = u32x4{a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3]};
    } else if (UN == Units::Whole || n == kUnit) {
#pragma unroll
        for (int i = 0; i < kUnit / row_vec<T>(); ++i) r.a[i] = load16b<NT>(p + 16 * i);
    } else if constexpr (UN == Units::WholeOrEmpty) {
#pragma unroll
        for (int i = 0; i < kUnit / row_vec<T>(); ++i) r.a[i] = u32x4{0, 0, 0, 0};
    } else if constexpr (T == MI_TYPE_F32) {
        const u32x4 p4 = n & 4 ? load16b<NT>(p) : u32x4{0, 0, 0, 0};
        const u32x2 p2 = n & 2 ? load_piece<u32x2>(p + (n & 4) * 4) : u32x2{0, 0};
        const uint32_t p1 = n & 1 ? load_piece<uint32_t>(p + (n & 6) * 4) : 0;
        const u32x4 rest = {n & 2 ? p2.x : p1, p2.y, n & 2 ? p1 : 0, 0};
        r.a[0] = n & 4 ? p4 : rest;
        r.a[1] = n & 4 ? rest : p4;
    } else {
        const u32x2 p4 = n & 4 ? load_piece<u32x2>(p) : u32x2{0, 0};
        const uint32_t p2 = n & 2 ? load_piece<uint32_t>(p + (n & 4) * 2) : 0;
        const uint32_t p1 = n & 1 ? load_piece<uint16_t>(p + (n & 6) * 2) : 0;
        const u32x2 rest = {n & 2 ? p2 : p1, n & 2 ? p1 : 0};
        r.a[0] = n & 4 ? u32x4{p4.x, p4.y, rest.x, rest.y} : u32x4{rest.x, rest.y, 0, 0};
    }
    return r;
}

template <int T>
__device__ __forceinline__ void unpack_unit(const RawUnit<T>& r, float (&v)[kUnit]) {
#pragma unroll
    for (int i = 0; i < kUnit / row_vec<T>(); ++i) {
        float part[row_vec<T>()];
        row_unpack<T>(r.a[i], part);
#pragma unroll
        for (int e = 0; e < row_vec<T>(); ++e) v[i * row_vec<T>() + e] = part[e];
    }
}

template <int T, Units UN>
__device__ __forceinline__ void store_unit(char* row, const Unit& un, const float (&v)[kUnit]) {
    char* p = row + static_cast<size_t>(un.col) * sizeof(row_elem<T>);
    const int n = un.n;
    u32x4 a[kUnit / row_vec<T>()];
#pragma unroll
    for (int i = 0; i < kUnit / row_vec<T>(); ++i) {
        float part[row_vec<T>()];
#pragma unroll
        for (int e = 0; e < row_vec<T>(); ++e) part[e] = v[i * row_vec<T>() + e];
        a[i] = row_pack<T>(part);
    }
    if (UN == Units::Whole || n == kUnit) {
#pragma unroll
        for (int i = 0; i < kUnit / row_vec<T>(); ++i) store16b(p + 16 * i, a[i]);
    } else if constexpr (UN == Units::WholeOrEmpty) {
        return;
    } else if constexpr (T == MI_TYPE_F32) {
        const u32x4 rest = n & 4 ? a[1] : a[0];
        if (n & 4) store16b(p, a[0]);
        if (n & 2) store_piece(p + (n & 4) * 4, u32x2{rest.x, rest.y});
        if (n & 1) store_piece<uint32_t>(p + (n & 6) * 4, n & 2 ? rest.z : rest.x);
    } else {
        const uint32_t x = n & 4 ? a[0].z : a[0].x, y = n & 4 ? a[0].w : a[0].y;
        if (n & 4) store_piece(p, u32x2{a[0].x, a[0].y});
        if (n & 2) store_piece<uint32_t>(p + (n & 4) * 2, x);
        if (n & 1) store_piece(p + (n & 6) * 2, static_cast<uint16_t>(n & 2 ? y : x));
    }
}

template <Units UN>
__device__ __forceinline__ u32x2 load_codes(const uint8_t* row, const Unit& un) {
    const char* p = reinterpret_cast<const char*>(row) + un.col;
    const int n = un.n;
    if constexpr (UN == Units::Partial) {
        const u32x2 v = load_piece<u32x2>(reinterpret_cast<const char*>(row) + un.from);
        const uint64_t w = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(u32x2, un.back < kUnit ? w >> (8 * un.back) : 0);
    }
    if (UN == Units::Whole || n == kUnit) return load_piece<u32x2>(p);
    if constexpr (UN == Units::WholeOrEmpty) return u32x2{0, 0};
    const uint32_t p4 = n & 4 ? load_piece<uint32_t>(p) : 0;
    const uint32_t p2 = n & 2 ? load_piece<uint16_t>(p + (n & 4)) : 0;
    const uint32_t p1 = n & 1 ? load_piece<uint8_t>(p + (n & 6)) : 0;
    const uint32_t rest = n & 2 ? p2 | p1 << 16 : p1;
    return n & 4 ? u32x2{p4, rest} : u32x2{rest, 0};
}

template <Units UN>
__device__ __forceinline__ void store_codes(uint8_t* row, const Unit& un, const u32x2& q) {
    char* p = reinterpret_cast<char*>(row) + un.col;
    const int n = un.n;
    if (UN == Units::Whole || n == kUnit) {
        store_piece(p, q);
    } else if constexpr (UN == Units::Partial || UN == Units::Short) {
        const uint32_t rest = n & 4 ? q.y : q.x;
        if (n & 4) store_piece<uint32_t>(p, q.x);
        if (n & 2) store_piece(p + (n & 4), static_cast<uint16_t>(rest));
        if (n & 1) store_piece(p + (n & 6), static_cast<uint8_t>(n & 2 ? rest >> 16 : rest));
    }
}

// The scale byte of the block that the lane's quad holds.  Magnitudes compare
// as integers, with NaN and infinity above every number, and the exponent
// field of the largest is e + 127.  Two 16-bit magnitudes compare at a time.
template <int T>
__device__ __forceinline__ int block_scale(const RawUnit<T>& r) {
    int m = 0;
    if constexpr (T == MI_TYPE_F32) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) m = max(m, static_cast<int>(r.a[i][e] & 0x7fffffffu));
    } else {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        u16x2 p = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            p = __builtin_elementwise_max(p, __builtin_bit_cast(u16x2, r.a[0][e] & 0x7fff7fffu));
        m = max(p.x, p.y);
    }
    m = max(m, dpp_move_i<0xB1>(m));
    m = max(m, dpp_move_i<0x4E>(m));
    if constexpr (T == MI_TYPE_BF16) m <<= 16;
    if constexpr (T == MI_TYPE_F16)
        m = __float_as_int(
            static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(m))));
    return max(m >> 23, 9);
}

// The codes of a unit.  int8: adding 1.5 2^23 leaves rint(x 2^(6-e)) in the low
// bits of the sum, two's complement; the product is exact inside the FMA.
template <int FMT>
__device__ __forceinline__ u32x2 encode(const float (&v)[kUnit], int scale) {
    u32x2 q = {0, 0};
    if (scale == 255) return q;
    const float mul = __int_as_float(((FMT == MI_CKPT8_INT8 ? 260 : 262) - scale) << 23);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (FMT == MI_CKPT8_INT8) {
            uint32_t b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                b[e] = __float_as_uint(fminf(fmaf(v[4 * h + e], mul, 12582912.0f), 12583039.0f));
            const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u);
            const uint32_t hi = __builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u);
            q[h] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
        } else {
            float s[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                s[e] = __builtin_amdgcn_fmed3f(v[4 * h + e] * mul, -448.0f, 448.0f);
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], w, true);
            q[h] = static_cast<uint32_t>(w);
        }
    }
    return q;
}

// value + add: the product is exact, so this is one rounding, of the sum.
template <int FMT>
__device__ __forceinline__ void decode(const u32x2& q, int scale, const float (&add)[kUnit],
                                       float (&v)[kUnit]) {
    // hidden from the compiler, which else tests every element for the NaN
    const float step =
        rounded(scale == 255 ? __int_as_float(0x7fc00000)
                             : __builtin_ldexpf(1.0f, scale - (FMT == MI_CKPT8_INT8 ? 133 : 135)));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int w = static_cast<int>(q[h]);
        float x[4];
        if constexpr (FMT == MI_CKPT8_INT8) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[e] = static_cast<float>(static_cast<int8_t>(w >> (8 * e)));
        } else {
            x[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
            x[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
            x[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
            x[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * h + e] = fmaf(x[e], step, add[4 * h + e]);
    }
}

// ---------------------------------------------------------------------------
// Segments.  Group g's rows are offsets[g] .. offsets[g + 1] - 1; without
// offsets there is one group of all rows.  Values outside [0, rows] are cut,
// so that offsets which are not what they should be cannot lead out of the
// tensors.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int group_end(const int* offsets, int g, int rows) {
    return offsets == nullptr ? rows : max(0, min(offsets[g + 1], rows));
}

// The first row of any group.
__device__ __forceinline__ int first_row(const int* offsets, int rows) {
    return offsets == nullptr ? 0 : max(0, min(offsets[0], rows));
}

template <Units UN>
__device__ __forceinline__ void load_bias(const float* bias, int g, int cols, const Unit& un,
                                          float (&b)[kUnit]) {
    const float* row = bias + static_cast<size_t>(g) * cols;
    unpack_unit<MI_TYPE_F32>(
        load_unit<MI_TYPE_F32, UN, false>(reinterpret_cast<const char*>(row), un), b);
}

// f(g, a, b) for the rows a .. b - 1 of group g inside r0 .. r1 - 1.  Everything
// here is the same for a whole workgroup.  The ends of 64 groups are loaded at a
// time, one a lane: the first group that ends behind a row is the number of those
// that do not, so finding it costs one memory round trip per 64 groups instead of
// one per bit of a search, and the next groups' ends are at hand.
template <class F>
__device__ __forceinline__ void for_segments(const int* offsets, int groups, int rows, int r0,
                                             int r1, F f) {
    if (offsets == nullptr) {
        f(0, r0, r1);
        return;
    }
    const int lane = threadIdx.x & (kWave - 1);
    int a = max(r0, first_row(offsets, rows));
    for (int base = 0; base < groups && a < r1; base += kWave) {
        const int here = min(kWave, groups - base);
        const int end = group_end(offsets, base + min(lane, here - 1), rows);
        int i = static_cast<int>(__popcll(__ballot(lane < here && end <= a)));
        for (; i < here && a < r1; ++i) {
            const int b = min(__builtin_amdgcn_readlane(end, i), r1);
            if (b > a) {
                f(base + i, a, b);
                a = b;
            }
        }
    }
}

// Rows of a lane that are in hand together: their loads are issued before the
// first is computed.  Backward of [16384, 6400], [16384, 4096] bf16 by one 105.8,
// 64.0 us, two 103.9, 61.7, four 108.9, 61.9; with the next rows' loads issued before
// these are computed 115.8, 63.4 (fewer waves fit).
constexpr int kRowsInHand = 2;

// The kernels take first what they use first: their leading 14 dwords of arguments
// are in registers when a wave starts.

template <class F>
__device__ __forceinline__ void by_units(Units units, F body) {
    if (units == Units::Whole)
        body(std::integral_constant<Units, Units::Whole>());
    else if (units == Units::WholeOrEmpty)
        body(std::integral_constant<Units, Units::WholeOrEmpty>());
    else if (units == Units::Partial)
        body(std::integral_constant<Units, Units::Partial>());
    else
        body(std::integral_constant<Units, Units::Short>());
}

// GELU: out = gelu(in + bias) and the checkpoint of in; else the checkpoint.
// out may be in: a lane reads its units of the rows in hand before it writes
// them.
template <int T, int FMT, bool GELU, bool NT>
__global__ __launch_bounds__(kThreads) void to_ckpt8_kernel(
    int cols, int full_tiles, int last_lanes, int last_bands, int band, int rows, int groups,
    const char* in, const int* __restrict__ offsets, const float* __restrict__ bias, char* out,
    uint8_t* __restrict__ q, uint8_t* __restrict__ scales) {
    constexpr int U = kRowsInHand;
    const Task t = workgroup_task(cols, full_tiles, last_lanes, last_bands);
    const Unit un = t.un;
    const size_t row_bytes = static_cast<size_t>(cols) * sizeof(row_elem<T>);
    const int blocks = (cols + kBlock - 1) / kBlock;
    const int r0 = t.band * band, r1 = min(r0 + band, rows);
    by_units(t.units, [&](auto units) {
        constexpr Units UN = decltype(units)::value;
        for_segments(offsets, groups, rows, r0, r1, [&](int g, int a, int end) {
            float b[kUnit];
            if constexpr (GELU) load_bias<UN>(bias, g, cols, un, b);
            for (int r = a + t.row_lane; r < end; r += U * t.row_lanes) {
                RawUnit<T> raw[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int rr = r + u * t.row_lanes;
                    raw[u] = load_unit<T, UN, NT>(in + (rr < end ? rr : r) * row_bytes, un);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int rr = r + u * t.row_lanes;
                    if (rr >= end) break;
                    const int scale = block_scale<T>(raw[u]);
                    float v[kUnit];
                    unpack_unit<T>(raw[u], v);
                    store_codes<UN>(q + static_cast<size_t>(rr) * cols, un,
                                      encode<FMT>(v, scale));
                    if (un.n > 0 && un.col % kBlock == 0)
                        scales[static_cast<size_t>(rr) * blocks + un.col / kBlock] =
                            static_cast<uint8_t>(scale);
                    if constexpr (GELU) {
#pragma unroll
                        for (int e = 0; e < kUnit; ++e) v[e] = gelu_pair(v[e] + b[e]).y;
                        store_unit<T, UN>(out + rr * row_bytes, un, v);
                    }
                }
            }
        });
    });
}

// Memory-bound: [16384, 6400] to bf16 54.8 us (5.8 TB/s), the checkpoint alone of it 59.9
// (5.3).  fp32 rows are slower in every kernel here: to fp32 120.1 us (4.4), the checkpoint
// of it 104.5 (5.05).  A unit of them is two accesses of 16 bytes, 32 bytes from those
// of the next lane; a plain copy in this form reaches 3.98 TB/s, with each access side by
// side 6.5.
template <int T, int FMT>
__global__ __launch_bounds__(kThreads) void from_ckpt8_kernel(
    const uint8_t* __restrict__ q, const uint8_t* __restrict__ scales, char* __restrict__ out,
    int rows, int cols, int band, int full_tiles, int last_lanes, int last_bands) {
    const Task t = workgroup_task(cols, full_tiles, last_lanes, last_bands);
    const Unit un = t.un;
    if (un.n == 0) return;
    const size_t row_bytes = static_cast<size_t>(cols) * sizeof(row_elem<T>);
    const int blocks = (cols + kBlock - 1) / kBlock;
    const int r0 = t.band * band, r1 = min(r0 + band, rows);
    const float none[kUnit] = {};
    // the empty lanes are gone
    by_units(t.units == Units::WholeOrEmpty ? Units::Whole : t.units, [&](auto units) {
        constexpr Units UN = decltype(units)::value;
        for (int r = r0 + t.row_lane; r < r1; r += t.row_lanes) {
            float v[kUnit];
            decode<FMT>(load_codes<UN>(q + static_cast<size_t>(r) * cols, un),
                        scales[static_cast<size_t>(r) * blocks + un.col / kBlock], none, v);
            store_unit<T, UN>(out + r * row_bytes, un, v);
        }
    });
}

// What the backward pass reads of a row.
template <int T>
struct HeldRow {
    RawUnit<T> grad;
    u32x2 code;
    int scale;
};

// u = value of the checkpoint + bias; grad_in = grad_out gelu'(u); act =
// gelu(u); the column sums of grad_in over the band's rows of group g, added
// over the row lanes in order, go to partial row band + g.  Going down the
// rows, band and g only grow, and one of them does with every new pair, so no
// two pairs share a partial row.  With part == nullptr there is one band, and its
// sums are added to dbias at once.  grad_in may be grad_out.
template <int T, int FMT, bool ACT, bool NT>
__global__ __launch_bounds__(kThreads) void gelu_bwd_ckpt8_kernel(
    int cols, int full_tiles, int last_lanes, int last_bands, int band, int rows, int groups,
    const int* __restrict__ offsets, const float* __restrict__ bias,
    const uint8_t* __restrict__ q, const uint8_t* __restrict__ scales, const char* grad_out,
    char* grad_in, char* __restrict__ act, float* __restrict__ part,
    float* __restrict__ dbias) {
    constexpr int U = kRowsInHand;
    __shared__ float red[kThreads * kUnit];
    const Task t = workgroup_task(cols, full_tiles, last_lanes, last_bands);
    const Unit un = t.un;
    const size_t row_bytes = static_cast<size_t>(cols) * sizeof(row_elem<T>);
    const int blocks = (cols + kBlock - 1) / kBlock;
    const int scale_at = min(un.col / kBlock, blocks - 1);
    const int r0 = t.band * band, r1 = min(r0 + band, rows);
    auto segment = [&](auto units, int g, int a, int end) {
        constexpr Units UN = decltype(units)::value;
        float b[kUnit], acc[kUnit];
#pragma unroll
        for (int e = 0; e < kUnit; ++e) b[e] = acc[e] = 0.0f;
        if (un.n > 0) load_bias<UN>(bias, g, cols, un, b);
        // The rows are taken in turn from a place that differs from band to band:
        // bands that are all at the same row of theirs touch the same memory
        // channels where a band is a power of two of bytes ([8192, 4096] fp32 85
        // us in step, 67 so; other sizes alike).
        const int trips = (end - a + U * t.row_lanes - 1) / (U * t.row_lanes);
        int trip = static_cast<int>(static_cast<unsigned>(t.band) * 3u % trips);
        auto row_of = [&](int of, int u) { return a + t.row_lane + (of * U + u) * t.row_lanes; };
        // Rows behind the segment's last read the last one and are not used.
        auto load = [&](int of, HeldRow<T> (&h)[U]) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const size_t r = min(row_of(of, u), end - 1);
                h[u].code = load_codes<UN>(q + r * cols, un);
                h[u].scale = scales[r * blocks + scale_at];
                h[u].grad = load_unit<T, UN, NT>(grad_out + r * row_bytes, un);
            }
        };
        auto use = [&](int of, const HeldRow<T> (&h)[U]) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = row_of(of, u);
                if (r >= end) break;
                float v[kUnit], d[kUnit];
                unpack_unit<T>(h[u].grad, d);
                decode<FMT>(h[u].code, h[u].scale, b, v);
#pragma unroll
                for (int e = 0; e < kUnit; ++e) {
                    const GeluPair p = gelu_pair(v[e]);
                    acc[e] = fmaf(d[e], p.d, acc[e]);
                    d[e] *= p.d;
                    v[e] = p.y;
                }
                store_unit<T, UN>(grad_in + r * row_bytes, un, d);
                if constexpr (ACT) store_unit<T, UN>(act + r * row_bytes, un, v);
            }
        };
        if (un.n > 0)
            for (int i = 0; i < trips; ++i, trip = trip + 1 < trips ? trip + 1 : 0) {
                HeldRow<T> held[U];
                load(trip, held);
                use(trip, held);
            }
        const int width = t.lanes * kUnit;
        float* mine = red + threadIdx.x * kUnit;
#pragma unroll
        for (int e = 0; e < kUnit; ++e) mine[e] = acc[e];
        __syncthreads();
        for (int c = threadIdx.x; c < width; c += kThreads) {
            float sum = red[c];
            for (int l = 1; l < t.row_lanes; ++l) sum += red[l * width + c];
            const int col = t.first_col + c;
            if (col >= cols) continue;
            if (part == nullptr)
                dbias[static_cast<size_t>(g) * cols + col] += sum;
            else
                part[static_cast<size_t>(t.band + g) * cols + col] = sum;
        }
        __syncthreads();
    };
    // empty lanes only take part in the sums, so units are whole or partial
    by_units(t.units == Units::WholeOrEmpty ? Units::Whole : t.units, [&](auto units) {
        for_segments(offsets, groups, rows, r0, r1,
                     [&](int g, int a, int end) { segment(units, g, a, end); });
    });
}

// dbias[g][c] += sum of group g's partial rows: 64 columns a workgroup, its
// waves each a consecutive slice of the partial rows in order, then the waves
// in order.  Loads are issued 16 at a time.  Latency-bound: 4 to 7 us where segments are of
// about one length.  The slices go by the average: a segment that holds nine tenths
// of [16384, 1600] in 128 groups has one slice for its 950 partial rows, 47 us (5 where
// the groups are even).  32 or 16 columns a workgroup and more slices were no faster, and
// slower for many groups.
__global__ __launch_bounds__(1024) void group_sum_kernel(const float* __restrict__ part,
                                                         const int* __restrict__ offsets,
                                                         float* __restrict__ dbias, int rows,
                                                         int cols, int band, int slices) {
    constexpr int CH = 16;
    __shared__ float tot[1024 / kWave][kWave];
    const int g = blockIdx.y;
    const int start = g == 0 ? first_row(offsets, rows) : group_end(offsets, g - 1, rows);
    const int end = group_end(offsets, g, rows);
    if (start >= end) return;
    const int lane = threadIdx.x & (kWave - 1);
    const int slice = threadIdx.x / kWave;
    const int c = blockIdx.x * kWave + lane;
    const int first = start / band, n = (end - 1) / band - first + 1;
    const int p0 = static_cast<int>(static_cast<long long>(slice) * n / slices);
    const int p1 = static_cast<int>(static_cast<long long>(slice + 1) * n / slices);
    float* o = dbias + static_cast<size_t>(g) * cols + c;
    const float old = slice == 0 && c < cols ? *o : 0.0f;
    float s = 0.0f;
    if (c < cols) {
        const float* col = part + static_cast<size_t>(first + g) * cols + c;
        for (int p = p0; p < p1; p += CH) {
            float v[CH];
#pragma unroll
            for (int i = 0; i < CH; ++i)
                v[i] = p + i < p1 ? col[static_cast<size_t>(p + i) * cols] : 0.0f;
#pragma unroll
            for (int i = 0; i < CH; ++i)
                if (p + i < p1) s += v[i];
        }
    }
    tot[slice][lane] = s;
    __syncthreads();
    if (slice == 0 && c < cols) {
        float sum = tot[0][lane];
        for (int w = 1; w < slices; ++w) sum += tot[w][lane];
        *o = old + sum;
    }
}

struct Plan {
    int band, bands, full_tiles, last_lanes, last_bands;
    unsigned grid;
};

// Rows of a band: as many as make `waves` waves of the tensor, at least least_trips
// for each row lane while that leaves 256 workgroups, and at most most_trips; in no
// more than `most` bands.
Plan plan_ckpt8(int rows, int cols, int waves, int least_trips, int most_trips, int most) {
    Plan p;
    int left = cols % kTile;
    p.full_tiles = cols / kTile;
    // A tile of 64 units that are whole or empty goes with the full ones where these
    // take bands side by side: step of [20000, 2000] bf16 101.1 -> 96.6 us, [30000, 776]
    // 70.4 -> 67.5; with a partial unit [30000, 777] 77.0 -> 74.3, but [9000, 777] 28.3 ->
    // 30.2.
    if (cols % kLine != 0 && cols % kUnit == 0 && left > kTile / 2) {
        left = 0;
        ++p.full_tiles;
    }
    p.last_lanes = 0;
    if (left) {
        p.last_lanes = 4;
        while (p.last_lanes * kUnit < left) p.last_lanes *= 2;
    }
    const int tiles = p.full_tiles + (left ? 1 : 0);
    const long long row_lanes = kThreads / (p.full_tiles ? kWave : p.last_lanes);
    const long long work = static_cast<long long>(rows) * tiles;
    long long band = std::max(work * (kThreads / kWave) / waves,
                              std::min(least_trips * row_lanes, work / 256));
    band = std::min(std::max(band, row_lanes), most_trips * row_lanes);
    most = std::min(most, (1 << 23) / tiles);  // a legal grid
    band = std::max(band, (static_cast<long long>(rows) + most - 1) / most);
    band = std::min<long long>(band, rows);
    p.band = static_cast<int>(band);
    p.bands = static_cast<int>((rows + band - 1) / band);
    p.last_bands = left ? p.bands : 0;
    p.grid = static_cast<unsigned>(static_cast<long long>(p.bands) * tiles);
    return p;
}

// Forward: bands are short (16 rows of a full tile), so that the workgroups,
// started in order, sweep through memory; 8 rows a lane were as fast on most
// sizes and slower on [8192, 4096] fp32 (71 -> 87 us), one was slower on all
// ([16384, 6400] bf16 104 -> 122 us: every band reads its biases).
Plan plan_forward(int rows, int cols) { return plan_ckpt8(rows, cols, 4096, 2, 4, INT_MAX); }

// Backward: every band leaves a partial row to write and add up, so bands are
// longer: [4096, 1024] bf16 in 2048 workgroups of one row a lane 13.8 + 5.9 us (the
// sums), in 512 of four 8.8 + 3.9.  Too few workgroups starve the memory: [16384,
// 6400] bf16 in 520 198 us, 1027 159, 2054 153, 3328 148 (of an earlier kernel); and
// 8192 waves or 32768 as the target: bf16 with act [16384, 6400] 148 -> 139 us, 8192
// columns 178 -> 165.  Six trips a row lane instead of four where the tensor is large:
// fp32 [8192, 4096] with act 101 -> 94 us, but [4096, 1024] bf16 step 15.4 -> 16.5.
// Few rows are one band, whose sums go to dbias without the second launch: step of
// [16, 4096] bf16 10.0 -> 7.7 us, of 32 rows 10.0 -> 10.4.
Plan plan_backward(int rows, int cols, int groups) {
    if (rows <= 16 && groups <= 4) return plan_ckpt8(rows, cols, 1, 1, INT_MAX, 1);
    const bool large = static_cast<long long>(rows) * cols >= 65536ll * kTile;
    return plan_ckpt8(rows, cols, 32768, large ? 6 : 4, INT_MAX, 1024);
}

int check_args(const char* name, int rows, int cols, int groups, int format, int type) {
    if (rows < 0 || rows > kMaxRows || cols < 1 || cols > kMaxCols || groups < 1 ||
        groups > kMaxGroups)
        return set_error(MI_ERR_INVALID_ARG,
                         "%s: invalid shape rows=%d cols=%d groups=%d (rows is 0 to %d, cols 1 to "
                         "%d, groups 1 to %d)",
                         name, rows, cols, groups, kMaxRows, kMaxCols, kMaxGroups);
    if (format != MI_CKPT8_INT8 && format != MI_CKPT8_E4M3)
        return set_error(MI_ERR_INVALID_ARG, "%s: unknown format %d", name, format);
    if (!row_type_ok(type))
        return set_error(MI_ERR_INVALID_ARG, "%s: unknown type %d", name, type);
    return MI_OK;
}

template <class F>
void with_format(int format, F f) {
    if (format == MI_CKPT8_INT8)
        f(std::integral_constant<int, MI_CKPT8_INT8>());
    else
        f(std::integral_constant<int, MI_CKPT8_E4M3>());
}

template <bool GELU>
int launch_to_ckpt8(const char* name, const void* in, const float* bias, const int* offsets,
                    void* out, void* q, void* scales, int rows, int cols, int groups, int format,
                    int type, hipStream_t st) {
    const Plan p = plan_forward(rows, cols);
    const double bytes =
        static_cast<double>(rows) * cols * ((GELU ? 2 : 1) * row_type_size(type) + 1);
    with_row_type(type, [&](auto t) {
        with_format(format, [&](auto f) {
            constexpr int T = decltype(t)::value, F = decltype(f)::value;
            with_flag(stream_loads(bytes), [&](auto nt) {
                hipLaunchKernelGGL((to_ckpt8_kernel<T, F, GELU, decltype(nt)::value>), dim3(p.grid),
                                   dim3(kThreads), 0, st, cols, p.full_tiles, p.last_lanes,
                                   p.last_bands, p.band, rows, groups,
                                   static_cast<const char*>(in), offsets, bias,
                                   static_cast<char*>(out), static_cast<uint8_t*>(q),
                                   static_cast<uint8_t*>(scales));
            });
        });
    });
    return check_launch(name);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" {

int mi_float_to_ckpt8(const void* in, void* q, void* scales, int rows, int cols, int format,
                      int type, void* stream) {
    const char* name = "mi_float_to_ckpt8";
    if (int rc = check_args(name, rows, cols, 1, format, type)) return rc;
    if (rows == 0) return MI_OK;
    if (!in || !q || !scales) return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    return launch_to_ckpt8<false>(name, in, nullptr, nullptr, nullptr, q, scales, rows, cols, 1,
                                  format, type, to_stream(stream));
}

int mi_ckpt8_to_float(const void* q, const void* scales, void* out, int rows, int cols, int format,
                      int type, void* stream) {
    const char* name = "mi_ckpt8_to_float";
    if (int rc = check_args(name, rows, cols, 1, format, type)) return rc;
    if (rows == 0) return MI_OK;
    if (!q || !scales || !out) return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    const Plan p = plan_forward(rows, cols);
    with_row_type(type, [&](auto t) {
        with_format(format, [&](auto f) {
            constexpr int T = decltype(t)::value, F = decltype(f)::value;
            hipLaunchKernelGGL((from_ckpt8_kernel<T, F>), dim3(p.grid), dim3(kThreads), 0,
                               to_stream(stream), static_cast<const uint8_t*>(q),
                               static_cast<const uint8_t*>(scales), static_cast<char*>(out), rows,
                               cols, p.band, p.full_tiles, p.last_lanes, p.last_bands);
        });
    });
    return check_launch(name);
}

int mi_bias_gelu_forward_ckpt8(const void* in, const float* bias, const int* offsets, void* out,
                               void* q, void* scales, int rows, int cols, int groups, int format,
                               int type, void* stream) {
    const char* name = "mi_bias_gelu_forward_ckpt8";
    if (int rc = check_args(name, rows, cols, groups, format, type)) return rc;
    if (rows == 0) return MI_OK;
    if (!in || !bias || !out || !q || !scales)
        return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    if (groups > 1 && !offsets)
        return set_error(MI_ERR_INVALID_ARG, "%s: %d groups need offsets", name, groups);
    return launch_to_ckpt8<true>(name, in, bias, offsets, out, q, scales, rows, cols, groups,
                                 format, type, to_stream(stream));
}

size_t mi_gelu_backward_ckpt8_workspace(int rows, int cols, int groups) {
    if (rows <= 0 || cols <= 0 || groups <= 0) return 0;
    const int bands = plan_backward(rows, cols, groups).bands;
    return bands > 1 ? colsum_bytes(bands + groups - 1, cols) : 0;
}

int mi_gelu_backward_with_bias_backward_ckpt8(const void* q, const void* scales, const float* bias,
                                              const int* offsets, const void* grad_out,
                                              void* grad_in, void* act, float* dbias, int rows,
                                              int cols, int groups, int format, int type,
                                              void* stream) {
    const char* name = "mi_gelu_backward_with_bias_backward_ckpt8";
    if (int rc = check_args(name, rows, cols, groups, format, type)) return rc;
    if (rows == 0) return MI_OK;
    if (!q || !scales || !bias || !grad_out || !grad_in || !dbias)
        return set_error(MI_ERR_INVALID_ARG, "%s: NULL pointer", name);
    if (groups > 1 && !offsets)
        return set_error(MI_ERR_INVALID_ARG, "%s: %d groups need offsets", name, groups);
    hipStream_t st = to_stream(stream);
    const Plan p = plan_backward(rows, cols, groups);
    float* part = nullptr;
    if (p.bands > 1) {
        int err = MI_OK;
        char* ws = static_cast<char*>(
            workspace_get(mi_gelu_backward_ckpt8_workspace(rows, cols, groups), st, &err));
        if (!ws) return err;
        part = reinterpret_cast<float*>(ws + colsum_part_offset());
    }
    const double bytes = static_cast<double>(rows) * cols *
                         ((act != nullptr ? 3 : 2) * row_type_size(type) + 1);
    with_row_type(type, [&](auto t) {
        with_format(format, [&](auto f) {
            constexpr int T = decltype(t)::value, F = decltype(f)::value;
            with_flag(act != nullptr, [&](auto a) {
                with_flag(stream_loads(bytes), [&](auto nt) {
                    constexpr bool A = decltype(a)::value, NT = decltype(nt)::value;
                    hipLaunchKernelGGL((gelu_bwd_ckpt8_kernel<T, F, A, NT>), dim3(p.grid),
                                       dim3(kThreads), 0, st, cols, p.full_tiles, p.last_lanes,
                                       p.last_bands, p.band, rows, groups, offsets, bias,
                                       static_cast<const uint8_t*>(q),
                                       static_cast<const uint8_t*>(scales),
                                       static_cast<const char*>(grad_out),
                                       static_cast<char*>(grad_in), static_cast<char*>(act), part,
                                       dbias);
                });
            });
        });
    });
    if (p.bands == 1) return check_launch(name);
    if (int rc = check_launch(name)) return rc;
    const int each = p.bands / groups;  // partial rows of a group, about
    int slices = each >= 64 ? 16 : each >= 16 ? 8 : each >= 8 ? 4 : 1;
    // many waves of few rows each take their latency in several rounds: step of [16384,
    // 6400] bf16, 32 groups, 228.9 -> 225.6 us, gradient of [16384, 1600], 128 groups, 44.8
    // -> 43.5
    const long long column_waves = static_cast<long long>((cols + kWave - 1) / kWave) * groups;
    while (slices > 1 && column_waves * slices > 4096 && each < 32 * slices) slices /= 2;
    hipLaunchKernelGGL(group_sum_kernel, dim3((cols + kWave - 1) / kWave, groups),
                       dim3(slices * kWave), 0, st, part, offsets, dbias, rows, cols, p.band,
                       slices);
    return check_launch(name);
}

}  // extern "C"

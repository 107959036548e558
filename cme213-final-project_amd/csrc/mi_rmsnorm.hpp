// The RMS norm's calls with their row type as a constant: compiled in one source for each type
// (rmsnorm_f32.hip, rmsnorm_f16.hip, rmsnorm_bf16.hip), called from rmsnorm.hip.
#pragma once

#include <algorithm>

#include "mi_rowtype.hpp"

namespace mi {
namespace rms {

struct Forward {
    const void *a, *b;  // b: NULL without the residual
    const float* gamma;
    void *residual_out, *out;
    float* inv_rms;
    void* q;  // NULL: rows alone
    float* scales;
    int rows, cols;
    float eps;
    int block, format, type;
};

struct Backward {
    const void *grad_out, *x;
    const float *inv_rms, *gamma;
    void* dx;
    bool add;  // dx is added to
    int rows, cols, type;
    float* part;
};

template <int T>
void forward(const Forward& c, hipStream_t stream);
template <int T>
void backward(const Backward& c, hipStream_t stream);

inline int units_of(int cols, int type) {
    const int v = 16 / row_type_size(type);
    return (cols + v - 1) / v;
}

inline bool walked(int cols, int type, int most_units) {
    return cols < 16 / row_type_size(type) || units_of(cols, type) > most_units;
}

// Units of a thread, at most: 32 elements in the forward kernel, 24 in the backward kernel,
// whose registers hold gamma and the sums beside the row's inputs; fewer in a workgroup of 1024
// threads, which has half as many registers a thread.
constexpr int fwd_steps(int type) { return type == MI_TYPE_F32 ? 8 : 4; }
constexpr int bwd_steps(int type) { return type == MI_TYPE_F32 ? 6 : 3; }
constexpr int wide_steps(int type) { return type == MI_TYPE_F32 ? 3 : 2; }

constexpr int kBwdThreads = 512;

// Many rows whose units leave a wave's lanes idle share a wave, 16 or 32 lanes each with as many
// units as this, at most.
constexpr int kManyRows = 8192;
constexpr int kFwdNarrowSteps = 4;
constexpr int bwd_narrow_steps(int type) { return type == MI_TYPE_F32 ? 3 : 2; }

// Nine tenths of a wave's lanes have a unit in every step.
inline bool fills_wave(int units) { return units * 10 >= (units + 63) / 64 * 64 * 9; }

// Threads of a row's group in the backward kernel.  [245487, 139] fp32, 35 units: a wave 108 us, 16
// lanes 92; [88599, 342] fp16, 43 units: a wave 44.6, 32 lanes 37.5, 16 lanes 40.1; but [65536, 512]
// bf16, 64 units: a wave 45.2, 32 lanes 47.1.
inline int bwd_threads(int rows, int units, int type) {
    const int steps = bwd_steps(type);
    const int narrow = rows >= kManyRows && !fills_wave(units) ? bwd_narrow_steps(type) : 1;
    return units <= 16 * narrow ? 16 : units <= 32 * narrow ? 32 : units <= 64 * steps ? 64
           : units <= 256 * steps ? 256 : 1024;
}

// Workgroups of the backward kernel, each of which leaves a partial row: one a CU.  Rows of four
// waves take two a CU where their registers fit twice and there are rows enough to pay for twice
// the partial rows (bf16 [32768, 1600] 85.7 -> 59.4 us, [8192, 1600] 23.8 -> 20.6; but [1024, 4096]
// 12.7 -> 13.9, and fp32 rows of 4096 columns, whose four units a thread do not fit twice, 355 ->
// 375).  Rows of one wave keep one: [65536, 768] bf16 68.7, 75.0 with two.
inline int backward_blocks(int rows, int cols, int type) {
    int per = 1, most = 256;
    if (!walked(cols, type, 1024 * wide_steps(type))) {
        const int units = units_of(cols, type), threads = bwd_threads(rows, units, type);
        per = std::max(1, kBwdThreads / threads);
        const int steps = (units + threads - 1) / threads, values = 16 / row_type_size(type);
        if (threads == 256 && steps * (2 * values + 12) <= 64 && rows >= 4096) most = 512;
    } else {
        most = std::max(16, std::min(256, (1 << 25) / cols));  // 128 MB of partial rows, or 16
    }
    return static_cast<int>(
        std::min<long long>((static_cast<long long>(rows) + per - 1) / per, most));
}

}  // namespace rms
}  // namespace mi

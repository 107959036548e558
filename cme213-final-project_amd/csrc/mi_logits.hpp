// A router's logits [tokens, experts] in registers: the layout that the router's and the
// balance loss's kernels share.
#pragma once

#include <climits>
#include <type_traits>

#include "mi_rowtype.hpp"

namespace mi {

constexpr int kMaxExperts = 1024;
constexpr int kMaxChoices = 16;
constexpr float kLog2e = 1.4426950408889634f;

// A lane's logits of a row: P, in pieces of one access that it takes in turn with the row's
// other lanes.  Their experts are gl * N, N = kPiece, and the steps that step_expert gives.
template <int T, int P>
constexpr int kPiece = P < row_vec<T>() ? P : row_vec<T>();

template <int T, int L, int P>
constexpr int step_expert(int p) {
    constexpr int N = kPiece<T, P>;
    return p / N * (N * L) + p % N;
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

inline int check_gate_args(const char* name, int tokens, int experts, int k, int type) {
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

}  // namespace mi

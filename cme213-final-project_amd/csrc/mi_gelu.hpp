// tanh-approximation GELU and its derivative, shared by the element-wise
// kernels and the 8-bit checkpoint kernels.
#pragma once

#include <hip/hip_runtime.h>

namespace mi {

namespace {

// ---------------------------------------------------------------------------
// tanh-approximation GELU (Hendrycks & Gimpel 2016):
//   gelu(u) = 0.5 u (1 + tanh z),  z = sqrt(2/pi) (u + 0.044715 u^3).
// With s = 0.5 (1 + tanh z) = 1 / (1 + e^{-2z}) (logistic of 2z):
//   gelu(u)  = u s
//   gelu'(u) = s + 2 u s (1 - s) z',  z' = sqrt(2/pi) (1 + 3*0.044715 u^2)
//            = s (1 + 2 u (e s) z'),  since 1 - s = e s with e = e^{-2z}.
// Neither form has the cancellation of 1 + tanh z for very negative u.
// e^{-2z} is one v_exp_f32 (2^x) on -2 z log2(e), its exponent clamped at
// 126 so that e, s and e*s stay finite; 1 / (1 + e) is one v_rcp_f32.
// Where the exponent reaches 126 (u below about -10, and u = -inf) gelu and
// gelu' are below 1e-36 in magnitude and are returned as 0, their limit: u*s
// with the clamped s = 2^-126 would grow like u (gelu(-1e38) = -1.2) and the
// derivative like u^3.  Where e underflows to 0 (u above about 10.5, and
// u = +inf) gelu' is exactly 1 = s, and the u*(e*s)*z' term, 0 * inf for
// |u| > 1.8e19, is skipped.  NaN propagates through both.
// ---------------------------------------------------------------------------
// Folded constants: -2 z log2(e) = u * (kT0 + kT1 u^2), and
// 2 z' = kD0 + kD1 u^2.
constexpr float kT0 = -2.302208198144325f;    // -2 * sqrt(2/pi) * log2(e)
constexpr float kT1 = -0.1029432395800235f;   // -2 * sqrt(2/pi) * 0.044715 * log2(e)
constexpr float kD0 = 1.5957691216057308f;    // 2 * sqrt(2/pi)
constexpr float kD1 = 0.21406444881780076f;   // 2 * sqrt(2/pi) * 3 * 0.044715
constexpr float kTMax = 126.0f;

struct GeluTerms {
    float s;     // 1 / (1 + e^{-2z})
    float e;     // e^{-2z}, exponent clamped at kTMax
    bool zero;   // the exponent reached kTMax: gelu and gelu' are 0
};

__device__ __forceinline__ GeluTerms gelu_terms(float u, float u2) {
    const float t = u * fmaf(kT1, u2, kT0);
    const float e = __builtin_amdgcn_exp2f(fminf(t, kTMax));
    return {__builtin_amdgcn_rcpf(1.0f + e), e, t >= kTMax};
}

__device__ __forceinline__ float gelu_fwd(float u) {
    const GeluTerms g = gelu_terms(u, u * u);
    return g.zero ? 0.0f : u * g.s;
}

__device__ __forceinline__ float gelu_grad(float u) {
    const float u2 = u * u;
    const GeluTerms g = gelu_terms(u, u2);
    // s (1 + 2 u (1 - s) z') with 1 - s = e s
    const float d = g.s * fmaf(u * (g.e * g.s), fmaf(kD1, u2, kD0), 1.0f);
    return g.zero ? 0.0f : (g.e == 0.0f ? g.s : d);
}

// The same two functions where both are wanted, or where instructions count: u
// is clamped, NaN kept, instead of the exponent, so no case is set apart.  Past
// +-10 the exponent stays at +-125.97: above, s is 1 and gelu' is 1 to the last
// bit; below, gelu and gelu' come out under 1e-34 in magnitude instead of 0.
struct GeluPair {
    float y;  // gelu(u)
    float d;  // gelu'(u)
};

__device__ __forceinline__ GeluPair gelu_pair(float u) {
    const float lo = __builtin_elementwise_maximum(u, -10.0f);
    const float c = __builtin_elementwise_minimum(lo, 10.0f);
    const float c2 = c * c;
    const float e = __builtin_amdgcn_exp2f(c * fmaf(kT1, c2, kT0));
    const float s = __builtin_amdgcn_rcpf(1.0f + e);
    return {lo * s, s * fmaf(c * (e * s), fmaf(kD1, c2, kD0), 1.0f)};
}

}  // namespace

}  // namespace mi

// The gate of a gated layer: y = a(g) * u with a one of AGH_ACT_*, and the derivatives that its backward pass takes.
#pragma once
#include <limits.h>

#include "agh_internal.h"

namespace agh {

inline bool gate_known(int act) { return act >= AGH_ACT_NONE && act <= AGH_ACT_SIGMOID; }

// Results that are rounded to bf16 (FAST) take the hardware's exponential and reciprocal; for f32 the library's exponential and a division that rounds once.
// FAST: the rounding of x log2(e) makes e^x about |x| 2^-23 of its size off, 31 steps of f32 at |x| = 85, and the instructions add a few: at most 2^-11 of a step of bf16.
// Where e^-g passes f32 or its reciprocal is subnormal, g < -87, silu and sigmoid come out as 0 in place of values of less than 2^-119.
template <bool FAST>
__device__ __forceinline__ float gate_exp(float x) {
    if constexpr (FAST) return __builtin_amdgcn_exp2f(x * 1.44269504f);
    else return expf(x);
}
template <bool FAST>
__device__ __forceinline__ float gate_divide(float a, float b) {
    if constexpr (FAST) return a * __builtin_amdgcn_rcpf(b);
    else return a / b;
}

// P(Z <= g) = erfc(-g / sqrt 2) / 2, Z standard normal: through erfc, since 1 + erf would cancel where g is negative.
// FAST: erfc(x) = t e^(-x^2 + p(t)), x >= 0, t = 1 / (1 + x / 2), the form given by Press, Teukolsky, Vetterling and Flannery, Numerical Recipes, 6.2, with a polynomial of our own: p of
// degree 7, fitted to log2(e^(x^2) erfc(x) / t) for x up to 14 (7e-7 of the value in exact
// arithmetic; with x^2's rounding 4e-6 up to |g| = 6 and 2e-5 at 13, where the value is 1e-38).  The library's erfcf is three times as long: a gated product of 16384x4096x4096 903 us instead of 756.
template <bool FAST>
__device__ __forceinline__ float gate_share(float g) {
    if constexpr (!FAST) return 0.5f * erfcf(g * -0.707106781f);
    const float t = __builtin_amdgcn_rcpf(1.0f + 0.353553391f * fabsf(g));
    float p = -0.270306896f;
    p = __builtin_fmaf(p, t, 1.08222683f);
    p = __builtin_fmaf(p, t, -1.44170175f);
    p = __builtin_fmaf(p, t, 0.50364644f);
    p = __builtin_fmaf(p, t, -0.0574269161f);
    p = __builtin_fmaf(p, t, 0.568701731f);
    p = __builtin_fmaf(p, t, 1.44054569f);
    p = __builtin_fmaf(p, t, -1.82568612f);
    const float e = 0.5f * t * __builtin_amdgcn_exp2f(__builtin_fmaf(g * g, -0.72134752f, p));
    return g < 0.0f ? e : 1.0f - e;
}

// a(g)
template <bool FAST>
__device__ __forceinline__ float gate_value(float g, int act) {
    if (act == AGH_ACT_SILU) return gate_divide<FAST>(g, 1.0f + gate_exp<FAST>(-g));
    if (act == AGH_ACT_GELU) return g * gate_share<FAST>(g);
    if (act == AGH_ACT_SIGMOID) return gate_divide<FAST>(1.0f, 1.0f + gate_exp<FAST>(-g));
    if (act == AGH_ACT_RELU) return g >= 0.0f ? g : 0.0f;  // as the Relu layer has it
    return g;
}

// of N values, one look at which activation it is
template <bool FAST, int N>
__device__ __forceinline__ void gate_values(const float (&g)[N], int act, float (&value)[N]) {
    auto all = [&](int known) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < N; ++i) value[i] = gate_value<FAST>(g[i], known);
    };
    if (act == AGH_ACT_SILU) all(AGH_ACT_SILU);
    else if (act == AGH_ACT_GELU) all(AGH_ACT_GELU);
    else if (act == AGH_ACT_SIGMOID) all(AGH_ACT_SIGMOID);
    else if (act == AGH_ACT_RELU) all(AGH_ACT_RELU);
    else all(AGH_ACT_NONE);
}

// a(g) and a'(g).  The sigmoid and its complement come from one exponential of -|g|, which neither overflows nor cancels.
template <bool FAST>
__device__ __forceinline__ void gate_slope(float g, int act, float &value, float &slope) {
    if (act == AGH_ACT_SILU || act == AGH_ACT_SIGMOID) {
        const float e = gate_exp<FAST>(-fabsf(g)), large = gate_divide<FAST>(1.0f, 1.0f + e), small = e * large;
        const float s = g >= 0.0f ? large : small, rest = g >= 0.0f ? small : large;
        value = act == AGH_ACT_SILU ? g * s : s;
        slope = act == AGH_ACT_SILU ? s * (1.0f + g * rest) : s * rest;
        if (g != g) value = slope = g;
    } else if (act == AGH_ACT_GELU) {
        const float share = gate_share<FAST>(g);
        value = g * share;
        slope = share + g * (gate_exp<FAST>(-0.5f * g * g) * 0.398942280f);
    } else if (act == AGH_ACT_RELU) {
        value = g >= 0.0f ? g : 0.0f;
        slope = g >= 0.0f ? 1.0f : 0.0f;
    } else {
        value = g;
        slope = 1.0f;
    }
}

template <bool FAST, int N>
__device__ __forceinline__ void gate_slopes(const float (&g)[N], int act, float (&value)[N], float (&slope)[N]) {
    auto all = [&](int known) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < N; ++i) gate_slope<FAST>(g[i], known, value[i], slope[i]);
    };
    if (act == AGH_ACT_SILU) all(AGH_ACT_SILU);
    else if (act == AGH_ACT_GELU) all(AGH_ACT_GELU);
    else if (act == AGH_ACT_SIGMOID) all(AGH_ACT_SIGMOID);
    else if (act == AGH_ACT_RELU) all(AGH_ACT_RELU);
    else all(AGH_ACT_NONE);
}

// what a gated layer does with the product of its input and its weight [k, 2 n]; see gated_product
struct GatedOut {
    const void *bias;  // 2 n values, or null
    int64_t bias_stride;
    int act;
    void *y, *h;  // [m, n], and [m, 2 n] or null
    size_t sums;  // bytes of f32 sums that may go through the workspace: a product that needs more of it is not made, and the answer is kGatedSumsShort
};
constexpr int kGatedSumsShort = INT_MIN;  // (no error's code)
// x [m, k] times w [k, 2 n] with bias, then the gate (agh_gemm_bf16.hip, agh_gemm_f32.hip); arguments have been checked, n > 0 and m > 0
template <typename T>
int gated_product(const char *name, int64_t m, int64_t k, int64_t n, const T *x, int64_t rsx, int64_t csx, const T *w, int64_t rsw, int64_t csw, const GatedOut &out);

}  // namespace agh

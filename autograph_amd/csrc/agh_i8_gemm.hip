// Product of two 8-bit integer operands: c[i][j] = act(s_i t_j sum_x a[i][x] b[j][x] + bias[j]), with a scale for each row of a and of b, and the gated form, whose
// second operand b2 gives u beside b's g: c = act(g) * u.
//
// v_mfma_i32_16x16x64_i8 forms the sums: 64 products deep, in whole numbers, exact.  It is fed D[p][q] = sum_k P[p][k] Q[q][k] with P = b's rows and Q = a's, so that a
// lane's four results, p = 4 (l / 16) + r and q = l % 16, are neighbours in a row of c.  The result is rounded once: scales, bias and activation are applied in f32.
#include "agh_i8_rows.h"
#include "agh_i8_tile.h"

using namespace agh;
using namespace agh::i8;

namespace {

// Whether c's rows leave with the streaming hint.  Rows on whole lines of memory do.  Of others two workgroups share lines: where c stays in the caches it
// still gains, beyond them it loses, as the MXFP4 product's rows do.
template <typename T>
bool rows_stream(const T *c, int64_t rs, int64_t m, int64_t n) {
    const int64_t pitch = rs * (int64_t)sizeof(T);
    if (((uintptr_t)c | (uint64_t)pitch) % 16 != 0) return false;
    return ((uintptr_t)c | (uint64_t)pitch) % 128 == 0 || m * n * (int64_t)sizeof(T) <= (24 << 20);
}

// The kernels' tiles (p: columns of c, q: rows) and what a product takes in them, fitted to measured times in us: `start`, and for each tile that a CU takes in turn
// `tile` (half as much again for f32 results of the kernels out of LDS) + `step` for every 64 of k, but at least `least`.  Of the small tiles, straight from memory, and of the largest a
// CU's turns are its share of them; of the two in between a CU holds several, and its turns are `first` + `more` times its share.  Over 1750 products, sizes drawn at random, both types,
// operands out of several copies in turn, the form chosen takes 1.015 of the best one's time in the mean, plain and gated, and more than 1.12 of it in 4 and 3 of 100.
// (Tiles of 32x16 and 32x64 straight from memory, of 256x128 and of 128x128 with four waves instead of eight, 1999x2047x1001 12.6 / 11.2 us, are left out: with them it is 1.01 to 1.02.)
struct Form {
    int bp, bq, threads;
    double start, tile, step, least, first, more;
};
constexpr int kFormCount = 6;
constexpr Form kForms[2][kFormCount] = {{{16, 16, 512, 3.0, 0.32, 0.023, 0.34, 0, 1}, {16, 32, 512, 2.8, 0.58, 0.033, 0.59, 0, 1}, {32, 32, 256, 2.8, 0.66, 0.049, 0.73, 0, 1},
                                         {128, 64, 256, 3.7, 1.22, 0.154, 0.0, 0.43, 1.01}, {128, 128, 512, 3.8, 1.56, 0.186, 0.0, 0.34, 1.39}, {256, 256, 512, 3.2, 9.2, 0.604, 0.0, 0, 1}},
                                        {{16, 16, 512, 3.2, 0.62, 0.041, 0.21, 0, 1}, {16, 32, 512, 2.5, 1.48, 0.050, 1.02, 0, 1}, {32, 32, 256, 3.1, 0.90, 0.092, 1.02, 0, 1},
                                         {64, 64, 256, 3.0, 1.80, 0.178, 0.0, 0.56, 0.70}, {64, 128, 512, 2.9, 2.20, 0.202, 0.0, 0.59, 0.98}, {128, 256, 512, 1.8, 11.6, 0.606, 0.0, 0, 1}}};
int64_t tiles_of(const Form &o, int64_t m, int64_t n) { return ((n + o.bp - 1) / o.bp) * ((m + o.bq - 1) / o.bq); }
bool launches(const Form &o, int64_t m, int64_t n) { return tiles_of(o, m, n) <= 0xFFFFFFFFll / o.threads; }  // a launch counts its work items in 32 bits

int choose_form(bool gated, int64_t m, int64_t n, int64_t steps, size_t element) {
    int best = kFormCount - 1;
    double least = 1e30;
    for (int f = 0; f < kFormCount; ++f) {
        const Form &o = kForms[gated][f];
        if (!launches(o, m, n)) continue;
        const double share = (double)tiles_of(o, m, n) / compute_units();
        double turns = share <= 1.0 ? 1.0 : f == kFormCount - 1 ? (double)((tiles_of(o, m, n) + compute_units() - 1) / compute_units()) : o.first + o.more * share;
        if (turns < 1.0) turns = 1.0;
        const double each = o.tile * (f >= 3 && element == 4 ? 1.5 : 1.0) + o.step * (double)steps, us = o.start + turns * (each > o.least ? each : o.least);
        if (us < least) least = us, best = f;
    }
    return best;
}

// AGH_I8_FORM, an override for experiments: the number of a form that every product takes, few rows too; -1 where it is not set
int forced_form() {
    const char *s = setting("AGH_I8_FORM");
    return s && *s ? atoi(s) : -1;
}

// Whether x's rows are quantised in the product's launch, by every workgroup again (agh_i8_rows.h), instead of by a launch of its own (one / two, bf16: 1x4096x4096 5.9 /
// 9.8 us, 1x16384x4096 15.8 / 30, 4x1000x16000 6.7 / 8.3, 16x1000x2000 6.3 / 6.9, 16x4096x4096 12.0 / 10.4; f32: 1x8192x8192 15.3 / 24.3, 16x1000x2000 9.4 / 7.9).  Its codes lie
// in LDS.
constexpr int kFewRowsMostK = 16384, kFewRowsMostBytes = 32768;
bool quantises_itself(int64_t m, int64_t k, size_t element) { return m <= 4 ? k <= kFewRowsMostK : m <= 16 && m * k * (int64_t)element <= kFewRowsMostBytes; }

template <typename T>
struct Launch {
    const char *name;
    Problem p;
    const T *x;  // null, or a before its quantisation, which the kernel does itself
    int64_t rsx;
    int k;

    template <bool GATED, int TP, int TQ, int WK, int U>
    int direct() {
        p.tiles_p = (p.n + 16 * TP - 1) / (16 * TP);
        p.tiles_q = (p.m + 16 * TQ - 1) / (16 * TQ);
        if ((int64_t)p.tiles_p * p.tiles_q > 0xFFFFFFFFll / (WK * 64)) return fail(AGH_ERANGE, "%s: a result of %d x %d: too many tiles", name, p.m, p.n);
        hipLaunchKernelGGL((i8_direct_kernel<T, GATED, TP, TQ, WK, U>), dim3((unsigned)(p.tiles_p * p.tiles_q)), dim3(WK * 64), 0, stream(), p);
        AGH_LAUNCH_CHECK(name);
        return AGH_OK;
    }
    template <bool GATED, int R, int TP>
    int rows() {
        constexpr int WK = 8;
        const int pitch = rows_pitch(p.steps, WK);
        p.tiles_p = (p.n + 16 * TP - 1) / (16 * TP);
        if (p.tiles_p > (int)(0xFFFFFFFFll / (WK * 64))) return fail(AGH_ERANGE, "%s: a result of %d x %d: too many tiles", name, p.m, p.n);
        auto kern = i8_rows_kernel<T, GATED, R, TP, WK, 2>;
        const size_t bytes = (size_t)(WK * R * pitch);
        // the codes of as many rows as quantises_itself lets through, beside 32 KB of sums
        constexpr int kMostCodes = 72 * 1024;
        static_assert(WK * 4 * ((kFewRowsMostK / kStep + WK - 1) / WK * kStep + 16) <= kMostCodes, "up to four rows");
        static_assert(WK * 16 * ((kFewRowsMostBytes / 5 / (int)sizeof(T) / kStep + WK) / WK * kStep + 16) <= kMostCodes, "five rows and more, of which sixteen have room");
        if (bytes > 48 * 1024) AGH_HIP(hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, kMostCodes));
        hipLaunchKernelGGL(kern, dim3((unsigned)p.tiles_p), dim3(WK * 64), bytes, stream(), p, x, rsx, k, pitch);
        AGH_LAUNCH_CHECK(name);
        return AGH_OK;
    }
    template <bool GATED, int BP, int BQ, int WGP, int WGQ, int NS>
    int tile() {
        constexpr int BO = GATED ? BP / 2 : BP;
        p.tiles_p = (p.n + BO - 1) / BO;
        p.tiles_q = (p.m + BQ - 1) / BQ;
        if ((int64_t)p.tiles_p * p.tiles_q > 0xFFFFFFFFll / (WGP * WGQ * 64)) return fail(AGH_ERANGE, "%s: a result of %d x %d: too many tiles", name, p.m, p.n);
        hipLaunchKernelGGL((i8_tile_kernel<T, GATED, BP, BQ, WGP, WGQ, NS>), dim3((unsigned)(p.tiles_p * p.tiles_q)), dim3(WGP * WGQ * 64), 0, stream(), p);
        AGH_LAUNCH_CHECK(name);
        return AGH_OK;
    }
    template <bool GATED>
    int run() {
        const int forced = forced_form();
        if (forced >= kFormCount) return fail(AGH_EINVAL, "%s: AGH_I8_FORM=%d: no such form", name, forced);
        switch (forced >= 0 ? forced : choose_form(GATED, p.m, p.n, p.steps, sizeof(T))) {
            case 0: return direct<GATED, 1, 1, 8, 4>();
            case 1: return direct<GATED, 1, 2, 8, 4>();
            case 2: return direct<GATED, 2, 2, 4, 2>();
            case 3: return tile<GATED, 128, 64, 2, 2, 4>();
            case 4: return tile<GATED, 128, 128, 2, 4, 4>();
            default: return tile<GATED, 256, 256, 4, 2, 4>();
        }
    }
    template <bool GATED>
    int few() {
        // Two tiles a workgroup where that leaves more than one a CU: half as many quantise the rows (one tile / two, bf16: 1x4096x16384 16.0 / 13.7 us, 4x1000x16000 8.1 / 6.7;
        // 1x8192x8192 15.0 / 16.4, and gated, which is two tiles already, 1x4096x16384 28.1 / 28.5)
        if constexpr (!GATED)
            if (p.m <= 4 && p.n > 3 * 16 * compute_units()) return p.m == 1 ? rows<GATED, 1, 2>() : rows<GATED, 4, 2>();
        if (p.m == 1) return rows<GATED, 1, 1>();
        if (p.m <= 4) return rows<GATED, 4, 1>();
        return rows<GATED, 16, 1>();
    }
};

int check_operand(const char *name, const char *what, const void *codes, const void *scales) {
    if (!codes || !scales) return fail(AGH_ENULL, "%s: null codes or scales of %s", name, what);
    if (((uintptr_t)codes & 15) || ((uintptr_t)scales & 3))
        return fail(AGH_EINVAL, "%s: codes must be 16-byte and scales 4-byte aligned (%s)", name, what);
    return AGH_OK;
}

int check_product(const char *name, int64_t m, int64_t k, int64_t n, const void *c, int64_t rsc, int64_t csc, int act, bool gated) {
    if (m < 0 || k < 0 || n < 0) return fail(AGH_EINVAL, "%s: negative size (m %lld, k %lld, n %lld)", name, (long long)m, (long long)k, (long long)n);
    if (k > kMostK) return fail(AGH_ERANGE, "%s: k %lld: the sums of more than %lld products of codes do not fit 32 bits", name, (long long)k, (long long)kMostK);
    if (!rows_fit(m, k) || !rows_fit(n, k)) return fail(AGH_ERANGE, "%s: m %lld, k %lld, n %lld: too large", name, (long long)m, (long long)k, (long long)n);
    if (gated ? !gate_known(act) : act != AGH_ACT_NONE && act != AGH_ACT_RELU) return fail(AGH_EINVAL, "%s: unknown activation %d", name, act);
    if (m == 0 || n == 0) return AGH_OK;
    if (!c) return fail(AGH_ENULL, "%s: null output", name);
    if ((m > 1 && rsc == 0) || (n > 1 && csc == 0)) return fail(AGH_EINVAL, "%s: the elements of c must be distinct addresses", name);
    return AGH_OK;
}

// what the entry points have in common: a is given in codes, or as x, which is quantised here
template <typename T, bool GATED>
int product(const char *name, int64_t m, int64_t k, int64_t n, const void *a_codes, const void *a_scales, const T *x, int64_t rsx, int64_t csx, const void *b_codes,
            const void *b_scales, const void *b2_codes, const void *b2_scales, T *c, int64_t rsc, int64_t csc, const T *bias, const T *bias2, int64_t bias_stride, int act) {
    Launch<T> l = {name, {}, nullptr, 0, (int)k};
    Problem &p = l.p;
    if (k > 0) {
        if (int rc = check_operand(name, GATED ? "gate" : "b", b_codes, b_scales)) return rc;
        if constexpr (GATED)
            if (int rc = check_operand(name, "up", b2_codes, b2_scales)) return rc;
        if (x) {
            if (csx == 1 && forced_form() < 0 && quantises_itself(m, k, sizeof(T))) {
                // few rows: quantised by every workgroup for itself, in one launch
                l.x = x;
                l.rsx = rsx;
            } else {
                void *codes;
                const size_t bytes = codes_bytes(m, k);
                if (int rc = workspace(bytes + scales_bytes(m) + scratch_bytes<T>(m, k, csx), &codes)) return rc;
                float *scales = (float *)((unsigned char *)codes + bytes);
                if (int rc = quantize_launch<T>(name, x, rsx, csx, m, k, codes, scales, scales + m)) return rc;
                a_codes = codes;
                a_scales = scales;
            }
        } else if (int rc = check_operand(name, "a", a_codes, a_scales)) return rc;
        p.a = (const unsigned char *)a_codes;
        p.b = (const unsigned char *)b_codes;
        p.b2 = (const unsigned char *)b2_codes;
        p.sa = (const float *)a_scales;
        p.sb = (const float *)b_scales;
        p.sb2 = (const float *)b2_scales;
    }
    p.c = c;
    p.rsc = rsc;
    p.csc = csc;
    p.bias = bias;
    p.bias2 = bias2;
    p.bias_stride = bias_stride;
    p.m = (int)m;
    p.n = (int)n;
    p.steps = (int)steps_of(k);
    p.act = act;
    p.streamed = rows_stream(c, rsc, m, n);
    return l.x ? l.template few<GATED>() : l.template run<GATED>();
}

template <typename T>
int gemm_entry(const char *name, int64_t m, int64_t k, int64_t n, const void *a_codes, const void *a_scales, const void *b_codes, const void *b_scales,
               void *c, int64_t off_c, int64_t rsc, int64_t csc, const void *bias, int64_t off_bias, int64_t bias_stride, int act) {
    if (int rc = check_product(name, m, k, n, c, rsc, csc, act, false)) return rc;
    if (m == 0 || n == 0) return AGH_OK;
    return product<T, false>(name, m, k, n, a_codes, a_scales, nullptr, 0, 0, b_codes, b_scales, nullptr, nullptr, (T *)c + off_c, rsc, csc,
                             bias ? (const T *)bias + off_bias : nullptr, nullptr, bias_stride, act);
}

template <typename T>
int dense_entry(const char *name, int64_t m, int64_t k, int64_t n, const void *x, int64_t off_x, int64_t rsx, int64_t csx, const void *w_codes,
                const void *w_scales, void *c, int64_t off_c, int64_t rsc, int64_t csc, const void *bias, int64_t off_bias, int64_t bias_stride, int act) {
    if (int rc = check_product(name, m, k, n, c, rsc, csc, act, false)) return rc;
    if (m == 0 || n == 0) return AGH_OK;
    if (k > 0 && !x) return fail(AGH_ENULL, "%s: null input", name);
    return product<T, false>(name, m, k, n, nullptr, nullptr, (const T *)x + off_x, rsx, csx, w_codes, w_scales, nullptr, nullptr, (T *)c + off_c, rsc, csc,
                             bias ? (const T *)bias + off_bias : nullptr, nullptr, bias_stride, act);
}

template <typename T>
int gated_entry(const char *name, int64_t m, int64_t k, int64_t n, const void *x, int64_t off_x, int64_t rsx, int64_t csx, const void *gate_codes,
                const void *gate_scales, const void *up_codes, const void *up_scales, void *c, int64_t off_c, int64_t rsc, int64_t csc, const void *bias,
                int64_t off_bias, int64_t bias_stride, int act) {
    if (int rc = check_product(name, m, k, n, c, rsc, csc, act, true)) return rc;
    if (m == 0 || n == 0) return AGH_OK;
    if (k > 0 && !x) return fail(AGH_ENULL, "%s: null input", name);
    const T *b = bias ? (const T *)bias + off_bias : nullptr;
    return product<T, true>(name, m, k, n, nullptr, nullptr, (const T *)x + off_x, rsx, csx, gate_codes, gate_scales, up_codes, up_scales, (T *)c + off_c, rsc, csc,
                            b, b ? b + n * bias_stride : nullptr, bias_stride, act);
}

}  // namespace

extern "C" {

#define AGH_I8_GEMM(SUFFIX, T)                                                                                                                  \
    int agh_gemm_int8_##SUFFIX(int64_t m, int64_t k, int64_t n, const void *a_codes, const void *a_scales, const void *b_codes,                 \
                               const void *b_scales, void *c, int64_t off_c, int64_t rsc, int64_t csc, const void *bias, int64_t off_bias,      \
                               int64_t bias_stride, int act) {                                                                                  \
        AGH_API_ENTER();                                                                                                                        \
        return gemm_entry<T>("agh_gemm_int8_" #SUFFIX, m, k, n, a_codes, a_scales, b_codes, b_scales, c, off_c, rsc, csc, bias, off_bias,       \
                             bias_stride, act);                                                                                                 \
    }                                                                                                                                           \
    int agh_dense_int8_##SUFFIX(int64_t m, int64_t k, int64_t n, const void *x, int64_t off_x, int64_t rsx, int64_t csx, const void *w_codes,   \
                                const void *w_scales, void *c, int64_t off_c, int64_t rsc, int64_t csc, const void *bias, int64_t off_bias,     \
                                int64_t bias_stride, int act) {                                                                                 \
        AGH_API_ENTER();                                                                                                                        \
        return dense_entry<T>("agh_dense_int8_" #SUFFIX, m, k, n, x, off_x, rsx, csx, w_codes, w_scales, c, off_c, rsc, csc, bias, off_bias,    \
                              bias_stride, act);                                                                                                \
    }                                                                                                                                           \
    int agh_gated_dense_int8_##SUFFIX(int64_t m, int64_t k, int64_t n, const void *x, int64_t off_x, int64_t rsx, int64_t csx,                  \
                                      const void *gate_codes, const void *gate_scales, const void *up_codes, const void *up_scales, void *c,    \
                                      int64_t off_c, int64_t rsc, int64_t csc, const void *bias, int64_t off_bias, int64_t bias_stride,         \
                                      int act) {                                                                                                \
        AGH_API_ENTER();                                                                                                                        \
        return gated_entry<T>("agh_gated_dense_int8_" #SUFFIX, m, k, n, x, off_x, rsx, csx, gate_codes, gate_scales, up_codes, up_scales, c,    \
                              off_c, rsc, csc, bias, off_bias, bias_stride, act);                                                               \
    }
AGH_I8_GEMM(f32, float)
AGH_I8_GEMM(bf16, uint16_t)

}  // extern "C"

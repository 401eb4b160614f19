// Product of two MXFP4 operands: c[i][j] = relu(sum_b 2^(sa[i][b] + sb[j][b]) * sum over the block of a * b + bias[j]), b over blocks of 32 along k.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 forms it: 128 products deep, each lane's 32 values with a scale of their own, sums in f32.  It is
// fed D[p][q] = sum_k P[p][k] Q[q][k] with P = b's rows and Q = a's, so that a lane's four results, p = 4 (l / 16) + r and q = l % 16, are
// neighbours in a row of c.
// The result is rounded once: bias and relu are applied in f32.  (agh_gemm_bf16_bias_act rounds between them, as the layers it fuses do.)
#include "agh_mx_direct.h"

using namespace agh;
using namespace agh::mx;

namespace {

// The kernels' tiles (p: columns of c, q: rows) and what a product takes in them, fitted to measured times in us: `start`, and for each tile that a CU takes in turn
// `tile` (half as much again for f32 results of the large tiles, which they are bound by) + `step` for every 128 of k, but at least `least` (fetching the kernel's code,
// storing the result).  Over 520 products, sizes drawn at random, both types, no operand in a cache from the call before, the form chosen takes 1.02 of the best one's
// time in the mean, and more than 1.12 of it in 4 of 100.  (128x128 tiles with k split between two halves of a workgroup took 11.5 instead of 12.4 us at 2048x4096x1000
// and lost where k is short; 64x64 tiles, straight from memory, are never the best of these. Neither is taken.)
struct Form {
    int bp, bq, threads;
    double start, tile, step, least;
};
constexpr Form kForms[] = {{16, 16, 512, 2.5, 0.2, 0.034, 0.4},   {32, 16, 512, 2.5, 0.2, 0.064, 0.5},   {16, 32, 512, 3.1, 0.13, 0.042, 0.73},
                           {32, 32, 256, 2.5, 0.2, 0.071, 0.48},  {32, 64, 256, 3.6, 0.65, 0.077, 1.25}, {128, 128, 256, 4.0, 1.6, 0.19, 0.0},
                           {256, 256, 512, 2.8, 5.9, 0.54, 0.0}};
constexpr int kFormCount = sizeof(kForms) / sizeof(kForms[0]);
int64_t tiles_of(const Form &o, int64_t m, int64_t n) { return ((n + o.bp - 1) / o.bp) * ((m + o.bq - 1) / o.bq); }
bool launches(const Form &o, int64_t m, int64_t n) { return tiles_of(o, m, n) <= 0xFFFFFFFFll / o.threads; }  // a launch counts its work items in 32 bits

// Whether Dense's input is quantised in the product's launch, by every workgroup again, instead of by a launch of its own, about 3 us and as much of the host's time.  What it
// costs a CU for every 128 of k, fitted in us to the difference: the conversion, and its rows' bytes at 50 bytes a ns (one launch / two, bf16: 1x4096x4096 4.6 / 6.2 us, 64x256x256
// 3.5 / 5.7, 100x1000x300 4.8 / 5.6, 16x4096x32000 23.3 / 16.0, 200x2000x100 6.8 / 5.8; f32: 1x4096x32000 17.9 / 16.0, 16x4096x32000 40 / 17.2).
bool quantises_itself(const Form &o, int64_t m, int64_t n, int64_t steps, size_t element) {
    if (o.bq != 16 && !(o.bp == 32 && o.bq == 32)) return false;
    const double tiles = (double)tiles_of(o, m, n), cus = compute_units(), turns = tiles > cus ? tiles / cus : 1.0;
    const double bytes = (double)((m < o.bq ? m : o.bq) * kStep * (int64_t)element);
    return turns * (double)steps * ((element == 4 ? 0.037 : 0.02) + bytes * 2e-5) < 3.2;
}

// The same for Dense as for the product, whose bits it gives.
int choose_form(int64_t m, int64_t n, int64_t steps, size_t element) {
    int best = kFormCount - 1;
    double least = 1e30;
    for (int f = 0; f < kFormCount; ++f) {
        const Form &o = kForms[f];
        // (up to 16 rows: the 32 of the others would be half empty, and Dense would need a second launch)
        if ((o.bp < 128 && (o.bq == 16) != (m <= 16)) || !launches(o, m, n)) continue;
        const double tiles = (double)tiles_of(o, m, n), cus = compute_units();
        // the tiled kernels' workgroups fill a CU, one or two at a time; many small ones share it evenly
        const bool large = o.bp >= 128;
        const double turns = large ? (double)(int64_t)((tiles + cus - 1) / cus) : tiles > cus ? tiles / cus : 1.0;
        const double each = o.tile * (large && element == 4 ? 1.5 : 1.0) + o.step * (double)steps, us = o.start + turns * (each > o.least ? each : o.least);
        if (us < least) least = us, best = f;
    }
    return best;
}

// Whether c's rows leave with the streaming hint.  Rows on whole lines of memory do (bf16 2048^3 9.1 -> 8.5 us, 16384x4096x4096 127.8 -> 125.4).  Of others two
// workgroups share lines: where c stays in the caches it still gains (f32 2048x2048x2056, 17 MB, 13.8 -> 12.7), beyond them it
// loses (34 MB, bf16 8192x640x2056 18.0 -> 20.4; 169 MB, f32 3616x26x11660 35.5 -> 61.5).
template <typename T>
bool rows_stream(const T *c, int64_t rs, int64_t m, int64_t n) {
    const int64_t pitch = rs * (int64_t)sizeof(T);
    if (((uintptr_t)c | (uint64_t)pitch) % 16 != 0) return false;
    return ((uintptr_t)c | (uint64_t)pitch) % 128 == 0 || m * n * (int64_t)sizeof(T) <= (24 << 20);
}

template <typename T>
struct Launch {
    const char *name;
    Problem p;
    const T *x;  // null, or a before its quantisation, which the kernel does itself
    int64_t rsx;
    int k;

    int grid(int form, unsigned &blocks) {
        const Form &o = kForms[form];
        p.tiles_p = (p.n + o.bp - 1) / o.bp;
        p.tiles_q = (p.m + o.bq - 1) / o.bq;
        if (!launches(o, p.m, p.n)) return fail(AGH_ERANGE, "%s: a result of %d x %d: too many tiles", name, p.m, p.n);
        blocks = (unsigned)(p.tiles_p * p.tiles_q);
        return AGH_OK;
    }
    template <bool RAW, int TP, int TQ, int WK, int U>
    void direct(unsigned blocks) const {
        hipLaunchKernelGGL((mx_direct_kernel<T, RAW, TP, TQ, WK, U>), dim3(blocks), dim3(WK * 64), 0, stream(), p, x, rsx, k);
    }
    int run(int form) {
        unsigned blocks;
        if (int rc = grid(form, blocks)) return rc;
        switch (form) {
            case 0: x ? direct<true, 1, 1, 8, 2>(blocks) : direct<false, 1, 1, 8, 4>(blocks); break;
            case 1: x ? direct<true, 2, 1, 8, 2>(blocks) : direct<false, 2, 1, 8, 4>(blocks); break;
            case 2: direct<false, 1, 2, 8, 4>(blocks); break;
            case 3: x ? direct<true, 2, 2, 4, 1>(blocks) : direct<false, 2, 2, 4, 2>(blocks); break;
            case 4: direct<false, 2, 4, 4, 2>(blocks); break;
            case 5: hipLaunchKernelGGL((mx_tile_kernel<T, 128, 128, 2, 2, 4>), dim3(blocks), dim3(256), 0, stream(), p); break;
            default: hipLaunchKernelGGL((mx_tile_kernel<T, 256, 256, 4, 2, 4>), dim3(blocks), dim3(512), 0, stream(), p); break;
        }
        AGH_LAUNCH_CHECK(name);
        return AGH_OK;
    }
};

int check_operand(const char *name, const char *what, const void *codes, const void *scales) {
    if (!codes || !scales) return fail(AGH_ENULL, "%s: null codes or scales of %s", name, what);
    if (((uintptr_t)codes & 15) || ((uintptr_t)scales & 3))
        return fail(AGH_EINVAL, "%s: codes must be 16-byte and scales 4-byte aligned (%s)", name, what);
    return AGH_OK;
}

int check_product(const char *name, int64_t m, int64_t k, int64_t n, const void *c, int64_t rsc, int64_t csc, int act) {
    if (m < 0 || k < 0 || n < 0) return fail(AGH_EINVAL, "%s: negative size (m %lld, k %lld, n %lld)", name, (long long)m, (long long)k, (long long)n);
    if (!sizes_fit(m, k) || !sizes_fit(n, k)) return fail(AGH_ERANGE, "%s: m %lld, k %lld, n %lld: too large", name, (long long)m, (long long)k, (long long)n);
    if (act != AGH_ACT_NONE && act != AGH_ACT_RELU) return fail(AGH_EINVAL, "%s: unknown activation %d", name, act);
    if (m == 0 || n == 0) return AGH_OK;
    if (!c) return fail(AGH_ENULL, "%s: null output", name);
    if ((m > 1 && rsc == 0) || (n > 1 && csc == 0)) return fail(AGH_EINVAL, "%s: the elements of c must be distinct addresses", name);
    return AGH_OK;
}

template <typename T>
int gemm_entry(const char *name, int64_t m, int64_t k, int64_t n, const void *a_codes, const void *a_scales, const void *b_codes, const void *b_scales,
               void *c, int64_t off_c, int64_t rsc, int64_t csc, const void *bias, int64_t off_bias, int64_t bias_stride, int act) {
    if (int rc = check_product(name, m, k, n, c, rsc, csc, act)) return rc;
    if (m == 0 || n == 0) return AGH_OK;
    if (k > 0) {
        if (int rc = check_operand(name, "a", a_codes, a_scales)) return rc;
        if (int rc = check_operand(name, "b", b_codes, b_scales)) return rc;
    }
    const int64_t steps = steps_of(k);
    Launch<T> l = {name, {(const unsigned char *)a_codes, (const unsigned char *)a_scales, (const unsigned char *)b_codes, (const unsigned char *)b_scales,
                          (T *)c + off_c, rsc, csc, bias ? (const T *)bias + off_bias : nullptr, bias_stride, (int)m, (int)n, (int)steps, act,
                          rows_stream<T>((T *)c + off_c, rsc, m, n), 0, 0}, nullptr, 0, 0};
    return l.run(choose_form(m, n, steps, sizeof(T)));
}

template <typename T>
int dense_entry(const char *name, int64_t m, int64_t k, int64_t n, const void *x, int64_t off_x, int64_t rsx, int64_t csx, const void *w_codes,
                const void *w_scales, void *c, int64_t off_c, int64_t rsc, int64_t csc, const void *bias, int64_t off_bias, int64_t bias_stride, int act) {
    if (int rc = check_product(name, m, k, n, c, rsc, csc, act)) return rc;
    if (m == 0 || n == 0) return AGH_OK;
    void *codes = nullptr, *scales = nullptr;
    if (k > 0) {
        if (!x) return fail(AGH_ENULL, "%s: null input", name);
        if (int rc = check_operand(name, "w", w_codes, w_scales)) return rc;
        const int64_t steps = steps_of(k);
        const int form = choose_form(m, n, steps, sizeof(T));
        if (csx == 1 && quantises_itself(kForms[form], m, n, steps, sizeof(T))) {
            // few rows: quantised by every workgroup for itself, in one launch
            Launch<T> l = {name, {nullptr, nullptr, (const unsigned char *)w_codes, (const unsigned char *)w_scales, (T *)c + off_c, rsc, csc,
                                  bias ? (const T *)bias + off_bias : nullptr, bias_stride, (int)m, (int)n, (int)steps, act, false, 0, 0}, (const T *)x + off_x, rsx, (int)k};
            return l.run(form);
        }
        const size_t bytes = codes_bytes(m, k);
        if (int rc = workspace(bytes + scales_bytes(m, k), &codes)) return rc;
        scales = (unsigned char *)codes + bytes;
        if (int rc = quantize_launch<T>(name, (const T *)x + off_x, rsx, csx, m, k, codes, scales)) return rc;
    }
    return gemm_entry<T>(name, m, k, n, codes, scales, w_codes, w_scales, c, off_c, rsc, csc, bias, off_bias, bias_stride, act);
}

}  // namespace

extern "C" {

#define AGH_MX_GEMM(SUFFIX, T)                                                                                                                  \
    int agh_gemm_mxfp4_##SUFFIX(int64_t m, int64_t k, int64_t n, const void *a_codes, const void *a_scales, const void *b_codes,                \
                                const void *b_scales, void *c, int64_t off_c, int64_t rsc, int64_t csc, const void *bias, int64_t off_bias,     \
                                int64_t bias_stride, int act) {                                                                                 \
        AGH_API_ENTER();                                                                                                                        \
        return gemm_entry<T>("agh_gemm_mxfp4_" #SUFFIX, m, k, n, a_codes, a_scales, b_codes, b_scales, c, off_c, rsc, csc, bias, off_bias,      \
                             bias_stride, act);                                                                                                 \
    }                                                                                                                                           \
    int agh_dense_mxfp4_##SUFFIX(int64_t m, int64_t k, int64_t n, const void *x, int64_t off_x, int64_t rsx, int64_t csx, const void *w_codes,  \
                                 const void *w_scales, void *c, int64_t off_c, int64_t rsc, int64_t csc, const void *bias, int64_t off_bias,    \
                                 int64_t bias_stride, int act) {                                                                                \
        AGH_API_ENTER();                                                                                                                        \
        return dense_entry<T>("agh_dense_mxfp4_" #SUFFIX, m, k, n, x, off_x, rsx, csx, w_codes, w_scales, c, off_c, rsc, csc, bias, off_bias,   \
                              bias_stride, act);                                                                                                \
    }
AGH_MX_GEMM(f32, float)
AGH_MX_GEMM(bf16, uint16_t)

}  // extern "C"

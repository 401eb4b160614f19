// Product of two MXFP4 operands: c[i][j] = relu(sum_b 2^(sa[i][b] + sb[j][b]) * sum over the block of a * b + bias[j]), b over blocks of 32 along k.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 forms it: 128 products deep, each lane's 32 values with a scale of their own, sums in f32.  It is
// fed D[p][q] = sum_k P[p][k] Q[q][k] with P = b's rows and Q = a's, so that a lane's four results, p = 4 (l / 16) + r and q = l % 16, are
// neighbours in a row of c.
// The result is rounded once: bias and relu are applied in f32.  (agh_gemm_bf16_bias_act rounds between them, as the layers it fuses do.)
#include "agh_mx.h"

using namespace agh;
using namespace agh::mx;

namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

struct Problem {
    const unsigned char *a, *sa, *b, *sb;  // codes and scales: a of m rows, b of n rows
    void *c;
    int64_t rsc, csc;  // of c, elements
    const void *bias;  // or null
    int64_t bias_stride;
    int m, n, steps, act;
};

__device__ __forceinline__ i32x8_t widen(u32x4_t v) { return i32x8_t{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; }

// both operands fp4 (format 4); S: which byte of the scale registers
template <int SP, int SQ>
__device__ __forceinline__ f32x4_t mfma(u32x4_t p, u32x4_t q, f32x4_t acc, uint32_t sp, uint32_t sq) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(p), widen(q), acc, 4, 4, SP, (int)sp, SQ, (int)sq);
}

template <typename T>
__device__ __forceinline__ T finish(float v, float bias, int act) {
    v += bias;
    if (act == AGH_ACT_RELU && !(v >= 0.0f)) v = 0.0f;  // x >= 0 ? x : 0, as the Relu layer has it
    return Elem<T>::from_f32(v);
}

// four results of a lane: columns j .. j+3 of row i
template <typename T>
__device__ __forceinline__ void store4(const Problem &p, f32x4_t v, int i, int j) {
    if (i >= p.m) return;
    T *c = (T *)p.c + i * p.rsc;
    const T *bias = (const T *)p.bias;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (j + r < p.n) c[(j + r) * p.csc] = finish<T>(v[r], bias ? Elem<T>::raw(bias[(j + r) * p.bias_stride]) : 0.0f, p.act);
}

// Straight from memory: a wave forms 64x64 of c, a workgroup of 2x2 waves 128x128.
template <typename T>
__global__ __launch_bounds__(256) void mx_direct_kernel(Problem p) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int p0 = (blockIdx.x * 2 + (wave & 1)) * 64, q0 = (blockIdx.y * 2 + (wave >> 1)) * 64;
    if (p0 >= p.n || q0 >= p.m) return;
    const int last_p = (p.n - 1) / 16, last_q = (p.m - 1) / 16;
    const u32x4_t *fp[4], *fq[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        fp[i] = (const u32x4_t *)(p.b + (int64_t)min(p0 / 16 + i, last_p) * p.steps * kFragBytes) + lane;
        fq[i] = (const u32x4_t *)(p.a + (int64_t)min(q0 / 16 + i, last_q) * p.steps * kFragBytes) + lane;
    }
    const uint32_t *sp = (const uint32_t *)(p.sb + (int64_t)(p0 / 64) * p.steps * kPieceBytes) + lane;
    const uint32_t *sq = (const uint32_t *)(p.sa + (int64_t)(q0 / 64) * p.steps * kPieceBytes) + lane;
    f32x4_t acc[4][4] = {};
    for (int s = 0; s < p.steps; ++s) {
        u32x4_t vp[4], vq[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) vp[i] = fp[i][s * 64], vq[i] = fq[i][s * 64];
        const uint32_t xp = sp[s * 64], xq = sq[s * 64];
#define AGH_MX_ROW(I)                                          \
    acc[I][0] = mfma<I, 0>(vp[I], vq[0], acc[I][0], xp, xq);   \
    acc[I][1] = mfma<I, 1>(vp[I], vq[1], acc[I][1], xp, xq);   \
    acc[I][2] = mfma<I, 2>(vp[I], vq[2], acc[I][2], xp, xq);   \
    acc[I][3] = mfma<I, 3>(vp[I], vq[3], acc[I][3], xp, xq);
        AGH_MX_ROW(0) AGH_MX_ROW(1) AGH_MX_ROW(2) AGH_MX_ROW(3)
#undef AGH_MX_ROW
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) store4<T>(p, acc[i][j], q0 + j * 16 + (lane & 15), p0 + i * 16 + (lane >> 4) * 4);
}

template <typename T>
int product_launch(const char *name, const Problem &p) {
    const int64_t gp = ((int64_t)p.n + 127) / 128, gq = ((int64_t)p.m + 127) / 128;
    if (gq > 65535) return fail(AGH_ERANGE, "%s: %d rows: too many", name, p.m);
    hipLaunchKernelGGL(mx_direct_kernel<T>, dim3((unsigned)gp, (unsigned)gq), dim3(256), 0, stream(), p);
    AGH_LAUNCH_CHECK(name);
    return AGH_OK;
}

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
    const Problem p = {(const unsigned char *)a_codes, (const unsigned char *)a_scales, (const unsigned char *)b_codes, (const unsigned char *)b_scales,
                       (T *)c + off_c, rsc, csc, bias ? (const T *)bias + off_bias : nullptr, bias_stride, (int)m, (int)n, (int)steps_of(k), act};
    return product_launch<T>(name, p);
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

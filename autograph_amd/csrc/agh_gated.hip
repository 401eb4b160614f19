// The gated layer: y = a(x Wg + bg) * (x Wu + bu), and its backward pass.  The products are the GEMM kernels'.
//
// Backward, from the pre-activations h = (g | u) that the forward pass kept: dg = dy u a'(g), du = dy a(g), dh = (dg | du); then dx = dh W^T, dW = x^T dh as two
// products, and db the sum of dh's rows.  dh is rounded to T for the products, which take their operands in that type, as the layers' gradients are; db is summed in f32
// from the values before that rounding, in an order that depends on the sizes alone.
#include <algorithm>

#include "agh_gated_kernel.h"
#include "agh_gated_rows.h"

using namespace agh;

namespace {

constexpr int kThreads = 256;

// A workgroup takes a strip of 64 VE columns and a share of the rows, its W waves every W-th of them; a lane VE neighbouring columns of both halves, U rows at a time
// so that their loads are in flight together.  Its share of db goes to shares[blockIdx.y][2 n]; of few rows, whose share is the whole, to db.
// Bounded by memory, three values in and two out an output: with the shares' sum bf16 4096x4096 32 us, 5.2 TB/s.
template <typename T, int U, int W>
__global__ __launch_bounds__(W * 64) void gated_backward_kernel(const T *h, const T *__restrict__ dy, int m, int n, int rows, int act, T *dh, float *__restrict__ shares,
                                                                  T *__restrict__ db) {
    constexpr int VE = Group<T>::VE;
    __shared__ float sums[W][2][VE][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int p = ((int)blockIdx.x * 64 + lane) * VE, at = min(p, n - VE);
    const bool live = p < n, whole = p + VE <= n;
    float sg[VE] = {}, su[VE] = {};
    const int64_t first = (int64_t)blockIdx.y * rows, last = first + rows < m ? first + rows : m;
    if (live)
        for (int64_t q0 = first + wave; q0 < last; q0 += U * W) {
            u32x4_t vg[U], vu[U], vd[U];
            if (n >= VE) {
                // a group that would pass the last column is read from where it would end there, and shifted behind all the loads: none of them waits for another
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int64_t q = min(q0 + i * W, last - 1);
                    vg[i] = *(const typename Group<T>::vec *)(h + q * 2 * n + at);
                    vu[i] = *(const typename Group<T>::vec *)(h + q * 2 * n + n + at);
                    vd[i] = *(const typename Group<T>::vec *)(dy + q * n + at);
                }
                if (p != at)
#pragma unroll
                    for (int i = 0; i < U; ++i) {
                        vg[i] = Group<T>::shifted(vg[i], p - at);
                        vu[i] = Group<T>::shifted(vu[i], p - at);
                        vd[i] = Group<T>::shifted(vd[i], p - at);
                    }
            } else
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int64_t q = min(q0 + i * W, last - 1);
                    vg[i] = Group<T>::load(h + q * 2 * n, p, n);
                    vu[i] = Group<T>::load(h + q * 2 * n + n, p, n);
                    vd[i] = Group<T>::load(dy + q * n, p, n);
                }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int64_t q = q0 + i * W;
                if (q >= last) break;
                float dg[VE], du[VE], gate[VE];
#pragma unroll
                for (int e = 0; e < VE; ++e) gate[e] = Group<T>::get(vg[i], e);
                gate_slopes<sizeof(T) == 2, VE>(gate, act, du, dg);
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float d = Group<T>::get(vd[i], e);
                    dg[e] = d * dg[e] * Group<T>::get(vu[i], e);  // (the slope first: d u alone may pass f32 where it is 0 or small)
                    du[e] = d * du[e];
                    sg[e] += dg[e];
                    su[e] += du[e];
                }
                T *to = dh + q * 2 * n + p;
                const u32x4_t a = Group<T>::pack(dg), b = Group<T>::pack(du);
                if (whole) {
                    *(typename Group<T>::vec *)to = a;
                    *(typename Group<T>::vec *)(to + n) = b;
                } else {
                    typename Group<T>::Bits ba, bb;
                    ba.q = a;
                    bb.q = b;
#pragma unroll
                    for (int e = 0; e < VE - 1; ++e)
                        if (p + e < n) {
                            to[e] = ba.e[e];
                            to[n + e] = bb.e[e];
                        }
                }
            }
        }
    if (!shares && !db) return;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
        sums[wave][0][e][lane] = sg[e];
        sums[wave][1][e][lane] = su[e];
    }
    __syncthreads();
    const int64_t p0 = (int64_t)blockIdx.x * 64 * VE;
    const int count = min(64 * VE, n - (int)blockIdx.x * 64 * VE);
    for (int v = threadIdx.x; v < 2 * 64 * VE; v += W * 64) {
        const int half = v / (64 * VE), c = v % (64 * VE);
        if (c >= count) continue;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) s += sums[w][half][c % VE][c / VE];
        if (db) db[p0 + (int64_t)half * n + c] = Elem<T>::from_f32(s);
        else shares[(int64_t)blockIdx.y * 2 * n + p0 + (int64_t)half * n + c] = s;
    }
}

// db from the shares, which a workgroup adds for 16 columns: 16 threads a column, each every 16th share, and their sums in order
__global__ __launch_bounds__(kThreads) void gated_bias_kernel(const float *__restrict__ shares, int count, int columns, void *__restrict__ db, bool bf16) {
    __shared__ float sums[16][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4, p = (int)blockIdx.x * 16 + c;
    float s = 0.0f;
    if (p < columns)
#pragma unroll 4
        for (int i = r; i < count; i += 16) s += shares[(int64_t)i * columns + p];
    sums[r][c] = s;
    __syncthreads();
    if (r != 0 || p >= columns) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) s += sums[i][c];
    if (bf16) ((uint16_t *)db)[p] = f32_to_bf16(s);
    else ((float *)db)[p] = s;
}

constexpr int64_t kMost = ((int64_t)1 << 31) - 512;

int check_sizes(const char *name, int64_t m, int64_t k, int64_t n, int act) {
    if (m < 0 || k < 0 || n < 0) return fail(AGH_EINVAL, "%s: negative size (m %lld, k %lld, n %lld)", name, (long long)m, (long long)k, (long long)n);
    if (m > kMost || k > kMost || n > kMost / 2) return fail(AGH_ERANGE, "%s: m %lld, k %lld, n %lld: too large", name, (long long)m, (long long)k, (long long)n);
    if (!gate_known(act)) return fail(AGH_EINVAL, "%s: unknown activation %d", name, act);
    return AGH_OK;
}

// How few rows are taken: groups of a strip, splits of k; no groups: not at all.  bf16, one split of the GEMM kernels' tiles or their splits and the join / here, 1 row in us: 1024x1024
// 5.9 / 4.7, 64x16384 6.9 / 4.4, 1000x16000 22 / 13.3, 16384x64 23 / 12.3; but 4096x1000 10 / 11.3, 2048x4096 10.8 / 11.9, 4096x8192 31.1 / 32.3.  f32: 1024x1024 10.5 / 6.9,
// 4096x1000 17.8 / 12.3, 4096x8192 80 / 50, 16384x64 43 / 12.8.  From 3 rows on in bf16, 5 in f32, the vector units are behind (8 rows, 1024x1024: bf16 6.0 / 13, f32 11.2 / 12.6).
struct FewPlan { int groups, splits; };
template <typename T>
FewPlan few_plan(int64_t m, int64_t k, int64_t n) {
    constexpr bool f32 = sizeof(T) == 4;
    if (m > (f32 ? 4 : 2) || n < Group<T>::VE || k == 0) return {0, 0};
    if (k <= 1024) return {n > 8192 ? (f32 ? 16 : 8) : 4, 1};
    if (f32) return n >= 4096 ? FewPlan{16, 4} : FewPlan{8, (int)std::max<int64_t>(2, std::min<int64_t>(8, k / 1024))};
    return n <= 512 ? FewPlan{8, (int)std::min<int64_t>(16, k / 1024)} : FewPlan{0, 0};
}

template <typename T>
int rows_launch(const char *name, GatedFew<T> g, const FewPlan &plan) {
    const int strip = plan.groups * Group<T>::VE;
    const unsigned strips = (unsigned)((g.n + strip - 1) / strip);
    if (strips > 0xFFFFFFFFu / 512 / (unsigned)plan.splits) return fail(AGH_ERANGE, "%s: %d columns: too many", name, g.n);
    if (plan.splits > 1) {
        void *ws = nullptr;
        if (int rc = workspace((size_t)plan.splits * g.m * 2 * g.n * sizeof(float), &ws)) return rc;
        g.ws = (float *)ws;
    }
    auto launch = [&](auto mc) {
        constexpr int M = decltype(mc)::value;
        const dim3 grid(strips, (unsigned)plan.splits);
        if (plan.groups == 4) hipLaunchKernelGGL((gated_rows_kernel<T, M, 8, 4>), grid, dim3(512), 0, stream(), g);
        else if (sizeof(T) == 2 || plan.groups == 8) hipLaunchKernelGGL((gated_rows_kernel<T, M, 8, 8>), grid, dim3(512), 0, stream(), g);
        else if constexpr (sizeof(T) == 4) hipLaunchKernelGGL((gated_rows_kernel<T, M, 8, 16>), grid, dim3(512), 0, stream(), g);
    };
    if (g.m == 1) launch(std::integral_constant<int, 1>{});
    else if (g.m == 2) launch(std::integral_constant<int, 2>{});
    else if constexpr (sizeof(T) == 4) launch(std::integral_constant<int, 4>{});
    AGH_LAUNCH_CHECK(name);
    if (plan.splits > 1) {
        hipLaunchKernelGGL(gemm::gated_join_kernel<T>, dim3((unsigned)((g.n + 1023) / 1024), (unsigned)g.m), dim3(256), 0, stream(), g.ws, plan.splits, (int64_t)g.m * 2 * g.n,
                           2 * g.n, g.m, g.n, g.bias, g.bias_stride, g.act, g.y, g.h);
        AGH_LAUNCH_CHECK(name);
    }
    return AGH_OK;
}

template <typename T>
int forward_entry(const char *name, int64_t m, int64_t k, int64_t n, const void *x, int64_t off_x, int64_t rsx, int64_t csx, const void *w, int64_t off_w,
                  int64_t rsw, int64_t csw, const void *bias, int64_t off_bias, int64_t bias_stride, int act, void *y, void *h) {
    if (int rc = check_sizes(name, m, k, n, act)) return rc;
    if (m == 0 || n == 0) return AGH_OK;
    if (!y) return fail(AGH_ENULL, "%s: null output", name);
    if (k > 0 && (!x || !w)) return fail(AGH_ENULL, "%s: null input or weight", name);
    if (const FewPlan plan = few_plan<T>(m, k, n); plan.groups && csx == 1 && csw == 1) {
        const GatedFew<T> g = {(const T *)x + off_x, (const T *)w + off_w, bias ? (const T *)bias + off_bias : nullptr, rsx, rsw, bias_stride, (T *)y, (T *)h, (int)m, (int)k, (int)n, act, nullptr};
        return rows_launch<T>(name, g, plan);
    }
    const GatedOut out = {bias ? (const T *)bias + off_bias : nullptr, bias_stride, act, y, h, 0};
    return gated_product<T>(name, m, k, n, (const T *)x + off_x, rsx, csx, (const T *)w + off_w, rsw, csw, out);
}

template <typename T>
int backward_entry(const char *name, int64_t m, int64_t k, int64_t n, const void *x, int64_t off_x, int64_t rsx, int64_t csx, const void *w, int64_t off_w,
                   int64_t rsw, int64_t csw, const void *h, const void *dy, int act, void *dh, void *dx, void *dw, void *db) {
    if (int rc = check_sizes(name, m, k, n, act)) return rc;
    if (m > 0 && n > 0 && (!h || !dy || !dh)) return fail(AGH_ENULL, "%s: null pre-activations, output gradient or their gradient", name);
    if (m > 0 && k > 0 && n > 0 && ((dx && !w) || (dw && !x))) return fail(AGH_ENULL, "%s: null input or weight", name);
    if (n > 0) {
        const int columns = (int)(2 * n);
        int count = 0;
        void *ws = nullptr;
        if (m > 0) {
            constexpr int VE = Group<T>::VE, U = 4;
            const int64_t strips = (n + 64 * VE - 1) / (64 * VE);
            // a share: at least U rows for each of four waves, and eight workgroups a CU; few rows are one share of sixteen waves, which saves the launch that adds
            // them (bf16, shares / one, with both products: 32 rows 16.7 / 13.8 us, 64 of 4096 columns 23.5 / 25.7; f32 64 rows 16.0 / 13.2, 100 16.1 / 15.7)
            const bool whole = db && m <= 256 / VE;
            const int64_t shares = whole ? 1 : std::max<int64_t>(1, std::min<int64_t>((m + U * 4 - 1) / (U * 4), (int64_t)compute_units() * 8 / strips));
            const int64_t rows = (m + shares - 1) / shares;
            count = (int)((m + rows - 1) / rows);
            if (db && count > 1)
                if (int rc = workspace((size_t)count * columns * sizeof(float), &ws)) return rc;
            const dim3 grid((unsigned)strips, (unsigned)count);
            T *direct = count == 1 ? (T *)db : nullptr;
            if (whole)
                hipLaunchKernelGGL((gated_backward_kernel<T, U, 16>), grid, dim3(1024), 0, stream(), (const T *)h, (const T *)dy, (int)m, (int)n, (int)rows, act, (T *)dh, nullptr, direct);
            else
                hipLaunchKernelGGL((gated_backward_kernel<T, U, 4>), grid, dim3(256), 0, stream(), (const T *)h, (const T *)dy, (int)m, (int)n, (int)rows, act, (T *)dh, (float *)ws,
                                   direct);
            AGH_LAUNCH_CHECK(name);
        }
        if (db && count != 1) {
            hipLaunchKernelGGL(gated_bias_kernel, dim3((unsigned)((columns + 15) / 16)), dim3(kThreads), 0, stream(), (const float *)ws, count, columns, db, sizeof(T) == 2);
            AGH_LAUNCH_CHECK(name);
        }
    }
    auto gemm = sizeof(T) == 2 ? agh_gemm_bf16 : agh_gemm_f32;
    if (dx)
        if (int rc = gemm(m, 2 * n, k, 1.0f, dh, 0, 2 * n, 1, w, off_w, csw, rsw, 0.0f, dx, 0, k, 1)) return rc;
    if (dw)
        if (int rc = gemm(k, m, 2 * n, 1.0f, x, off_x, csx, rsx, dh, 0, 2 * n, 1, 0.0f, dw, 0, 2 * n, 1)) return rc;
    return AGH_OK;
}

}  // namespace

extern "C" {

#define AGH_GATED(SUFFIX, T)                                                                                                                     \
    int agh_gated_dense_##SUFFIX(int64_t m, int64_t k, int64_t n, const void *x, int64_t off_x, int64_t rsx, int64_t csx, const void *w,         \
                                 int64_t off_w, int64_t rsw, int64_t csw, const void *bias, int64_t off_bias, int64_t bias_stride, int act,      \
                                 void *y, void *h) {                                                                                             \
        AGH_API_ENTER();                                                                                                                         \
        return forward_entry<T>("agh_gated_dense_" #SUFFIX, m, k, n, x, off_x, rsx, csx, w, off_w, rsw, csw, bias, off_bias, bias_stride, act,   \
                                y, h);                                                                                                           \
    }                                                                                                                                            \
    int agh_gated_dense_backward_##SUFFIX(int64_t m, int64_t k, int64_t n, const void *x, int64_t off_x, int64_t rsx, int64_t csx,               \
                                          const void *w, int64_t off_w, int64_t rsw, int64_t csw, const void *h, const void *dy, int act,        \
                                          void *dh, void *dx, void *dw, void *db) {                                                              \
        AGH_API_ENTER();                                                                                                                         \
        return backward_entry<T>("agh_gated_dense_backward_" #SUFFIX, m, k, n, x, off_x, rsx, csx, w, off_w, rsw, csw, h, dy, act, dh, dx, dw,   \
                                 db);                                                                                                            \
    }
AGH_GATED(f32, float)
AGH_GATED(bf16, uint16_t)

}  // extern "C"

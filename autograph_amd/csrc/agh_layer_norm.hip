// Layer norm over the rows of a matrix, forward and backward.
//
//   mean = sum x / C, rstd = 1 / sqrt(sum (x - mean)^2 / C + eps), y = (x - mean) rstd w + b
//   with h = (x - mean) rstd and g = dy w:  dx = rstd (g - sum g / C - h sum (g h) / C), dw = sum over rows dy h, db = sum over rows dy
// All sums are f32, whatever the element type, and every result is rounded to it once.
#include "agh_internal.h"

using namespace agh;

namespace {

constexpr int kThreads = 256;

// sum over the workgroup, the same bits in every thread; `part`: one f32 a wave
__device__ __forceinline__ float workgroup_sum(float v, float *part) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.0f;
    for (int i = 0; i < kThreads / 64; ++i) s += part[i];
    return s;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_kernel(const T *x, const T *__restrict__ w, const T *__restrict__ b, float eps,
                                                              T *y, float *__restrict__ mean_out, float *__restrict__ rstd_out, int64_t cols) {
    __shared__ float part[kThreads / 64];
    const int64_t row = blockIdx.x;
    x += row * cols;
    y += row * cols;
    float s = 0.0f;
    for (int64_t i = threadIdx.x; i < cols; i += kThreads) s += Elem<T>::raw(x[i]);
    const float mean = workgroup_sum(s, part) / (float)cols;
    s = 0.0f;
    for (int64_t i = threadIdx.x; i < cols; i += kThreads) {
        const float d = Elem<T>::raw(x[i]) - mean;
        s += d * d;
    }
    const float rstd = 1.0f / sqrtf(workgroup_sum(s, part) / (float)cols + eps);
    for (int64_t i = threadIdx.x; i < cols; i += kThreads) {
        float v = (Elem<T>::raw(x[i]) - mean) * rstd;
        if (w) v *= Elem<T>::raw(w[i]);
        if (b) v += Elem<T>::raw(b[i]);
        y[i] = Elem<T>::from_f32(v);
    }
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_backward_kernel(const T *x, const T *dy, const T *__restrict__ w,
                                                                       const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                                                                       T *dx, int64_t cols) {
    __shared__ float part[kThreads / 64];
    const int64_t row = blockIdx.x;
    const float mean = mean_in[row], rstd = rstd_in[row];
    x += row * cols;
    dy += row * cols;
    dx += row * cols;
    float sg = 0.0f, sgh = 0.0f;
    for (int64_t i = threadIdx.x; i < cols; i += kThreads) {
        const float g = Elem<T>::raw(dy[i]) * (w ? Elem<T>::raw(w[i]) : 1.0f);
        sg += g;
        sgh += g * ((Elem<T>::raw(x[i]) - mean) * rstd);
    }
    sg = workgroup_sum(sg, part) / (float)cols;
    sgh = workgroup_sum(sgh, part) / (float)cols;
    for (int64_t i = threadIdx.x; i < cols; i += kThreads) {
        const float g = Elem<T>::raw(dy[i]) * (w ? Elem<T>::raw(w[i]) : 1.0f);
        dx[i] = Elem<T>::from_f32(rstd * (g - sg - (Elem<T>::raw(x[i]) - mean) * rstd * sgh));
    }
}

// one thread a column
template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_parameters_kernel(const T *__restrict__ x, const T *__restrict__ dy, const float *__restrict__ mean,
                                                                         const float *__restrict__ rstd, T *__restrict__ dw, T *__restrict__ db, int64_t rows,
                                                                         int64_t cols) {
    const int64_t col = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (col >= cols) return;
    float sw = 0.0f, sb = 0.0f;
    for (int64_t r = 0; r < rows; ++r) {
        const float g = Elem<T>::raw(dy[r * cols + col]);
        sb += g;
        sw += g * ((Elem<T>::raw(x[r * cols + col]) - mean[r]) * rstd[r]);
    }
    if (dw) dw[col] = Elem<T>::from_f32(sw);
    if (db) db[col] = Elem<T>::from_f32(sb);
}

int check_sizes(const char *name, int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 1) return fail(AGH_EINVAL, "%s: %lld rows of %lld elements", name, (long long)rows, (long long)cols);
    if (rows >= (int64_t)1 << 31 || cols >= (int64_t)1 << 31) return fail(AGH_ERANGE, "%s: %lld rows of %lld elements: too many", name, (long long)rows, (long long)cols);
    return AGH_OK;
}

template <typename T>
int forward_entry(const char *name, const void *x, const void *w, const void *b, float eps, void *y, void *mean, void *rstd, int64_t rows, int64_t cols) {
    if (int rc = check_sizes(name, rows, cols)) return rc;
    if (!(eps >= 0.0f)) return fail(AGH_EINVAL, "%s: eps %g is negative or no number", name, (double)eps);
    if (rows == 0) return AGH_OK;
    if (!x || !y) return fail(AGH_ENULL, "%s: null input or output", name);
    hipLaunchKernelGGL(layer_norm_kernel<T>, dim3((unsigned)rows), dim3(kThreads), 0, stream(), (const T *)x, (const T *)w, (const T *)b, eps, (T *)y,
                       (float *)mean, (float *)rstd, cols);
    AGH_LAUNCH_CHECK(name);
    return AGH_OK;
}

template <typename T>
int backward_entry(const char *name, const void *x, const void *dy, const void *w, const void *mean, const void *rstd, void *dx, void *dw, void *db,
                   int64_t rows, int64_t cols) {
    if (int rc = check_sizes(name, rows, cols)) return rc;
    if (rows > 0 && (!x || !dy || !mean || !rstd)) return fail(AGH_ENULL, "%s: null input", name);
    // (the parameters' gradients first: dx may overwrite x or dy)
    if (dw || db) {
        hipLaunchKernelGGL(layer_norm_parameters_kernel<T>, dim3((unsigned)((cols + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream(), (const T *)x,
                           (const T *)dy, (const float *)mean, (const float *)rstd, (T *)dw, (T *)db, rows, cols);
        AGH_LAUNCH_CHECK(name);
    }
    if (rows > 0 && dx) {
        hipLaunchKernelGGL(layer_norm_backward_kernel<T>, dim3((unsigned)rows), dim3(kThreads), 0, stream(), (const T *)x, (const T *)dy, (const T *)w,
                           (const float *)mean, (const float *)rstd, (T *)dx, cols);
        AGH_LAUNCH_CHECK(name);
    }
    return AGH_OK;
}

}  // namespace

extern "C" {

#define AGH_LAYER_NORM(SUFFIX, T)                                                                                                                  \
    int agh_layer_norm_##SUFFIX(const void *x, const void *weight, const void *bias, float eps, void *y, void *mean, void *rstd, int64_t rows,     \
                                int64_t cols) {                                                                                                    \
        AGH_API_ENTER();                                                                                                                           \
        return forward_entry<T>("agh_layer_norm_" #SUFFIX, x, weight, bias, eps, y, mean, rstd, rows, cols);                                       \
    }                                                                                                                                              \
    int agh_layer_norm_backward_##SUFFIX(const void *x, const void *dy, const void *weight, const void *mean, const void *rstd, void *dx,          \
                                         void *dweight, void *dbias, int64_t rows, int64_t cols) {                                                 \
        AGH_API_ENTER();                                                                                                                           \
        return backward_entry<T>("agh_layer_norm_backward_" #SUFFIX, x, dy, weight, mean, rstd, dx, dweight, dbias, rows, cols);                   \
    }
AGH_LAYER_NORM(f32, float)
AGH_LAYER_NORM(bf16, uint16_t)

}  // extern "C"

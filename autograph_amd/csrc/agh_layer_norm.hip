// Layer norm over the rows of a matrix, forward and backward.
//
//   mean = sum x / C, rstd = 1 / sqrt(sum (x - mean)^2 / C + eps), y = (x - mean) rstd w + b
//   with h = (x - mean) rstd and g = dy w:  dx = rstd (g - sum g / C - h sum (g h) / C), dw = sum over rows dy h, db = sum over rows dy
// All sums are f32, whatever the element type, and every result is rounded to it once.
//
// Bounded by memory: each element is read once and written once.  A row stays in the registers of the threads that share it, in 16-byte
// groups, between its sums and its result; so the squares can be taken of deviations from the finished mean.  Up to 4 groups a lane a row belongs to
// one wave, whose sums need neither LDS nor a barrier, longer ones to a workgroup.  Threads keep their columns from row to row: weight and bias are read
// once, and the backward pass adds its columns' shares of dw and db in registers.  bf16 16384x4096: 47.8 us forward (5.6 TB/s), 81 backward (5.0).
#include "agh_groups.h"

using namespace agh;

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;

// sum over TPR neighbouring lanes (16 or 64), the same bits in each of them
template <int TPR>
__device__ __forceinline__ float lanes_sum(float v) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, true));   // quad_perm 1 0 3 2
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, true));   // quad_perm 2 3 0 1
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, true));  // row_half_mirror
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, true));  // row_mirror
    if constexpr (TPR == 64) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
        v = __int_as_float(a[0]) + __int_as_float(a[1]);
        const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
        v = __int_as_float(b[0]) + __int_as_float(b[1]);
    }
    return v;
}

// N sums over the TPR threads of a row; beyond a wave through `part` (N floats a wave, not the memory of the sums before: its readers may still be at it)
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float *part) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lanes_sum<(TPR < 64 ? TPR : 64)>(v[i]);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) part[(threadIdx.x >> 6) * N + i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < TPR / 64; ++j) s += part[j * N + i];
            v[i] = s;
        }
    }
}

// A row's groups: those that pass its end behind a branch where a thread holds many (without one, each takes registers for an address of its own: bf16 4096x16384,
// 4 groups, forward 66 us against 52), else not.
template <typename T, bool MANY>
__device__ __forceinline__ u32x4_t load_row(const T *row, int e, int cols) {
    if constexpr (MANY)
        if (e + Group<T>::VE <= cols) return *(const typename Group<T>::vec *)(row + e);
    return Group<T>::load(row, e, cols);
}
// the elements of a weight that may be absent: `none` is what it stands for then
template <typename T>
__device__ __forceinline__ u32x4_t load_or(const T *row, int e, int cols, float none) {
    if (row) return Group<T>::load(row, e, cols);
    float f[Group<T>::VE];
#pragma unroll
    for (int i = 0; i < Group<T>::VE; ++i) f[i] = none;
    return Group<T>::pack(f);
}
// with the streaming hint: forward bf16 16384x1024 15.2 -> 12.6 us, 2048x4096 8.8 -> 7.5, 16384x4096 50.4 -> 48.5
template <typename T>
__device__ __forceinline__ void store_group(T *row, int e, int cols, u32x4_t v) {
    if (e + Group<T>::VE <= cols) {
        __builtin_nontemporal_store(v, (typename Unaligned<T>::vec *)(row + e));
        return;
    }
    typename Group<T>::Bits b;
    b.q = v;
#pragma unroll
    for (int i = 0; i < Group<T>::VE; ++i)
        if (e + i < cols) row[e + i] = b.e[i];
}

// Values that stay packed: without this the compiler widens them once for all their uses, which takes a bf16 row twice the registers
__device__ __forceinline__ void keep_packed(u32x4_t &v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w = v[i];
        asm("" : "+v"(w));
        v[i] = w;
    }
}

// Whether a row spreads so little around its mean that the mean's own error, a few steps of f32, counts against the deviations (rows of one value came out as far as 1 from
// their bias).  Such a row adds its deviations too, moves the mean by what is left, and takes the squares again.
// (By the root, to the instruction's accuracy: the mean's square may vanish.  Rows that are not of this kind pay for the question where they are short, f32 65536x84 17.5 -> 18.2 us,
// and for nothing at 16384x1001, 24.0.  The squares and this in one loop of up to two turns: bf16 16384x2048 24.7 -> 27.1, 4096x16384 53.7 -> 60.)
__device__ __forceinline__ bool far_from_zero(float var, float mean) { return __builtin_amdgcn_sqrtf(var) * 16.0f < fabsf(mean); }

constexpr int wg_threads(int tpr) { return tpr > kThreads ? tpr : kThreads; }

// rows of at most TPR * VPT groups, TPR threads a row
template <typename T, int TPR, int VPT>
__global__ __launch_bounds__(wg_threads(TPR)) void layer_norm_kernel(const T *x, const T *__restrict__ w, const T *__restrict__ b, float eps, T *y,
                                                                     float *__restrict__ mean_out, float *__restrict__ rstd_out, int64_t rows, int cols) {
    using G = Group<T>;
    constexpr int VE = G::VE, ROWS = wg_threads(TPR) / TPR;
    __shared__ float part[2][wg_threads(TPR) / 64];
    const int t = threadIdx.x % TPR;
    const float per = 1.0f / (float)cols;
    u32x4_t wv[VPT], bv[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int e = (t + j * TPR) * VE;
        wv[j] = load_or(w, e, cols, 1.0f);
        bv[j] = load_or(b, e, cols, 0.0f);
    }
    for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR; row < rows; row += (int64_t)gridDim.x * ROWS) {
        const T *xr = x + row * cols;
        u32x4_t xv[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            xv[j] = load_row<T, (VPT > 3 && TPR > 64)>(xr, (t + j * TPR) * VE, cols);
        }
        float s[1] = {0.0f};
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
#pragma unroll
            for (int i = 0; i < VE; ++i) s[0] += G::get(xv[j], i);
        }
        row_sums<TPR>(s, part[0]);
        float mean = s[0] * per;
        s[0] = 0.0f;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int left = cols - (t + j * TPR) * VE;
            keep_packed(xv[j]);
            if (left >= VE) {
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    const float d = G::get(xv[j], i) - mean;
                    s[0] += d * d;
                }
            } else {
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    const float d = G::get(xv[j], i) - mean;
                    s[0] += i < left ? d * d : 0.0f;
                }
            }
        }
        row_sums<TPR>(s, part[1]);
        float rstd = 1.0f / sqrtf(s[0] * per + eps);
        if (__builtin_expect(far_from_zero(s[0] * per, mean), 0)) {
            const float first = mean;
            s[0] = 0.0f;
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                keep_packed(xv[j]);
#pragma unroll
                for (int i = 0; i < VE; ++i) s[0] += (t + j * TPR) * VE + i < cols ? G::get(xv[j], i) - first : 0.0f;
            }
            row_sums<TPR>(s, part[0]);
            mean = first + s[0] * per;
            s[0] = 0.0f;
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                keep_packed(xv[j]);
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    const float d = (t + j * TPR) * VE + i < cols ? G::get(xv[j], i) - mean : 0.0f;
                    s[0] += d * d;
                }
            }
            row_sums<TPR>(s, part[1]);
            rstd = 1.0f / sqrtf(s[0] * per + eps);
        }
        T *yr = y + row * cols;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int e = (t + j * TPR) * VE;
            float f[VE];
            keep_packed(xv[j]);
            keep_packed(wv[j]);
            keep_packed(bv[j]);
#pragma unroll
            for (int i = 0; i < VE; ++i) f[i] = (G::get(xv[j], i) - mean) * rstd * G::get(wv[j], i) + G::get(bv[j], i);
            if (e < cols) store_group(yr, e, cols, G::pack(f));
        }
        if (t == 0) {
            if (mean_out) mean_out[row] = mean;
            if (rstd_out) rstd_out[row] = rstd;
        }
    }
}

// rstd as the factor of the deviations.  Behind a row's end x is 0 and h = -mean rstd, which has to be finite: 0 * inf would be a NaN in all of dx.  It is, unless all the
// row's values are one: else some value deviates from the mean by half a step of it, and rstd is at most 2^25 sqrt(C) / |mean|.  The deviations of a row of one value are 0,
// and so is h whatever the factor is.  (Places behind the end left out, by a branch or a select for each group: 2 to 10 % of the time.)
__device__ __forceinline__ float deviations_rstd(float mean, float rstd) { return __builtin_isinf(mean * rstd) && !__builtin_isinf(rstd) ? 0.0f : rstd; }

// Backward: dx, and this workgroup's shares of dw and db.  shares [gridDim.x][2][pitch]: f32, or with one workgroup nothing, then dw and db are written here.
template <typename T, int THREADS, int TPR, int VPT>
__global__ __launch_bounds__(THREADS, THREADS == 512 && VPT == 2 ? 4 : 1) void layer_norm_backward_kernel(
    const T *x, const T *dy, const T *__restrict__ w, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
    T *dx, float *__restrict__ shares, T *__restrict__ dw, T *__restrict__ db, int64_t rows, int cols, int pitch) {
    using G = Group<T>;
    constexpr int VE = G::VE, ROWS = THREADS / TPR;
    static_assert(TPR <= 64 || ROWS == 1, "the waves of a row meet at the workgroup's barrier");
    __shared__ float part[TPR > 64 ? 2 * 2 * (THREADS / 64) : 1];
    __shared__ float added[ROWS > 1 ? ROWS / 2 * TPR * 2 * VE : 1];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const float per = 1.0f / (float)cols;
    u32x4_t wv[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) wv[j] = load_or(w, (t + j * TPR) * VE, cols, 1.0f);
    float aw[VPT][VE] = {}, ab[VPT][VE] = {};
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * ROWS + sub; row < rows; row += (int64_t)gridDim.x * ROWS) {
        u32x4_t xv[VPT], gv[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int e = (t + j * TPR) * VE;
            xv[j] = load_row<T, (VPT > 3 && TPR > 64)>(x + row * cols, e, cols);
            gv[j] = load_row<T, (VPT > 3 && TPR > 64)>(dy + row * cols, e, cols);
        }
        const float mean = mean_in[row], rstd = rstd_in[row], rstd_h = deviations_rstd(mean, rstd);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            keep_packed(wv[j]);
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                // (behind the row's end dy is 0 and so is every term, or a NaN where the whole row is NaN: h is finite there)
                const float d = G::get(gv[j], i), h = (G::get(xv[j], i) - mean) * rstd_h, g = d * G::get(wv[j], i);
                ab[j][i] += d;
                aw[j][i] += d * h;
                s[0] += g;
                s[1] += g * h;
            }
        }
        if (dx) {
            row_sums<TPR>(s, part + (TPR > 64 ? turn * 2 * (THREADS / 64) + sub * (TPR / 64) * 2 : 0));
            turn ^= 1;
            s[0] *= per;
            s[1] *= per;
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int e = (t + j * TPR) * VE;
                float f[VE];
                keep_packed(xv[j]);
                keep_packed(gv[j]);
                keep_packed(wv[j]);
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    const float d = G::get(gv[j], i), h = (G::get(xv[j], i) - mean) * rstd_h, g = d * G::get(wv[j], i);
                    f[i] = rstd * (g - s[0] - h * s[1]);
                }
                if (e < cols) store_group(dx + row * cols, e, cols, G::pack(f));
            }
        }
    }
    if (!shares && !dw && !db) return;
    // the rows that ran side by side: the upper half adds its sums to the lower half's, until one is left
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
#pragma unroll
        for (int half = ROWS / 2; half; half /= 2) {
            float *at = added + ((sub % half) * TPR + t) * 2 * VE;
            __syncthreads();
            if (sub >= half && sub < 2 * half)
#pragma unroll
                for (int i = 0; i < VE; ++i) at[i] = aw[j][i], at[VE + i] = ab[j][i];
            __syncthreads();
            if (sub < half)
#pragma unroll
                for (int i = 0; i < VE; ++i) aw[j][i] += at[i], ab[j][i] += at[VE + i];
        }
        const int e = (t + j * TPR) * VE;
        if (sub != 0 || e >= cols) continue;
        if (shares) {
            float *mine = shares + (int64_t)blockIdx.x * 2 * pitch + e;  // pitch: whole groups
#pragma unroll
            for (int i = 0; i < VE; i += 4) {
                *(f32x4_t *)(mine + i) = f32x4_t{aw[j][i], aw[j][i + 1], aw[j][i + 2], aw[j][i + 3]};
                *(f32x4_t *)(mine + pitch + i) = f32x4_t{ab[j][i], ab[j][i + 1], ab[j][i + 2], ab[j][i + 3]};
            }
        } else {
            if (dw) store_group(dw, e, cols, G::pack(aw[j]));
            if (db) store_group(db, e, cols, G::pack(ab[j]));
        }
    }
}

// dw (blockIdx.y 0) and db out of n workgroups' shares: a workgroup adds kAddColumns columns at a time, a line of memory of each share, a thread 4 columns of every
// PARTS-th share.  (16 columns, half a line, by 64 threads: with the pass before bf16 16384x4096 77.2 us against 75.1, 2048x2048 15.7 against 14.6; 32 by 32: 65536x84
// 17.9 against 16.6.)
constexpr int kAddColumns = 32, kAddThreads = kAddColumns / 4;
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void add_shares_kernel(const float *__restrict__ shares, int n, int pitch, T *__restrict__ dw, T *__restrict__ db, int cols) {
    constexpr int PARTS = THREADS / kAddThreads;
    __shared__ f32x4_t part[THREADS / 64][kAddThreads];
    const int c = threadIdx.x % kAddThreads, p = threadIdx.x / kAddThreads;
    T *out = blockIdx.y ? db : dw;
    if (!out) return;
    for (int64_t col = (int64_t)blockIdx.x * kAddColumns + c * 4; col - c * 4 < cols; col += (int64_t)gridDim.x * kAddColumns) {
        f32x4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
        if (col < cols) {
            const float *from = shares + blockIdx.y * (int64_t)pitch + col;
#pragma unroll 8
            for (int i = p; i < n; i += PARTS) s += *(const f32x4_t *)(from + (int64_t)i * 2 * pitch);
        }
#pragma unroll
        for (int d = kAddThreads; d < 64; d *= 2)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += __shfl_xor(s[i], d);
        __syncthreads();  // the turn before has been read
        if ((threadIdx.x & 63) < kAddThreads) part[threadIdx.x >> 6][c] = s;
        __syncthreads();
        if (threadIdx.x >= kAddThreads || col >= cols) continue;
        s = part[0][c];
#pragma unroll
        for (int i = 1; i < THREADS / 64; ++i) s += part[i][c];
        for (int i = 0; i < 4 && col + i < cols; ++i) out[col + i] = Elem<T>::from_f32(s[i]);
    }
}

// ---- rows longer than a workgroup's registers hold: read again for every sum, from the caches where they fit, 16 bytes a lane (element by element: f32 1638x20480 126
// us against 63, backward bf16 127 against 74) ----

__device__ __forceinline__ float workgroup_sum(float v, float *part) {
    v = lanes_sum<64>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.0f;
    for (int i = 0; i < (int)blockDim.x / 64; ++i) s += part[i];
    return s;
}

constexpr int kLongThreads = 1024;
constexpr int64_t kMostWorkgroups = 1 << 20;  // of a launch (its work items are counted in 32 bits): what lies behind takes further turns

template <typename T>
__global__ __launch_bounds__(kLongThreads) void layer_norm_long_kernel(const T *x, const T *__restrict__ w, const T *__restrict__ b, float eps, T *y,
                                                                       float *__restrict__ mean_out, float *__restrict__ rstd_out, int64_t rows, int cols) {
    using G = Group<T>;
    constexpr int VE = G::VE, TURN = kLongThreads * VE;
    __shared__ float part[kLongThreads / 64];
    const float per = 1.0f / (float)cols;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * cols;
        T *yr = y + row * cols;
        float s = 0.0f;
#pragma unroll 4
        for (int e = threadIdx.x * VE; e < cols; e += TURN) {
            const u32x4_t v = G::load(xr, e, cols);
#pragma unroll
            for (int i = 0; i < VE; ++i) s += G::get(v, i);
        }
        float mean = workgroup_sum(s, part) * per;
        const auto variance = [&]() {
            float v2 = 0.0f;
#pragma unroll 4
            for (int e = threadIdx.x * VE; e < cols; e += TURN) {
                const u32x4_t v = G::load(xr, e, cols);
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    const float d = e + i < cols ? G::get(v, i) - mean : 0.0f;
                    v2 += d * d;
                }
            }
            return workgroup_sum(v2, part) * per;
        };
        float var = variance();
        if (__builtin_expect(far_from_zero(var, mean), 0)) {
            s = 0.0f;
            for (int e = threadIdx.x * VE; e < cols; e += TURN) {
                const u32x4_t v = G::load(xr, e, cols);
#pragma unroll
                for (int i = 0; i < VE; ++i) s += e + i < cols ? G::get(v, i) - mean : 0.0f;
            }
            mean += workgroup_sum(s, part) * per;
            var = variance();
        }
        const float rstd = 1.0f / sqrtf(var + eps);
#pragma unroll 2
        for (int e = threadIdx.x * VE; e < cols; e += TURN) {
            const u32x4_t v = G::load(xr, e, cols), wv = load_or(w, e, cols, 1.0f), bv = load_or(b, e, cols, 0.0f);
            float f[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) f[i] = (G::get(v, i) - mean) * rstd * G::get(wv, i) + G::get(bv, i);
            store_group(yr, e, cols, G::pack(f));
        }
        if (threadIdx.x == 0) {
            if (mean_out) mean_out[row] = mean;
            if (rstd_out) rstd_out[row] = rstd;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kLongThreads) void layer_norm_backward_long_kernel(const T *x, const T *dy, const T *__restrict__ w, const float *__restrict__ mean_in,
                                                                                const float *__restrict__ rstd_in, T *dx, int64_t rows, int cols) {
    using G = Group<T>;
    constexpr int VE = G::VE, TURN = kLongThreads * VE;
    __shared__ float part[kLongThreads / 64];
    const float per = 1.0f / (float)cols;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float mean = mean_in[row], rstd = rstd_in[row], rstd_h = deviations_rstd(mean, rstd);
        const T *xr = x + row * cols, *dyr = dy + row * cols;
        T *dxr = dx + row * cols;
        float sg = 0.0f, sgh = 0.0f;
#pragma unroll 2
        for (int e = threadIdx.x * VE; e < cols; e += TURN) {
            const u32x4_t xv = G::load(xr, e, cols), gv = G::load(dyr, e, cols), wv = load_or(w, e, cols, 1.0f);
#pragma unroll
            for (int i = 0; i < VE; ++i) {  // (behind the row's end dy is 0)
                const float g = G::get(gv, i) * G::get(wv, i);
                sg += g;
                sgh += g * ((G::get(xv, i) - mean) * rstd_h);
            }
        }
        sg = workgroup_sum(sg, part) * per;
        sgh = workgroup_sum(sgh, part) * per;
#pragma unroll 2
        for (int e = threadIdx.x * VE; e < cols; e += TURN) {
            const u32x4_t xv = G::load(xr, e, cols), gv = G::load(dyr, e, cols), wv = load_or(w, e, cols, 1.0f);
            float f[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) f[i] = rstd * (G::get(gv, i) * G::get(wv, i) - sg - (G::get(xv, i) - mean) * rstd_h * sgh);
            store_group(dxr, e, cols, G::pack(f));
        }
    }
}

// a thread a group of columns, a share for every gridDim.y-th row; without shares (one for all rows) the results themselves
template <typename T>
__global__ __launch_bounds__(kThreads) void column_shares_kernel(const T *__restrict__ x, const T *__restrict__ dy, const float *__restrict__ mean,
                                                                 const float *__restrict__ rstd, float *__restrict__ shares, T *__restrict__ dw, T *__restrict__ db,
                                                                 int64_t rows, int cols, int pitch) {
    using G = Group<T>;
    constexpr int VE = G::VE;
    const int64_t e = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * VE;
    if (e >= cols) return;
    float sw[VE] = {}, sb[VE] = {};
#pragma unroll 4
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const u32x4_t gv = G::load(dy + r * cols, (int)e, cols), xv = G::load(x + r * cols, (int)e, cols);
        const float m = mean[r], s = rstd[r];
#pragma unroll
        for (int i = 0; i < VE; ++i) {
            const float g = G::get(gv, i);
            sb[i] += g;
            sw[i] += g * ((G::get(xv, i) - m) * s);
        }
    }
    if (!shares) {
        if (dw) store_group(dw, (int)e, cols, G::pack(sw));
        if (db) store_group(db, (int)e, cols, G::pack(sb));
        return;
    }
    float *mine = shares + (int64_t)blockIdx.y * 2 * pitch + e;  // pitch: whole groups
#pragma unroll
    for (int i = 0; i < VE; i += 4) {
        *(f32x4_t *)(mine + i) = f32x4_t{sw[i], sw[i + 1], sw[i + 2], sw[i + 3]};
        *(f32x4_t *)(mine + pitch + i) = f32x4_t{sb[i], sb[i + 1], sb[i + 2], sb[i + 3]};
    }
}

int check_sizes(const char *name, int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 1) return fail(AGH_EINVAL, "%s: %lld rows of %lld elements", name, (long long)rows, (long long)cols);
    if (rows >= (int64_t)1 << 31 || cols >= ((int64_t)1 << 31) - 65536)
        return fail(AGH_ERANGE, "%s: %lld rows of %lld elements: too many", name, (long long)rows, (long long)cols);
    return AGH_OK;
}

template <typename T>
struct Forward {
    const T *x, *w, *b;
    float eps;
    T *y;
    float *mean, *rstd;
    int64_t rows;
    int cols;
    template <int TPR, int VPT>
    void run() const {
        constexpr int per_wg = wg_threads(TPR) / TPR;
        // As many workgroups as run together, or a few times that: weight and bias are read once for several rows (a workgroup for each row: f32
        // 16384x1001 29.4 us against 27.8, bf16 4096x16384 58 against 52), the others' loads cover what a row waits for.
        const int64_t wgs = (rows + per_wg - 1) / per_wg, most = (int64_t)compute_units() * (TPR <= 64 || VPT > 2 ? 4 : 16);
        hipLaunchKernelGGL((layer_norm_kernel<T, TPR, VPT>), dim3((unsigned)(wgs < most ? wgs : most)), dim3(wg_threads(TPR)), 0, stream(), x, w, b, eps, y, mean,
                           rstd, rows, cols);
    }
};

template <typename T>
int forward_entry(const char *name, const void *x, const void *w, const void *b, float eps, void *y, void *mean, void *rstd, int64_t rows, int64_t cols) {
    if (int rc = check_sizes(name, rows, cols)) return rc;
    if (!(eps >= 0.0f)) return fail(AGH_EINVAL, "%s: eps %g is negative or no number", name, (double)eps);
    if (rows == 0) return AGH_OK;
    if (!x || !y) return fail(AGH_ENULL, "%s: null input or output", name);
    const Forward<T> f = {(const T *)x, (const T *)w, (const T *)b, eps, (T *)y, (float *)mean, (float *)rstd, rows, (int)cols};
    const int64_t groups = (cols + Group<T>::VE - 1) / Group<T>::VE;
    // the fewest threads that hold the row, but a workgroup beyond 256 groups (bf16 16384x4096, 512 groups: a wave with 8 each 54.7 us, 256 threads
    // with 2 48.5, 1024 threads, half of them idle, 76) and 512 threads beyond 768 (8192x8192: 256 with 4 51.1, 512 with 2 49.5, 1024 with 1 52.7)
    if (groups <= 16) f.template run<16, 1>();
    else if (groups <= 64) f.template run<64, 1>();
    else if (groups <= 128) f.template run<64, 2>();
    else if (groups <= 192) f.template run<64, 3>();
    else if (groups <= 256) f.template run<64, 4>();
    else if (groups <= 512) f.template run<256, 2>();
    else if (groups <= 768) f.template run<256, 3>();
    else if (groups <= 1024) f.template run<512, 2>();
    else if (groups <= 1536) f.template run<512, 3>();
    else if (groups <= 2048) f.template run<512, 4>();
    else if (groups <= 4096) f.template run<1024, 4>();
    else
        hipLaunchKernelGGL(layer_norm_long_kernel<T>, dim3((unsigned)(rows < kMostWorkgroups ? rows : kMostWorkgroups)), dim3(kLongThreads), 0, stream(), f.x, f.w, f.b, eps, f.y,
                           f.mean, f.rstd, rows, f.cols);
    AGH_LAUNCH_CHECK(name);
    return AGH_OK;
}

template <typename T>
struct Backward {
    const char *name;
    const T *x, *dy, *w;
    const float *mean, *rstd;
    T *dx, *dw, *db;
    int64_t rows;
    int cols, pitch;

    int add(const float *shares, int64_t n) const {
        const int64_t wgs = ((int64_t)cols + kAddColumns - 1) / kAddColumns;
        const dim3 grid((unsigned)(wgs < kMostWorkgroups ? wgs : kMostWorkgroups), 2);
        // (few shares of many columns: smaller workgroups, more of them side by side; with the pass before bf16 16x16384 11.9 us, by 1024 threads 15.5)
        if (n <= 64) hipLaunchKernelGGL((add_shares_kernel<T, 256>), grid, dim3(256), 0, stream(), shares, (int)n, pitch, dw, db, cols);
        else hipLaunchKernelGGL((add_shares_kernel<T, 1024>), grid, dim3(1024), 0, stream(), shares, (int)n, pitch, dw, db, cols);
        AGH_LAUNCH_CHECK(name);
        return AGH_OK;
    }
    template <int THREADS, int TPR, int VPT>
    int run() const {
        constexpr int per_wg = THREADS / TPR;
        // A workgroup's shares of dw and db, written and read again, cost what two to four rows do: no more workgroups than keep memory busy (bf16
        // 16384x4096, 512 threads: 256 workgroups 98.5 us, 512 76.6, 1024 87.7; 4096x16384: 256 89.8, 512 97.7), and two turns each at least.
        // Where a quarter of the threads has no columns, a third fills the gap (512 threads by 1, f32 21845x1536 86.2 -> 78.5, bf16 13107x2560 55.6 -> 53.1; all at work, 8192x4096 bf16 46.2 -> 47.4).
        const bool gaps = cols <= TPR * VPT * Group<T>::VE / 4 * 3;
        constexpr int each = TPR <= 64 ? (VPT <= 2 ? 3 : 2) : TPR == 512 && VPT <= 2 ? 2 : 1;
        const int64_t turns = (rows + per_wg - 1) / per_wg, most = (int64_t)compute_units() * (TPR == 512 && VPT == 1 && gaps ? 3 : each);
        int64_t wgs = THREADS == 1024 && TPR <= 64 ? 1 : (turns + 1) / 2;
        if (wgs > most) wgs = most;
        float *shares = nullptr;
        if (wgs > 1 && (dw || db))
            if (int rc = workspace((size_t)wgs * 2 * pitch * sizeof(float), (void **)&shares)) return rc;
        hipLaunchKernelGGL((layer_norm_backward_kernel<T, THREADS, TPR, VPT>), dim3((unsigned)wgs), dim3(THREADS), 0, stream(), x, dy, w, mean, rstd, dx, shares, dw, db,
                           rows, cols, pitch);
        AGH_LAUNCH_CHECK(name);
        return shares ? add(shares, wgs) : AGH_OK;
    }
    int run_long() const {
        if (dw || db) {  // (before dx, which may overwrite x or dy)
            // Shares of 16 rows, and no more of them than the workgroups that keep the chip busy: their memory, which the library keeps, stays below 34 MB however long a row is.
            // Where the columns alone are workgroups enough, one share, which is the result.
            const int64_t groups = pitch / Group<T>::VE, wgs = (groups + kThreads - 1) / kThreads, most = (int64_t)compute_units() * 8 / wgs;
            int64_t n = rows < 16 ? rows : rows / 16 < 64 ? rows / 16 : 64;
            if (n > most) n = most > 1 ? most : 1;
            float *shares = nullptr;
            if (n > 1)
                if (int rc = workspace((size_t)n * 2 * pitch * sizeof(float), (void **)&shares)) return rc;
            hipLaunchKernelGGL(column_shares_kernel<T>, dim3((unsigned)wgs, (unsigned)n), dim3(kThreads), 0, stream(), x, dy, mean, rstd, shares, dw, db, rows, cols, pitch);
            AGH_LAUNCH_CHECK(name);
            if (shares)
                if (int rc = add(shares, n)) return rc;
        }
        if (dx) {
            hipLaunchKernelGGL(layer_norm_backward_long_kernel<T>, dim3((unsigned)(rows < kMostWorkgroups ? rows : kMostWorkgroups)), dim3(kLongThreads), 0, stream(), x, dy, w,
                               mean, rstd, dx, rows, cols);
            AGH_LAUNCH_CHECK(name);
        }
        return AGH_OK;
    }
};

template <typename T>
int backward_entry(const char *name, const void *x, const void *dy, const void *w, const void *mean, const void *rstd, void *dx, void *dw, void *db,
                   int64_t rows, int64_t cols) {
    if (int rc = check_sizes(name, rows, cols)) return rc;
    if (rows > 0 && (!x || !dy || !mean || !rstd)) return fail(AGH_ENULL, "%s: null input", name);
    if (!dw && !db && (!dx || rows == 0)) return AGH_OK;
    constexpr int VE = Group<T>::VE;
    const int64_t groups = (cols + VE - 1) / VE;
    const Backward<T> f = {name, (const T *)x, (const T *)dy, (const T *)w, (const float *)mean, (const float *)rstd, (T *)dx, (T *)dw, (T *)db, rows, (int)cols,
                           (int)(groups * VE)};
    if (rows == 0) return f.add(nullptr, 0);
    // as the forward pass, but 512 threads beyond 256 groups: a thread's columns take their sums' registers too (16384x4096: bf16, 512 groups, a wave with 8 each
    // 111 us, 256 threads with 2 79.7, 512 with 1 76.6; f32, 1024 groups, 512 with 2 145.6, 1024 with 1 147)
    // Few short rows: one workgroup of 1024 threads, which needs no second launch and, called after another from Python, saves 2 us of the host's time.  It is taken as far as such
    // calls gain; replayed from a graph it loses before that.  us, one workgroup / two launches, in calls and in a graph: f32 64x84 7.2 / 9.4 and 6.1 / 5.7, 96x84 8.1 / 9.3 and 7.9 / 5.8,
    // 128x84 9.7 / 9.4 and 9.6 / 5.9, 256x60 7.1 / 9.4 and 6.2 / 6.0, 512x60 9.6 / 9.3 and 9.5 / 6.0; bf16 32x512 7.3 / 9.2 and 6.1 / 5.8, 64x512 8.5 / 9.4 and 8.4 / 5.9, 96x512 11.0 / 9.3,
    // 128x128 6.7 / 9.4 and 6.1 / 6.0, 192x84 8.5 / 9.2 and 8.3 / 7.0, 256x84 9.8 / 9.4.  So few that 256 threads are one workgroup too, and have
    // one turn, bf16 up to two: those (in a graph f32 4x10 2.9 for 3.3, bf16 32x128 3.8 for 4.5; f32 with two turns 32x60 3.6 for 3.5).
    constexpr int turns = VE == 8 ? 2 : 1;
    if (groups <= 16 && rows > 16 * turns && rows <= (VE == 8 ? 192 : 256)) return f.template run<1024, 16, 1>();
    if (groups > 16 && groups <= 64 && rows > 4 * turns && rows <= (VE == 8 ? 64 : 128)) return f.template run<1024, 64, 1>();
    if (groups <= 16) return f.template run<256, 16, 1>();
    if (groups <= 64) return f.template run<256, 64, 1>();
    if (groups <= 128) return f.template run<256, 64, 2>();
    if (groups <= 192) return f.template run<256, 64, 3>();
    if (groups <= 256) return f.template run<256, 64, 4>();
    if (groups <= 512) return f.template run<512, 512, 1>();
    // (bf16 4096x8192: 512 threads with 2 in 135 registers, one workgroup a unit, 62.8 us; in 128, two, 53.0; 1024 threads 49.9.  5461x6144: 62.2, 53.7, 52.9; 7281x4608: 71.7, 55.6, 60.5.
    // f32 8192x4096: 512 threads 69.3, 1024 76.7)
    if (groups <= (VE == 8 ? 768 : 1024)) return f.template run<512, 512, 2>();
    if constexpr (VE == 8)
        if (groups <= 1024) return f.template run<1024, 1024, 1>();
    if (groups <= 1536) return f.template run<512, 512, 3>();
    if (groups <= 2048) return f.template run<512, 512, 4>();
    // (bf16 has twice the sums for each group, which leaves the compiler no registers: 1638x20480 190 us against 74 when the rows are read again)
    if constexpr (VE == 4) {
        if (groups <= 3 * 1024) return f.template run<1024, 1024, 3>();  // f32 3276x10240 85.7 us, 512 threads with 8 96
        // (spills 40 registers, and is still the fastest of three by a wide margin: 4096x16384 178 us, 1024 threads with 4 224, read again 289; 4096x12292 141, 196, 217; one row 7.1, 10.7, 8.3)
        if (groups <= 4096) return f.template run<512, 512, 8>();
    }
    return f.run_long();
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

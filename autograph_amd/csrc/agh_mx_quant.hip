// MXFP4: quantisation of f32 and bf16 matrices along either axis, and its inverse.
//
//   s = clamp(floor(log2 max |v|) - 2, -127, 127) over a block of 32, code = E2M1(v / 2^s) rounded half to even, magnitudes above 6 to 6.
// A block with an infinity or a NaN gets the scale byte 255 and stands for 32 NaNs: E2M1 has neither, and clipping would hide them.
// v / 2^s is a product with a power of two between 2^-125 and 2^127: exact, but where it falls below f32's smallest numbers, far below half a code.
#include "agh_mx_quant.h"

using namespace agh;
using namespace agh::mx;

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int64_t code_at(int64_t row, int64_t block, int64_t steps) {
    return (((row >> 4) * steps + (block >> 2)) * 64 + (block & 3) * 16 + (row & 15)) * 16;
}
__device__ __forceinline__ int64_t scale_at(int64_t row, int64_t block, int64_t steps) {
    return (((row >> 6) * steps + (block >> 2)) * 64 + (block & 3) * 16 + (row & 15)) * 4 + ((row >> 4) & 3);
}

// k contiguous: a wave takes a fragment, lane l the block l / 16 of row l % 16
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(const T *__restrict__ x, int64_t rs, int rows, int k, int steps, int64_t frags,
                                                                 unsigned char *__restrict__ codes, unsigned char *__restrict__ scales) {
    const int64_t frag = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (frag >= frags) return;
    const int lane = threadIdx.x & 63;
    const int64_t rt = frag / steps;
    const int64_t row = rt * 16 + (lane & 15), block = (frag - rt * steps) * 4 + (lane >> 4), k0 = block * kBlock;
    Block<T> v;
    v.load(x + row * rs + k0, row < rows ? (int)max((int64_t)0, k - k0) : 0);
    u32x4_t c;
    uint32_t s;
    v.quantize(c, s);
    *(u32x4_t *)(codes + frag * kFragBytes + lane * 16) = c;
    scales[scale_at(row, block, steps)] = (unsigned char)s;
}

// any strides, meant for rows that are neighbours in memory: a wave takes a block of 64 rows, lane l row l
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_columns_kernel(const T *__restrict__ x, int64_t rs, int64_t cs, int rows, int k, int steps,
                                                                    int64_t items, unsigned char *__restrict__ codes,
                                                                    unsigned char *__restrict__ scales) {
    const int64_t item = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (item >= items) return;
    const int64_t rt64 = item / (steps * 4), block = item - rt64 * (steps * 4), row = rt64 * 64 + (threadIdx.x & 63), k0 = block * kBlock;
    if (row >= ((int64_t)rows + 15) / 16 * 16) return;
    const T *p = x + row * rs + k0 * cs;
    Block<T> v;
#pragma unroll
    for (int i = 0; i < Block<T>::NV; ++i) {
        typename Block<T>::Bits u;
#pragma unroll
        for (int j = 0; j < Block<T>::VE; ++j) u.e[j] = row < rows && k0 + i * Block<T>::VE + j < k ? p[(i * Block<T>::VE + j) * cs] : (T)0;
        v.v[i] = u.q;
    }
    u32x4_t c;
    uint32_t s;
    v.quantize(c, s);
    *(u32x4_t *)(codes + code_at(row, block, steps)) = c;
    scales[scale_at(row, block, steps)] = (unsigned char)s;
}

// 2^(s - 127) as f32, 255 as NaN
__device__ __forceinline__ float scale_value(uint32_t s) {
    return s == 255u ? __uint_as_float(0x7FC00000u) : s ? __uint_as_float(s << 23) : __uint_as_float(0x00400000u);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const unsigned char *__restrict__ codes, const unsigned char *__restrict__ scales, int rows,
                                                              int k, int steps, int64_t items, bool by_column, T *__restrict__ y, int64_t rs, int64_t cs) {
    const int64_t item = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (item >= items) return;
    const int lane = threadIdx.x & 63;
    int64_t row, block;
    if (by_column) {
        const int64_t rt64 = item / (steps * 4);
        row = rt64 * 64 + lane;
        block = item - rt64 * (steps * 4);
    } else {
        const int64_t rt = item / steps;
        row = rt * 16 + (lane & 15);
        block = (item - rt * steps) * 4 + (lane >> 4);
    }
    const int64_t k0 = block * kBlock;
    if (row >= rows || k0 >= k) return;
    const u32x4_t c = *(const u32x4_t *)(codes + code_at(row, block, steps));
    const float by = scale_value(scales[scale_at(row, block, steps)]);
    float v[kBlock];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const auto p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], 1.0f, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], 1.0f, 1);
        const auto p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], 1.0f, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], 1.0f, 3);
        v[8 * i] = p0[0], v[8 * i + 1] = p0[1], v[8 * i + 2] = p1[0], v[8 * i + 3] = p1[1];
        v[8 * i + 4] = p2[0], v[8 * i + 5] = p2[1], v[8 * i + 6] = p3[0], v[8 * i + 7] = p3[1];
    }
    T *p = y + row * rs + k0 * cs;
    if (cs == 1 && k0 + kBlock <= k) {
        constexpr int VE = 16 / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < kBlock / VE; ++i) {
            union { u32x4_t q; T e[VE]; } u;
#pragma unroll
            for (int j = 0; j < VE; ++j) u.e[j] = Elem<T>::from_f32(v[i * VE + j] * by);
            *(typename Unaligned<T>::vec *)(p + i * VE) = u.q;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kBlock; ++i)
            if (k0 + i < k) p[i * cs] = Elem<T>::from_f32(v[i] * by);
    }
}

int check_sizes(const char *name, int64_t rows, int64_t k) {
    if (rows < 0 || k < 0) return fail(AGH_EINVAL, "%s: negative size (%lld rows, %lld values each)", name, (long long)rows, (long long)k);
    if (!sizes_fit(rows, k)) return fail(AGH_ERANGE, "%s: %lld rows of %lld values: too many", name, (long long)rows, (long long)k);
    return AGH_OK;
}
int check_quantized(const char *name, const void *codes, const void *scales) {
    if (!codes || !scales) return fail(AGH_ENULL, "%s: null codes or scales", name);
    if (((uintptr_t)codes & 15) || ((uintptr_t)scales & 3)) return fail(AGH_EINVAL, "%s: codes must be 16-byte and scales 4-byte aligned", name);
    return AGH_OK;
}
int waves_grid(const char *name, int64_t items, unsigned &blocks) {
    const int64_t n = (items + kThreads / 64 - 1) / (kThreads / 64);
    if (n > 0x7FFFFFFFll) return fail(AGH_ERANGE, "%s: too many blocks", name);
    blocks = (unsigned)n;
    return AGH_OK;
}

template <typename T>
int quantize_entry(const char *name, const void *x, int64_t off, int64_t rs, int64_t cs, int64_t rows, int64_t k, void *codes, void *scales) {
    if (int rc = check_sizes(name, rows, k)) return rc;
    if (rows == 0 || k == 0) return AGH_OK;
    if (!x) return fail(AGH_ENULL, "%s: null input", name);
    if (int rc = check_quantized(name, codes, scales)) return rc;
    return quantize_launch<T>(name, (const T *)x + off, rs, cs, rows, k, codes, scales);
}

template <typename T>
int dequantize_entry(const char *name, const void *codes, const void *scales, int64_t rows, int64_t k, void *y, int64_t off, int64_t rs, int64_t cs) {
    if (int rc = check_sizes(name, rows, k)) return rc;
    if (rows == 0 || k == 0) return AGH_OK;
    if (!y) return fail(AGH_ENULL, "%s: null output", name);
    if ((rows > 1 && rs == 0) || (k > 1 && cs == 0)) return fail(AGH_EINVAL, "%s: the elements of y must be distinct addresses", name);
    if (int rc = check_quantized(name, codes, scales)) return rc;
    const int steps = (int)steps_of(k);
    const bool by_column = (rs < 0 ? -rs : rs) < (cs < 0 ? -cs : cs);
    const int64_t items = by_column ? (rows + 63) / 64 * steps * 4 : (rows + 15) / 16 * steps;
    unsigned blocks;
    if (int rc = waves_grid(name, items, blocks)) return rc;
    hipLaunchKernelGGL(dequantize_kernel<T>, dim3(blocks), dim3(kThreads), 0, stream(), (const unsigned char *)codes, (const unsigned char *)scales,
                       (int)rows, (int)k, steps, items, by_column, (T *)y + off, rs, cs);
    AGH_LAUNCH_CHECK(name);
    return AGH_OK;
}

}  // namespace

namespace agh {
namespace mx {

template <typename T>
int quantize_launch(const char *name, const T *x, int64_t rs, int64_t cs, int64_t rows, int64_t k, void *codes, void *scales) {
    const int steps = (int)steps_of(k);
    unsigned blocks;
    if (cs == 1) {
        const int64_t frags = (rows + 15) / 16 * steps;
        if (int rc = waves_grid(name, frags, blocks)) return rc;
        hipLaunchKernelGGL(quantize_rows_kernel<T>, dim3(blocks), dim3(kThreads), 0, stream(), x, rs, (int)rows, (int)k, steps, frags,
                           (unsigned char *)codes, (unsigned char *)scales);
    } else {
        const int64_t items = (rows + 63) / 64 * steps * 4;
        if (int rc = waves_grid(name, items, blocks)) return rc;
        hipLaunchKernelGGL(quantize_columns_kernel<T>, dim3(blocks), dim3(kThreads), 0, stream(), x, rs, cs, (int)rows, (int)k, steps, items,
                           (unsigned char *)codes, (unsigned char *)scales);
    }
    AGH_LAUNCH_CHECK(name);
    return AGH_OK;
}
template int quantize_launch<float>(const char *, const float *, int64_t, int64_t, int64_t, int64_t, void *, void *);
template int quantize_launch<uint16_t>(const char *, const uint16_t *, int64_t, int64_t, int64_t, int64_t, void *, void *);

}  // namespace mx
}  // namespace agh

extern "C" {

int agh_mxfp4_bytes(int64_t rows, int64_t k, size_t *codes, size_t *scales) {
    if (int rc = check_sizes("agh_mxfp4_bytes", rows, k)) return rc;
    if (!codes || !scales) return fail(AGH_ENULL, "agh_mxfp4_bytes: null argument");
    *codes = codes_bytes(rows, k);
    *scales = scales_bytes(rows, k);
    return AGH_OK;
}

#define AGH_MX_QUANT(SUFFIX, T)                                                                                                                   \
    int agh_quantize_mxfp4_##SUFFIX(const void *x, int64_t off_x, int64_t rs, int64_t cs, int64_t rows, int64_t k, void *codes, void *scales) {   \
        AGH_API_ENTER();                                                                                                                         \
        return quantize_entry<T>("agh_quantize_mxfp4_" #SUFFIX, x, off_x, rs, cs, rows, k, codes, scales);                                       \
    }                                                                                                                                            \
    int agh_dequantize_mxfp4_##SUFFIX(const void *codes, const void *scales, int64_t rows, int64_t k, void *y, int64_t off_y, int64_t rs,        \
                                      int64_t cs) {                                                                                              \
        AGH_API_ENTER();                                                                                                                         \
        return dequantize_entry<T>("agh_dequantize_mxfp4_" #SUFFIX, codes, scales, rows, k, y, off_y, rs, cs);                                   \
    }
AGH_MX_QUANT(f32, float)
AGH_MX_QUANT(bf16, uint16_t)

}  // extern "C"

// MXFP4: quantisation of f32 and bf16 matrices along either axis, and its inverse.
//
//   s = clamp(floor(log2 max |v|) - 2, -127, 127) over a block of 32, code = E2M1(v / 2^s) rounded half to even, magnitudes above 6 to 6.
// A block with an infinity or a NaN gets the scale byte 255 and stands for 32 NaNs: E2M1 has neither, and clipping would hide them.
// Bounded by memory: bf16 16384x4096 27 us along the rows (6.3 TB/s), its inverse 25 (6.8).
// The conversion instruction divides by 2^s, rounds and saturates; its results are compared with the formula's at every border between codes, under scales from the smallest to the largest.
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
    if (row < rows) v.load(x + row * rs, (int)k0, k);
    else v.clear();
    u32x4_t c;
    uint32_t s;
    v.quantize(c, s);
    *(u32x4_t *)(codes + frag * kFragBytes + lane * 16) = c;
    scales[scale_at(row, block, steps)] = (unsigned char)s;
}

// bf16 rows that are neighbours in memory (a matrix quantised along its columns): a workgroup takes 64 rows x 128 k, whose 128 pieces of memory, 64 values each, it
// copies to LDS in 16-byte groups.  A wave then reads a fragment of it with the reads that transpose: within 16 lanes, lanes 4 j .. 4 j + 3 name the 16 rows of k + j, and
// lane i receives row i's values of k .. k + 3; so lane l ends with the block l / 16 of row l % 16.
constexpr int kTilePitch = 160;  // bytes of 64 rows at one k: four neighbouring k lie in different banks
__global__ __launch_bounds__(kThreads) void quantize_columns_kernel(const uint16_t *__restrict__ x, int64_t cs, int rows, int k, int steps,
                                                                    unsigned char *__restrict__ codes, unsigned char *__restrict__ scales) {
    __shared__ __align__(16) unsigned char tile[kStep * kTilePitch];
    // (neighbouring workgroups take neighbouring rows: what they read together are whole rows of memory)
    const int64_t groups = ((int64_t)rows + 63) / 64, ks = blockIdx.x / groups, rt64 = blockIdx.x - ks * groups;
    const int row0 = (int)rt64 * 64, k0 = (int)ks * kStep, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int kk = i * 32 + (threadIdx.x >> 3), e = (threadIdx.x & 7) * 8;
        u32x4_t v = {0, 0, 0, 0};
        if (k0 + kk < k) v = Group<uint16_t>::load(x + (int64_t)(k0 + kk) * cs, row0 + e, rows);
        *(u32x4_t *)(tile + kk * kTilePitch + e * 2) = v;
    }
    __syncthreads();
    const int row = row0 + wave * 16 + (lane & 15);
    if (row0 + wave * 16 >= rows) return;
    typedef short s16x4_t __attribute__((ext_vector_type(4)));
    Block<uint16_t> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned char *at = tile + ((lane >> 4) * kBlock + i * 4 + (lane & 15) / 4) * kTilePitch + wave * 32 + (lane & 3) * 8;
        const s16x4_t r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t *)at);
        const u32x2_t q = __builtin_bit_cast(u32x2_t, r);
        v.v[i / 2][i % 2 * 2] = q[0];
        v.v[i / 2][i % 2 * 2 + 1] = q[1];
    }
    u32x4_t c;
    uint32_t s;
    v.quantize(c, s);
    *(u32x4_t *)(codes + (((rt64 * 4 + wave) * steps + ks) * 64 + lane) * 16) = c;
    scales[scale_at(row, ks * 4 + (lane >> 4), steps)] = (unsigned char)s;
}

// any strides: a wave takes a block of 64 rows, lane l row l
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_strided_kernel(const T *__restrict__ x, int64_t rs, int64_t cs, int rows, int k, int steps,
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
        typename Group<T>::Bits u;
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
// codes 2 I and 2 I + 1 of a dword
template <int I>
__device__ __forceinline__ void decode(uint32_t c, float by, float &lo, float &hi) {
    const auto v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, I);
    lo = v[0] * by;
    hi = v[1] * by;
}

// y's rows contiguous: a wave takes a fragment and writes whole rows of it, 128 values each, 16 bytes a lane.  Rows on whole lines of memory leave with the streaming
// hint (16384x4096 bf16 36.4 -> 26.1 us, f32 68 -> 48.7, 4096x4096 bf16 10.4 -> 8.4); of others two waves share lines, and they lose by it (bf16 16384x1032 9.0 -> 12.8,
// f32 4096x2056 8.2 -> 10.2) or gain little (f32 16384x4104 77 -> 70).
template <typename T>
__global__ __launch_bounds__(kThreads) void dequantize_rows_kernel(const unsigned char *__restrict__ codes, const unsigned char *__restrict__ scales, int rows,
                                                                   int k, int steps, int64_t frags, T *__restrict__ y, int64_t rs, bool streamed) {
    constexpr int VE = 16 / (int)sizeof(T), LANES = kStep / VE, ROWS = 64 / LANES;  // values a lane, lanes a row, rows a store instruction
    typedef typename std::conditional<VE == 8, uint32_t, uint16_t>::type Codes;     // of VE values
    const int64_t frag = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (frag >= frags) return;
    const int lane = threadIdx.x & 63, at = lane % LANES * VE, block = at / kBlock;
    const int64_t rt = frag / steps, ks = frag - rt * steps, k0 = ks * kStep + at;
    const unsigned char *from = codes + frag * kFragBytes + block * 256 + at % kBlock / 2;
    uint32_t c[16 / ROWS], s[16 / ROWS];
#pragma unroll
    for (int i = 0; i < 16 / ROWS; ++i) {
        const int r = i * ROWS + lane / LANES;
        c[i] = *(const Codes *)(from + r * 16);
        s[i] = rt * 16 + r < rows ? scales[scale_at(rt * 16 + r, ks * 4 + block, steps)] : 0;
    }
#pragma unroll
    for (int i = 0; i < 16 / ROWS; ++i) {
        const int64_t row = rt * 16 + i * ROWS + lane / LANES;
        const float by = scale_value(s[i]);
        float f[8];
        decode<0>(c[i], by, f[0], f[1]);
        decode<1>(c[i], by, f[2], f[3]);
        if constexpr (VE == 8) decode<2>(c[i], by, f[4], f[5]), decode<3>(c[i], by, f[6], f[7]);
        union { u32x4_t q; T e[VE]; } u;
#pragma unroll
        for (int j = 0; j < VE; ++j) u.e[j] = Elem<T>::from_f32(f[j]);
        if (row >= rows || k0 >= k) continue;
        T *to = y + row * rs + k0;
        if (streamed && k0 + VE <= k) __builtin_nontemporal_store(u.q, (u32x4_t *)to);
        else if (k0 + VE <= k) *(typename Unaligned<T>::vec *)to = u.q;
        else
#pragma unroll
            for (int j = 0; j < VE; ++j)
                if (k0 + j < k) to[j] = u.e[j];
    }
}

// any strides: a wave takes a block of 64 rows, lane l row l
template <typename T>
__global__ __launch_bounds__(kThreads) void dequantize_strided_kernel(const unsigned char *__restrict__ codes, const unsigned char *__restrict__ scales, int rows,
                                                                      int k, int steps, int64_t items, T *__restrict__ y, int64_t rs, int64_t cs) {
    const int64_t item = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (item >= items) return;
    const int64_t rt64 = item / (steps * 4), block = item - rt64 * (steps * 4), row = rt64 * 64 + (threadIdx.x & 63), k0 = block * kBlock;
    if (row >= rows || k0 >= k) return;
    const u32x4_t c = *(const u32x4_t *)(codes + code_at(row, block, steps));
    const float by = scale_value(scales[scale_at(row, block, steps)]);
    T *p = y + row * rs + k0 * cs;
    agh::gemm::static_for<kBlock / 2>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        float lo, hi;
        decode<i % 4>(c[i / 4], by, lo, hi);
        if (k0 + 2 * i < k) p[2 * i * cs] = Elem<T>::from_f32(lo);
        if (k0 + 2 * i + 1 < k) p[(2 * i + 1) * cs] = Elem<T>::from_f32(hi);
    });
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
// workgroups of four waves; sizes_fit keeps them below 2^24
unsigned waves_grid(int64_t items) { return (unsigned)((items + kThreads / 64 - 1) / (kThreads / 64)); }

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
    const unsigned char *c = (const unsigned char *)codes, *s = (const unsigned char *)scales;
    T *to = (T *)y + off;
    const int64_t items = cs == 1 ? (rows + 15) / 16 * steps : (rows + 63) / 64 * steps * 4;
    const unsigned blocks = waves_grid(items);
    if (cs == 1)
        hipLaunchKernelGGL(dequantize_rows_kernel<T>, dim3(blocks), dim3(kThreads), 0, stream(), c, s, (int)rows, (int)k, steps, items, to, rs,
                           ((uintptr_t)to | (uint64_t)rs * sizeof(T)) % 128 == 0);
    else
        hipLaunchKernelGGL(dequantize_strided_kernel<T>, dim3(blocks), dim3(kThreads), 0, stream(), c, s, (int)rows, (int)k, steps, items, to, rs, cs);
    AGH_LAUNCH_CHECK(name);
    return AGH_OK;
}

}  // namespace

namespace agh {
namespace mx {

template <typename T>
int quantize_launch(const char *name, const T *x, int64_t rs, int64_t cs, int64_t rows, int64_t k, void *codes, void *scales) {
    const int steps = (int)steps_of(k);
    if (cs == 1) {
        const int64_t frags = (rows + 15) / 16 * steps;
        hipLaunchKernelGGL(quantize_rows_kernel<T>, dim3(waves_grid(frags)), dim3(kThreads), 0, stream(), x, rs, (int)rows, (int)k, steps, frags,
                           (unsigned char *)codes, (unsigned char *)scales);
        AGH_LAUNCH_CHECK(name);
        return AGH_OK;
    }
    if constexpr (sizeof(T) == 2) {
        if (rs == 1 && rows >= 16) {
            hipLaunchKernelGGL(quantize_columns_kernel, dim3((unsigned)((rows + 63) / 64 * steps)), dim3(kThreads), 0, stream(), x, cs, (int)rows, (int)k, steps, (unsigned char *)codes,
                               (unsigned char *)scales);
            AGH_LAUNCH_CHECK(name);
            return AGH_OK;
        }
    }
    const int64_t items = (rows + 63) / 64 * steps * 4;
    hipLaunchKernelGGL(quantize_strided_kernel<T>, dim3(waves_grid(items)), dim3(kThreads), 0, stream(), x, rs, cs, (int)rows, (int)k, steps, items, (unsigned char *)codes,
                       (unsigned char *)scales);
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

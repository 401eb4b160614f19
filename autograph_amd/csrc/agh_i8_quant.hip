// 8-bit integers with a scale for each row: quantisation of f32 and bf16 matrices along either axis, and its inverse.
//
//   scale = max |x| / 127 over a row, code = 127 x / max |x| to the nearest whole number (agh_i8_quant.h)
// A row with an infinity or a NaN gets the scale NaN and codes 0: it stands for NaNs.  A row of zeros gets the scale 0.
// A row is passed over twice, for its largest magnitude and for its codes: once out of memory, and then out of registers or, where it is longer than a workgroup holds, out of memory again.  Bounded
// by memory: bf16 16384x4096 along the rows 32.5 us (6.2 TB/s), f32 65; 16384x8192, read twice, 104 and 175; along the columns, k 4096 of 16384, 47 and 90, where a lane's 16 values of a
// chunk are as many loads.
#include "agh_i8_quant.h"

using namespace agh;
using namespace agh::i8;

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

__device__ __forceinline__ int64_t code_at(int64_t row, int64_t chunk, int64_t steps) {
    return (((row >> 4) * steps + (chunk >> 2)) * 64 + (chunk & 3) * 16 + (row & 15)) * 16;
}

// k contiguous: a workgroup takes R rows, lane l row l % R and the chunk l / R of 64 / R neighbours; four rows' chunks lie next to each other in a fragment.  A thread
// holds HELD chunks, so that rows of up to HELD * kThreads / R chunks are read once.
template <typename T, int R, int HELD>
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(const T *__restrict__ x, int64_t rs, int rows, int k, int steps, unsigned char *__restrict__ codes,
                                                                 float *__restrict__ scales) {
    __shared__ uint32_t tops[kWaves][R];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane % R;
    const int64_t row = (int64_t)blockIdx.x * R + r;
    const bool live = row < rows;
    const T *p = x + (live ? row : (int64_t)rows - 1) * rs;
    const int padded = steps * kStep;
    // the thread's i-th chunk starts at k
    auto at = [&](int i) __attribute__((always_inline)) { return ((i * kWaves + wave) * (64 / R) + lane / R) * kChunk; };
    Chunk<T> v[HELD];
    auto hold = [&](int first) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            if (at(first + i) < k) v[i].load(p, at(first + i), k);
            else v[i].clear();
        }
    };
    const int chunks = (padded / kChunk + kWaves * (64 / R) - 1) / (kWaves * (64 / R));  // a thread's
    uint32_t top = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < chunks; i0 += HELD) {
        hold(i0);
#pragma unroll
        for (int i = 0; i < HELD; ++i) top = max(top, v[i].most());
    }
#pragma unroll
    for (int o = R; o < 64; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    if (lane < R) tops[wave][lane] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = max(top, tops[w][r]);
    const RowScale s(top);
    if (!live) return;
    if (threadIdx.x < R) scales[row] = s.scale;
#pragma unroll 1
    for (int i0 = 0; i0 < chunks; i0 += HELD) {
        if (chunks > HELD) hold(i0);
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (at(i0 + i) < padded) *(u32x4_t *)(codes + code_at(row, at(i0 + i) / kChunk, steps)) = v[i].quantize(s);
    }
}

// any strides: a workgroup takes 64 rows, lane l row l (rows that are neighbours in memory are read together), the waves share the chunks
template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_strided_kernel(const T *__restrict__ x, int64_t rs, int64_t cs, int rows, int k, int steps,
                                                                    unsigned char *__restrict__ codes, float *__restrict__ scales) {
    __shared__ uint32_t tops[kWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * 64 + lane;
    const bool live = row < rows;
    const T *p = x + (live ? row : (int64_t)rows - 1) * rs;
    uint32_t top = 0;
    Chunk<T> v;
    for (int c = wave; c * kChunk < k; c += kWaves) {
        v.load_strided(p, cs, c * kChunk, k);
        top = max(top, v.most());
    }
    tops[wave][lane] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = max(top, tops[w][lane]);
    const RowScale s(top);
    if (!live) return;
    if (wave == 0) scales[row] = s.scale;
    for (int c = wave; c < steps * (kStep / kChunk); c += kWaves) {
        if (c * kChunk < k) v.load_strided(p, cs, c * kChunk, k);
        else v.clear();
        *(u32x4_t *)(codes + code_at(row, c, steps)) = v.quantize(s);
    }
}

// The same where k is short enough for one workgroup of 16 waves to hold the values of R rows, a thread HELD chunks, which are read once (ColumnForm).
template <typename T, int R, int HELD>
__global__ __launch_bounds__(kColumnThreads) void quantize_columns_kernel(const T *__restrict__ x, int64_t rs, int64_t cs, int rows, int k, int steps,
                                                                          unsigned char *__restrict__ codes, float *__restrict__ scales) {
    constexpr int WAVES = kColumnThreads / 64;
    __shared__ uint32_t tops[WAVES][R];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane % R;
    // a run of groups for every XCD (workgroup id mod 8): neighbours share lines of memory
    int id = blockIdx.x;
    {
        const int n = gridDim.x, xcd = id & 7;
        id = xcd * (n >> 3) + min(xcd, n & 7) + (id >> 3);
    }
    const int64_t row = (int64_t)id * R + r;
    const bool live = row < rows;
    const T *p = x + (live ? row : (int64_t)rows - 1) * rs;
    auto at = [&](int i) __attribute__((always_inline)) { return (i * WAVES + wave) * (64 / R) + lane / R; };  // the thread's i-th chunk
    Chunk<T> v[HELD];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        if (at(i) * kChunk < k) v[i].load_strided(p, cs, at(i) * kChunk, k);
        else v[i].clear();
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i) top = max(top, v[i].most());
#pragma unroll
    for (int o = R; o < 64; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
    if (lane < R) tops[wave][lane] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = max(top, tops[w][r]);
    const RowScale s(top);
    if (!live) return;
    if (threadIdx.x < R) scales[row] = s.scale;
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (at(i) < steps * (kStep / kChunk)) *(u32x4_t *)(codes + code_at(row, at(i), steps)) = v[i].quantize(s);
}

// The same in two launches, for few rows that are long: a workgroup takes a share of k of 64 rows.  The first finds the shares' largest magnitudes, tops[share][row], the
// second the codes.
template <typename T, bool CODES>
__global__ __launch_bounds__(kThreads) void quantize_shares_kernel(const T *__restrict__ x, int64_t rs, int64_t cs, int rows, int k, int steps, Shares shares,
                                                                   uint32_t *__restrict__ tops, unsigned char *__restrict__ codes, float *__restrict__ scales) {
    __shared__ uint32_t mine[kWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, groups = (rows + 63) / 64;
    // (neighbouring workgroups take neighbouring rows: what they read together are whole rows of memory)
    const int share = (int)blockIdx.x / groups, first = share * shares.each, last = first + shares.each;
    const int64_t row = (int64_t)((int)blockIdx.x - share * groups) * 64 + lane;
    const bool live = row < rows;
    const T *p = x + (live ? row : (int64_t)rows - 1) * rs;
    uint32_t top = 0;
    Chunk<T> v;
    if constexpr (!CODES) {
        for (int c = first + wave; c < last && c * kChunk < k; c += kWaves) {
            v.load_strided(p, cs, c * kChunk, k);
            top = max(top, v.most());
        }
    } else if (live) {
        for (int i = wave; i < shares.count; i += kWaves) top = max(top, tops[(int64_t)i * rows + row]);
    }
    mine[wave][lane] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = max(top, mine[w][lane]);
    if (!live) return;
    if constexpr (!CODES) {
        if (wave == 0) tops[(int64_t)share * rows + row] = top;
    } else {
        const RowScale s(top);
        if (wave == 0 && share == 0) scales[row] = s.scale;
        for (int c = first + wave; c < last && c < steps * (kStep / kChunk); c += kWaves) {
            if (c * kChunk < k) v.load_strided(p, cs, c * kChunk, k);
            else v.clear();
            *(u32x4_t *)(codes + code_at(row, c, steps)) = v.quantize(s);
        }
    }
}

// value i of a dword of codes
template <typename T>
__device__ __forceinline__ T value_of(uint32_t codes, int i, float scale) { return Elem<T>::from_f32((float)((int32_t)(codes << (24 - 8 * i)) >> 24) * scale); }

// y's rows contiguous: a workgroup takes 8 rows' share of a few hundred values, lane l row l % 8 and a 16-byte group of y, the l / 8 th of 8 neighbours (a line of memory), U
// of them together.  Rows on whole lines of memory leave with the streaming hint.  (bf16 16384x4096 30.2 us, 6.7 TB/s; four rows and 16 neighbours 40.6; whole rows
// instead of shares of them 34.2, and 300x16384 17.6 instead of 4.6.)
template <typename T>
struct Dequantize {
    static constexpr int ROWS = 8, VE = 16 / (int)sizeof(T), U = 4, SPAN = 64 / ROWS * VE, SHARE = U * kWaves * SPAN;
};
template <typename T>
__global__ __launch_bounds__(kThreads) void dequantize_rows_kernel(const unsigned char *__restrict__ codes, const float *__restrict__ scales, int rows, int k, int steps, int shares,
                                                                   T *__restrict__ y, int64_t rs, bool streamed) {
    constexpr int ROWS = Dequantize<T>::ROWS, VE = Dequantize<T>::VE, U = Dequantize<T>::U, SPAN = Dequantize<T>::SPAN, SHARE = Dequantize<T>::SHARE;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = (int)blockIdx.x / shares, share = (int)blockIdx.x - group * shares;
    const int64_t row = (int64_t)group * ROWS + lane % ROWS;
    const int64_t at = (int64_t)share * SHARE + wave * SPAN + lane / ROWS * VE;
    if (row >= rows || at >= k) return;
    const int first = (int)at;
    const float s = scales[row];
    T *to = y + row * rs;
    uint32_t c[U][VE / 4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int k0 = min(first + u * kWaves * SPAN, k - 1) / VE * VE;
        const unsigned char *from = codes + code_at(row, k0 / kChunk, steps) + k0 % kChunk;
        if constexpr (VE == 8) {
            const uint2 v = *(const uint2 *)from;
            c[u][0] = v.x;
            c[u][1] = v.y;
        } else c[u][0] = *(const uint32_t *)from;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int k0 = first + u * kWaves * SPAN;
        if (k0 >= k) break;
        union { u32x4_t q; T e[VE]; } v;
#pragma unroll
        for (int j = 0; j < VE; ++j) v.e[j] = value_of<T>(c[u][j / 4], j % 4, s);
        if (k0 + VE <= k) {
            if (streamed) __builtin_nontemporal_store(v.q, (u32x4_t *)(to + k0));
            else *(typename Unaligned<T>::vec *)(to + k0) = v.q;
        } else
#pragma unroll
            for (int j = 0; j < VE; ++j)
                if (k0 + j < k) to[k0 + j] = v.e[j];
    }
}

// any strides: a wave takes a chunk of 64 rows, lane l row l
template <typename T>
__global__ __launch_bounds__(kThreads) void dequantize_strided_kernel(const unsigned char *__restrict__ codes, const float *__restrict__ scales, int rows, int k, int steps,
                                                                      int64_t items, T *__restrict__ y, int64_t rs, int64_t cs) {
    const int64_t item = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6), groups = ((int64_t)rows + 63) / 64;
    if (item >= items) return;
    const int64_t chunk = item / groups, row = (item - chunk * groups) * 64 + (threadIdx.x & 63);
    if (row >= rows) return;
    const float s = scales[row];
    const u32x4_t c = *(const u32x4_t *)(codes + code_at(row, chunk, steps));
    T *to = y + row * rs + chunk * kChunk * cs;
#pragma unroll
    for (int i = 0; i < kChunk; ++i)
        if (chunk * kChunk + i < k) to[i * cs] = value_of<T>(c[i / 4], i % 4, s);
}

int check_sizes(const char *name, int64_t rows, int64_t k) {
    if (rows < 0 || k < 0) return fail(AGH_EINVAL, "%s: negative size (%lld rows, %lld values each)", name, (long long)rows, (long long)k);
    if (k >= ((int64_t)1 << 31) - 512 || !rows_fit(rows, k)) return fail(AGH_ERANGE, "%s: %lld rows of %lld values: too many", name, (long long)rows, (long long)k);
    return AGH_OK;
}
int check_quantized(const char *name, const void *codes, const void *scales) {
    if (!codes || !scales) return fail(AGH_ENULL, "%s: null codes or scales", name);
    if ((codes != scales && ((uintptr_t)codes & 15)) || ((uintptr_t)scales & 3)) return fail(AGH_EINVAL, "%s: codes must be 16-byte and scales 4-byte aligned", name);
    return AGH_OK;
}

template <typename T>
int quantize_entry(const char *name, const void *x, int64_t off, int64_t rs, int64_t cs, int64_t rows, int64_t k, void *codes, void *scales) {
    if (int rc = check_sizes(name, rows, k)) return rc;
    if (rows == 0) return AGH_OK;
    if (k > 0 && !x) return fail(AGH_ENULL, "%s: null input", name);
    if (int rc = check_quantized(name, k > 0 ? codes : scales, scales)) return rc;  // (without values there are no codes either)
    void *scratch = nullptr;
    if (const size_t bytes = scratch_bytes<T>(rows, k, cs))
        if (int rc = workspace(bytes, &scratch)) return rc;
    return quantize_launch<T>(name, k > 0 ? (const T *)x + off : nullptr, rs, cs, rows, k, codes, (float *)scales, scratch);
}

template <typename T>
int dequantize_entry(const char *name, const void *codes, const void *scales, int64_t rows, int64_t k, void *y, int64_t off, int64_t rs, int64_t cs) {
    if (int rc = check_sizes(name, rows, k)) return rc;
    if (rows == 0 || k == 0) return AGH_OK;
    if (!y) return fail(AGH_ENULL, "%s: null output", name);
    if ((rows > 1 && rs == 0) || (k > 1 && cs == 0)) return fail(AGH_EINVAL, "%s: the elements of y must be distinct addresses", name);
    if (int rc = check_quantized(name, codes, scales)) return rc;
    const int steps = (int)steps_of(k);
    T *to = (T *)y + off;
    if (cs == 1) {
        const int64_t groups = (rows + Dequantize<T>::ROWS - 1) / Dequantize<T>::ROWS, shares = (k + Dequantize<T>::SHARE - 1) / Dequantize<T>::SHARE;
        hipLaunchKernelGGL(dequantize_rows_kernel<T>, dim3((unsigned)(groups * shares)), dim3(kThreads), 0, stream(), (const unsigned char *)codes,
                           (const float *)scales, (int)rows, (int)k, steps, (int)shares, to, rs, ((uintptr_t)to | (uint64_t)rs * sizeof(T)) % 128 == 0);
    } else {
        const int64_t items = (rows + 63) / 64 * ((k + kChunk - 1) / kChunk);
        hipLaunchKernelGGL(dequantize_strided_kernel<T>, dim3((unsigned)((items + kWaves - 1) / kWaves)), dim3(kThreads), 0, stream(), (const unsigned char *)codes,
                           (const float *)scales, (int)rows, (int)k, steps, items, to, rs, cs);
    }
    AGH_LAUNCH_CHECK(name);
    return AGH_OK;
}

}  // namespace

namespace agh {
namespace i8 {

template <typename T>
int quantize_launch(const char *name, const T *x, int64_t rs, int64_t cs, int64_t rows, int64_t k, void *codes, float *scales, void *scratch) {
    const int steps = (int)steps_of(k);
    if (cs == 1) {
        // a row a workgroup where that leaves CUs to spare, else four
        auto launch = [&](auto rc, auto hc) {
            constexpr int R = decltype(rc)::value;
            hipLaunchKernelGGL((quantize_rows_kernel<T, R, decltype(hc)::value>), dim3((unsigned)((rows + R - 1) / R)), dim3(kThreads), 0, stream(), x, rs, (int)rows, (int)k, steps,
                               (unsigned char *)codes, scales);
        };
        typedef std::integral_constant<int, 1> One;
        typedef std::integral_constant<int, 2> Two;
        typedef std::integral_constant<int, 4> Four;
        if (rows <= 2 * compute_units()) launch(One{}, Two{});
        else if (k <= 2048) launch(Four{}, Two{});
        else launch(Four{}, Four{});
    } else if (const ColumnForm<T> form(rows, k); form.rows) {
        auto launch = [&](auto rc, auto hc) {
            constexpr int R = decltype(rc)::value;
            hipLaunchKernelGGL((quantize_columns_kernel<T, R, decltype(hc)::value>), dim3((unsigned)((rows + R - 1) / R)), dim3(kColumnThreads), 0, stream(), x, rs, cs, (int)rows, (int)k,
                               steps, (unsigned char *)codes, scales);
        };
        auto held = [&](auto rc) {
            if (form.held == 1) {
                if constexpr (decltype(rc)::value == ColumnForm<T>::NARROW) launch(rc, std::integral_constant<int, 1>{});
            } else if (form.held == 2) launch(rc, std::integral_constant<int, 2>{});
            else launch(rc, std::integral_constant<int, 4>{});
        };
        constexpr int NARROW = ColumnForm<T>::NARROW;
        if (form.rows == NARROW) held(std::integral_constant<int, NARROW>{});
        else held(std::integral_constant<int, 2 * NARROW>{});
    } else if (const Shares shares(rows, k); shares.count <= 2) {
        hipLaunchKernelGGL(quantize_strided_kernel<T>, dim3((unsigned)((rows + 63) / 64)), dim3(kThreads), 0, stream(), x, rs, cs, (int)rows, (int)k, steps, (unsigned char *)codes,
                           scales);
    } else {
        const dim3 grid((unsigned)((rows + 63) / 64 * shares.count));
        hipLaunchKernelGGL((quantize_shares_kernel<T, false>), grid, dim3(kThreads), 0, stream(), x, rs, cs, (int)rows, (int)k, steps, shares, (uint32_t *)scratch,
                           (unsigned char *)codes, scales);
        AGH_LAUNCH_CHECK(name);
        hipLaunchKernelGGL((quantize_shares_kernel<T, true>), grid, dim3(kThreads), 0, stream(), x, rs, cs, (int)rows, (int)k, steps, shares, (uint32_t *)scratch,
                           (unsigned char *)codes, scales);
    }
    AGH_LAUNCH_CHECK(name);
    return AGH_OK;
}
template int quantize_launch<float>(const char *, const float *, int64_t, int64_t, int64_t, int64_t, void *, float *, void *);
template int quantize_launch<uint16_t>(const char *, const uint16_t *, int64_t, int64_t, int64_t, int64_t, void *, float *, void *);

}  // namespace i8
}  // namespace agh

extern "C" {

int agh_int8_bytes(int64_t rows, int64_t k, size_t *codes, size_t *scales) {
    if (int rc = check_sizes("agh_int8_bytes", rows, k)) return rc;
    if (!codes || !scales) return fail(AGH_ENULL, "agh_int8_bytes: null argument");
    *codes = codes_bytes(rows, k);
    *scales = scales_bytes(rows);
    return AGH_OK;
}

#define AGH_I8_QUANT(SUFFIX, T)                                                                                                                  \
    int agh_quantize_int8_##SUFFIX(const void *x, int64_t off_x, int64_t rs, int64_t cs, int64_t rows, int64_t k, void *codes, void *scales) {   \
        AGH_API_ENTER();                                                                                                                        \
        return quantize_entry<T>("agh_quantize_int8_" #SUFFIX, x, off_x, rs, cs, rows, k, codes, scales);                                       \
    }                                                                                                                                           \
    int agh_dequantize_int8_##SUFFIX(const void *codes, const void *scales, int64_t rows, int64_t k, void *y, int64_t off_y, int64_t rs,        \
                                     int64_t cs) {                                                                                              \
        AGH_API_ENTER();                                                                                                                        \
        return dequantize_entry<T>("agh_dequantize_int8_" #SUFFIX, codes, scales, rows, k, y, off_y, rs, cs);                                   \
    }
AGH_I8_QUANT(f32, float)
AGH_I8_QUANT(bf16, uint16_t)

}  // extern "C"

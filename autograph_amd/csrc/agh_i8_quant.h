// 8-bit integer operands: a chunk of 16 values in one lane's registers, and its quantisation by a row's largest magnitude.
//
//   code = 127 x / most, to the nearest whole number, half to even: decided exactly.
// bf16: 127 x has 15 bits and is exact; the quotient of that and `most` is corrected once by its remainder, which is exact too, so that it is rounded once.  A quotient
// of two such numbers that is no half lies at least 2^-17 of its size beside it, so it does not round to one.
// f32: t = 127 x * (1 / most) is within 2^-15 of the quotient (three roundings of at most 127).  Where it lies that near to a half n + 1/2, the sign of
// 127 x - (n + 1/2) most decides: with 127 x as a sum p + rest of two floats, p - (n + 1/2) most is a small multiple of the last bits of both and exact in one fma, and the
// sum with `rest` keeps its sign.
#pragma once
#include "agh_gemm_kernel.h"
#include "agh_i8.h"

namespace agh {
namespace i8 {

// what a row's largest magnitude says: as bits of f32, so that a NaN's are above infinity's and those above every number's
struct RowScale {
    float most, inv;  // the largest magnitude and its reciprocal, of x * up
    float times;      // 127 up: up = 2^100 where the reciprocal would pass f32 or the remainder lose its last bits, 2^-60 where 127 x would pass it, else 1
    float scale;      // most / 127, or NaN for a row that holds an infinity or a NaN: it stands for NaNs
                      // (of f32's largest value the f32 below that quotient: 127 times the nearest one is infinity)
    uint32_t keep;    // of the codes: none of such a row
    __device__ __forceinline__ explicit RowScale(uint32_t bits) {
        const bool bad = bits >= 0x7F800000u;
        const float m = bad ? 0.0f : __uint_as_float(bits), up = m < 0x1p-90f ? 0x1p100f : m > 0x1p90f ? 0x1p-60f : 1.0f;
        scale = bad ? __uint_as_float(0x7FC00000u) : fminf(m / 127.0f, 0x1.020406p+121f);
        keep = bad ? 0u : 0xFFFFFFFFu;
        most = m * up;
        inv = most > 0.0f ? 1.0f / most : 0.0f;  // (a row of zeros: codes 0)
        times = 127.0f * up;
    }
};

// the codes of N neighbouring values of one row, four in a dword
template <typename T, int N, typename Get>
__device__ __forceinline__ void codes_of(Get get, const RowScale &r, uint32_t (&codes)[N / 4]) {
    // adding 1.5 * 2^23 rounds to a whole number, half to even, and leaves it in the low bits in two's complement
    constexpr float kWhole = 12582912.0f;
    uint32_t q[N];
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float p = get(i) * r.times, t = p * r.inv;
            q[i] = __float_as_uint(__builtin_fmaf(__builtin_fmaf(-t, r.most, p), r.inv, t) + kWhole);
        }
    } else {
        float far = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float t = get(i) * r.times * r.inv, whole = t + kWhole;
            q[i] = __float_as_uint(whole);
            far = fmaxf(far, fabsf(t - (whole - kWhole)));
        }
        if (far > 0.5f - 0x1p-15f)  // some value next to a half
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float x = get(i), p = x * r.times, rest = __builtin_fmaf(x, r.times, -p), t = p * r.inv, n = floorf(t);
                const float over = __builtin_fmaf(-(n + 0.5f), r.most, p) + rest;
                if (fabsf(t - n - 0.5f) < 0x1p-14f) q[i] = (uint32_t)(int)n + (over > 0.0f || (over == 0.0f && ((int)n & 1)) ? 1u : 0u);
            }
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
        codes[i] = r.keep & __builtin_amdgcn_perm(__builtin_amdgcn_perm(q[4 * i + 3], q[4 * i + 2], 0x0C0C0400u), __builtin_amdgcn_perm(q[4 * i + 1], q[4 * i], 0x0C0C0400u), 0x05040100u);
}
// of a 16-byte group: 8 of bf16, 4 of f32
template <typename T>
__device__ __forceinline__ uint2 quantize8(u32x4_t v, const RowScale &r) {
    uint32_t c[2];
    codes_of<T, 8>([&](int i) { return Group<T>::get(v, i); }, r, c);
    return make_uint2(c[0], c[1]);
}
template <typename T>
__device__ __forceinline__ uint32_t quantize4(u32x4_t v, const RowScale &r) {
    uint32_t c[1];
    codes_of<T, 4>([&](int i) { return Group<T>::get(v, i); }, r, c);
    return c[0];
}

template <typename T>
struct Chunk {
    static constexpr int VE = Group<T>::VE, NV = kChunk / VE;
    u32x4_t v[NV];
    // elements k0 .. of a row of k, zeros behind its end
    __device__ __forceinline__ void load(const T *row, int k0, int k) {
        if (k0 + kChunk <= k) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = *(const typename Group<T>::vec *)(row + k0 + i * VE);
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = Group<T>::load(row, k0 + i * VE, k);
        }
    }
    __device__ __forceinline__ void load_strided(const T *row, int64_t cs, int k0, int k) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            typename Group<T>::Bits u;
#pragma unroll
            for (int j = 0; j < VE; ++j) u.e[j] = k0 + i * VE + j < k ? row[(k0 + i * VE + j) * cs] : (T)0;
            v[i] = u.q;
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = u32x4_t{0, 0, 0, 0};
    }
    __device__ __forceinline__ float get(int i) const { return Group<T>::get(v[i / VE], i % VE); }
    // the bits of the largest magnitude, as f32
    __device__ __forceinline__ uint32_t most() const {
        if constexpr (sizeof(T) == 4) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < kChunk; ++i) m = max(m, v[i / 4][i % 4] & 0x7FFFFFFFu);
            return m;
        } else {  // two at a time
            typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
            u16x2_t m = {0, 0};
#pragma unroll
            for (int i = 0; i < kChunk / 2; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, v[i / 4][i % 4] & 0x7FFF7FFFu));
            return (uint32_t)max(m[0], m[1]) << 16;
        }
    }
    // its 16 codes, in order
    __device__ __forceinline__ u32x4_t quantize(const RowScale &r) const {
        uint32_t c[kChunk / 4];
        codes_of<T, kChunk>([&](int i) { return get(i); }, r, c);
        return u32x4_t{c[0], c[1], c[2], c[3]};
    }
};

}  // namespace i8
}  // namespace agh

// MXFP4: a block of 32 values in one lane's registers, and its quantisation.
#pragma once
#include "agh_gemm_kernel.h"
#include "agh_mx.h"

namespace agh {
namespace mx {

// the 16-byte groups of a block, as they were loaded
template <typename T>
struct Block {
    static constexpr int VE = Group<T>::VE, NV = kBlock / VE;
    u32x4_t v[NV];
    // elements k0 .. of a row of k, zeros behind its end
    __device__ __forceinline__ void load(const T *row, int k0, int k) {
        if (k0 + kBlock <= k) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = *(const typename Group<T>::vec *)(row + k0 + i * VE);
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = Group<T>::load(row, k0 + i * VE, k);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = u32x4_t{0, 0, 0, 0};
    }
    __device__ __forceinline__ float get(int i) const { return Group<T>::get(v[i / VE], i % VE); }
    // the bits of the largest magnitude, as f32: a NaN's are above infinity's, those above every number's
    __device__ __forceinline__ uint32_t most() const {
        if constexpr (sizeof(T) == 4) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < kBlock; ++i) m = max(m, v[i / 4][i % 4] & 0x7FFFFFFFu);
            return m;
        } else {  // two at a time
            typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
            u16x2_t m = {0, 0};
#pragma unroll
            for (int i = 0; i < kBlock / 2; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, v[i / 4][i % 4] & 0x7FFF7FFFu));
            return (uint32_t)max(m[0], m[1]) << 16;
        }
    }
    // its 32 codes and its scale byte
    __device__ __forceinline__ void quantize(u32x4_t &codes, uint32_t &scale) const {
        const uint32_t e = most() >> 23;                       // 0: zero or subnormal, below 2^-126: the scale is held to 2^-127
        scale = e == 255u ? 255u : e < 2u ? 0u : e - 2u;
        // the conversion divides by 2^(scale - 127), which it takes from the exponent bits of a float, and rounds half to even, larger values to 6
        const bool bad = scale == 255u;
        const float by = __uint_as_float(bad ? 0u : scale << 23);
        agh::gemm::static_for<4>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            uint32_t c = 0;
            if constexpr (sizeof(T) == 4) {
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, get(8 * i), get(8 * i + 1), by, 0);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, get(8 * i + 2), get(8 * i + 3), by, 1);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, get(8 * i + 4), get(8 * i + 5), by, 2);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, get(8 * i + 6), get(8 * i + 7), by, 3);
            } else {
                // (the pairs by value: a bit cast of a vector's element takes the vector's first)
                typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
                const uint32_t p0 = v[i][0], p1 = v[i][1], p2 = v[i][2], p3 = v[i][3];
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, p0), by, 0);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, p1), by, 1);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, p2), by, 2);
                c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, p3), by, 3);
            }
            codes[i] = bad ? 0u : c;
        });
    }
};

}  // namespace mx
}  // namespace agh

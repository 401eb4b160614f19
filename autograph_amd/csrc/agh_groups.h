// 16-byte groups of a row that may start at any element's address and end inside a group.
#pragma once
#include "agh_internal.h"

namespace agh {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// 16 bytes at any element's address
template <typename T> struct Unaligned;
template <> struct Unaligned<float> { typedef u32x4_t vec __attribute__((aligned(4))); };
template <> struct Unaligned<uint16_t> { typedef u32x4_t vec __attribute__((aligned(2))); };

template <typename T>
struct Group {
    static constexpr int VE = 16 / (int)sizeof(T);
    typedef typename Unaligned<T>::vec vec;
    union Bits { u32x4_t q; T e[VE]; };

    // Elements e .. e + VE - 1 of a row of `cols`, zeros behind its end.  A group that passes the end is read from where it would end there, and shifted: one load
    // whatever the group, behind no branch, so that many can be in flight (element by element, each load of a short group waited for the one
    // before: layer norm of bf16 16384x1022 20 us).
    static __device__ __forceinline__ u32x4_t load(const T *row, int e, int cols) {
        if (cols < VE) {
            Bits b;
            b.q = u32x4_t{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < VE; ++i)
                if (e + i < cols) b.e[i] = row[e + i];
            return b.q;
        }
        const int at = min(e, cols - VE);
        u32x4_t v = *(const vec *)(row + at);
        if (at != e) v = shifted(v, e - at);
        return v;
    }
    // by s >= 1 elements towards the first
    static __device__ __forceinline__ u32x4_t shifted(u32x4_t v, int s) {
        const int d = s * (int)sizeof(T) / 4;  // whole dwords
        if (d & 2) v = u32x4_t{v[2], v[3], 0, 0};
        if (d & 1) v = u32x4_t{v[1], v[2], v[3], 0};
        if (sizeof(T) == 2 && (s & 1))
            v = u32x4_t{__builtin_amdgcn_alignbit(v[1], v[0], 16), __builtin_amdgcn_alignbit(v[2], v[1], 16), __builtin_amdgcn_alignbit(v[3], v[2], 16), v[3] >> 16};
        return s >= VE ? u32x4_t{0, 0, 0, 0} : v;
    }
    static __device__ __forceinline__ float get(u32x4_t v, int i) {
        if constexpr (sizeof(T) == 4) return __uint_as_float(v[i]);
        else return __uint_as_float(i & 1 ? v[i / 2] & 0xFFFF0000u : v[i / 2] << 16);
    }
    static __device__ __forceinline__ u32x4_t pack(const float (&f)[VE]) {
        u32x4_t v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) v[i] = __float_as_uint(f[i]);
            else v[i] = f32x2_to_bf16x2(f[2 * i], f[2 * i + 1]);
        }
        return v;
    }
};

}  // namespace agh

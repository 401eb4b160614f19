// MXFP4 operands: how they lie in memory, shared by the quantiser and the product.
//
// A matrix of `rows` rows quantised along k (blocks of 32 values, one scale byte each) is two arrays:
//   codes   fragments of 16 rows x 128 k, 1024 bytes each, row tile by row tile, k ascending: the 16 bytes (32 codes, the even k in the low
//           half of a byte) of row r, block b are at ((r / 16 * steps + b / 4) * 64 + b % 4 * 16 + r % 16) * 16, steps = ceil(k / 128)
//   scales  pieces of 64 rows x 128 k, 256 bytes each: the byte of row r, block b is at
//           ((r / 64 * steps + b / 4) * 64 + b % 4 * 16 + r % 16) * 4 + r / 16 % 4
// A fragment is what one v_mfma_scale_f32_16x16x128_f8f6f4 takes of an operand, lane l (row l % 16, block l / 16) at byte 16 l: a wave reads it with
// one 16-byte load a lane, from memory or from LDS, without gaps, bank conflicts or address arithmetic.  The instruction takes a lane's scale from
// a byte of a register that it names itself, so the dword that lane l reads of a piece serves the four fragments of 64 rows.
// Blocks behind k (the last 128 are always whole) hold zeros and the scale byte 0; what rows behind the last one hold is never used.
#pragma once
#include "agh_groups.h"

namespace agh {
namespace mx {

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kBlock = 32;    // values that share a scale
constexpr int kStep = 128;    // k of a fragment
constexpr int kFragBytes = 1024, kPieceBytes = 256;

inline int64_t steps_of(int64_t k) { return (k + kStep - 1) / kStep; }
inline size_t codes_bytes(int64_t rows, int64_t k) { return (size_t)((rows + 15) / 16) * (size_t)steps_of(k) * kFragBytes; }
inline size_t scales_bytes(int64_t rows, int64_t k) { return (size_t)((rows + 63) / 64) * (size_t)steps_of(k) * kPieceBytes; }

// rows and k of a quantised matrix: int indexes of fragments, rows and k, and a workgroup of 256 for each 64 rows x 128 k (a launch counts its work items in 32 bits)
inline bool sizes_fit(int64_t rows, int64_t k) {
    return rows < ((int64_t)1 << 31) - 512 && k < ((int64_t)1 << 31) - 512 && (rows + 63) / 64 * steps_of(k) < (1 << 24);
}

// quantises x (rows x k, element strides) into codes and scales on the current stream; arguments have been checked
template <typename T>
int quantize_launch(const char *name, const T *x, int64_t rs, int64_t cs, int64_t rows, int64_t k, void *codes, void *scales);

}  // namespace mx
}  // namespace agh

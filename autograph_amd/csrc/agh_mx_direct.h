// MXFP4 product straight from memory, for results of few tiles: a workgroup's WK waves share one tile of 16 TP x 16 TQ and split k among themselves, so nothing that
// one of them reads is of use to another, and fragments go from memory into the registers that the matrix instruction reads.  Their sums meet in LDS, added
// in the waves' order.  With few rows of a (one token, a handful of requests) this is one pass over b: 1x4096x4096 with the
// quantisation 4.7 us, 1.9 TB/s.  A wave has 4 steps there and takes U = 2 at a time: two waits for memory, in each of which the second step's weights are requested
// behind the first step's values of a, and then the quantisation and the joining of the sums, one behind the other.
//
// RAW: a is not quantised yet.  A lane quantises what its place in the fragment holds, 32 neighbours of one row, so the values never leave its
// registers; every workgroup does it again, which for few rows is less than a launch of its own.
#pragma once
#include "agh_mx_quant.h"
#include "agh_mx_tile.h"

namespace agh {
namespace mx {

template <typename T, bool RAW, int TP, int TQ, int WK, int U>
__global__ __launch_bounds__(WK * 64) void mx_direct_kernel(Problem g, const T *__restrict__ x, int64_t rsx, int k) {
    static_assert((TP == 1 || TP == 2 || TP == 4) && (TQ == 1 || TQ == 2 || TQ == 4), "a tile's rows lie in one piece of the scales");
    __shared__ f32x4_t sums[WK][TP * TQ][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // a run of tiles for every XCD (workgroup id mod 8), p fastest: neighbours share pieces of scales, and a
    int id = blockIdx.x;
    {
        const int n = gridDim.x, xcd = id & 7;
        id = xcd * (n >> 3) + min(xcd, n & 7) + (id >> 3);
    }
    const int tq = id / g.tiles_p, tp = id - tq * g.tiles_p;
    const int p0 = tp * 16 * TP, q0 = tq * 16 * TQ;
    const int first = (int)((int64_t)g.steps * wave / WK), last = (int)((int64_t)g.steps * (wave + 1) / WK);

    const u32x4_t *fp[TP], *fq[TQ];
#pragma unroll
    for (int i = 0; i < TP; ++i) fp[i] = (const u32x4_t *)(g.b + (int64_t)min(p0 / 16 + i, (g.n - 1) / 16) * g.steps * kFragBytes) + lane;
#pragma unroll
    for (int j = 0; j < TQ; ++j) fq[j] = RAW ? nullptr : (const u32x4_t *)(g.a + (int64_t)min(q0 / 16 + j, (g.m - 1) / 16) * g.steps * kFragBytes) + lane;
    const uint32_t *sp = (const uint32_t *)(g.sb + (int64_t)(p0 / 64) * g.steps * kPieceBytes) + lane;
    const uint32_t *sq = RAW ? nullptr : (const uint32_t *)(g.sa + (int64_t)(q0 / 64) * g.steps * kPieceBytes) + lane;
    const int shift_p = p0 / 16 % 4 * 8, shift_q = q0 / 16 % 4 * 8;
    const int row = q0 + (lane & 15);  // (RAW) of the first fragment of a

    f32x4_t acc[TP][TQ];
#pragma unroll
    for (int i = 0; i < TP; ++i)
#pragma unroll
        for (int j = 0; j < TQ; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    // `count` steps from s on: all loads, then all products
    auto steps = [&](int s, auto countc) __attribute__((always_inline)) {
        constexpr int count = decltype(countc)::value;
        u32x4_t vp[count][TP], vq[count][TQ];
        uint32_t xp[count], xq[count];
        Block<T> raw[RAW ? count : 1][TQ];
#pragma unroll
        for (int c = 0; c < count; ++c) {
            if constexpr (RAW) {
#pragma unroll
                for (int j = 0; j < TQ; ++j) {
                    if (row + 16 * j < g.m) raw[c][j].load(x + (int64_t)(row + 16 * j) * rsx, (s + c) * kStep + (lane >> 4) * kBlock, k);
                    else raw[c][j].clear();
                }
            }
#pragma unroll
            for (int i = 0; i < TP; ++i) vp[c][i] = fp[i][(int64_t)(s + c) * 64];
            xp[c] = sp[(int64_t)(s + c) * 64];
            if constexpr (!RAW) {
#pragma unroll
                for (int j = 0; j < TQ; ++j) vq[c][j] = fq[j][(int64_t)(s + c) * 64];
                xq[c] = sq[(int64_t)(s + c) * 64];
            }
        }
#pragma unroll
        for (int c = 0; c < count; ++c) {
            if constexpr (RAW) {
                xq[c] = 0;
#pragma unroll
                for (int j = 0; j < TQ; ++j) {
                    uint32_t scale;
                    raw[c][j].quantize(vq[c][j], scale);
                    xq[c] |= scale << (8 * j);
                }
            } else {
                xq[c] >>= shift_q;
            }
            xp[c] >>= shift_p;
            mfma_written(xp[c]);
            mfma_written(xq[c]);
            if constexpr (RAW)
#pragma unroll
                for (int j = 0; j < TQ; ++j) mfma_written(vq[c][j]);
            mfma_ready();
            agh::gemm::static_for<TP>([&](auto ic) {
                agh::gemm::static_for<TQ>([&](auto jc) {
                    constexpr int i = decltype(ic)::value, j = decltype(jc)::value;
                    mfma<i, j>(acc[i][j], vp[c][i], vq[c][j], xp[c], xq[c]);
                });
            });
        }
        mfma_done(acc);  // (here and not behind the loops: between them the compiler may move accumulators)
    };
    int s = first;
    for (; s + U <= last; s += U) steps(s, std::integral_constant<int, U>{});
    for (; s < last; ++s) steps(s, std::integral_constant<int, 1>{});
#pragma unroll
    for (int i = 0; i < TP; ++i)
#pragma unroll
        for (int j = 0; j < TQ; ++j) sums[wave][i * TQ + j][lane] = acc[i][j];
    __syncthreads();
    const T *bias = (const T *)g.bias;
#pragma unroll 1
    for (int v = threadIdx.x; v < TP * TQ * 64; v += WK * 64) {
        const int l = v & 63, ij = v >> 6, q = q0 + ij % TQ * 16 + (l & 15), p = p0 + ij / TQ * 16 + (l >> 4) * 4;
        f32x4_t sum = sums[0][ij][l];
#pragma unroll
        for (int w = 1; w < WK; ++w) sum += sums[w][ij][l];
        if (q >= g.m) continue;
        T *c = (T *)g.c + q * g.rsc;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (p + r >= g.n) break;
            float f = sum[r] + (bias ? Elem<T>::raw(bias[(p + r) * g.bias_stride]) : 0.0f);
            f = g.act == AGH_ACT_RELU && !(f >= 0.0f) ? 0.0f : f;
            c[(p + r) * g.csc] = Elem<T>::from_f32(f);
        }
    }
}

}  // namespace mx
}  // namespace agh

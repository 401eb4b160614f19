// 8-bit integer product out of LDS: the tiled kernel, one workgroup a tile of BP x BQ of D[p][q] = sum_k P[p][k] Q[q][k] (P = b, Q = a, so D's p runs along c's rows).
//
// A step of 64 along k is BP / 16 + BQ / 16 fragments of 1 KB, copied from memory straight into one of NS stages of LDS (global_load_lds, no registers in between)
// NS - 1 steps ahead.  As the operands lie in fragments already, each load is one contiguous KB and each LDS read 16 bytes a lane in order: no bank conflicts, no
// address arithmetic beyond a scalar addition a load.
// A wave holds two sets of Q's fragments and one of P's: while step s is multiplied, the reads of step s + 1 go into the other set, and into P's fragment i as soon as
// row i of the tile is done, spread over the MFMAs.  Behind the barrier early in step s, the stage that step s was read from is refilled.
// Bounded by power where the result is large: 8192x8192x8192 bf16 369 to 390 us, call after call (2.8 to 3.0 PTOP/s), matrix pipes busy 75 % of the cycles at a clock of 1.69 GHz (waves as 2x2 of
// 128x128 433, tiles of 128x128 496; 16384x4096x4096 205); where it is small, by one workgroup a CU: 1999x2047x1001 has 256 tiles of
// 128x64, four waves each, so that nothing covers a wave's barrier, its six LDS reads a step and its wait for memory: f32 9.6 to 10.4, bf16 8.7 to 9.4, eight stages instead of four 0.2 more.
// Gated 16384x4096x8192 854 to 880, in 256x256 tiles, whose bf16 form keeps one register in scratch memory in
// the epilogue (all 256 are in use), read again for each of a wave's columns of tiles.
//
// GATED: the tile's BP rows of P are BP / 2 of b (the gate's) and the same BP / 2 of b2; a wave holds the accumulators of both in the same lanes, and the tile of c is BP / 2 wide.
#pragma once
#include "agh_i8_direct.h"

namespace agh {
namespace i8 {

// Issued from inline assembly with the accumulator tied to the accumulation registers and updated in place: given the builtin, the register allocator moves
// accumulators between the two register files inside the loop.  Between two of these no wait is needed: an accumulator is C and D in the same registers, and the
// hardware hands such a result on to the next instruction that adds to exactly those; their operands come out of LDS reads, whose arrival is waited for.
__device__ __forceinline__ void mfma_tied(i32x4_t &c, u32x4_t p, u32x4_t q) {
    asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(c) : "v"(p), "v"(q));
}
// Behind the last of them, before the accumulators are read: more wait states than the instruction has passes.  The accumulators pass through it too.
template <int N, int M>
__device__ __forceinline__ void mfma_done(i32x4_t (&acc)[N][M]) {
    asm volatile("s_nop 15" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < M; ++j) asm volatile("" : "+a"(acc[i][j]));
}

// 16 bytes a lane from a wave-uniform address plus a lane's offset to LDS, lane after lane; awaited by s_waitcnt vmcnt
__device__ __forceinline__ void load_fragment(const unsigned char *base, uint32_t lane16, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(lane16), "s"(base), "s"(lds) : "memory", "m0");
}

template <typename T, bool GATED, int BP, int BQ, int WGP, int WGQ, int NS>
__global__ __launch_bounds__(WGP * WGQ * 64) void i8_tile_kernel(Problem g) {
    using agh::gemm::static_for;
    constexpr int NW = WGP * WGQ, WP = BP / WGP, WQ = BQ / WGQ, TP = WP / 16, TQ = WQ / 16;
    constexpr int FP = BP / 16, FQ = BQ / 16, STAGE = (FP + FQ) * kFragBytes;
    constexpr int NL = (FP + FQ) / NW;                            // loads a wave issues for a step
    constexpr int HALVES = GATED ? 2 : 1, TO = TP / HALVES, BO = BP / HALVES, WO = WP / HALVES;  // of c's tile
    static_assert(TP % HALVES == 0 && (FP + FQ) % NW == 0 && (NS - 1) * NL < 64 && NS % 2 == 0, "every wave issues as many loads; the sets alternate with the stages");
    __shared__ __align__(16) unsigned char lds[NS * STAGE];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wave % WGP, wq = wave / WGP;
    // every XCD (workgroup id mod 8) takes a run of tiles, which share panels
    int id = blockIdx.x;
    {
        const int n = gridDim.x, xcd = id & 7;
        id = xcd * (n >> 3) + min(xcd, n & 7) + (id >> 3);
    }
    int tp, tq;
    agh::gemm::tile_walk(id, g.tiles_p, g.tiles_q, tp, tq);
    const int p0 = tp * BO, q0 = tq * BQ, KT = g.steps;

    // this wave's loads: fragments wave * NL .. of the stage, P's (b's, b2's) first; one behind the last row repeats the last
    const unsigned char *src[NL];
#pragma unroll
    for (int l = 0; l < NL; ++l) {
        const int f = wave * NL + l;
        const bool is_p = f < FP, second = GATED && f >= FP / 2;
        const int row = is_p ? p0 / 16 + (second ? f - FP / 2 : f) : q0 / 16 + (f - FP), last = ((is_p ? g.n : g.m) - 1) / 16;
        src[l] = (is_p ? second ? g.b2 : g.b : g.a) + (int64_t)min(row, last) * KT * kFragBytes;
    }
    const uint32_t base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const unsigned char *)lds);
    const uint32_t lane16 = lane * 16;
    // issues load l of the next step into stage s; `more`: move on to the step behind it
    auto load = [&](auto lc, int s, bool more) __attribute__((always_inline)) {
        constexpr int l = decltype(lc)::value;
        load_fragment(src[l], lane16, base + s * STAGE + (wave * NL + l) * kFragBytes);
        src[l] += more ? kFragBytes : 0;
    };

    u32x4_t fp[TP], fa[TQ], fb[TQ];
    auto read_p = [&](int s, int i) __attribute__((always_inline)) {
        const int f = i / TO * (FP / HALVES) + wp * TO + i % TO;
        fp[i] = *(const u32x4_t *)(lds + s * STAGE + f * kFragBytes + lane16);
    };
    auto read_q = [&](u32x4_t (&set)[TQ], int s, int j) __attribute__((always_inline)) {
        set[j] = *(const u32x4_t *)(lds + s * STAGE + (FP + wq * TQ + j) * kFragBytes + lane16);
    };

    i32x4_t acc[TP][TQ];
#pragma unroll
    for (int i = 0; i < TP; ++i)
#pragma unroll
        for (int j = 0; j < TQ; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};

    // Step kt, out of `set`; its stage is kt % NS, and the loads of steps kt + 1 .. kt + NS - 1 are in flight.
    constexpr int NM = TP * TQ, NB = TQ / 2, RSTEP = (NM - NB) / TQ > 3 ? 3 : (NM - NB) / TQ > 1 ? (NM - NB) / TQ : 1, LSTEP = (NM - NB) / NL > 1 ? (NM - NB) / NL : 1;
    auto step = [&](u32x4_t (&set)[TQ], u32x4_t (&next)[TQ], auto sc, bool more) __attribute__((always_inline)) {
        constexpr int s = decltype(sc)::value;
        static_for<NM>([&](auto nc) {
            constexpr int n = decltype(nc)::value, i = n / TQ, j = n % TQ;
            if constexpr (n == NB) {
                // step kt + 1 has landed, for all waves; and none of them reads the stage of step kt any more
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * NL) : "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
            }
            mfma_tied(acc[i][j], fp[i], set[j]);
            if constexpr (j == TQ - 1) read_p((s + 1) % NS, i);
            // (what does not fit behind the MFMAs one by one goes out behind the last)
            static_for<TQ>([&](auto uc) {
                constexpr int u = decltype(uc)::value, at = NB + u * RSTEP < NM ? NB + u * RSTEP : NM - 1;
                if constexpr (at == n) read_q(next, (s + 1) % NS, u);
            });
            static_for<NL>([&](auto lc) {
                constexpr int l = decltype(lc)::value, at = NB + l * LSTEP < NM ? NB + l * LSTEP : NM - 1;
                if constexpr (at == n) load(lc, s, more);
            });
            __builtin_amdgcn_sched_barrier(0);
        });
    };

    if (KT > 0) {
        static_for<NS>([&](auto sc) { static_for<NL>([&](auto lc) { load(lc, decltype(sc)::value, decltype(sc)::value + 1 < KT); }); });
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * NL) : "memory");
        __syncthreads();
        static_for<TQ>([&](auto jc) { read_q(fa, 0, decltype(jc)::value); });
        static_for<TP>([&](auto ic) { read_p(0, decltype(ic)::value); });
        // a step requests step kt + NS, the last one again where there is none
        auto turn = [&](int kt, auto sc) __attribute__((always_inline)) {
            constexpr int s = decltype(sc)::value;
            step(s % 2 ? fb : fa, s % 2 ? fa : fb, sc, kt + NS + 1 < KT);
        };
        int kt = 0;
        for (; kt + NS <= KT; kt += NS) static_for<NS>([&](auto sc) { turn(kt + decltype(sc)::value, sc); });
        static_for<NS - 1>([&](auto sc) {
            if (kt + decltype(sc)::value < KT) turn(kt + decltype(sc)::value, sc);
        });
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    }
    mfma_done(acc);
    __syncthreads();  // the stages are free: no load is in flight, no wave reads

    // Element r of lane l of acc[i][j] is D[.. 16 i + 4 (l / 16) + r][q0 + wq WQ + 16 j + l % 16]: four neighbours in a row of c, the 16 lanes of a group in as
    // many rows.  Stored like that, an instruction would touch 64 lines; so a wave turns 16 rows at a time in LDS and stores whole 16-byte chunks.
    constexpr int VE = 16 / (int)sizeof(T), PITCH = WO * (int)sizeof(T) + 16, CHUNKS = WO / VE;
    static_assert(NW * 16 * PITCH <= NS * STAGE && 16 * CHUNKS % 64 == 0, "the turned rows must fit in the stages");
    unsigned char *mine = lds + wave * 16 * PITCH;
    const int l16 = lane & 15, lg = lane >> 4, pw = p0 + wp * WO, qw = q0 + wq * WQ;
    T *c = (T *)g.c;
    const bool relu = g.act == AGH_ACT_RELU;
    Scale sp[TP][4];
    float bv[TP][4];
#pragma unroll
    for (int i = 0; i < TP; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int p = min(pw + 16 * (i % TO) + 4 * lg + r, g.n - 1);
            const float *scales = i < TO ? g.sb : g.sb2;
            const T *bias = (const T *)(i < TO ? g.bias : g.bias2);
            sp[i][r] = Scale(scales ? scales[p] : 0.0f);
            bv[i][r] = bias ? Elem<T>::raw(bias[p * g.bias_stride]) : 0.0f;
        }
    static_for<TQ>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        const int q = qw + 16 * j;
        const Scale sq(g.sa ? g.sa[min(q + l16, g.m - 1)] : 0.0f);
#pragma unroll
        for (int i = 0; i < TO; ++i) {
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = value_of(acc[i][j][r], sq, sp[i][r]) + bv[i][r];
            if constexpr (GATED) {
                float a[4];
                gate_values<sizeof(T) == 2, 4>(v, g.act, a);
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = a[r] * (value_of(acc[TO + i][j][r], sq, sp[TO + i][r]) + bv[TO + i][r]);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = relu && !(v[r] >= 0.0f) ? 0.0f : v[r];  // x >= 0 ? x : 0, as the Relu layer has it
            }
            unsigned char *at = mine + l16 * PITCH + (16 * i + 4 * lg) * (int)sizeof(T);
            if constexpr (sizeof(T) == 4) *(u32x4_t *)at = u32x4_t{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
            else *(uint2 *)at = make_uint2(f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]));
        }
        // (one wave, whose LDS accesses are in order: these reads see the writes, the next writes come behind them)
        if (g.csc == 1) {
#pragma unroll
            for (int t = 0; t < 16 * CHUNKS / 64; ++t) {
                const int at = t * 64 + lane, row = at / CHUNKS, chunk = at % CHUNKS, p = pw + chunk * VE;
                const unsigned char *from = mine + row * PITCH + chunk * 16;
                if (q + row < g.m) {
                    T *to = c + (q + row) * g.rsc + p;
                    if (p + VE <= g.n) {
                        if (g.streamed) __builtin_nontemporal_store(*(const u32x4_t *)from, (u32x4_t *)to);
                        else *(typename Unaligned<T>::vec *)to = *(const u32x4_t *)from;
                    } else
#pragma unroll 1
                        for (int e = 0; p + e < g.n; ++e) to[e] = ((const T *)from)[e];
                }
            }
        } else {
#pragma unroll 1
            for (int t = 0; t < 16 * WO / 64; ++t) {
                const int at = t * 64 + lane, row = at % 16, p = pw + at / 16;
                if (q + row < g.m && p < g.n) c[(q + row) * g.rsc + p * g.csc] = *(const T *)(mine + row * PITCH + at / 16 * (int)sizeof(T));
            }
        }
    });
}

}  // namespace i8
}  // namespace agh

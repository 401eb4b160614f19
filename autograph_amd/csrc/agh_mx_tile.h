// MXFP4 product out of LDS: the tiled kernel, one workgroup a BP x BQ tile of D[p][q] = sum_k P[p][k] Q[q][k] (P = b, Q = a, so D's p runs along c's rows).
//
// A step of 128 along k is BP / 16 + BQ / 16 fragments of 1 KB and a piece of scales for every 64 rows, copied from memory straight into one of NS stages
// of LDS (global_load_lds, no registers in between) NS - 1 steps ahead.  As the operands lie in fragments already, each load is one contiguous KB
// and each LDS read 16 bytes a lane in order: no bank conflicts, no address arithmetic beyond a scalar addition a load.
// A wave holds two sets of fragments: while step s is multiplied out of one, the reads of step s + 1 go into the other, spread over the MFMAs (all
// at once they would ask the LDS for twice what it gives).  Behind the barrier early in step s, the stage that step s was read from is refilled.
//
// 8192^3 with 256x256 tiles, 8 waves: 222 us, 4.9 PFLOP/s, 73 % of a loop of nothing but these instructions on such codes.  A step reads 96 KB of LDS and writes 32 KB, 1024
// cycles, as long as its instructions take; left out for timing, one operand's reads give 203 us, the loads 189, both operands' reads and the loads 149.  Four waves
// of 128x128, with a third less to read, have no second wave to hide what they wait for: 289.
#pragma once
#include "agh_gemm_kernel.h"
#include "agh_mx.h"

namespace agh {
namespace mx {

struct Problem {
    const unsigned char *a, *sa, *b, *sb;  // codes and scales: a of m rows, b of n rows
    void *c;
    int64_t rsc, csc;  // of c, elements
    const void *bias;  // or null
    int64_t bias_stride;
    int m, n, steps, act;
    bool streamed;  // c's rows start on 16 bytes and leave with the streaming hint
    int tiles_p, tiles_q;
};

// Issued from inline assembly with the accumulator tied to the accumulation registers and updated in place: given the builtin, the register allocator
// moves accumulators between the two register files inside the loop.  SP, SQ: which byte of the scale registers.  Between two of these no wait is needed: an accumulator is C
// and D in the same registers, and the hardware hands such a result on to the next instruction that adds to exactly those (the direct kernels do so back to back);
// what it does not hand on, another overlap or a result as operand A or B, does not occur.
template <int SP, int SQ>
__device__ __forceinline__ void mfma(f32x4_t &c, u32x4_t p, u32x4_t q, uint32_t sp, uint32_t sq) {
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] cbsz:4 blgp:4"
                 : "+a"(c)
                 : "v"(p), "v"(q), "v"(sp), "v"(sq), "n"(SP & 1), "n"(SQ & 1), "n"(SP >> 1), "n"(SQ >> 1));
}
// The compiler does not see matrix instructions in these, so what it keeps to around its own is kept to here.
// Operands that vector instructions wrote: two wait states before the first matrix instruction that reads them.  Each operand passes through the wait, so what writes it
// stays in front.
__device__ __forceinline__ void mfma_ready() { asm volatile("s_nop 1" ::: "memory"); }
template <typename V>
__device__ __forceinline__ void mfma_written(V &operand) { asm volatile("" : "+v"(operand)); }
// Behind the last of them, before the accumulators are read: their passes, which are 8 at most.  The accumulators pass through it too.
template <int N, int M>
__device__ __forceinline__ void mfma_done(f32x4_t (&acc)[N][M]) {
    asm volatile("s_nop 15" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < M; ++j) asm volatile("" : "+a"(acc[i][j]));
}

// 16 (4) bytes a lane from a wave-uniform address plus a lane's offset to LDS, lane after lane; awaited by s_waitcnt vmcnt
__device__ __forceinline__ void load_fragment(const unsigned char *base, uint32_t lane16, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(lane16), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void load_piece(const unsigned char *base, uint32_t lane4, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(lane4), "s"(base), "s"(lds) : "memory", "m0");
}

template <typename T, int BP, int BQ, int WGP, int WGQ, int NS>
__global__ __launch_bounds__(WGP * WGQ * 64) void mx_tile_kernel(Problem g) {
    using agh::gemm::static_for;
    constexpr int NW = WGP * WGQ, WP = BP / WGP, WQ = BQ / WGQ, TP = WP / 16, TQ = WQ / 16;
    constexpr int FP = BP / 16, FQ = BQ / 16, PP = BP / 64, PQ = BQ / 64;  // fragments and pieces of a stage
    constexpr int SCALES = (FP + FQ) * kFragBytes, STAGE = SCALES + (PP + PQ) * kPieceBytes;
    constexpr int NF = (FP + FQ) / NW, NP = (PP + PQ + NW - 1) / NW, NL = NF + NP;  // loads a wave issues for a step
    static_assert(WP % 64 == 0 && WQ % 64 == 0, "the rows of a wave are whole pieces");
    static_assert((FP + FQ) % NW == 0 && (NS - 1) * NL < 64 && NS % 2 == 0, "every wave issues as many loads; the sets alternate with the stages");
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
    const int p0 = tp * BP, q0 = tq * BQ, KT = g.steps;

    // this wave's loads: fragments wave * NF .. of the stage, then pieces wave * NP .. (one that does not exist repeats the last)
    const unsigned char *src[NL];
    uint32_t dst[NL];
#pragma unroll
    for (int l = 0; l < NL; ++l) {
        if (l < NF) {
            const int f = wave * NF + l;
            const bool is_p = f < FP;
            const int row = is_p ? p0 / 16 + f : q0 / 16 + (f - FP), last = ((is_p ? g.n : g.m) - 1) / 16;
            src[l] = (is_p ? g.b : g.a) + (int64_t)min(row, last) * KT * kFragBytes;
            dst[l] = (uint32_t)f * kFragBytes;
        } else {
            const int f = min(wave * NP + l - NF, PP + PQ - 1);
            const bool is_p = f < PP;
            const int row = is_p ? p0 / 64 + f : q0 / 64 + (f - PP), last = ((is_p ? g.n : g.m) - 1) / 64;
            src[l] = (is_p ? g.sb : g.sa) + (int64_t)min(row, last) * KT * kPieceBytes;
            dst[l] = (uint32_t)(SCALES + f * kPieceBytes);
        }
    }
    const uint32_t base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const unsigned char *)lds);
    const uint32_t lane16 = lane * 16, lane4 = lane * 4;
    // issues load l of the next step into stage s; `more`: move on to the step behind it
    auto load = [&](auto lc, int s, bool more) __attribute__((always_inline)) {
        constexpr int l = decltype(lc)::value;
        if constexpr (l < NF) load_fragment(src[l], lane16, base + s * STAGE + dst[l]);
        else load_piece(src[l], lane4, base + s * STAGE + dst[l]);
        src[l] += more ? (l < NF ? kFragBytes : kPieceBytes) : 0;
    };

    // P's fragments: fragment i of the next step takes the place of this step's as soon as row i of the tile is done.  Q's are in use until the end, so there
    // are two sets of them, as of the scales.
    struct Set {
        u32x4_t q[TQ];
        uint32_t sp[TP / 4], sq[TQ / 4];
    };
    u32x4_t fp[TP];
    Set A, B;
    constexpr int NSC = TP / 4 + TQ / 4, NR = NSC + TQ;  // LDS reads of a step into a set
    auto read_p = [&](int s, int i) __attribute__((always_inline)) { fp[i] = *(const u32x4_t *)(lds + s * STAGE + (wp * TP + i) * kFragBytes + lane16); };
    auto read = [&](Set &set, int s, auto uc) __attribute__((always_inline)) {
        constexpr int u = decltype(uc)::value;
        const unsigned char *at = lds + s * STAGE;
        if constexpr (u < TP / 4) set.sp[u] = *(const uint32_t *)(at + SCALES + (wp * (TP / 4) + u) * kPieceBytes + lane4);
        else if constexpr (u < NSC) set.sq[u - TP / 4] = *(const uint32_t *)(at + SCALES + (PP + wq * (TQ / 4) + u - TP / 4) * kPieceBytes + lane4);
        else set.q[u - NSC] = *(const u32x4_t *)(at + (FP + wq * TQ + u - NSC) * kFragBytes + lane16);
    };

    f32x4_t acc[TP][TQ];
#pragma unroll
    for (int i = 0; i < TP; ++i)
#pragma unroll
        for (int j = 0; j < TQ; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

    // Step kt, out of `set`; its stage is kt % NS, and the loads of steps kt + 1 .. kt + NS - 1 are in flight.
    constexpr int NM = TP * TQ, NB = TQ / 2, RSTEP = (NM - NB) / NR > 1 ? (NM - NB) / NR > 3 ? 3 : (NM - NB) / NR : 1, LSTEP = (NM - NB) / NL > 1 ? (NM - NB) / NL : 1;
    auto step = [&](Set &set, Set &next, auto sc, bool more) __attribute__((always_inline)) {
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
            mfma<i % 4, j % 4>(acc[i][j], fp[i], set.q[j], set.sp[i / 4], set.sq[j / 4]);
            if constexpr (j == TQ - 1) read_p((s + 1) % NS, i);
            // (what does not fit behind the MFMAs one by one goes out behind the last)
            static_for<NR>([&](auto uc) {
                constexpr int u = decltype(uc)::value, at = NB + u * RSTEP < NM ? NB + u * RSTEP : NM - 1;
                if constexpr (at == n) read(next, (s + 1) % NS, uc);
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
        static_for<NR>([&](auto uc) { read(A, 0, uc); });
        static_for<TP>([&](auto ic) { read_p(0, decltype(ic)::value); });
        // a step requests step kt + NS, the last one again where there is none
        auto turn = [&](int kt, auto sc) __attribute__((always_inline)) {
            constexpr int s = decltype(sc)::value;
            step(s % 2 ? B : A, s % 2 ? A : B, sc, kt + NS + 1 < KT);
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

    // Element r of lane l of acc[i][j] is D[p0 + wp WP + 16 i + 4 (l / 16) + r][q0 + wq WQ + 16 j + l % 16]: four neighbours in a row of c, the 16 lanes of a group in as
    // many rows.  Stored like that, an instruction would touch 64 lines; so a wave turns 16 rows at a time in LDS and stores whole 16-byte chunks.
    // (Kept short: the code of an epilogue is fetched for every workgroup anew, and written out in full it took longer than the products of 16 steps.)
    constexpr int VE = 16 / (int)sizeof(T), PITCH = WP * (int)sizeof(T) + 16, CHUNKS = WP / VE;
    static_assert(NW * 16 * PITCH <= NS * STAGE && 16 * CHUNKS % 64 == 0, "the turned rows must fit in the stages");
    unsigned char *mine = lds + wave * 16 * PITCH;
    const int l16 = lane & 15, lg = lane >> 4, pw = p0 + wp * WP, qw = q0 + wq * WQ;
    T *c = (T *)g.c;
    const T *bias = (const T *)g.bias;
    const bool relu = g.act == AGH_ACT_RELU;
    float bv[TP][4] = {};
    if (bias)
#pragma unroll
        for (int i = 0; i < TP; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) bv[i][r] = Elem<T>::raw(bias[min(pw + 16 * i + 4 * lg + r, g.n - 1) * g.bias_stride]);
    static_for<TQ>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
#pragma unroll
        for (int i = 0; i < TP; ++i) {
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                v[r] = acc[i][j][r] + bv[i][r];
                v[r] = relu && !(v[r] >= 0.0f) ? 0.0f : v[r];  // x >= 0 ? x : 0, as the Relu layer has it
            }
            unsigned char *at = mine + l16 * PITCH + (16 * i + 4 * lg) * (int)sizeof(T);
            if constexpr (sizeof(T) == 4) *(f32x4_t *)at = f32x4_t{v[0], v[1], v[2], v[3]};
            else *(uint2 *)at = make_uint2(f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]));
        }
        // (one wave, whose LDS accesses are in order: these reads see the writes, the next writes come behind them)
        const int q = qw + 16 * j;
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
            for (int t = 0; t < 16 * WP / 64; ++t) {
                const int at = t * 64 + lane, row = at % 16, p = pw + at / 16;
                if (q + row < g.m && p < g.n) c[(q + row) * g.rsc + p * g.csc] = *(const T *)(mine + row * PITCH + at / 16 * (int)sizeof(T));
            }
        }
    });
}

}  // namespace mx
}  // namespace agh

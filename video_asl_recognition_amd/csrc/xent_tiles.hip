// The products of the cross entropy operator for bf16 problems on gfx950: tiles of 256 x 256 (or 128 x 128, where those are
// too few for 256 CUs), 64 or 32 deep.
//
// Four waves of 128 x 128, one a SIMD: at 64 FLOP per LDS byte a tile of that shape asks the LDS for 3/4 of its rate (reads
// and the DMA's writes) while the matrix pipe runs at its own; two waves a SIMD on 128 x 64 each ask for all of it.  The 256
// accumulators leave each wave alone on its SIMD, so it hides its own latencies: while the MFMAs of one 16-deep slice run,
// the next slice's fragments are read into a second set of registers, and the stages after this one are on their way from
// memory by LDS-DMA.  A K step has one barrier, placed where a wave holds the last slice's fragments and has that slice's MFMAs
// still to issue: behind it the next stage is whole and this one is free for the DMA.  Of the 128 x 128 form two workgroups
// fit a CU.
//
// Operands contiguous along k are staged as [tile][step] and read as 16-byte fragments.  Operands contiguous along their own
// index (W for dx, x and G for dW) are staged as they lie, [step][tile], and read with the transposing LDS read, which hands a
// group of 16 lanes four k of 16 indices; no transposed copy of anything is made.
//
// fp32 operands come as three bf16 planes, x = h + m + l to all its 24 bits (rounded to nearest one after the other), and the
// contraction runs over six pairs of planes, h l + l h + m m + h m + m h + h h, smallest first.  What is left out, m l + l m +
// l l, is below 2^-23 of the product of the absolute values at worst and 2^-25 of it in the mean: the fp32 sums' own
// rounding.  Six bf16 products still take less time than one fp32 product on this card's matrix pipe (2048 x 8192 x 1024: 170 us
// each, 203 TFLOP/s; a library's fp32 product 134 TFLOP/s).
//
// Measured, 8192 x 32768 x 2048 (1.10 PFLOP a product): logits 1016 to 1067 us (1.03 to 1.08 PFLOP/s), dx 826 to 847 (1.30 to
// 1.33), dW 794 to 826 (1.33 to 1.38); a library's plain products of the same shapes 1.20, 1.12 and 0.99 PFLOP/s.  dW keeps the
// matrix pipe 86 % busy at the clock that its power leaves it, dx 78 to 82 % and the logits 60 %: a logits tile adds 8 us of exponentials
// and 6 us of first loads to 32 steps of 1.6 us, alone on its CU.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "asl_hip.h"
#include "patch_args.h"
#include "xent_args.h"

namespace asl_detail {

// k a step, by whether the operands are contiguous along k.  Four stages of 32 hide more of the memory's latency than two of
// 64 (dW of 8192 x 32768 x 2048: 794 us against 900), but rows contiguous along k are then read 64 bytes at a time, half of
// each line twice (logits of the same: 1127 us against 1066).
constexpr int step_depth(bool pkc, bool qkc) { return pkc || qkc ? 64 : 32; }

// LDS of a tile kernel: the stages of both operands, 128 k in all; over them, behind the K loop, the results on their way out:
// all rows in 16 bits, or 128 of them in 32 (padded, so that consecutive rows start in different banks); then a tile's bias
// and targets
template <int TILE, int BK>
struct TileLds {
    static constexpr int kStages = 128 / BK;
    static constexpr int kPanel = TILE * BK * 2;         // one operand's tile
    static constexpr int kStaged = 2 * kStages * kPanel;
    static constexpr int kRow16 = TILE * 2 + 16;         // bytes
    static constexpr int kRow32 = TILE * 4 + 16;
    static constexpr int kOut = TILE * kRow16 > 128 * kRow32 ? TILE * kRow16 : 128 * kRow32;
    static constexpr int kMain = kStaged > kOut ? kStaged : kOut;
    static constexpr int kLogits = kMain + TILE * 8;
};

#if defined(__HIP_DEVICE_COMPILE__)
// 1 KiB (16 bytes a lane) from a buffer into LDS at `lds` (wave-uniform).  Written out because the compiler, which knows
// only that the builtin writes LDS somewhere, drains the whole queue ahead of the next transposing read; it has no result in
// registers, and the kernel's own counted waits and barriers are what orders it (LDS addresses go through M0, which wants
// one instruction between its write and its use; nothing else in these kernels uses it).
template <int AT>
__device__ __forceinline__ void dma_1k(i32x4 rsrc, unsigned voff, unsigned lds) {
    asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc), "n"(AT) : "scc");
}

// One operand's way from memory to registers.  Its stages lie behind one another in LDS, so that a fragment's address is
// one register and an immediate.
template <int TILE, int BK, bool KC>
struct Panel {
    static constexpr int kPanel = TileLds<TILE, BK>::kPanel, ND = TILE * BK / 2048, F = TILE / 64;   // DMA instructions and fragments a wave
    const char* at;          // first byte of the K step to be staged next
    const char* origin;      // of the first step, and how far apart planes lie
    long long plane;
    int kall;
    long long row_bytes;
    int idx;                 // rows (KC) or columns of the stored matrix that belong to this tile
    int krem;                // k left from `at` on
    unsigned lds;            // this wave's part of stage 0
    unsigned voff[ND];
    unsigned rd[KC ? BK / 16 : F]; // fragment addresses in stage 0: by slice (KC) or by fragment

    // 16-byte chunks of rows contiguous along k change places with the row, so that eight consecutive rows' same chunk lies in
    // different banks
    static __device__ __forceinline__ int swizzle(int row) { return BK == 64 ? (row >> 1) & 7 : (row >> 2) & 3; }

    __device__ __forceinline__ void init(const void* base, long long ld, int i0, int n, int kb, int ke, int wave, int lane,
                                         int w0, unsigned stages) {
        row_bytes = ld * 2;
        idx = n - i0 < TILE ? n - i0 : TILE;
        krem = kall = ke - kb;
        origin = at = (const char*)base + (KC ? (long long)i0 * row_bytes + kb * 2LL : (long long)kb * row_bytes + i0 * 2LL);
        lds = stages + wave * (kPanel / 4);
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            if constexpr (KC) {                          // eight rows of 128 bytes a DMA instruction, or sixteen of 64
                constexpr int L = BK / 8;                // lanes a row
                const int row = wave * (TILE / 4) + i * (64 / L) + lane / L, c = (lane % L) ^ swizzle(row);
                voff[i] = (unsigned)(row * row_bytes + c * 16);
            } else {                                     // two or four k rows; their 32-byte units swapped by k's low bits
                constexpr int L = TILE / 8;              // lanes a row
                const int k = wave * (BK / 4) + i * (64 / L) + lane / L, u = ((lane % L) >> 1) ^ ((k & 3) << 1);
                voff[i] = (unsigned)(k * row_bytes + u * 32 + (lane & 1) * 16);
            }
        }
        if constexpr (KC) {
            const int r = w0 + (lane & 31);
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk) rd[kk] = stages + r * (BK * 2) + (((kk * 2 + (lane >> 5)) ^ swizzle(r)) << 4);
        } else {
            const int g = lane >> 4, s = lane & 15, x = (s >> 2) << 1;
#pragma unroll
            for (int u = 0; u < F; ++u)
                rd[u] = stages + ((g >> 1) * 8 + (s >> 2)) * (TILE * 2) + (((w0 >> 4) + u * 2 + (g & 1)) ^ x) * 32 + (s & 3) * 8;
        }
    }
    // The descriptor of the step at `at`: everything past the operand's last element reads as nought, all of it behind the
    // last step.  Rows that are contiguous along k hold noughts up to a whole step (the caller sees to that).
    __device__ __forceinline__ i32x4 rsrc() const {
        // (32 bits: a tile's rows are at most 2^22 bytes and some apart, G's of 2^21 classes)
        const int k = krem < BK ? krem : BK;
        const int n = KC ? (idx - 1) * (int)row_bytes + BK * 2 : (k - 1) * (int)row_bytes + idx * 2;
        const unsigned long long p = (unsigned long long)at;
        return i32x4{__builtin_amdgcn_readfirstlane((int)p), __builtin_amdgcn_readfirstlane((int)(p >> 32) & 0xffff),
                     __builtin_amdgcn_readfirstlane(krem > 0 ? (n + 3) & ~3 : 0), 0x00020000};
    }
    __device__ __forceinline__ void advance() {
        at += KC ? BK * 2 : BK * row_bytes;
        krem -= BK;
    }
    __device__ __forceinline__ void to_plane(int which, bool turn, bool more) {
        at = turn ? origin + which * plane : at;
        krem = turn ? (more ? kall : 0) : krem;
    }
    template <int STAGE, int I>
    __device__ __forceinline__ void dma(i32x4 r) const {
        dma_1k<STAGE * kPanel + I * 1024>(r, voff[I], lds);
    }
    // fragment u (32 indices) of the 16-deep slice kk
    __device__ __forceinline__ bf16x8 frag(int stage, int kk, int u) const {
        typedef __attribute__((address_space(3))) char* P1;
        if constexpr (KC) {
            return *(const __attribute__((address_space(3))) bf16x8*)((P1)(unsigned long long)rd[kk] + (stage * kPanel + u * (BK * 64)));
        } else {
            typedef __attribute__((address_space(3))) bf16x4* P4;
            const P1 a = (P1)(unsigned long long)rd[u];
            const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P4)(a + (stage * kPanel + kk * (TILE * 32))));
            const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P4)(a + (stage * kPanel + kk * (TILE * 32) + TILE * 8)));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// those of TOTAL things that fall to place I of N when they are spread evenly over the places
template <int TOTAL, int N, int I, typename F>
__device__ __forceinline__ void paced(F&& f) {
    constexpr int first = (I * TOTAL + N - 1) / N, last = ((I + 1) * TOTAL + N - 1) / N;
    if constexpr (last > first) f(std::integral_constant<int, first>{});
    if constexpr (last > first + 1) f(std::integral_constant<int, first + 1>{});
    static_assert(last <= first + 2, "at most two a place");
}

template <int N, typename F>
__device__ __forceinline__ void unroll(F&& f) {
    if constexpr (N > 0) {
        unroll<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}
#endif

// tile order: XCD-contiguous ranges (workgroups go to the XCDs in turn), within which tiles run in blocks of 8 j by all i
// of a strip of 4, so that the tiles an XCD's 32 CUs hold at a time share panels in its L2
__device__ __forceinline__ void tile_of(int id, int ti, int tj, int& i, int& j) {
    const int n = ti * tj, q = n >> 3, r = n & 7, xcd = id & 7;
    const int l = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (id >> 3);
    constexpr int GJ = 8;
    const int strip = l / (GJ * ti), first = strip * GJ, w = tj - first < GJ ? tj - first : GJ, in = l - strip * GJ * ti;
    i = in / w;
    j = first + in % w;
}

#if defined(__HIP_DEVICE_COMPILE__)
// One tile of a product: workgroup `id` of ti * tj * splits.
template <int TILE, int BK, bool PKC, bool QKC, bool LOGITS, bool WIDE>
__device__ __forceinline__ void tile_body(const XentGemm& a, int id, int ti, int tj) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    using Lds = TileLds<TILE, BK>;
    constexpr int F = TILE / 64, W = TILE / 2;       // fragments of 32 and indices a wave has of either operand
    float* const bias_row = (float*)(smem + Lds::kMain);
    int* const target_at = (int*)(smem + Lds::kMain + TILE * 4);             // within the tile, or -1
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = (wave >> 1) * W, wj = (wave & 1) * W;
    int bi, bj;
    const int slice = id / (ti * tj);
    tile_of(id % (ti * tj), ti, tj, bi, bj);
    const int i0 = bi * TILE, j0 = bj * TILE;
    const int kb = slice * a.k_per_split, ke = kb + a.k_per_split < a.K ? kb + a.k_per_split : a.K;
    const int steps = ke > kb ? (ke - kb + BK - 1) / BK * (WIDE ? 6 : 1) : 0;

    const unsigned lds0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)smem;
    Panel<TILE, BK, PKC> P;
    Panel<TILE, BK, QKC> Q;
    P.init(a.p, a.ld_p, i0, a.I, kb, ke, wave, lane, wi, lds0);
    Q.init(a.q, a.ld_q, j0, a.Jn, kb, ke, wave, lane, wj, lds0 + Lds::kStaged / 2);
    int pair = 0;
    constexpr int kPlaneP = 0 << 0 | 2 << 2 | 1 << 4 | 0 << 6 | 1 << 8 | 0 << 10, kPlaneQ = 2 << 0 | 0 << 2 | 1 << 4 | 1 << 6 | 0 << 8 | 0 << 10;
    if constexpr (WIDE) {
        P.plane = a.plane_p * 2;
        Q.plane = a.plane_q * 2;
        Q.at += 2 * Q.plane;                         // h l first
    }
    const auto next = [&]() {
        P.advance();
        Q.advance();
        if constexpr (WIDE) {
            const bool turn = P.krem <= 0;
            pair += turn;
            P.to_plane(kPlaneP >> (pair * 2) & 3, turn, pair < 6);
            Q.to_plane(kPlaneQ >> (pair * 2) & 3, turn, pair < 6);
        }
    };
    const auto dma = [&](i32x4 pr, i32x4 qr, auto stage, auto n) {  // the n-th of a stage's DMA instructions
        constexpr int N = decltype(n)::value, S = decltype(stage)::value;
        if constexpr (N & 1) Q.template dma<S, N / 2>(qr);
        else P.template dma<S, N / 2>(pr);
    };
    i32x4 pr, qr;                                    // of the stage that is being filled
    constexpr int kDma = 2 * Panel<TILE, BK, PKC>::ND;        // DMA instructions a stage
    const auto fill = [&](auto stage) {
        pr = P.rsrc();
        qr = Q.rsrc();
        unroll<decltype(stage)::value == Lds::kStages - 1 ? kDma / 2 : kDma>([&](auto n) { dma(pr, qr, stage, n); });
        next();
    };
    unroll<Lds::kStages>(fill);                      // past the end: nought, and no memory touched; the last one half

    if constexpr (LOGITS) {
        const int at = threadIdx.x % TILE, i = i0 + at, j = j0 + at;
        float b = -INFINITY;                         // classes behind the last are masked like any other
        if (i < a.I) b = !a.bias ? 0.f : a.bias_bf16 ? load1((const short*)a.bias + i) : load1((const float*)a.bias + i);
        bias_row[at] = b;
        const long long t = j < a.Jn ? a.target[j] : -1;
        target_at[at] = t >= i0 && t < i0 + TILE && t < a.I ? (int)(t - i0) : -1;
    }

    f32x16 acc[F][F];
    if constexpr (LOGITS) {
        // the sums start from the bias, while the first stages are on their way
        __syncthreads();
#pragma unroll
        for (int u = 0; u < F; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const f32x4 b = *(const f32x4*)(bias_row + wi + u * 32 + r * 8 + (lane >> 5) * 4);
#pragma unroll
                for (int v = 0; v < F; ++v)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[u][v][r * 4 + e] = b[e];
            }
    } else {
#pragma unroll
        for (int u = 0; u < F; ++u)
#pragma unroll
            for (int v = 0; v < F; ++v)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[u][v][e] = 0.f;
    }

    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((Lds::kStages - 2) * kDma + kDma / 2) : "memory");
    bf16x8 pf[2][F], qf[2][F];
    const auto read = [&](int set, int stage, int kk, int n) {      // the n-th of a slice's fragments
        if (n & 1) qf[set][n >> 1] = Q.frag(stage, kk, n >> 1);
        else pf[set][n >> 1] = P.frag(stage, kk, n >> 1);
    };
    const auto mma = [&](int set, int n) {                          // the n-th of its products, in the fragments' order
        constexpr unsigned char U[16] = {0, 1, 0, 1, 2, 2, 0, 1, 2, 3, 3, 3, 0, 1, 2, 3};
        constexpr unsigned char V[16] = {0, 0, 1, 1, 0, 1, 2, 2, 2, 0, 1, 2, 3, 3, 3, 3};
        f32x16& c = acc[U[n]][V[n]];
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(pf[set][U[n]], qf[set][V[n]], c, 0, 0, 0);
    };
#pragma unroll
    for (int n = 0; n < 2 * F; ++n) read(0, 0, 0, n);
    // A step is BK / 16 slices.  The DMA goes out at an even pace over two of them, an instruction every few MFMAs: in one
    // burst a stage's 64 instructions hold the waves up at the address unit, which takes 16 cycles each.
    const auto step = [&](auto stage) {
        constexpr int S = decltype(stage)::value, N = F * F, kSlices = BK / 16;
        constexpr std::integral_constant<int, (S + Lds::kStages - 1) % Lds::kStages> before{};
        i32x4 next_p, next_q;
        // all slices but the last: under each the fragments of the next, and under the first the rest of the stage that the
        // last step began to fill
        unroll<(kSlices - 1) * N>([&](auto n) {
            constexpr int M = decltype(n)::value, K = M / N, R = M % N;
            if (R < 2 * F) read((K + 1) & 1, S, K + 1, R);
            if constexpr (K == 0) paced<kDma / 2, N, R>([&](auto d) { dma(pr, qr, before, std::integral_constant<int, kDma / 2 + decltype(d)::value>{}); });
            // the next stage's descriptors between the last MFMAs (the empty asm holds them there: left to itself the
            // compiler computes them where they are used, in one gap behind the barrier)
            constexpr bool kEnd = K == kSlices - 2;
            if constexpr (kEnd && R == N - 3 && F == 4) next_p = P.rsrc();
            if constexpr (kEnd && R == N - 2) next_q = Q.rsrc();
            if constexpr (kEnd && R == N - 2 && F == 2) next_p = P.rsrc();
            if constexpr (kEnd && R == N - 1) next();
            mma(K & 1, R);
            if constexpr (kEnd && R == N - 3 && F == 4) asm volatile("" : "+s"(next_p));
            if constexpr (kEnd && R == N - 2) asm volatile("" : "+s"(next_q));
            __builtin_amdgcn_sched_barrier(0);
        });
        pr = next_p;
        qr = next_q;
        // this wave has read all it needs of this stage, and its part of the next one has landed
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((Lds::kStages - 2) * kDma) : "memory");
        // the last slice, under it the next stage's first fragments and half of this stage's next filling
        unroll<N>([&](auto n) {
            constexpr int M = decltype(n)::value;
            if (M < 2 * F) read(0, (S + 1) % Lds::kStages, 0, M);
            paced<kDma / 2, N, M>([&](auto d) { dma(pr, qr, stage, d); });
            mma(1, M);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
#pragma unroll 1
    for (int s = 0; s < steps; s += Lds::kStages) unroll<Lds::kStages>(step);      // behind the last step: noughts
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

    // ---- results.  Lane: i = wi + u*32 + 8*(r/4) + 4*(lane/32) + r%4, j = wj + v*32 + lane%32 -------------------------
    const int h4 = (lane >> 5) * 4;
    if constexpr (LOGITS) {
        // Maxima and sums are kept per W classes, a wave's own: nothing is exchanged but between a row's two lanes.  The
        // exponential is the hardware's power of two of a fused multiply-add, which makes it 2^15 times as large for the 16-bit
        // form on the way.
        constexpr float kLog2e = 1.44269504088896341f;
        const int block = bi * 2 + (wi ? 1 : 0);
#pragma unroll
        for (int v = 0; v < F; ++v) {
            const int jl = wj + v * 32 + (lane & 31), j = j0 + jl;
            float m = -INFINITY;
#pragma unroll
            for (int u = 0; u < F; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[u][v][r]);
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            const float ref = m == -INFINITY ? 0.f : m;            // classes that are all masked: sum nought, not NaN
            float s = 0.f, lin = 0.f;
#pragma unroll
            for (int u = 0; u < F; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    f32x4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float l = acc[u][v][r * 4 + e];
                        x[e] = WIDE ? expf(l - ref) : __builtin_amdgcn_exp2f(fmaf(l - ref, kLog2e, 15.f));
                        s += x[e];
                    }
                    const int at = wi + u * 32 + r * 8 + h4;
                    if constexpr (WIDE) {
                        if (a.store_e && j < a.Jn) *(f32x4*)((float*)a.out + j * a.ld_out + i0 + at) = x;
                    } else {
                        half4 o;
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[e] = (_Float16)x[e];
                        *(half4*)(smem + jl * Lds::kRow16 + at * 2) = o;
                    }
                }
            s += __shfl_xor(s, 32, 64);
            if (!WIDE) s *= 1.f / kExpScale16;
            if (a.smooth) {
#pragma unroll
                for (int u = 0; u < F; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) lin += i0 + wi + u * 32 + (r >> 2) * 8 + h4 + (r & 3) < a.I ? acc[u][v][r] : 0.f;
                lin += __shfl_xor(lin, 32, 64);
            }
            if (lane < 32 && j < a.Jn && block < a.tiles) {
                const long long o = (long long)j * a.tiles + block;
                a.tile_max[o] = m;
                a.tile_sum[o] = s;
                if (a.smooth) a.tile_lin[o] = lin;
            }
            const int t = target_at[jl] - wi;
            const bool mine = t >= 0 && t < W && ((t >> 2) & 1) * 4 == h4;
            if (__any(mine)) {
                float l = 0.f;
#pragma unroll
                for (int u = 0; u < F; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) l = (t & ~4) == u * 32 + (r >> 2) * 8 + (r & 3) ? acc[u][v][r] : l;
                if (mine) a.target_logit[j] = l;
            }
        }
        if (WIDE || !a.store_e) return;
        __syncthreads();
    } else if (a.slabs) {                              // rows padded to whole tiles: nothing to cut
        const long long ld = (long long)ti * TILE;
#pragma unroll
        for (int v = 0; v < F; ++v) {
            const int j = j0 + wj + v * 32 + (lane & 31);
            float* row = (float*)a.out + ((long long)slice * a.Jn + j) * ld + i0 + wi + h4;
            if (j < a.Jn) {
                if (a.add) {
#pragma unroll
                    for (int u = 0; u < F; ++u)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const f32x4 q = *(const f32x4*)(row + u * 32 + r * 8);
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[u][v][r * 4 + e] += q[e];
                        }
                }
#pragma unroll
                for (int u = 0; u < F; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        *(f32x4*)(row + u * 32 + r * 8) = f32x4{acc[u][v][r * 4], acc[u][v][r * 4 + 1], acc[u][v][r * 4 + 2], acc[u][v][r * 4 + 3]};
            }
        }
        return;
    } else {
        const float c = *a.factor;
        if constexpr (WIDE) {                          // fp32 rows through LDS, 128 at a time
#pragma unroll 1
            for (int half = 0; half < TILE / 128; ++half) {
                if (half) __syncthreads();
                if (TILE == 128 || wj == half * 128) {
#pragma unroll
                    for (int v = 0; v < F; ++v)
#pragma unroll
                        for (int u = 0; u < F; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                *(f32x4*)(smem + (wj % 128 + v * 32 + (lane & 31)) * Lds::kRow32 + (wi + u * 32 + r * 8 + h4) * 4) =
                                    f32x4{acc[u][v][r * 4] * c, acc[u][v][r * 4 + 1] * c, acc[u][v][r * 4 + 2] * c, acc[u][v][r * 4 + 3] * c};
                }
                __syncthreads();
                constexpr int L = TILE / 4;            // four results a lane
#pragma unroll 4
                for (int n = 0; n < 128 * L / 256; ++n) {
                    const int row = n * (256 / L) + threadIdx.x / L, at = (threadIdx.x % L) * 4, j = j0 + half * 128 + row;
                    const f32x4 x = *(const f32x4*)(smem + row * Lds::kRow32 + at * 4);
                    float* dst = (float*)a.out + j * a.ld_out + i0 + at;
                    if (j < a.Jn && i0 + at < a.I) {
                        if (i0 + at + 4 <= a.I) {
                            *(f32x4u*)dst = x;
                        } else {
                            dst[0] = x[0];
                            if (i0 + at + 1 < a.I) dst[1] = x[1];
                            if (i0 + at + 2 < a.I) dst[2] = x[2];
                        }
                    }
                }
            }
            return;
        }
#pragma unroll
        for (int v = 0; v < F; ++v)
#pragma unroll
            for (int u = 0; u < F; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    bf16x4 o;
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = f32_to_bf16(acc[u][v][r * 4 + e] * c);
                    *(bf16x4*)(smem + (wj + v * 32 + (lane & 31)) * Lds::kRow16 + (wi + u * 32 + r * 8 + h4) * 2) = o;
                }
        __syncthreads();
    }
    // 16-bit rows out of LDS, 16 bytes a lane
    constexpr int L = TILE / 8;
    const int at = (threadIdx.x % L) * 8, left = LOGITS ? 8 : a.I - i0 - at;   // (the exponentials' rows are padded to whole tiles)
    short* out = (short*)a.out + (j0 + threadIdx.x / L) * a.ld_out + i0 + at;
    const char* src = smem + threadIdx.x / L * Lds::kRow16 + at * 2;
    const int rows = a.Jn - j0 - (int)threadIdx.x / L;             // this lane's first row is there if positive
    if (left >= 8) {
#pragma unroll 4
        for (int n = 0; n < TILE * L / 256; ++n)
            if (n * (256 / L) < rows) *(bf16x8u*)(out + (long long)n * (256 / L) * a.ld_out) = *(const bf16x8*)(src + n * (256 / L) * Lds::kRow16);
    } else if (left > 0) {
#pragma unroll 1
        for (int n = 0; n < TILE * L / 256; ++n)
            if (n * (256 / L) < rows) {
                const bf16x8 x = *(const bf16x8*)(src + n * (256 / L) * Lds::kRow16);
#pragma unroll
                for (int e = 0; e < 7; ++e)
                    if (e < left) out[(long long)n * (256 / L) * a.ld_out + e] = x[e];
            }
    }
}
#endif

template <int TILE, bool PKC, bool QKC, bool LOGITS, bool WIDE>
__global__ __launch_bounds__(256, TILE == 256 ? 1 : 2) void xent_tile_kernel(const XentGemm a, int ti, int tj) {
#if defined(__HIP_DEVICE_COMPILE__)
    tile_body<TILE, step_depth(PKC, QKC), PKC, QKC, LOGITS, WIDE>(a, blockIdx.x, ti, tj);
#endif
}

// Both gradient products in one launch, dx's workgroups first: they do not depend on one another, and where neither fills
// the CUs they fill them together.  (128 x 128 only: two bodies of the large tile in one kernel leave the compiler no way to
// keep 256 accumulators where they are, and products that take it fill the CUs alone.)
template <int TILE, bool WIDE>
__global__ __launch_bounds__(256, 2) void xent_tile_pair_kernel(const XentGemm dx, const XentGemm dw, int dx_ti, int dx_tj, int dw_ti, int dw_tj,
                                                                int dx_blocks) {
#if defined(__HIP_DEVICE_COMPILE__)
    if ((int)blockIdx.x < dx_blocks) tile_body<TILE, step_depth(false, true), false, true, false, WIDE>(dx, blockIdx.x, dx_ti, dx_tj);
    else tile_body<TILE, step_depth(false, false), false, false, false, WIDE>(dw, blockIdx.x - dx_blocks, dw_ti, dw_tj);
#endif
}

template <int TILE, bool PKC, bool QKC, bool LOGITS, bool WIDE>
static int launch_tiles(const XentGemm& a, hipStream_t s) {
    const int ti = ceil_div(a.I, TILE), tj = ceil_div(a.Jn, TILE);
    if ((long long)ti * tj * a.splits > 0x7fffffffLL) return ASL_ETOOBIG;
    constexpr int lds = LOGITS ? TileLds<TILE, step_depth(PKC, QKC)>::kLogits : TileLds<TILE, step_depth(PKC, QKC)>::kMain;
    static unsigned char lds_done[64];
    const int rc = ensure_dynamic_lds((const void*)xent_tile_kernel<TILE, PKC, QKC, LOGITS, WIDE>, lds, lds_done);
    if (rc != ASL_OK) return rc;
    hipLaunchKernelGGL((xent_tile_kernel<TILE, PKC, QKC, LOGITS, WIDE>), dim3((unsigned)(ti * tj * a.splits)), dim3(256), lds, s, a, ti, tj);
    return (int)hipGetLastError();
}
template <int TILE, bool WIDE>
static int launch_pair(const XentGemm& dx, const XentGemm& dw, hipStream_t s) {
    const int xi = ceil_div(dx.I, TILE), xj = ceil_div(dx.Jn, TILE), wi = ceil_div(dw.I, TILE), wj = ceil_div(dw.Jn, TILE);
    const long long nx = (long long)xi * xj * dx.splits, nw = (long long)wi * wj * dw.splits;
    if (nx + nw > 0x7fffffffLL) return ASL_ETOOBIG;
    constexpr int lds = TileLds<TILE, 32>::kMain;
    static_assert(TileLds<TILE, 32>::kMain == TileLds<TILE, 64>::kMain, "both bodies' LDS");
    static unsigned char lds_done[64];
    const int rc = ensure_dynamic_lds((const void*)xent_tile_pair_kernel<TILE, WIDE>, lds, lds_done);
    if (rc != ASL_OK) return rc;
    hipLaunchKernelGGL((xent_tile_pair_kernel<TILE, WIDE>), dim3((unsigned)(nx + nw)), dim3(256), lds, s, dx, dw, xi, xj, wi, wj, (int)nx);
    return (int)hipGetLastError();
}
template <bool PKC, bool QKC, bool LOGITS>
static int launch_any(const XentGemm& a, int tile, hipStream_t s) {
    if (a.plane_p)
        return tile == 256 ? launch_tiles<256, PKC, QKC, LOGITS, true>(a, s) : launch_tiles<128, PKC, QKC, LOGITS, true>(a, s);
    return tile == 256 ? launch_tiles<256, PKC, QKC, LOGITS, false>(a, s) : launch_tiles<128, PKC, QKC, LOGITS, false>(a, s);
}

int xent_tiles_pair(const XentGemm& dx, const XentGemm& dw, hipStream_t s) {
    return dx.plane_p ? launch_pair<128, true>(dx, dw, s) : launch_pair<128, false>(dx, dw, s);
}
int xent_tiles_logits(const XentGemm& a, int tile, hipStream_t s) { return launch_any<true, true, true>(a, tile, s); }
int xent_tiles_dx(const XentGemm& a, int tile, hipStream_t s) { return launch_any<false, true, false>(a, tile, s); }
int xent_tiles_dw(const XentGemm& a, int tile, hipStream_t s) { return launch_any<false, false, false>(a, tile, s); }

}  // namespace asl_detail

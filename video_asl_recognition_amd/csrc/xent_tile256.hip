// The products of the cross entropy operator for large bf16 problems on gfx950: 256 x 256 tiles, 64 deep.
//
// Four waves of 128 x 128, one a SIMD: at 64 FLOP per LDS byte a tile of that shape asks the LDS for 3/4 of its rate (reads
// and the DMA's writes) while the matrix pipe runs at its own; two waves a SIMD on 128 x 64 each ask for all of it.  The 256
// accumulators leave each wave alone on its SIMD, so it hides its own latencies: while the MFMAs of one 16-deep slice run,
// the next slice's fragments are read into a second set of registers, and the tile after next is on its way from memory by
// LDS-DMA.  A K step has one barrier, placed where a wave holds the last slice's fragments and has that slice's MFMAs still
// to issue: behind it the other buffer is whole and this one is free for the DMA.
//
// Operands contiguous along k are staged as [256][64] and read as 16-byte fragments.  Operands contiguous along their own
// index (W for dx, x and G for dW) are staged as they lie, [64][256], and read with the transposing LDS read, which hands a
// group of 16 lanes four k of 16 indices; no transposed copy of anything is made.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "asl_hip.h"
#include "patch_args.h"
#include "xent_args.h"

namespace asl_detail {

constexpr int kBK = 64;
constexpr int kPanelBytes = kBigTile * kBK * 2;          // one operand's tile
constexpr int kStageBytes = 2 * kPanelBytes;
constexpr int kOutRow = kBigTile * 2 + 16;               // an output row in LDS: the pad walks the banks from row to row
constexpr int kBigLds = kBigTile * kOutRow;              // 132 KiB: covers the two stages as well
static_assert(kBigLds >= 2 * kStageBytes, "stages fit");

#if defined(__HIP_DEVICE_COMPILE__)
// 1 KiB (16 bytes a lane) from a buffer into LDS at `lds` (wave-uniform).  Written out because the compiler, which knows
// only that the builtin writes LDS somewhere, drains the whole queue ahead of the next transposing read; it has no result in
// registers, and the kernel's own counted waits and barriers are what orders it (LDS addresses go through M0, which wants
// one instruction between its write and its use;
// nothing else in these kernels uses it).
__device__ __forceinline__ void dma_1k(i32x4 rsrc, unsigned voff, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc));
}

// One operand's way from memory to registers.
template <bool KC>
struct Panel {
    const char* at;          // first byte of the K step to be staged next
    long long row_bytes;
    int idx;                 // rows (KC) or columns of the stored matrix that belong to this tile
    int krem;                // k left from `at` on
    unsigned voff[8];
    unsigned dead[2];        // KC: what a chunk's offset is or-ed with in the last K step (bit 31: past the end, reads nought)
    int rd[4];               // fragment addresses within a panel

    __device__ __forceinline__ void init(const void* base, long long ld, int i0, int n, int kb, int ke, int wave, int lane,
                                         int w128) {
        row_bytes = ld * 2;
        idx = n - i0 < kBigTile ? n - i0 : kBigTile;
        krem = ke - kb;
        at = (const char*)base + (KC ? (long long)i0 * row_bytes + kb * 2LL : (long long)kb * row_bytes + i0 * 2LL);
        dead[0] = dead[1] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (KC) {                          // eight rows of 128 bytes a DMA instruction
                const int row = wave * 64 + i * 8 + (lane >> 3), c = (lane & 7) ^ ((row >> 1) & 7);
                voff[i] = (unsigned)(row * row_bytes + c * 16);
            } else {                                     // two k rows of 512 bytes; 32-byte units swapped by k's low bits
                const int k = wave * 16 + i * 2 + (lane >> 5), u = ((lane & 31) >> 1) ^ ((k & 3) << 1);
                voff[i] = (unsigned)(k * row_bytes + u * 32 + (lane & 1) * 16);
            }
        }
        if constexpr (KC) {
            const int r = w128 + (lane & 31), sw = (r >> 1) & 7;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) rd[kk] = r * 128 + (((kk * 2 + (lane >> 5)) ^ sw) << 4);
        } else {
            const int g = lane >> 4, s = lane & 15, x = (s >> 2) << 1;
#pragma unroll
            for (int u = 0; u < 4; ++u)
                rd[u] = ((g >> 1) * 8 + (s >> 2)) * 512 + ((w128 >> 4) + ((u * 2) ^ x) + (g & 1)) * 32 + (s & 3) * 8;
        }
    }

    // the descriptor of the step at `at`: everything past the operand's last element reads as nought
    __device__ __forceinline__ i32x4 rsrc() const {
        // (32 bits: a tile's rows are at most 2^21 bytes apart)
        const int k = krem < kBK ? krem : kBK;
        const int n = KC ? (idx - 1) * (int)row_bytes + krem * 2 : (k - 1) * (int)row_bytes + idx * 2;
        const unsigned long long p = (unsigned long long)at;
        return i32x4{__builtin_amdgcn_readfirstlane((int)p), __builtin_amdgcn_readfirstlane((int)(p >> 32) & 0xffff),
                     __builtin_amdgcn_readfirstlane(krem > 0 ? (n + 3) & ~3 : 0), 0x00020000};
    }
    __device__ __forceinline__ void advance(int lane) {
        at += KC ? kBK * 2 : kBK * row_bytes;
        krem -= kBK;
        if constexpr (KC) {
            // chunks behind the last k of a row hold the next row, or nothing
#pragma unroll
            for (int o = 0; o < 2; ++o) {
                const int c = (lane & 7) ^ ((o * 4 + (lane >> 4)) & 7);
                dead[o] = c * 8 >= krem ? 0x80000000u : 0u;
            }
        }
    }
    __device__ __forceinline__ void dma(i32x4 r, int i, int lds, int wave) const {
        dma_1k(r, KC ? voff[i] | dead[i & 1] : voff[i], (unsigned)(lds + wave * 8192 + i * 1024));
    }
    // fragment u (32 indices) of the 16-deep slice kk; `lds` is the panel's LDS byte address
    __device__ __forceinline__ bf16x8 frag(int lds, int kk, int u) const {
        if constexpr (KC) {
            return *(const __attribute__((address_space(3))) bf16x8*)(unsigned long long)(unsigned)(lds + rd[kk] + u * 4096);
        } else {
            typedef __attribute__((address_space(3))) bf16x4* P4;
            const unsigned a = (unsigned)(lds + rd[u] + kk * 8192);
            const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P4)(unsigned long long)a);
            const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P4)(unsigned long long)(a + 2048));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};
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

template <bool PKC, bool QKC, bool LOGITS>
__global__ __launch_bounds__(256, 1) void xent_big_kernel(const XentGemm a, int ti, int tj) {
#if defined(__HIP_DEVICE_COMPILE__)
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    float* const bias_row = (float*)(smem + kBigLds);
    float (*const red)[kBigTile][3] = (float (*)[kBigTile][3])(smem + kBigLds + kBigTile * 4);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = (wave >> 1) * 128, wj = (wave & 1) * 128;
    int bi, bj;
    tile_of(blockIdx.x, ti, tj, bi, bj);
    const int i0 = bi * kBigTile, j0 = bj * kBigTile;
    const int kb = blockIdx.y * a.k_per_split, ke = kb + a.k_per_split < a.K ? kb + a.k_per_split : a.K;
    const int steps = ke > kb ? (ke - kb + kBK - 1) / kBK : 0;

    if constexpr (LOGITS) {
        const int i = i0 + threadIdx.x;              // classes behind the last are masked like any other: by -inf
        float b = -INFINITY;
        if (i < a.I) b = !a.bias ? 0.f : a.bias_bf16 ? load1((const short*)a.bias + i) : load1((const float*)a.bias + i);
        bias_row[threadIdx.x] = b;
    }

    Panel<PKC> P;
    Panel<QKC> Q;
    P.init(a.p, a.ld_p, i0, a.I, kb, ke, wave, lane, wi);
    Q.init(a.q, a.ld_q, j0, a.Jn, kb, ke, wave, lane, wj);
    if constexpr (PKC) {                             // a single short step
        P.at -= kBK * 2; P.krem += kBK; P.advance(lane);
    }
    if constexpr (QKC) {
        Q.at -= kBK * 2; Q.krem += kBK; Q.advance(lane);
    }
    const int lds0 = (int)(unsigned long long)(__attribute__((address_space(3))) char*)smem;
    const auto dma = [&](i32x4 pr, i32x4 qr, int buf, int n) {     // the n-th of a stage's eight pairs of DMA instructions
        const int l = lds0 + buf * kStageBytes;
        P.dma(pr, n, l, wave);
        Q.dma(qr, n, l + kPanelBytes, wave);
    };
    const auto stage = [&](int buf) {
        const i32x4 pr = P.rsrc(), qr = Q.rsrc();
#pragma unroll
        for (int n = 0; n < 8; ++n) dma(pr, qr, buf, n);
        P.advance(lane);
        Q.advance(lane);
    };

    f32x16 acc[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[u][v][e] = 0.f;

    stage(0);
    stage(1);                                        // past the end: nought, and no memory touched
    asm volatile("s_waitcnt vmcnt(16)\n\ts_barrier" ::: "memory");
    bf16x8 pf[2][4], qf[2][4];
    const auto read = [&](int set, int l, int kk, int n) {         // the n-th of a slice's eight fragments
        if (n & 1) qf[set][n >> 1] = Q.frag(l + kPanelBytes, kk, n >> 1);
        else pf[set][n >> 1] = P.frag(l, kk, n >> 1);
    };
    const auto mma = [&](int set, int n) {                         // the n-th of its sixteen products, in the fragments' order
        constexpr unsigned char U[16] = {0, 1, 0, 1, 2, 2, 0, 1, 2, 3, 3, 3, 0, 1, 2, 3};
        constexpr unsigned char V[16] = {0, 0, 1, 1, 0, 1, 2, 2, 2, 0, 1, 2, 3, 3, 3, 3};
        f32x16& c = acc[U[n]][V[n]];
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(pf[set][U[n]], qf[set][V[n]], c, 0, 0, 0);
    };
#pragma unroll
    for (int n = 0; n < 8; ++n) read(0, lds0, 0, n);
    int buf = 0;
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
        const int l = lds0 + buf * kStageBytes;
        // slices 0 .. 2: the next slice's fragments under the first half of this one's MFMAs
#pragma unroll
        for (int kk = 0; kk < 3; ++kk) {
#pragma unroll
            for (int n = 0; n < 16; ++n) {
                if (n < 8) read((kk + 1) & 1, l, kk + 1, n);
                mma(kk & 1, n);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // this wave has read all it needs of this buffer, and its part of the next one has landed
        const i32x4 pr = P.rsrc(), qr = Q.rsrc();
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int ln = lds0 + (buf ^ 1) * kStageBytes;
#pragma unroll
        for (int n = 0; n < 16; ++n) {
            if (n < 8) read(0, ln, 0, n);
            else dma(pr, qr, buf, n - 8);
            mma(1, n);
            __builtin_amdgcn_sched_barrier(0);
        }
        P.advance(lane);
        Q.advance(lane);
        buf ^= 1;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

    // ---- lane: i = wi + u*32 + 8*(r/4) + 4*(lane/32) + r%4, j = wj + v*32 + lane%32 ------------------------------
    const int h4 = (lane >> 5) * 4;
    if constexpr (!LOGITS) {
        if (a.slabs) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int j = j0 + wj + v * 32 + (lane & 31);
                if (j >= a.Jn) continue;
                float* row = (float*)a.out + ((long long)blockIdx.y * a.Jn + j) * a.I;
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int i = i0 + wi + u * 32 + r * 8 + h4;
                        f32x4 d = {acc[u][v][r * 4], acc[u][v][r * 4 + 1], acc[u][v][r * 4 + 2], acc[u][v][r * 4 + 3]};
                        if (i + 3 < a.I) {
                            if (a.add) d += *(const f32x4u*)(row + i);
                            *(f32x4u*)(row + i) = d;
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (i + e < a.I) row[i + e] = a.add ? row[i + e] + d[e] : d[e];
                        }
                    }
            }
            return;
        }
        const float c = *a.factor;
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    bf16x4 o;
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = f32_to_bf16(acc[u][v][r * 4 + e] * c);
                    *(bf16x4*)(smem + (wj + v * 32 + (lane & 31)) * kOutRow + (wi + u * 32 + r * 8 + h4) * 2) = o;
                }
    } else {
        float m[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) m[v] = -INFINITY;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const f32x4 b = *(const f32x4*)(bias_row + wi + u * 32 + r * 8 + h4);
#pragma unroll
                for (int v = 0; v < 4; ++v)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        acc[u][v][r * 4 + e] += b[e];
                        m[v] = fmaxf(m[v], acc[u][v][r * 4 + e]);
                    }
            }
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int jl = wj + v * 32 + (lane & 31), j = j0 + jl;
            m[v] = fmaxf(m[v], __shfl_xor(m[v], 32, 64));
            if (lane < 32) red[wave >> 1][jl][0] = m[v];
            const long long t = j < a.Jn ? a.target[j] - i0 - wi : -1;
            const bool mine = t >= 0 && t < 128 && t + i0 + wi < a.I;
            if (__any(mine)) {
                float l = 0.f;
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) l = (int)t == u * 32 + (r >> 2) * 8 + h4 + (r & 3) ? acc[u][v][r] : l;
                if (mine && (((int)t >> 2) & 1) * 4 == h4) a.target_logit[j] = l;
            }
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int jl = wj + v * 32 + (lane & 31);
            const float mm = fmaxf(red[0][jl][0], red[1][jl][0]);
            const float ref = mm == -INFINITY ? 0.f : mm;          // a tile whose classes are all masked: sum nought, not NaN
            float s = 0.f, lin = 0.f;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    half4 o;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float l = acc[u][v][r * 4 + e], x = __expf(l - ref);
                        if (a.smooth && i0 + wi + u * 32 + r * 8 + h4 + e < a.I) lin += l;
                        s += x;
                        o[e] = (_Float16)(x * kExpScale16);
                    }
                    *(half4*)(smem + jl * kOutRow + (wi + u * 32 + r * 8 + h4) * 2) = o;
                }
            s += __shfl_xor(s, 32, 64);
            lin += __shfl_xor(lin, 32, 64);
            if (lane < 32) {
                red[wave >> 1][jl][1] = s;
                red[wave >> 1][jl][2] = lin;
            }
        }
    }
    __syncthreads();
    if constexpr (LOGITS) {
        const int jl = threadIdx.x, j = j0 + jl;
        if (j < a.Jn) {
            const long long at = (long long)j * a.tiles + bi;
            a.tile_max[at] = fmaxf(red[0][jl][0], red[1][jl][0]);
            a.tile_sum[at] = red[0][jl][1] + red[1][jl][1];
            if (a.smooth) a.tile_lin[at] = red[0][jl][2] + red[1][jl][2];
        }
        if (!a.store_e) return;
    }
    // rows out of LDS, 512 bytes a half wave
#pragma unroll 8
    for (int n = 0; n < 32; ++n) {
        const int jl = n * 8 + (threadIdx.x >> 5), c = (threadIdx.x & 31) * 8, j = j0 + jl;
        if (j >= a.Jn) break;
        const bf16x8 o = *(const bf16x8*)(smem + jl * kOutRow + c * 2);
        short* dst = (short*)a.out + j * a.ld_out + i0 + c;
        if (LOGITS || i0 + c + 8 <= a.I) {           // the exponentials' rows are padded to whole tiles
            *(bf16x8u*)dst = o;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i0 + c + e < a.I) dst[e] = o[e];
        }
    }
#endif
}

template <bool PKC, bool QKC, bool LOGITS>
static int launch_big(const XentGemm& a, hipStream_t s) {
    const int ti = ceil_div(a.I, kBigTile), tj = ceil_div(a.Jn, kBigTile);
    if ((long long)ti * tj > 0x7fffffffLL) return ASL_ETOOBIG;
    constexpr int lds = kBigLds + (LOGITS ? kBigTile * 4 * 7 : 0);
    static unsigned char lds_done[64];
    const int rc = ensure_dynamic_lds((const void*)xent_big_kernel<PKC, QKC, LOGITS>, lds, lds_done);
    if (rc != ASL_OK) return rc;
    hipLaunchKernelGGL((xent_big_kernel<PKC, QKC, LOGITS>), dim3((unsigned)(ti * tj), a.splits), dim3(256), lds, s, a, ti, tj);
    return (int)hipGetLastError();
}

int xent_big_logits(const XentGemm& a, hipStream_t s) { return launch_big<true, true, true>(a, s); }
int xent_big_dx(const XentGemm& a, hipStream_t s) { return launch_big<false, true, false>(a, s); }
int xent_big_dw(const XentGemm& a, hipStream_t s) { return launch_big<false, false, false>(a, s); }

}  // namespace asl_detail

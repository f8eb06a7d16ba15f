// Linear + softmax cross entropy for a handful of rows (up to 32: clips of one small batch), with gradients, for gfx950.
//
// Such a call is a chain of dependent launches over a weight matrix of a few megabytes, bound by latency: what counts is how
// few launches there are and that each has all its loads in flight at once.  Four launches: logits with per-tile maxima and
// sums; statistics, loss, G and the bias's gradient together (every workgroup takes all rows' statistics for itself: 32 rows
// of at most 512 tiles); both gradient products side by side; the sum of dx's slices.  All products run on fp32 MFMAs, bf16
// operands widened on load, because nothing here is bound by the matrix pipe; G stays fp32.  8 x 2000 x 512 fp32 with gradients
// takes 20 us as a graph (its launches 6.8, 4.8, 4.6 and 2.9 us): 8 MB, 2 us of this card's memory rate.
//
// The MFMA (16 x 16 x 4) wants one k of one index a lane.  A lane loads four consecutive elements and deals them to four
// MFMAs, with the same assignment of k (or of the index) on both sides, so every load is 16 bytes (8 for bf16).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "asl_hip.h"
#include "xent_args.h"

namespace asl_detail {

// A workgroup takes 32 classes; its four waves take every fourth 16 k and meet in LDS.  NB: 16-row halves of the batch.
template <typename T, int NB>
__global__ __launch_bounds__(256) void xent_few_logits_kernel(const XentFew a) {
    __shared__ __attribute__((aligned(16))) float part[4][32][33];           // [wave][row][class]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    const int c0 = blockIdx.x * kFewTile;
    f32x4 acc[2][NB];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const T* wr[2];
    const T* xr[NB];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int c = c0 + i * 16 + fr;
        wr[i] = (const T*)a.w + (c < a.classes ? c : a.classes - 1) * a.ld_w;     // surplus rows repeat one and are dropped
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int r = j * 16 + fr;
        xr[j] = (const T*)a.x + (r < a.n ? r : a.n - 1) * a.ld_x;
    }
    constexpr int U = 4;                                                     // 16-k chunks on their way at once
    for (int k0 = wave * 16; k0 < a.d; k0 += 64 * U) {
        f32x4 wf[U][2], xf[U][NB];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + u * 64 + fq * 4, n = a.d - k;
#pragma unroll
            for (int i = 0; i < 2; ++i) wf[u][i] = load4(wr[i] + (n > 0 ? k : 0), n);
#pragma unroll
            for (int j = 0; j < NB; ++j) xf[u][j] = load4(xr[j] + (n > 0 ? k : 0), n);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < NB; ++j) acc[i][j] = mma4(wf[u][i][e], xf[u][j][e], acc[i][j]);
    }
    // lane: class i*16 + fq*4 + r, row j*16 + fr
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) part[wave][j * 16 + fr][i * 16 + fq * 4 + r] = acc[i][j][r];
    __syncthreads();
    // eight lanes a row, four classes each
    const int row = threadIdx.x >> 3, cl = (threadIdx.x & 7) * 4;
    if (row >= a.n) return;                                                  // whole groups of eight leave
    float l[4], m = -INFINITY;
    const long long t = a.target[row];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int c = c0 + cl + e;
        float v = -INFINITY;
        if (c < a.classes) {
            v = part[0][row][cl + e] + part[1][row][cl + e] + part[2][row][cl + e] + part[3][row][cl + e];
            if (a.bias) v += a.bias_bf16 ? load1((const short*)a.bias + c) : load1((const float*)a.bias + c);
            if (c == t) a.target_logit[row] = v;
        }
        l[e] = v;
        m = fmaxf(m, v);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    const float ref = m == -INFINITY ? 0.f : m;          // a tile whose classes are all masked: sum nought, not NaN
    float s = 0.f, lin = 0.f;
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[e] = expf(l[e] - ref);
        s += x[e];
        if (c0 + cl + e < a.classes) lin += l[e];
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        s += __shfl_xor(s, o, 64);
        lin += __shfl_xor(lin, o, 64);
    }
    if (a.e) *(f32x4*)(a.e + row * a.ld_e + c0 + cl) = x;
    if ((threadIdx.x & 7) == 0) {
        const long long at = (long long)row * a.tiles + blockIdx.x;
        a.tile_max[at] = m;
        a.tile_sum[at] = s;
        if (a.smoothing != 0.f) a.tile_lin[at] = lin;
    }
}

// Statistics, loss, G and db: 256 columns and all rows a workgroup.
__global__ __launch_bounds__(256) void xent_few_g_kernel(const XentFew a) {
    constexpr int R = kFewRows / 8, TPB = 256 / kFewTile;
    __shared__ float fac[kFewRows][TPB], target_g[kFewRows], row_g[kFewRows], loss_row[kFewRows];
    __shared__ __attribute__((aligned(16))) float cols[8][256];
    const int lane = threadIdx.x & 63, cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const long long col = (long long)blockIdx.x * 256 + cl * 8;
    const bool in = a.e && col < a.ld_e;
    F8 g[R];
#pragma unroll
    for (int u = 0; u < R; ++u)
        if (in && rl + u * 8 < a.n) g[u] = load8_full(a.e + (rl + u * 8) * a.ld_e + col);
    const int kept_all = __popcll(__ballot(lane < a.n && a.target[lane < a.n ? lane : 0] != a.ignore));
    XentStats st = {};
    st.target = a.target; st.upstream = a.none ? a.upstream : nullptr; st.tile_max = a.tile_max; st.tile_sum = a.tile_sum;
    st.tile_lin = a.tile_lin; st.target_logit = a.target_logit; st.ignore = a.ignore; st.smoothing = a.smoothing;
    st.inv_classes = a.inv_classes; st.rows = a.n; st.classes = a.classes; st.tiles = a.tiles;
    const int l16 = threadIdx.x & 15;                        // sixteen rows at once
    for (int row = threadIdx.x >> 4; row < a.n; row += 16) {
        const XentRow r = row_stats<16>(st, row, l16);
        if (l16 == 0) {
            loss_row[row] = r.loss;
            target_g[row] = r.target_g;
            row_g[row] = r.g;
            if (blockIdx.x == 0) {
                if (a.none) a.loss[row] = r.loss;
                if (a.lse) a.lse[row] = r.lse;
            }
        }
        if (a.e && l16 < TPB) {
            const int tile = blockIdx.x * TPB + l16;
            if (tile < a.tiles) fac[row][l16] = r.valid ? r.g * expf(a.tile_max[(long long)row * a.tiles + tile] - r.lse) : NAN;
        }
    }
    __syncthreads();
    const float up = a.upstream && !a.none ? *a.upstream : 1.f;
    const float c = !a.mean ? up : kept_all ? up / (float)kept_all : 0.f;    // no row with a label: gradients are nought
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        float v = 0.f;
        for (int r = 0; r < a.n; ++r) v += loss_row[r];
        if (!a.none) *a.loss = a.mean ? v / (float)kept_all : v;
        if (a.factor) *a.factor = c;
    }
    if (!a.e) return;
    F8 db;
#pragma unroll
    for (int e = 0; e < 8; ++e) db.v[e] = 0.f;
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int r = rl + u * 8;
        if (!in || r >= a.n) continue;
        const long long t = a.target[r];
        const float f = fac[r][(cl * 8) / kFewTile], even = a.smoothing * a.inv_classes * row_g[r];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = col + e < a.classes ? g[u].v[e] * f - even : 0.f;
            if (col + e == t) v = target_g[r];
            if (t == a.ignore) v = 0.f;                      // whatever the row held
            g[u].v[e] = v;
            db.v[e] += v;
        }
        store8_full(a.e + r * a.ld_e + col, g[u]);
    }
    if (a.db) {
        store8_full(&cols[rl][cl * 8], db);
        __syncthreads();
        const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
        if (at < a.classes) {
            float v = 0.f;
#pragma unroll
            for (int q = 0; q < 8; ++q) v += cols[q][threadIdx.x];
            if (a.bias_bf16) store1((short*)a.db + at, v * c);
            else store1((float*)a.db + at, v * c);
        }
    }
}

// Both gradient products.  Workgroups below `dw_blocks`: dW of 64 classes x 64 features; the others: dx of 64 features from
// one slice of the classes, into a slab.
template <typename T, int NB>
__global__ __launch_bounds__(256) void xent_few_grad_kernel(const XentFew a, int dw_blocks, int d_tiles, int slice) {
    __shared__ __attribute__((aligned(16))) float part[4][16 * NB][64 + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    if ((int)blockIdx.x < dw_blocks) {
        const int i0 = (blockIdx.x % d_tiles) * 64, c = (blockIdx.x / d_tiles) * 64 + wave * 16 + fr;
        f32x4 acc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int i = i0 + fr * 4;
        f32x4 xf[4 * NB];
        float gf[4 * NB];
#pragma unroll
        for (int u = 0; u < 4 * NB; ++u) {
            const int k = u * 4 + fq;
            const bool ok = k < a.n;
            xf[u] = load4((const T*)a.x + (ok ? k : 0) * a.ld_x + (i < a.d ? i : 0), ok ? a.d - i : 0);
            gf[u] = ok && c < a.classes ? a.e[k * a.ld_e + c] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 4 * NB; ++u)
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[t] = mma4(xf[u][t], gf[u], acc[t]);
        // tile t, register r: feature i0 + (fq*4 + r)*4 + t -- sixteen consecutive ones a lane
        if (c < a.classes) {
            const float f = *a.factor;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int at = i0 + fq * 16 + r * 4;
                if (at < a.d)
                    store4((T*)a.dw + (long long)c * a.d + at, a.d - at, f32x4{acc[0][r] * f, acc[1][r] * f, acc[2][r] * f, acc[3][r] * f});
            }
        }
        return;
    }
    const int b = blockIdx.x - dw_blocks, i0 = (b % d_tiles) * 64, s = b / d_tiles;
    const int v0 = s * slice, v1 = v0 + slice < a.classes ? v0 + slice : a.classes;
    f32x4 acc[4][NB];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int i = i0 + fr * 4;
    // a chunk of 16 classes: MFMA e takes class 4*fq + e of it
    constexpr int U = 2;
    for (int v = v0 + wave * 16; v < v1; v += 64 * U) {
        f32x4 wf[U][4], gf[U][NB];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int vq = v + u * 64 + fq * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool ok = vq + e < v1 && i < a.d;
                wf[u][e] = load4((const T*)a.w + (ok ? (vq + e) * a.ld_w + i : 0), ok ? a.d - i : 0);
            }
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int r = j * 16 + fr;
                gf[u][j] = load4(a.e + (r < a.n && vq < v1 ? r * a.ld_e + vq : 0), r < a.n ? v1 - vq : 0);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int j = 0; j < NB; ++j) acc[t][j] = mma4(wf[u][e][t], gf[u][j][e], acc[t][j]);
    }
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            *(f32x4*)&part[wave][j * 16 + fr][fq * 16 + r * 4] = f32x4{acc[0][j][r], acc[1][j][r], acc[2][j][r], acc[3][j][r]};
    __syncthreads();
    for (int q = threadIdx.x; q < 16 * NB * 16; q += 256) {
        const int row = q >> 4, at = (q & 15) * 4;
        if (row < a.n && i0 + at < a.d) {
            f32x4 o = *(const f32x4*)&part[0][row][at];
#pragma unroll
            for (int w = 1; w < 4; ++w) o += *(const f32x4*)&part[w][row][at];
            store4(a.slabs + ((long long)s * a.n + row) * a.d + i0 + at, a.d - i0 - at, o);
        }
    }
}

// dx from the slabs: four features a thread, all slabs on their way at once
template <typename T>
__global__ __launch_bounds__(64) void xent_few_dx_kernel(const XentFew a, int slabs) {
    const int at = (blockIdx.x * 64 + threadIdx.x) * 4, row = blockIdx.y;
    if (at >= a.d) return;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < slabs; ++s) o += load4(a.slabs + ((long long)s * a.n + row) * a.d + at, a.d - at);
    o *= *a.factor;
    store4((T*)a.dx + (long long)row * a.d + at, a.d - at, o);
}

template <typename T, int NB>
static int run_few(const XentFew& a, hipStream_t s) {
    hipLaunchKernelGGL((xent_few_logits_kernel<T, NB>), dim3(a.tiles), dim3(256), 0, s, a);
    hipLaunchKernelGGL(xent_few_g_kernel, dim3(a.e ? ceil_div(a.ld_e, 256) : 1), dim3(256), 0, s, a);
    if (a.dx || a.dw) {
        const int d_tiles = ceil_div(a.d, 64), dw_blocks = a.dw ? d_tiles * ceil_div(a.classes, 64) : 0;
        const int slabs = a.dx ? xent_few_slabs(a.classes) : 0, slice = slabs ? ceil_div(ceil_div(a.classes, slabs), 16) * 16 : 1;
        hipLaunchKernelGGL((xent_few_grad_kernel<T, NB>), dim3(dw_blocks + slabs * d_tiles), dim3(256), 0, s, a, dw_blocks, d_tiles, slice);
        if (a.dx) hipLaunchKernelGGL((xent_few_dx_kernel<T>), dim3(ceil_div(a.d, 256), a.n), dim3(64), 0, s, a, slabs);
    }
    return (int)hipGetLastError();
}

int xent_few(const XentFew& a, int type, hipStream_t s) {
    if (type) return a.n <= 16 ? run_few<short, 1>(a, s) : run_few<short, 2>(a, s);
    return a.n <= 16 ? run_few<float, 1>(a, s) : run_few<float, 2>(a, s);
}

}  // namespace asl_detail

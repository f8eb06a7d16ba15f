// Linear + softmax cross entropy for a handful of rows (up to 32: clips of one small batch), with gradients, for gfx950.
//
// Such a call is a chain of dependent launches over a weight matrix of a few megabytes, bound by latency: what counts is how
// few launches there are and that each has all its loads in flight at once.  Two launches for small weights: logits with
// per-tile maxima and sums, and the rest.  Four for larger: logits; statistics, loss, G and the bias's gradient together (every
// workgroup takes all rows' statistics for itself: 32 rows of at most 512 tiles); both gradient products side by side; the sum
// of dx's slices.  All products run on fp32 MFMAs, bf16
// operands widened on load, because nothing here is bound by the matrix pipe; G stays fp32.  8 x 2000 x 512 fp32 with gradients
// takes 19 us as a graph (its launches 6.6 and 12): 8 MB, 2 us of this card's memory rate.
//
// The MFMA (16 x 16 x 4) wants one k of one index a lane.  A lane loads four consecutive elements and deals them to four
// MFMAs, with the same assignment of k (or of the index) on both sides, so every load is 16 bytes (8 for bf16).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "asl_hip.h"
#include "xent_args.h"

namespace asl_detail {

// A workgroup takes 32 classes; its eight waves take every eighth 16 k and meet in LDS (8 x 2000 x 512 forward 10.4 us, with four
// waves 11.2, with sixteen 11.6).  NB: 16-row halves of the batch.
constexpr int kLogitWaves = 8;
template <typename T, int NB>
__global__ __launch_bounds__(64 * kLogitWaves) void xent_few_logits_kernel(const XentFew a) {
    __shared__ __attribute__((aligned(16))) float part[kLogitWaves][32][33]; // [wave][row][class]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    const int c0 = blockIdx.x * kFewTile, row0 = blockIdx.y * kFewRows, n = a.n - row0 < kFewRows ? a.n - row0 : kFewRows;
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
        xr[j] = (const T*)a.x + (row0 + (r < n ? r : n - 1)) * a.ld_x;
    }
    constexpr int U = 4;                                                     // 16-k chunks on their way at once
    for (int k0 = wave * 16; k0 < a.d; k0 += 16 * kLogitWaves * U) {
        f32x4 wf[U][2], xf[U][NB];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + u * (16 * kLogitWaves) + fq * 4, left = a.d - k;
#pragma unroll
            for (int i = 0; i < 2; ++i) wf[u][i] = load4(wr[i] + (left > 0 ? k : 0), left);
#pragma unroll
            for (int j = 0; j < NB; ++j) xf[u][j] = load4(xr[j] + (left > 0 ? k : 0), left);
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
    const int at_row = threadIdx.x >> 3, cl = (threadIdx.x & 7) * 4;
    if (at_row >= n) return;                                                  // whole groups of eight leave, and waves behind the rows
    float l[4], m = -INFINITY;
    const int row = row0 + at_row;
    const long long t = a.target[row];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int c = c0 + cl + e;
        float v = -INFINITY;
        if (c < a.classes) {
            v = part[0][at_row][cl + e];
#pragma unroll
            for (int w = 1; w < kLogitWaves; ++w) v += part[w][at_row][cl + e];
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
    if (a.e) *(f32x4*)(a.e + (long long)row * a.ld_e + c0 + cl) = x;
    if ((threadIdx.x & 7) == 0) {
        const long long at = (long long)row * a.tiles + blockIdx.x;
        a.tile_max[at] = m;
        a.tile_sum[at] = s;
        if (a.smoothing != 0.f) a.tile_lin[at] = lin;
    }
}

// Statistics, loss, G and db: 256 columns and all rows a workgroup (32 x 16384: 22 us, its statistics' chain of loads).
__global__ __launch_bounds__(256) void xent_few_g_kernel(const XentFew a) {
    constexpr int R = kFewRows / 8, TPB = 256 / kFewTile;
    __shared__ float fac[kFewRows][TPB], target_g[kFewRows], row_g[kFewRows], loss_row[kFewRows];
    __shared__ __attribute__((aligned(16))) float cols[8][256];
    const int lane = threadIdx.x & 63, cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const long long col = (long long)blockIdx.x * 256 + cl * 8;
    const bool in = col < a.ld_e;
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
                if (a.lse) a.lse[row] = r.lse();
            }
        }
        if (l16 < TPB) {
            const int tile = blockIdx.x * TPB + l16;
            if (tile < a.tiles) fac[row][l16] = r.valid ? r.g * r.exp_of(a.tile_max[(long long)row * a.tiles + tile]) : NAN;
        }
    }
    __syncthreads();
    const float up = a.upstream && !a.none ? *a.upstream : 1.f;
    const float c = !a.mean ? up : kept_all ? up / (float)kept_all : 0.f;    // no row with a label: gradients are nought
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        float v = 0.f;
        for (int r = 0; r < a.n; ++r) v += loss_row[r];
        if (!a.none) *a.loss = a.mean ? v / (float)kept_all : v;
        *a.factor = c;
    }
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

// Both gradient products (32 x 16384 x 2048: 91 us, 2.9 TB/s).  Workgroups below `dw_blocks`: dW of 64 classes x 64 features;
// the others: dx of 64 features from one slice of the classes, into a slab.
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

// Everything behind the logits in one launch, for small weights: every workgroup takes the rows' statistics for itself, and G as
// it goes.  Workgroups below `dx_blocks`: dx of 16 features from all classes, a tile of 32 a wave at a time; the others: dW of
// 64 classes x 256 features, 16 x 64 a wave, and (those of the first features) db.
template <typename T, int NB>
__global__ __launch_bounds__(1024) void xent_few_rest_kernel(const XentFew a, int dx_blocks, int d_tiles) {
    __shared__ float top[kFewRows], rest[kFewRows], target_g[kFewRows], row_g[kFewRows], loss_row[kFewRows];
    __shared__ int label[kFewRows];                          // the target's class; -1: outside the vocabulary, -2: ignored
    __shared__ __attribute__((aligned(16))) float part[16][16 * NB][16 + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    const int kept_all = __popcll(__ballot(lane < a.n && a.target[lane < a.n ? lane : 0] != a.ignore));
    XentStats st = {};
    st.target = a.target; st.upstream = a.none ? a.upstream : nullptr; st.tile_max = a.tile_max; st.tile_sum = a.tile_sum;
    st.tile_lin = a.tile_lin; st.target_logit = a.target_logit; st.ignore = a.ignore; st.smoothing = a.smoothing;
    st.inv_classes = a.inv_classes; st.rows = a.n; st.classes = a.classes; st.tiles = a.tiles;
    const int mine = threadIdx.x >> 4;                       // sixteen lanes a row, all rows at once
    if (mine < kFewRows) {
        XentRow r = {0.f, 0.f, 0.f, 0.f, 0.f, true};
        if (mine < a.n) r = row_stats<16>(st, mine, fr);
        if (fr == 0) {
            top[mine] = r.top;
            rest[mine] = r.rest;
            target_g[mine] = r.target_g;
            row_g[mine] = r.valid ? r.g : NAN;
            loss_row[mine] = r.loss;
            label[mine] = mine >= a.n || a.target[mine] == a.ignore ? -2 : r.valid ? (int)a.target[mine] : -1;
            if (blockIdx.x == 0 && mine < a.n) {
                if (a.none) a.loss[mine] = r.loss;
                if (a.lse) a.lse[mine] = r.lse();
            }
        }
    }
    __syncthreads();
    const float up = a.upstream && !a.none ? *a.upstream : 1.f;
    const float c = !a.mean ? up : kept_all ? up / (float)kept_all : 0.f;    // no row with a label: gradients are nought
    if (blockIdx.x == 0 && threadIdx.x == 0 && !a.none) {
        float v = 0.f;
        for (int r = 0; r < a.n; ++r) v += loss_row[r];
        *a.loss = a.mean ? v / (float)kept_all : v;
    }
    if (!a.e) return;
    const float smooth = a.smoothing * a.inv_classes;
    // G from an exponential and its tile's maximum
    const auto grad = [&](float e, float f, int row, int col) {
        float v = col < a.classes ? e * f - smooth * row_g[row] : 0.f;
        if (col == label[row]) v = target_g[row];
        return label[row] == -2 ? 0.f : v;                   // whatever the row held
    };
    if ((int)blockIdx.x < dx_blocks) {
        const int i = blockIdx.x * 16 + fr, ic = i < a.d ? i : a.d - 1;      // surplus features repeat one and are dropped
        f32x4 acc[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        // MFMA s takes class 8*fq + s of a tile; two tiles on their way at once
        constexpr int U = 2;
        for (int t0 = wave; t0 < a.tiles; t0 += 16 * U) {
            float wf[U][8], m[U][NB];
            F8 e[U][NB];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int t = t0 + u * 16 < a.tiles ? t0 + u * 16 : t0, v = t * kFewTile + fq * 8;
#pragma unroll
                for (int s = 0; s < 8; ++s) wf[u][s] = load1((const T*)a.w + (v + s < a.classes ? v + s : 0) * a.ld_w + ic);
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    const int r = j * 16 + fr < a.n ? j * 16 + fr : 0;
                    e[u][j] = load8_full(a.e + r * a.ld_e + v);
                    m[u][j] = a.tile_max[(long long)r * a.tiles + t];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t0 + u * 16 >= a.tiles) break;
                const int v = (t0 + u * 16) * kFewTile + fq * 8;
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    const int row = j * 16 + fr;
                    const float f = row_g[row] * expf((m[u][j] - top[row]) - rest[row]);
#pragma unroll
                    for (int s = 0; s < 8; ++s) acc[j] = mma4(v + s < a.classes ? wf[u][s] : 0.f, grad(e[u][j].v[s], f, row, v + s), acc[j]);
                }
            }
        }
        // lane: feature fq*4 + r, row j*16 + fr
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) part[wave][j * 16 + fr][fq * 4 + r] = acc[j][r];
        __syncthreads();
        if (threadIdx.x < 256 * NB) {
            const int row = threadIdx.x >> 4;
            float o = 0.f;
#pragma unroll
            for (int w = 0; w < 16; ++w) o += part[w][row][fr];
            if (row < a.n && i < a.d) store1((T*)a.dx + (long long)row * a.d + i, o * c);
        }
        return;
    }
    const int b = blockIdx.x - dx_blocks, i0 = (b % d_tiles) * 256 + (wave >> 2) * 64, col = (b / d_tiles) * 64 + (wave & 3) * 16 + fr;
    const int cc = col < a.classes ? col : a.classes - 1, i = i0 + fr * 4;
    f32x4 xf[4 * NB];
    float gf[4 * NB], ef[4 * NB], mf[4 * NB];
#pragma unroll
    for (int u = 0; u < 4 * NB; ++u) {
        const int k = u * 4 + fq, r = k < a.n ? k : 0;
        xf[u] = load4((const T*)a.x + r * a.ld_x + (i < a.d ? i : 0), k < a.n ? a.d - i : 0);
        ef[u] = a.e[r * a.ld_e + cc];
        mf[u] = a.tile_max[(long long)r * a.tiles + cc / kFewTile];
    }
    float db = 0.f;
#pragma unroll
    for (int u = 0; u < 4 * NB; ++u) {
        const int k = u * 4 + fq;
        gf[u] = col < a.classes ? grad(ef[u], row_g[k] * expf((mf[u] - top[k]) - rest[k]), k, col) : 0.f;
        db += gf[u];
    }
    if (a.dw) {
        f32x4 acc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 4 * NB; ++u)
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[t] = mma4(xf[u][t], gf[u], acc[t]);
        // tile t, register r: feature i0 + (fq*4 + r)*4 + t -- sixteen consecutive ones a lane
        if (col < a.classes) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int at = i0 + fq * 16 + r * 4;
                if (at < a.d)
                    store4((T*)a.dw + (long long)col * a.d + at, a.d - at, f32x4{acc[0][r] * c, acc[1][r] * c, acc[2][r] * c, acc[3][r] * c});
            }
        }
    }
    if (a.db && b % d_tiles == 0 && wave < 4) {
        db += __shfl_xor(db, 16, 64);
        db += __shfl_xor(db, 32, 64);
        if (fq == 0 && col < a.classes) {
            if (a.bias_bf16) store1((short*)a.db + col, db * c);
            else store1((float*)a.db + col, db * c);
        }
    }
}

// One launch behind the logits for weights up to 2048 x 2048 or as many elements in fewer classes, or for none wanted; three
// for larger, where what every workgroup would do for itself adds up and strips of 16 features cost W's lines twice.  fp32 with
// gradients, as graphs: 8 x 100 x 512 13 us against 16, 8 x 2000 x 512 19 against 20 (as calls, which four launches bound, 20
// and 25), 8 x 2000 x 2048 36 against 39; 32 x 4000 x 512 42 against 36, 8 x 8000 x 1024 57 against 49, 32 x 16384 x 2048 222
// against 162.
static bool one_launch(const XentFew& a) { return !a.e || (a.classes <= 2048 && (double)a.classes * a.d <= (double)(1 << 22)); }

template <typename T, int NB>
static int run_few(const XentFew& a, hipStream_t s) {
    hipLaunchKernelGGL((xent_few_logits_kernel<T, NB>), dim3(a.tiles), dim3(64 * kLogitWaves), 0, s, a);
    if (one_launch(a)) {
        const int dx_blocks = a.e && a.dx ? ceil_div(a.d, 16) : 0, d_tiles = a.e && a.dw ? ceil_div(a.d, 256) : 1;
        const int dw_blocks = a.e && (a.dw || a.db) ? d_tiles * ceil_div(a.classes, 64) : 0, blocks = dx_blocks + dw_blocks;
        hipLaunchKernelGGL((xent_few_rest_kernel<T, NB>), dim3(blocks ? blocks : 1), dim3(1024), 0, s, a, dx_blocks, d_tiles);
        return (int)hipGetLastError();
    }
    hipLaunchKernelGGL(xent_few_g_kernel, dim3(ceil_div(a.ld_e, 256)), dim3(256), 0, s, a);
    if (a.dx || a.dw) {
        const int d_tiles = ceil_div(a.d, 64), dw_blocks = a.dw ? d_tiles * ceil_div(a.classes, 64) : 0;
        const int slabs = a.dx ? xent_few_slabs(a.classes) : 0, slice = slabs ? ceil_div(ceil_div(a.classes, slabs), 16) * 16 : 1;
        hipLaunchKernelGGL((xent_few_grad_kernel<T, NB>), dim3(dw_blocks + slabs * d_tiles), dim3(256), 0, s, a, dw_blocks, d_tiles, slice);
        if (a.dx) hipLaunchKernelGGL((xent_few_dx_kernel<T>), dim3(ceil_div(a.d, 256), a.n), dim3(64), 0, s, a, slabs);
    }
    return (int)hipGetLastError();
}

void xent_few_logits(const XentFew& a, hipStream_t s) {
    hipLaunchKernelGGL((xent_few_logits_kernel<float, 2>), dim3(a.tiles, ceil_div(a.n, kFewRows)), dim3(64 * kLogitWaves), 0, s, a);
}

int xent_few(const XentFew& a, int type, hipStream_t s) {
    static_assert(kFewRows16 <= 16 && kFewRows <= 32, "halves of 16 rows");
    if (a.n > (type ? kFewRows16 : kFewRows)) return ASL_EINVAL;
    if (type) return run_few<short, 1>(a, s);
    return a.n <= 16 ? run_few<float, 1>(a, s) : run_few<float, 2>(a, s);
}

}  // namespace asl_detail

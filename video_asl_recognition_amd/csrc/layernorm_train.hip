// LayerNorm for training on gfx950: forward with saved statistics, and backward with the reduction of the weight's and
// bias's gradients.
//
//   mu = mean x,  r = 1 / sqrt(mean (x - mu)^2 + eps),  h = (x - mu) r,  y = h w + b
//   g = dy w,  dx = r (g - mean g - h mean(g h)),  dw = sum over rows of dy h,  db = sum over rows of dy
//
// Both directions move bytes and little else, so a row is read once: a group of G lanes (a quarter wave up to a workgroup of
// 1024) holds it in registers, J vectors of eight elements a lane, and all sums are taken there, in fp32, the variance about
// the mean that was just found.  Backward keeps each lane's columns fixed while its group walks over rows, so the column
// sums dw and db also stay in registers; a workgroup leaves one partial row of each in the workspace and a second launch
// adds those up in a fixed order (no atomics: results do not vary from run to run).
//
// What bounds them is memory: 2^26 elements take, in bf16, 41 us forward and 76 us backward with rows of 1024 (x and y, or x,
// dy and dx, at 6.5 and 5.3 TB/s, part of it from the 256 MB cache; a copy of 2 GiB reaches 4.95) and 46 and 79 us with rows
// of 128 and 512, in fp32 102 to 112 us and 148 to 163 us with rows of 64 to 8192.  Small calls are two and three launches.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "asl_hip.h"
#include "train_common.h"

namespace asl_detail {

// eight of a weight or bias, or of the constant that stands for a missing one
__device__ __forceinline__ F8 load8_or(const void* base, int bf16, long long at, int n, float missing) {
    if (base) return load8_any(base, bf16, at, n);
    return {{missing, missing, missing, missing, missing, missing, missing, missing}};
}

struct LnArgs {
    const void* x;
    const void* dy;
    const void* w;
    const void* b;
    void* y;                 // forward: y; backward: dx
    float* mean;
    float* rstd;
    float* part;             // backward: [blocks][2][d] column sums
    long long ld_x, ld_y, ld_dy;
    int rows, d, w_bf16;
    float eps;
};

// a variance that rounding took below nought is nought; a NaN stays one (fmaxf would hide it)
__device__ __forceinline__ float not_below_nought(float v) { return v < 0.f ? 0.f : v; }

// Sum over the G lanes of a group, the same in every lane.  Groups wider than a wave meet in LDS: `slot` alternates from
// call to call, so one barrier a call is enough (a slot is written again only behind the next call's barrier).
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* lds, int& slot) {
    static_assert(G == 16 || G >= 64, "a quarter wave, or whole waves");
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = G == 16 ? row16_sum(v[k]) : wave64_sum(v[k]);
    if constexpr (G > 64) {
        constexpr int NW = G / 64;
        float* s = lds + slot * (NW * N);
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) s[(threadIdx.x >> 6) * N + k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) t += s[i * N + k];
            v[k] = t;
        }
        slot ^= 1;
    }
}

// Vector j of lane t begins at column (t + j G) 8, but the one that would reach over the row's end ends with it: it shares its
// first `lead` columns with its neighbour, which takes them for the sums, and both write them, the same.  So every access is a
// whole vector, in rows of at least eight elements, and none branches by lane (2^26 bf16 elements, backward: rows of 500 80 us,
// with a last vector loaded by element 214; rows of 2047 109 and 190).
template <int G, int J>
struct Columns {
    int at[J], lead[J];
    __device__ __forceinline__ Columns(int t, int d) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int k = (t + j * G) * 8;
            at[j] = k + 8 <= d ? k : d >= 8 ? d - 8 : 0;
            lead[j] = k - at[j];
        }
    }
    __device__ __forceinline__ bool any(int j) const { return lead[j] < 8; }
    __device__ __forceinline__ bool mine(int j, int e, int d) const { return e >= lead[j] && at[j] + e < d; }
};

// w and b stay in registers from row to row where a lane has at most two vectors of a row; with more, the registers go to
// occupancy and both come from the L1 with every row.  The next row is on its way while this one is worked on.
template <typename XT, typename YT, int G, int J>
__global__ __launch_bounds__(G > 256 ? G : 256) void ln_fwd_kernel(const LnArgs a) {
    constexpr int BLOCK = G > 256 ? G : 256, RPB = BLOCK / G;
    constexpr bool HOLD = J <= 2;
    __shared__ float lds[2 * 2 * (G > 64 ? G / 64 : 1)];
    int slot = 0;
    const int t = threadIdx.x % G;
    const Columns<G, J> c(t, a.d);
    const float inv_d = 1.0f / (float)a.d;
    F8 w[HOLD ? J : 1], b[HOLD ? J : 1];
    if constexpr (HOLD) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            w[j] = load8_or(a.w, a.w_bf16, c.at[j], a.d, 1.f);
            b[j] = load8_or(a.b, a.w_bf16, c.at[j], a.d, 0.f);
        }
    }
    typename RawOf<XT>::type next[J];
    const auto fetch = [&](long long row) {
        const XT* xr = (const XT*)a.x + row * a.ld_x;
#pragma unroll
        for (int j = 0; j < J; ++j) next[j] = load8_raw(xr + c.at[j], a.d);
    };
    const long long stride = (long long)gridDim.x * RPB;
    long long row = (long long)blockIdx.x * RPB + threadIdx.x / G;
    fetch(row < a.rows ? row : 0);
    // groups wider than a wave are one a workgroup, so all of its threads leave the loop together
    for (; row < a.rows; row += stride) {
        F8 x[J];
        float s[1] = {0.f};
#pragma unroll
        for (int j = 0; j < J; ++j) {
            x[j] = widen(next[j]);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[0] += c.mine(j, e, a.d) ? x[j].v[e] : 0.f;
        }
        if (row + stride < a.rows) fetch(row + stride);
        group_sum<G>(s, lds, slot);
        const float mean = s[0] * inv_d;
        // about the rounded mean; the rest of the mean that its rounding left comes out of the same pass, so a row of
        // equal large values has variance nought and not the square of its last bit
        float q[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < J; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[j].v[e] -= mean;
                const float m = c.mine(j, e, a.d) ? x[j].v[e] : 0.f;
                q[0] += m;
                q[1] += m * m;
            }
        }
        group_sum<G>(q, lds, slot);
        const float rest = q[0] * inv_d;
        const float rstd = 1.0f / sqrtf(not_below_nought(q[1] * inv_d - rest * rest) + a.eps);
        YT* yr = (YT*)a.y + row * a.ld_y;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (c.any(j)) {
                if constexpr (!HOLD) {
                    w[0] = load8_or(a.w, a.w_bf16, c.at[j], a.d, 1.f);
                    b[0] = load8_or(a.b, a.w_bf16, c.at[j], a.d, 0.f);
                }
                const F8 &wj = w[HOLD ? j : 0], &bj = b[HOLD ? j : 0];
                F8 o;
#pragma unroll
                for (int e = 0; e < 8; ++e) o.v[e] = (x[j].v[e] - rest) * rstd * wj.v[e] + bj.v[e];
                store8(yr + c.at[j], a.d, o);
            }
        }
        if (t == 0) {
            if (a.mean) a.mean[row] = mean + rest;
            if (a.rstd) a.rstd[row] = rstd;
        }
    }
}

// rows longer than the registers of a workgroup: the same sums in three passes over the row, the later two from L2
template <typename XT, typename YT>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(const LnArgs a) {
    constexpr int G = 1024;
    __shared__ float lds[2 * 2 * (G / 64)];
    int slot = 0;
    const int t = threadIdx.x;
    const float inv_d = 1.0f / (float)a.d;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const XT* xr = (const XT*)a.x + row * a.ld_x;
        float s[1] = {0.f};
#pragma unroll 4
        for (int k = t * 8; k < a.d; k += G * 8) {
            const F8 x = load8(xr + k, a.d - k);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[0] += x.v[e];
        }
        group_sum<G>(s, lds, slot);
        const float mean = s[0] * inv_d;
        float q[2] = {0.f, 0.f};
#pragma unroll 4
        for (int k = t * 8; k < a.d; k += G * 8) {
            const F8 x = load8(xr + k, a.d - k);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float c = k + e < a.d ? x.v[e] - mean : 0.f;
                q[0] += c;
                q[1] += c * c;
            }
        }
        group_sum<G>(q, lds, slot);
        const float rest = q[0] * inv_d;
        const float rstd = 1.0f / sqrtf(not_below_nought(q[1] * inv_d - rest * rest) + a.eps);
        YT* yr = (YT*)a.y + row * a.ld_y;
#pragma unroll 4
        for (int k = t * 8; k < a.d; k += G * 8) {
            const F8 x = load8(xr + k, a.d - k);
            const F8 w = load8_or(a.w, a.w_bf16, k, a.d - k, 1.f), b = load8_or(a.b, a.w_bf16, k, a.d - k, 0.f);
            F8 o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o.v[e] = (x.v[e] - mean - rest) * rstd * w.v[e] + b.v[e];
            store8(yr + k, a.d - k, o);
        }
        if (t == 0) {
            if (a.mean) a.mean[row] = mean + rest;
            if (a.rstd) a.rstd[row] = rstd;
        }
    }
}

// SUMS: with the column sums.  Rows too long for that (a lane's vectors, their sums and the next row's) leave them to
// ln_cols_kernel.
template <typename XT, typename YT, int G, int J, bool SUMS>
__global__ __launch_bounds__(G > 256 ? G : 256) void ln_bwd_kernel(const LnArgs a) {
    constexpr int BLOCK = G > 256 ? G : 256, RPB = BLOCK / G;
    constexpr bool HOLD = J <= 2 && G * J < 2048, AHEAD = G * J < 4096;
    __shared__ float lds[2 * 2 * (G > 64 ? G / 64 : 1)];
    __shared__ __attribute__((aligned(16))) float cols[RPB > 1 ? 4 * 2 * (G < 64 ? G : 64) * 8 : 1];
    int slot = 0;
    const int t = threadIdx.x % G;
    const Columns<G, J> c(t, a.d);
    const float inv_d = 1.0f / (float)a.d;
    F8 w[HOLD ? J : 1], dw[SUMS ? J : 1], db[SUMS ? J : 1];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        if constexpr (HOLD) w[j] = load8_or(a.w, a.w_bf16, c.at[j], a.d, 1.f);
        if constexpr (SUMS)
#pragma unroll
            for (int e = 0; e < 8; ++e) dw[j].v[e] = db[j].v[e] = 0.f;
    }
    typename RawOf<XT>::type next_x[J];
    typename RawOf<YT>::type next_dy[J];
    float next_mean, next_rstd;
    const auto fetch = [&](long long row) {
        const XT* xr = (const XT*)a.x + row * a.ld_x;
        const YT* dyr = (const YT*)a.dy + row * a.ld_dy;
        next_mean = a.mean[row];
        next_rstd = a.rstd[row];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            next_x[j] = load8_raw(xr + c.at[j], a.d);
            next_dy[j] = load8_raw(dyr + c.at[j], a.d);
        }
    };
    const long long stride = (long long)gridDim.x * RPB;
    long long row = (long long)blockIdx.x * RPB + threadIdx.x / G;
    if (AHEAD && row < a.rows) fetch(row);
    for (; row < a.rows; row += stride) {
        if (!AHEAD) fetch(row);
        const float mean = next_mean, rstd = next_rstd;
        F8 h[J], g[J];
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < J; ++j) {
            h[j] = widen(next_x[j]);
            g[j] = widen(next_dy[j]);
        }
        if (AHEAD && row + stride < a.rows) fetch(row + stride);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if constexpr (!HOLD) w[0] = load8_or(a.w, a.w_bf16, c.at[j], a.d, 1.f);
            const F8& wj = w[HOLD ? j : 0];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[j].v[e] = (h[j].v[e] - mean) * rstd;
                if constexpr (SUMS) {
                    dw[j].v[e] += g[j].v[e] * h[j].v[e];
                    db[j].v[e] += g[j].v[e];
                }
                g[j].v[e] *= wj.v[e];
                s[0] += c.mine(j, e, a.d) ? g[j].v[e] : 0.f;
                s[1] += c.mine(j, e, a.d) ? g[j].v[e] * h[j].v[e] : 0.f;
            }
        }
        group_sum<G>(s, lds, slot);
        const float m0 = s[0] * inv_d, m1 = s[1] * inv_d;
        XT* dxr = (XT*)a.y + row * a.ld_y;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (c.any(j)) {
                F8 o;
#pragma unroll
                for (int e = 0; e < 8; ++e) o.v[e] = (g[j].v[e] - m0 - h[j].v[e] * m1) * rstd;
                store8(dxr + c.at[j], a.d, o);
            }
        }
    }
    float* part = a.part + (long long)blockIdx.x * 2 * a.d;
    const auto leave = [&](float* row, int j, const F8& v) {      // a vector's own columns of a row that begins at `row`
        if (c.lead[j] == 0 && a.d >= 8) {
            store8_full(row + c.at[j], v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c.mine(j, e, a.d)) row[c.at[j] + e] = v.v[e];
        }
    };
    if constexpr (!SUMS) {
    } else if constexpr (RPB == 1) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            leave(part, j, dw[j]);
            leave(part + a.d, j, db[j]);
        }
    } else {
        // several groups a workgroup: within the wave by lane exchange, then the waves' sums through LDS, a vector at a time
        constexpr int L = G < 64 ? G : 64, COLS = L * 8, NW = BLOCK / 64;
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < J; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int o = 32; o >= G; o >>= 1) {
                    dw[j].v[e] += __shfl_xor(dw[j].v[e], o, 64);
                    db[j].v[e] += __shfl_xor(db[j].v[e], o, 64);
                }
            if (lane < L) {
                leave(cols + (wave * 2 + 0) * COLS - j * COLS, j, dw[j]);
                leave(cols + (wave * 2 + 1) * COLS - j * COLS, j, db[j]);
            }
            __syncthreads();
            for (int i = threadIdx.x; i < 2 * COLS; i += BLOCK) {
                const int which = i / COLS, k = i % COLS;
                float v = 0.f;
#pragma unroll
                for (int q = 0; q < NW; ++q) v += cols[(q * 2 + which) * COLS + k];
                if (j * COLS + k < a.d) part[which * a.d + j * COLS + k] = v;
            }
            __syncthreads();
        }
    }
}

// rows longer than the registers of a workgroup: sums, then dx, from re-read rows
template <typename XT, typename YT>
__global__ __launch_bounds__(1024) void ln_bwd_long_kernel(const LnArgs a) {
    constexpr int G = 1024;
    __shared__ float lds[2 * 2 * (G / 64)];
    int slot = 0;
    const int t = threadIdx.x;
    const float inv_d = 1.0f / (float)a.d;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const XT* xr = (const XT*)a.x + row * a.ld_x;
        const YT* dyr = (const YT*)a.dy + row * a.ld_dy;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s[2] = {0.f, 0.f};
#pragma unroll 4
        for (int k = t * 8; k < a.d; k += G * 8) {
            const int n = a.d - k;
            const F8 x = load8(xr + k, n), dy = load8(dyr + k, n), w = load8_or(a.w, a.w_bf16, k, n, 1.f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float g = dy.v[e] * w.v[e];                // dy is nought behind the row's end
                s[0] += g;
                s[1] += g * ((x.v[e] - mean) * rstd);
            }
        }
        group_sum<G>(s, lds, slot);
        const float m0 = s[0] * inv_d, m1 = s[1] * inv_d;
        XT* dxr = (XT*)a.y + row * a.ld_y;
#pragma unroll 4
        for (int k = t * 8; k < a.d; k += G * 8) {
            const int n = a.d - k;
            const F8 x = load8(xr + k, n), dy = load8(dyr + k, n), w = load8_or(a.w, a.w_bf16, k, n, 1.f);
            F8 o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o.v[e] = (dy.v[e] * w.v[e] - m0 - (x.v[e] - mean) * rstd * m1) * rstd;
            store8(dxr + k, n, o);
        }
    }
}

// The column sums of long rows from a second reading: 512 columns a workgroup, its four waves on rows in turn, four rows at a
// time on their way; blockIdx.y-th of the partial rows.
template <typename XT, typename YT>
__global__ __launch_bounds__(256) void ln_cols_kernel(const LnArgs a) {
    constexpr int U = 4;
    __shared__ __attribute__((aligned(16))) float cols[2][4][512];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int k = (blockIdx.x * 64 + lane) * 8, n = a.d - k;
    F8 dw, db;
#pragma unroll
    for (int e = 0; e < 8; ++e) dw.v[e] = db.v[e] = 0.f;
    const long long stride = gridDim.y * 4LL;
    for (long long row = blockIdx.y * 4LL + wave; row < a.rows; row += stride * U) {
        typename RawOf<XT>::type x[U];
        typename RawOf<YT>::type dy[U];
        float mean[U], rstd[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool there = row + u * stride < a.rows;
            const long long r = there ? row + u * stride : row;
            x[u] = load8_raw((const XT*)a.x + r * a.ld_x + (n > 0 ? k : 0), n);
            dy[u] = load8_raw((const YT*)a.dy + r * a.ld_dy + (n > 0 ? k : 0), there ? n : 0);
            mean[u] = a.mean[r];
            rstd[u] = a.rstd[r];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool there = row + u * stride < a.rows;
            const F8 h = widen(x[u]), g = widen(dy[u]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (there) dw.v[e] += g.v[e] * ((h.v[e] - mean[u]) * rstd[u]);
                if (there) db.v[e] += g.v[e];
            }
        }
    }
    store8_full(&cols[0][wave][lane * 8], dw);
    store8_full(&cols[1][wave][lane * 8], db);
    __syncthreads();
    float* part = a.part + (long long)blockIdx.y * 2 * a.d;
    for (int i = threadIdx.x; i < 1024; i += 256) {
        const int which = i >> 9, c = i & 511;
        if (blockIdx.x * 512 + c < a.d)
            part[which * (long long)a.d + blockIdx.x * 512 + c] = (cols[which][0][c] + cols[which][1][c]) + (cols[which][2][c] + cols[which][3][c]);
    }
}

// 64 columns a workgroup of 1024: 16 lanes of four columns by 64 row strides, so that the up to 512 partial rows, which other
// XCDs have just written and which come from memory, are all on their way at once
__global__ __launch_bounds__(1024) void column_sums_kernel(const float* __restrict__ part, int parts, int d, void* dw, void* db, int bf16) {
    __shared__ float s[64][64 + 1];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
    const long long cols = 2LL * d, c0 = (long long)blockIdx.x * 64 + c * 4;
    const int n = cols - c0 >= 4 ? 4 : cols > c0 ? (int)(cols - c0) : 0;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (n == 4) {
#pragma unroll 8
        for (int p = r; p < parts; p += 64) v += *(const f32x4u*)(part + p * cols + c0);
    } else if (n) {
        for (int p = r; p < parts; p += 64)
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < n) v[e] += part[p * cols + c0 + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s[r][c * 4 + e] = v[e];
    __syncthreads();
    // sixteen lanes a column, four rows each, then across the lanes
    const int k = threadIdx.x >> 4, q = threadIdx.x & 15;
    const float o = row16_sum((s[q][k] + s[q + 16][k]) + (s[q + 32][k] + s[q + 48][k]));
    const long long col = (long long)blockIdx.x * 64 + k;
    if (q == 0 && col < cols) {
        void* out = col < d ? dw : db;
        const long long at = col < d ? col : col - d;
        if (out) {
            if (bf16) store1((short*)out + at, o);
            else store1((float*)out + at, o);
        }
    }
}

// Lanes a row and vectors a lane, by the row's length.  Forward holds one row and the next (16 J registers), backward x, dy, two
// column sums and the next row's (48 J).  2^26 elements in bf16, forward and backward: rows of 200 on 16 lanes 48 and 83 us, on
// a wave that they leave more than half idle 95 and 165; rows of 2048 on four waves 45 and 79 us, on one wave, which then has
// a SIMD to itself but for one other, 50 and 90.  Rows above 8192: forward holds them with 256 threads up to 16384 (68 us, with 1024 threads 110), and reads
// longer ones three times, twice from the L2 (79 us; from the registers of 1024 threads, whose rows do not overlap, the same).
// Backward has no registers left for the column sums: from a second reading of x and dy, rows of 12288 take 131 us, with sums
// that spill 232; rows of 32768 162 us, with sums kept in memory 350.
struct LnShape {
    int g, j;
};
inline LnShape fwd_shape(int d) {
    if (d <= 128) return {16, 1};
    if (d <= 256) return {16, 2};
    if (d <= 512) return {64, 1};
    if (d <= 1024) return {64, 2};
    if (d <= 2048) return {256, 1};
    if (d <= 4096) return {256, 2};
    if (d <= 8192) return {256, 4};
    if (d <= 16384) return {256, 8};
    return {0, 0};
}
inline LnShape bwd_shape(int d) {
    if (d <= 128) return {16, 1};
    if (d <= 256) return {16, 2};
    if (d <= 512) return {64, 1};
    if (d <= 1024) return {64, 2};
    if (d <= 2048) return {256, 1};
    if (d <= 4096) return {256, 2};
    if (d <= 8192) return {1024, 1};
    if (d <= 16384) return {1024, 2};
    return {0, 0};
}
constexpr int kColsWith = 8192;           // longest row whose column sums go along
inline int rows_per_block(int g) { return g == 0 || g > 256 ? 1 : 256 / g; }

// Workgroups of a backward call = partial rows of its column sums: two a CU, so that the partial rows stay small against the
// tensors, or four for bf16 rows of 1025 to 1919, of which a workgroup has but one, and a short one, under way.  Two and four,
// 2^26 elements: bf16 rows of 1280 115 and 85 us, 1536 99 and 83, 1792 86 and 82, 1920 83 and 81, 2040 81 and 87, 2048 79 and 83;
// 2^23 elements: 1280 21.3 and 19.5, 1792 18.6 and 18.7, 2040 18.3 and 20.8.  fp32 x and bf16 dy: 1025 154 and 151, 1200 136
// and 141, 1800 141 and 140; fp32 both: 1280 152 and 160, 2048 149 and 159.
inline int bwd_blocks(const asl_layernorm_params& p) {
    const int rows = p.rows, d = p.d;
    if (d > kColsWith) {                  // ln_cols_kernel: eight workgroups a CU, each of at least 16 rows
        const int strips = (d + 511) / 512, most = strips < 2048 ? 2048 / strips : 1, need = (int)(((long long)rows + 15) / 16);
        return need < most ? need : most;
    }
    const LnShape sh = bwd_shape(d);
    const int rpb = rows_per_block(sh.g), most = sh.g == 256 && sh.j == 1 && p.x_type && p.y_type && d < 1920 ? 1024 : 512;
    const long long need = ((long long)rows + rpb - 1) / rpb;
    return (int)(need < most ? need : most);
}

template <typename XT, typename YT>
int launch_fwd(const LnArgs& a, hipStream_t s) {
    const LnShape sh = fwd_shape(a.d);
    const int rpb = rows_per_block(sh.g);
    const long long need = ((long long)a.rows + rpb - 1) / rpb;
    const dim3 grid((unsigned)(need < 4096 ? need : 4096)), b256(256), b1024(1024);
    switch (sh.g * 16 + sh.j) {
        case 16 * 16 + 1: hipLaunchKernelGGL((ln_fwd_kernel<XT, YT, 16, 1>), grid, b256, 0, s, a); break;
        case 16 * 16 + 2: hipLaunchKernelGGL((ln_fwd_kernel<XT, YT, 16, 2>), grid, b256, 0, s, a); break;
        case 64 * 16 + 1: hipLaunchKernelGGL((ln_fwd_kernel<XT, YT, 64, 1>), grid, b256, 0, s, a); break;
        case 64 * 16 + 2: hipLaunchKernelGGL((ln_fwd_kernel<XT, YT, 64, 2>), grid, b256, 0, s, a); break;
        case 256 * 16 + 1: hipLaunchKernelGGL((ln_fwd_kernel<XT, YT, 256, 1>), grid, b256, 0, s, a); break;
        case 256 * 16 + 2: hipLaunchKernelGGL((ln_fwd_kernel<XT, YT, 256, 2>), grid, b256, 0, s, a); break;
        case 256 * 16 + 4: hipLaunchKernelGGL((ln_fwd_kernel<XT, YT, 256, 4>), grid, b256, 0, s, a); break;
        case 256 * 16 + 8: hipLaunchKernelGGL((ln_fwd_kernel<XT, YT, 256, 8>), grid, b256, 0, s, a); break;
        default: hipLaunchKernelGGL((ln_fwd_long_kernel<XT, YT>), grid, b1024, 0, s, a); break;
    }
    return (int)hipGetLastError();
}

template <typename XT, typename YT>
int launch_bwd(const LnArgs& a, int blocks, bool want_cols, hipStream_t s) {
    const LnShape sh = bwd_shape(a.d);
    const bool apart = a.d > kColsWith;
    const dim3 grid((unsigned)(!apart ? blocks : a.rows < 4096 ? a.rows : 4096)), b256(256), b1024(1024);
    switch (sh.g * 16 + sh.j) {
        case 16 * 16 + 1: hipLaunchKernelGGL((ln_bwd_kernel<XT, YT, 16, 1, true>), grid, b256, 0, s, a); break;
        case 16 * 16 + 2: hipLaunchKernelGGL((ln_bwd_kernel<XT, YT, 16, 2, true>), grid, b256, 0, s, a); break;
        case 64 * 16 + 1: hipLaunchKernelGGL((ln_bwd_kernel<XT, YT, 64, 1, true>), grid, b256, 0, s, a); break;
        case 64 * 16 + 2: hipLaunchKernelGGL((ln_bwd_kernel<XT, YT, 64, 2, true>), grid, b256, 0, s, a); break;
        case 256 * 16 + 1: hipLaunchKernelGGL((ln_bwd_kernel<XT, YT, 256, 1, true>), grid, b256, 0, s, a); break;
        case 256 * 16 + 2: hipLaunchKernelGGL((ln_bwd_kernel<XT, YT, 256, 2, true>), grid, b256, 0, s, a); break;
        case 1024 * 16 + 1: hipLaunchKernelGGL((ln_bwd_kernel<XT, YT, 1024, 1, true>), grid, b1024, 0, s, a); break;
        case 1024 * 16 + 2: hipLaunchKernelGGL((ln_bwd_kernel<XT, YT, 1024, 2, false>), grid, b1024, 0, s, a); break;
        default: hipLaunchKernelGGL((ln_bwd_long_kernel<XT, YT>), grid, b1024, 0, s, a); break;
    }
    if (apart && want_cols)
        hipLaunchKernelGGL((ln_cols_kernel<XT, YT>), dim3((unsigned)((a.d + 511) / 512), (unsigned)blocks), b256, 0, s, a);
    return (int)hipGetLastError();
}

int ln_check(const asl_layernorm_params* p) {
    if (!p || p->rows < 0 || p->d <= 0) return ASL_EINVAL;
    if (p->x_type < 0 || p->x_type > 1 || p->w_type < 0 || p->w_type > 1 || p->y_type < 0 || p->y_type > 1) return ASL_EINVAL;
    if (p->ld_x < p->d || p->ld_y < p->d || p->ld_dx < p->d) return ASL_EINVAL;
    return p->d > (1 << 26) ? ASL_ETOOBIG : ASL_OK;       // a launch is fewer than 2^32 threads: 1024 per 64 column sums
}
inline bool misaligned(const void* p, int type) { return ((uintptr_t)p & (type ? 1 : 3)) != 0; }

}  // namespace asl_detail
using namespace asl_detail;

extern "C" int asl_layernorm_fwd(const asl_layernorm_params* p, const void* x, const void* gamma, const void* beta, void* y,
                                 float* mean, float* rstd, asl_stream_t stream) {
    const int rc = ln_check(p);
    if (rc != ASL_OK) return rc;
    if (p->rows == 0) return ASL_OK;
    if (!x || !y) return ASL_EINVAL;
    if (misaligned(x, p->x_type) || misaligned(y, p->y_type) || misaligned(gamma, p->w_type) || misaligned(beta, p->w_type) ||
        misaligned(mean, 0) || misaligned(rstd, 0))
        return ASL_EINVAL;
    LnArgs a = {};
    a.x = x; a.w = gamma; a.b = beta; a.y = y; a.mean = mean; a.rstd = rstd;
    a.ld_x = p->ld_x; a.ld_y = p->ld_y; a.rows = p->rows; a.d = p->d; a.w_bf16 = p->w_type; a.eps = p->eps;
    hipStream_t s = (hipStream_t)stream;
    if (p->x_type) return p->y_type ? launch_fwd<short, short>(a, s) : launch_fwd<short, float>(a, s);
    return p->y_type ? launch_fwd<float, short>(a, s) : launch_fwd<float, float>(a, s);
}

extern "C" int64_t asl_layernorm_bwd_workspace(const asl_layernorm_params* p) {
    const int rc = ln_check(p);
    if (rc != ASL_OK) return rc;
    return (int64_t)bwd_blocks(*p) * 2 * p->d * (int64_t)sizeof(float);
}

extern "C" int asl_layernorm_bwd(const asl_layernorm_params* p, const void* dy, const void* x, const void* gamma,
                                 const float* mean, const float* rstd, void* dx, void* dgamma, void* dbeta, float* workspace,
                                 asl_stream_t stream) {
    const int rc = ln_check(p);
    if (rc != ASL_OK) return rc;
    if (!dgamma && !dbeta && p->rows == 0) return ASL_OK;
    if (p->rows && (!dy || !x || !mean || !rstd || !dx || !workspace)) return ASL_EINVAL;
    if (misaligned(dy, p->y_type) || misaligned(x, p->x_type) || misaligned(gamma, p->w_type) || misaligned(dx, p->x_type) ||
        misaligned(dgamma, p->w_type) || misaligned(dbeta, p->w_type) || misaligned(mean, 0) || misaligned(rstd, 0) ||
        ((uintptr_t)workspace & 15))
        return ASL_EINVAL;
    hipStream_t s = (hipStream_t)stream;
    const int blocks = bwd_blocks(*p);
    if (blocks) {
        LnArgs a = {};
        a.x = x; a.dy = dy; a.w = gamma; a.y = dx; a.mean = (float*)mean; a.rstd = (float*)rstd; a.part = workspace;
        a.ld_x = p->ld_x; a.ld_y = p->ld_dx; a.ld_dy = p->ld_y; a.rows = p->rows; a.d = p->d; a.w_bf16 = p->w_type;
        int e;
        const bool cols = dgamma || dbeta;
        if (p->x_type) e = p->y_type ? launch_bwd<short, short>(a, blocks, cols, s) : launch_bwd<short, float>(a, blocks, cols, s);
        else e = p->y_type ? launch_bwd<float, short>(a, blocks, cols, s) : launch_bwd<float, float>(a, blocks, cols, s);
        if (e) return e;
    }
    if (dgamma || dbeta)
        hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)((2LL * p->d + 63) / 64)), dim3(1024), 0, s, workspace, blocks, p->d, dgamma, dbeta,
                           p->w_type);
    return (int)hipGetLastError();
}

// Linear + softmax cross entropy over a class vocabulary, with gradients, for gfx950.
//
//   l = x W^T + b,  lse = log sum_j exp l_j,  loss = lse - (1 - e) l_t - (e / V) sum_j l_j          (e: label smoothing)
//   G = g (softmax(l) - (1 - e) [j = t] - e / V),  dx = c G W,  dW = c G^T x,  db = c sum over rows of G
// with g the row's own weight (an upstream gradient a row, or 1) and c what all rows share (1 / rows, an upstream scalar).
// c is applied to the 32-bit sums: within G it would move every target's entry, -1 for an unsure row, to the same value
// between two bf16 numbers, and that one rounding would stand in all results.
//
// The logits are never held.  Rows are taken in pieces; the product x W^T leaves, for every row and every tile of classes, the
// tile's maximum m, the sum of exp(l - m) and, where gradients are asked for, exp(l - m) itself (fp32, or for bf16 operands
// fp16 of 2^15 times it: 11 bits of the value down to 2^-29 of the tile's largest, and 2^-40 of that below).  One pass over the per-tile numbers gives lse, the loss and
// the factors g exp(m - lse); one pass over the exponentials turns them into G in place, the target's entry from its own
// 32-bit logit (g expm1(l_t - lse), where p - 1 of a rounded p would cancel), and adds up db in 32 bits.  Then two products.
//
// Both gradient products have operands whose contraction index is not the contiguous one; see the tile kernels.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "asl_hip.h"
#include "xent_args.h"

namespace asl_detail {

template <typename T>
struct Mma;
template <>
struct Mma<short> {
    static constexpr int BK = 64, PAD = 8, KSTEP = 32;
    using Frag = bf16x8;
    static __device__ __forceinline__ Frag frag(const short* row, int k0, int q) { return *(const bf16x8*)(row + k0 + q * 8); }
    static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#else
        return c;
#endif
    }
    static __device__ __forceinline__ float exp_(float v) { return __expf(v); }
    using Exp = _Float16;                 // how exp(l - m) is held, times SCALE
    static constexpr float SCALE = kExpScale16;
};
template <>
struct Mma<float> {
    static constexpr int BK = 32, PAD = 4, KSTEP = 4;
    using Frag = float;
    static __device__ __forceinline__ Frag frag(const float* row, int k0, int q) { return row[k0 + q]; }
    static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
        return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
#else
        return c;
#endif
    }
    static __device__ __forceinline__ float exp_(float v) { return expf(v); }
    using Exp = float;
    static constexpr float SCALE = 1.f;
};

constexpr int kTile = 64;                 // of either index in the general kernel

// one thread's share of a 64 x BK operand tile: held in registers while the previous tile is multiplied
template <typename T, bool KC>
struct Stage {
    static constexpr int BK = Mma<T>::BK, LD = BK + Mma<T>::PAD, N = kTile * BK / 8 / 256;
    F8 r[N];
    __device__ __forceinline__ void load(const T* base, long long ld, int row0, int rows, int k0, int k1) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int v = u * 256 + threadIdx.x;
            const int a = KC ? v / (BK / 8) : v / (kTile / 8), c = (KC ? v % (BK / 8) : v % (kTile / 8)) * 8;
            // KC: stored row = operand index; else stored row = contraction index
            const int srow = (KC ? row0 : k0) + a, scol = (KC ? k0 : row0) + c;
            const bool ok = srow < (KC ? rows : k1);
            const int n = ok ? (KC ? k1 : rows) - scol : 0;
            r[u] = load8(base + (n > 0 ? srow * ld + scol : 0), n);
        }
    }
    __device__ __forceinline__ void store(T* lds) const {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int v = u * 256 + threadIdx.x;
            if constexpr (KC) {
                store8_full(lds + (v / (BK / 8)) * LD + (v % (BK / 8)) * 8, r[u]);
            } else {
                const int k = v / (kTile / 8), i = (v % (kTile / 8)) * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) store1(lds + (i + e) * LD + k, r[u].v[e]);
            }
        }
    }
};

// Any sizes, strides and alignment.  Four waves, 32 x 32 of the tile each.
template <typename T, bool PKC, bool QKC, bool LOGITS>
__global__ __launch_bounds__(256) void xent_gemm_kernel(const XentGemm a) {
    constexpr int BK = Mma<T>::BK, LD = BK + Mma<T>::PAD, KSTEP = Mma<T>::KSTEP;
    __shared__ __attribute__((aligned(16))) T lp[kTile * LD];
    __shared__ __attribute__((aligned(16))) T lq[kTile * LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
    const int i0 = blockIdx.x * kTile, j0 = blockIdx.y * kTile;
    const int kb = blockIdx.z * a.k_per_split, ke = kb + a.k_per_split < a.K ? kb + a.k_per_split : a.K;
    f32x4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    Stage<T, PKC> sp;
    Stage<T, QKC> sq;
    sp.load((const T*)a.p, a.ld_p, i0, a.I, kb, ke);
    sq.load((const T*)a.q, a.ld_q, j0, a.Jn, kb, ke);
    for (int k = kb; k < ke; k += BK) {
        sp.store(lp);
        sq.store(lq);
        __syncthreads();
        if (k + BK < ke) {
            sp.load((const T*)a.p, a.ld_p, i0, a.I, k + BK, ke);
            sq.load((const T*)a.q, a.ld_q, j0, a.Jn, k + BK, ke);
        }
#pragma unroll
        for (int ks = 0; ks < BK; ks += KSTEP) {
            typename Mma<T>::Frag fp[2], fqv[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                fp[u] = Mma<T>::frag(lp + (wi + u * 16 + fr) * LD, ks, fq);
                fqv[u] = Mma<T>::frag(lq + (wj + u * 16 + fr) * LD, ks, fq);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = Mma<T>::mma(fp[i], fqv[j], acc[i][j]);
        }
        __syncthreads();
    }
    // lane: i = i0 + wi + u*16 + fq*4 + e, j = j0 + wj + v*16 + fr
    if constexpr (!LOGITS) {
        const float c = a.slabs ? 1.f : *a.factor;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int j = j0 + wj + v * 16 + fr;
            if (j >= a.Jn) continue;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int i = i0 + wi + u * 16 + fq * 4;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (i + e >= a.I) continue;
                    if (a.slabs) {
                        float* o = (float*)a.out + ((long long)blockIdx.z * a.Jn + j) * a.I + i + e;
                        *o = a.add ? *o + acc[u][v][e] : acc[u][v][e];
                    } else {
                        store1((T*)a.out + j * a.ld_out + i + e, acc[u][v][e] * c);
                    }
                }
            }
        }
    } else {
        __shared__ float red[2][kTile][3];
        const int tile = blockIdx.x;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int j = j0 + wj + v * 16 + fr;
            float m = -INFINITY;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int i = i0 + wi + u * 16 + fq * 4;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float l = -INFINITY;
                    if (i + e < a.I) {
                        l = acc[u][v][e];
                        if (a.bias) l += a.bias_bf16 ? load1((const short*)a.bias + i + e) : load1((const float*)a.bias + i + e);
                    }
                    acc[u][v][e] = l;
                    m = fmaxf(m, l);
                }
            }
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            if (fq == 0) red[wave >> 1][wj + v * 16 + fr][0] = m;
            if (j < a.Jn) {
                const long long t = a.target[j];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = i0 + wi + u * 16 + fq * 4 + e;
                        if (i == t && i < a.I) a.target_logit[j] = acc[u][v][e];
                    }
            }
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int jl = wj + v * 16 + fr, j = j0 + jl;
            const float m = fmaxf(red[0][jl][0], red[1][jl][0]);
            const float ref = m == -INFINITY ? 0.f : m;      // a tile whose classes are all masked: sum nought, not NaN
            float s = 0.f, lin = 0.f;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int i = i0 + wi + u * 16 + fq * 4;
                F8 o;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float l = acc[u][v][e], x = Mma<T>::exp_(l - ref);
                    if (a.smooth && i + e < a.I) lin += l;
                    s += x;
                    o.v[e] = x;
                }
                if (a.store_e && j < a.Jn) {                 // the exponentials' rows are padded to whole tiles
                    typename Mma<T>::Exp* er = (typename Mma<T>::Exp*)a.out + j * a.ld_out + i;
#pragma unroll
                    for (int e = 0; e < 4; ++e) er[e] = (typename Mma<T>::Exp)(o.v[e] * Mma<T>::SCALE);
                }
            }
            s += __shfl_xor(s, 16, 64);
            s += __shfl_xor(s, 32, 64);
            lin += __shfl_xor(lin, 16, 64);
            lin += __shfl_xor(lin, 32, 64);
            if (fq == 0) {
                red[wave >> 1][jl][1] = s;
                red[wave >> 1][jl][2] = lin;
            }
        }
        __syncthreads();
        if (threadIdx.x < kTile) {
            const int j = j0 + threadIdx.x;
            if (j < a.Jn) {
                const long long at = (long long)j * a.tiles + tile;
                a.tile_max[at] = fmaxf(red[0][threadIdx.x][0], red[1][threadIdx.x][0]);
                a.tile_sum[at] = red[0][threadIdx.x][1] + red[1][threadIdx.x][1];
                if (a.smooth) a.tile_lin[at] = red[0][threadIdx.x][2] + red[1][threadIdx.x][2];
            }
        }
    }
}

struct XentRows {
    const long long* target;              // of this piece's rows
    const float* upstream;                // null: 1
    float* tile_max;                      // in: maxima; out (factors != 0): g exp(m - lse)
    const float* tile_sum;
    const float* tile_lin;
    const float* target_logit;
    float* target_g;                      // G at the target
    float* row_g;                         // g (label smoothing's even part)
    float* loss;
    float* lse;
    long long ignore;
    float smoothing, inv_classes, exp_unit;         // exp_unit: one over the scale the exponentials are held at
    int rows, classes, tiles, factors;
};

// one wave a row: the tiles' maxima and sums to lse, the loss, and the factors that turn exp(l - m) into G
__global__ __launch_bounds__(256) void xent_rows_kernel(const XentRows a) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= a.rows) return;
    float* mx = a.tile_max + (long long)row * a.tiles;
    const float* sm = a.tile_sum + (long long)row * a.tiles;
    float m = -INFINITY, lin = 0.f;
    for (int t = lane; t < a.tiles; t += 64) m = fmaxf(m, mx[t]);
    m = wave_max(m);
    const float ref = m == -INFINITY ? 0.f : m;
    float s = 0.f;
    for (int t = lane; t < a.tiles; t += 64) s += sm[t] * expf(mx[t] - ref);
    if (a.smoothing != 0.f) {
        const float* ln = a.tile_lin + (long long)row * a.tiles;
        for (int t = lane; t < a.tiles; t += 64) lin += ln[t];
        lin = wave_sum(lin);
    }
    s = wave_sum(s);
    const float lse = ref + logf(s);
    const long long t = a.target[row];
    const bool kept = t != a.ignore, valid = t >= 0 && t < a.classes;
    float g = 0.f;
    if (kept) g = a.upstream ? a.upstream[row] : 1.f;
    const float lt = valid ? a.target_logit[row] : NAN;       // a label outside the vocabulary makes loss and gradients NaN
    if (lane == 0) {
        float l = lse - lt;
        if (a.smoothing != 0.f) l = lse - (1.f - a.smoothing) * lt - a.smoothing * a.inv_classes * lin;
        a.loss[row] = kept ? l : 0.f;
        if (a.lse) a.lse[row] = lse;
        if (a.factors) {
            a.target_g[row] = g * (expm1f(lt - lse) + a.smoothing - a.smoothing * a.inv_classes);
            a.row_g[row] = g;
        }
    }
    if (a.factors)
        for (int t2 = lane; t2 < a.tiles; t2 += 64) mx[t2] = valid ? g * a.exp_unit * expf(mx[t2] - lse) : NAN;
}

// What concerns all of a call's rows, by one workgroup: the loss (the rows' sum, or their mean over those that carry a label;
// none of them: 0 / 0), and the factor c of the gradients.
struct XentAll {
    const long long* target;
    const float* loss_rows;               // null: the loss is not this launch's business
    float* loss;
    const float* upstream;                // null: 1
    float* factor;                        // null: not this launch's
    long long ignore;
    int n, mean;
};

__device__ __forceinline__ void over_all_rows(const XentAll& a) {
    __shared__ float lf[4];
    __shared__ int li[4];
    float v = 0.f;
    int kept = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < a.n; i += 256) {
        kept += a.target[i] != a.ignore;
        if (a.loss_rows) v += a.loss_rows[i];
    }
    v = wave_sum(v);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) kept += __shfl_xor(kept, o, 64);
    if ((threadIdx.x & 63) == 0) {
        lf[threadIdx.x >> 6] = v;
        li[threadIdx.x >> 6] = kept;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        v = lf[0] + lf[1] + lf[2] + lf[3];
        kept = li[0] + li[1] + li[2] + li[3];
        if (a.loss_rows) *a.loss = a.mean ? v / (float)kept : v;
        if (a.factor) {
            const float up = a.upstream ? *a.upstream : 1.f;
            *a.factor = !a.mean ? up : kept ? up / (float)kept : 0.f;      // no row with a label: gradients are nought
        }
    }
}

__global__ __launch_bounds__(256) void xent_loss_kernel(const XentAll a) { over_all_rows(a); }

constexpr int kGradRows = 32;             // rows a workgroup of the G pass takes; it leaves one partial row of db
constexpr int kGradCols = 256;            // and columns

struct XentG {
    void* e;                              // exp(l - m) in, G out
    long long ld;
    const float* factor;                  // [rows][tiles]
    const float* target_g;
    const float* row_g;
    const long long* target;
    float* db_part;                       // [row groups][ld], null: no bias gradient
    long long ignore;
    float smoothing, inv_classes;
    int rows, classes, tiles, tile_shift, db_add;
    short* planes;                        // not null: G goes here, as three bf16 planes
    long long plane;
    XentAll all;
};

__device__ __forceinline__ F8 load8_exp(const float* p) { return load8_full(p); }
__device__ __forceinline__ F8 load8_exp(const _Float16* p) {
    typedef _Float16 half8 __attribute__((ext_vector_type(8)));
    const half8 a = *(const half8*)p;
    F8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = (float)a[e];
    return r;
}

// fp32 as the sum of three bf16, each the rest's nearest.  Infinities and NaN lie in the first alone; a value that would round
// to infinity is cut instead.
__device__ __forceinline__ void store_planes(short* p, long long plane, const F8& v) {
    bf16x8 h, m, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float x = v.v[e];
        short a = f32_to_bf16(x);
        if (!(fabsf(bf16_to_f32(a)) < INFINITY)) a = fabsf(x) < INFINITY ? (short)(__builtin_bit_cast(unsigned, x) >> 16) : a;
        float rest = x - bf16_to_f32(a);
        if (!(fabsf(x) < INFINITY)) rest = 0.f;
        const short b = f32_to_bf16(rest);
        h[e] = a;
        m[e] = b;
        l[e] = f32_to_bf16(rest - bf16_to_f32(b));
    }
    *(bf16x8*)p = h;
    *(bf16x8*)(p + plane) = m;
    *(bf16x8*)(p + 2 * plane) = l;
}

// 256 columns x 32 rows a workgroup: half a wave on each row, four rows a lane, all of them on their way at once
template <typename T>
__global__ __launch_bounds__(256) void xent_g_kernel(const XentG a) {
    constexpr int R = kGradRows / 8;
    __shared__ __attribute__((aligned(16))) float cols[8][kGradCols];
    const int lane = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const long long col = (long long)blockIdx.x * kGradCols + lane * 8;
    const bool in = col < a.ld;
    const int r0 = blockIdx.y * kGradRows + rl;
    F8 g[R], db;
    float f[R], even[R], tg[R];
    long long t[R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int r = r0 + u * 8 < a.rows ? r0 + u * 8 : a.rows - 1;
        t[u] = a.target[r];
        if (in) {
            g[u] = load8_exp((const typename Mma<T>::Exp*)a.e + r * a.ld + col);
            f[u] = a.factor[(long long)r * a.tiles + (col >> a.tile_shift)];
        }
        even[u] = a.smoothing * a.inv_classes * a.row_g[r];
        tg[u] = a.target_g[r];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) db.v[e] = 0.f;
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int r = r0 + u * 8;
        if (!in || r >= a.rows) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = col + e < a.classes ? g[u].v[e] * f[u] - even[u] : 0.f;
            if (col + e == t[u]) v = tg[u];
            if (t[u] == a.ignore) v = 0.f;                   // whatever the row held
            g[u].v[e] = v;
            db.v[e] += v;
        }
        if (a.planes) store_planes(a.planes + r * a.ld + col, a.plane, g[u]);
        else store8_full((T*)a.e + r * a.ld + col, g[u]);
    }
    if (a.db_part) {
        store8_full(&cols[rl][lane * 8], db);
        __syncthreads();
        const long long c = (long long)blockIdx.x * kGradCols + threadIdx.x;
        if (c < a.ld) {
            float* o = a.db_part + blockIdx.y * a.ld + c;
            float v = a.db_add ? *o : 0.f;                   // on top of the earlier pieces' rows
#pragma unroll
            for (int q = 0; q < 8; ++q) v += cols[q][threadIdx.x];
            *o = v;
        }
    }
    if (blockIdx.x == 0 && blockIdx.y == 0 && (a.all.factor || a.all.loss_rows)) over_all_rows(a.all);
}

// out[r][c] = *factor times the sum over s of slab s, in the order of s; a row of `cols` values, slabs `stride` apart
template <typename U>
__global__ __launch_bounds__(256) void xent_slab_kernel(const float* in, int slabs, long long stride, long long ld_in, int rows,
                                                        int cols, U* out, long long ld_out, const float* factor) {
    const float f = *factor;
    const long long c = ((long long)blockIdx.x * 256 + threadIdx.x) * 8;
    if (c >= cols) return;
    const int n = (int)(cols - c < 8 ? cols - c : 8);
    for (int r = blockIdx.y; r < rows; r += gridDim.y) {
        F8 v = load8(in + r * ld_in + c, n);
#pragma unroll 4
        for (int s = 1; s < slabs; ++s) {
            const F8 q = load8(in + s * stride + r * ld_in + c, n);
#pragma unroll
            for (int e = 0; e < 8; ++e) v.v[e] += q.v[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v.v[e] *= f;
        store8(out + r * ld_out + c, n, v);
    }
}

// ---------------------------------------------------------------------------------------------
// Host side: how a call is cut up
// ---------------------------------------------------------------------------------------------
struct XentPlan {
    int esize, rows, pieces, tiles, tile, tile_shift, dx_tile, dw_tile, dx_splits, dw_splits, row_groups;
    long long ld_e, ld_pack;
    bool dw_slabs, pack_x, pack_w, wide, few;
    // workspace offsets, bytes
    long long shared, loss, lse, tmax, tsum, tlin, tlogit, tg, rg, e, dbp, dxs, dws, xp, wp, gp, total;
};

constexpr long long kPieceBytes = 1LL << 30;      // of exponentials held at a time
constexpr int kPieceRows = 1 << 17;               // and rows: what grids and per-tile numbers are sized by

inline int k_per_split(int k, int splits, int bk) { return ceil_div(ceil_div(k, splits), bk) * bk; }

// rows on 16 bytes, whole steps of 64 k, a tile's rows within 32-bit offsets
inline bool lies_well(const void* t, long long ld, int d) {
    return !((uintptr_t)t & 15) && !(ld & 7) && !(d & 63) && ld <= (1 << 20);
}

// Tile and slices of a product with `a` x `b` results over `k`: what its tiles take one after another on the 256 CUs, against
// what slabs of partial sums cost (written and read back at 4 TB/s, and one more launch).  Measured with one workgroup a CU:
// 1.65 us per 64 of k for 256 x 256, 0.65 for 128 x 128, 0.4 for 64 x 64 (fp32: 0.6), and about 8, 5 and 3 us around that a
// tile.  Products too narrow for the larger tiles, and fp32 ones too small to be worth taking apart into planes (128 M
// multiplications: 512 x 512 x 512), take 64 x 64.
struct TilePlan {
    int tile, splits;
};
inline TilePlan tiles_for(const asl_xent_params& p, long long a, long long b, int k, bool may_split) {
    const bool narrow = p.n < 64 || p.classes < 64 || p.d < 32 || (!p.type && (double)p.n * p.classes * p.d < (double)(1 << 27));
    TilePlan best = {kTile, 1};
    double least = 1e30;
    const int steps = ceil_div(k, 64);
    for (const int tile : {64, 128, 256}) {
        if (narrow != (tile == 64)) continue;
        const long long tiles = (long long)ceil_div(a, tile) * ceil_div(b, tile);
        const double us = tile == 256 ? 1.65 : tile == 128 ? 0.65 : p.type ? 0.4 : 0.6, around = tile == 256 ? 8.0 : tile == 128 ? 5.0 : 3.0;
        for (int s = 1; s <= (may_split ? 32 : 1) && (s == 1 || s * 2 <= steps); ++s) {
            const double t = ceil_div(tiles * s, 256) * (ceil_div(steps, s) * us * (p.type || tile == 64 ? 1 : 6) + around) +
                             (s > 1 ? 3.0 + s * (double)a * b * 8.0 / 4e6 : 0.0);
            if (t < least) {
                least = t;
                best = {tile, s};
            }
        }
    }
    return best;
}

XentPlan xent_plan(const asl_xent_params& p, const void* xp, const void* wp, bool grad, bool want_dx, bool want_dw, bool want_db) {
    XentPlan q = {};
    q.esize = p.type ? 2 : 4;
    q.few = p.n && p.n <= kFewRows && p.classes <= kFewClasses;
    q.tile = q.few ? kFewTile : tiles_for(p, p.n, p.classes, p.d, false).tile;
    q.tile_shift = q.tile == 256 ? 8 : q.tile == 128 ? 7 : 6;       // (few rows: not used)
    // the tile kernels read 16 bytes at a time and whole steps of 64 k: operands that do not allow it are laid out anew
    q.ld_pack = (p.d + 63LL) / 64 * 64;
    q.wide = q.tile > kTile && !p.type;
    q.pack_x = q.tile > kTile && (q.wide || !lies_well(xp, p.ld_x, p.d));
    q.pack_w = q.tile > kTile && (q.wide || !lies_well(wp, p.ld_w, p.d));
    const int planes = q.wide ? 3 : 1;
    q.tiles = ceil_div(p.classes, q.tile);
    q.ld_e = (long long)q.tiles * q.tile;
    long long rows = p.n < kPieceRows ? p.n : kPieceRows;
    if (grad) {
        const long long most = kPieceBytes / (q.ld_e * (q.wide ? 10 : q.esize)) / 256 * 256;
        if (rows > most) rows = most < 256 ? 256 : most;
    }
    q.rows = (int)rows;
    q.pieces = p.n ? ceil_div(p.n, rows) : 0;
    q.row_groups = ceil_div(rows, kGradRows);
    const int bk = p.type || q.wide ? Mma<short>::BK : Mma<float>::BK;
    q.dx_splits = q.dw_splits = 1;
    q.dx_tile = q.dw_tile = kTile;
    if (grad && p.n) {
        const TilePlan x = tiles_for(p, rows, p.d, p.classes, true), w = tiles_for(p, p.classes, p.d, (int)rows, true);
        q.dx_tile = x.tile; q.dx_splits = x.splits;
        q.dw_tile = w.tile; q.dw_splits = w.splits;
    }
    q.dx_splits = ceil_div(p.classes, k_per_split(p.classes, q.dx_splits, bk));
    q.dw_splits = rows ? ceil_div(rows, k_per_split((int)rows, q.dw_splits, bk)) : 1;
    q.dw_slabs = q.dw_splits > 1 || q.pieces > 1;
    if (q.few) {                          // exponentials and G in fp32 whatever the operands
        q.esize = 4;
        q.dx_splits = xent_few_slabs(p.classes) + 1;
        q.dw_slabs = false;
        want_db = false;
    }
    long long at = 0;
    const auto take = [&](long long bytes) {
        const long long r = at;
        at += (bytes + 255) / 256 * 256;
        return r;
    };
    q.shared = take(4);
    q.loss = take(4LL * p.n);
    q.lse = take(4LL * p.n);
    q.tmax = take(4LL * rows * q.tiles);
    q.tsum = take(4LL * rows * q.tiles);
    q.tlin = take(p.label_smoothing != 0.f ? 4LL * rows * q.tiles : 0);
    q.tlogit = take(4LL * rows);
    if (grad) {
        q.tg = take(4LL * rows);
        q.rg = take(4LL * rows);
        q.e = take(q.esize * rows * q.ld_e);
        q.dbp = take(want_db ? 4LL * q.row_groups * q.ld_e : 0);
        q.dxs = take(want_dx && q.dx_splits > 1 ? 4LL * q.dx_splits * rows * p.d : 0);
        q.dws = take(want_dw && q.dw_slabs ? 4LL * q.dw_splits * p.classes * p.d : 0);
    }
    q.xp = take(q.pack_x ? 2LL * planes * rows * q.ld_pack : 0);
    q.wp = take(q.pack_w ? 2LL * planes * p.classes * q.ld_pack : 0);
    q.gp = take(q.wide && grad ? 6LL * rows * q.ld_e : 0);
    q.total = at;
    return q;
}

int xent_check(const asl_xent_params* p) {
    if (!p || p->n < 0 || p->classes <= 0 || p->d <= 0) return ASL_EINVAL;
    if (p->type < 0 || p->type > 1 || p->bias_type < 0 || p->bias_type > 1) return ASL_EINVAL;
    if (p->reduction < ASL_REDUCE_NONE || p->reduction > ASL_REDUCE_MEAN) return ASL_EINVAL;
    if (p->ld_x < p->d || p->ld_w < p->d) return ASL_EINVAL;
    if (!(p->label_smoothing >= 0.f && p->label_smoothing <= 1.f)) return ASL_EINVAL;
    // grids take one of their 65535 rows of workgroups per 64 classes
    if (p->n > (1 << 28) || p->classes > (1 << 21) || p->d > (1 << 20)) return ASL_ETOOBIG;
    return ASL_OK;
}

// Rows of d elements at any alignment to rows of `per_row` 16-byte vectors of bf16, noughts behind d; fp32 to three planes of
// them.
template <typename T>
__global__ __launch_bounds__(256) void xent_pack_kernel(const T* src, long long ld, int rows, int d, short* dst, int per_row) {
    const long long vectors = (long long)rows * per_row;
    for (long long v = blockIdx.x * 256LL + threadIdx.x; v < vectors; v += gridDim.x * 256LL) {
        const long long r = v / per_row;
        const int c = (int)(v - r * per_row) * 8;
        const auto raw = load8_raw(src + r * ld + (c < d ? c : 0), d - c);
        if constexpr (std::is_same<T, short>::value) *(bf16x8*)(dst + v * 8) = raw;
        else store_planes(dst + v * 8, vectors * 8, widen(raw));
    }
}

int xent_run_few(const asl_xent_params& p, const XentPlan& q, bool grad, const void* x, const void* w, const void* bias,
                 const long long* target, const float* upstream, float* loss, float* lse, void* dx, void* dw, void* db, char* ws,
                 hipStream_t s) {
    XentFew a = {};
    a.x = x; a.w = w; a.bias = bias; a.target = target; a.upstream = upstream; a.loss = loss; a.lse = lse; a.dx = dx; a.dw = dw; a.db = db;
    a.e = grad ? (float*)(ws + q.e) : nullptr; a.tile_max = (float*)(ws + q.tmax); a.tile_sum = (float*)(ws + q.tsum);
    a.tile_lin = (float*)(ws + q.tlin); a.target_logit = (float*)(ws + q.tlogit); a.factor = grad ? (float*)(ws + q.shared) : nullptr;
    a.slabs = (float*)(ws + q.dxs); a.ld_x = p.ld_x; a.ld_w = p.ld_w; a.ld_e = q.ld_e; a.ignore = p.ignore_index;
    a.smoothing = p.label_smoothing; a.inv_classes = 1.f / (float)p.classes; a.n = p.n; a.classes = p.classes; a.d = p.d;
    a.tiles = q.tiles; a.bias_bf16 = p.bias_type; a.none = p.reduction == ASL_REDUCE_NONE; a.mean = p.reduction == ASL_REDUCE_MEAN;
    return xent_few(a, p.type, s);
}

template <typename T>
int xent_run(const asl_xent_params& p, const XentPlan& q, bool grad, const void* x, const void* w, const void* bias,
             const long long* target, const float* upstream, float* loss, float* lse, void* dx, void* dw, void* db, char* ws,
             hipStream_t s) {
    const int bk = q.wide ? Mma<short>::BK : Mma<T>::BK;
    const bool none = p.reduction == ASL_REDUCE_NONE, mean = p.reduction == ASL_REDUCE_MEAN;
    float* loss_rows = none ? loss : (float*)(ws + q.loss);
    float* shared = (float*)(ws + q.shared);
    XentAll all = {};
    all.target = target; all.loss = loss; all.upstream = none ? nullptr : upstream; all.ignore = p.ignore_index; all.n = p.n;
    all.mean = mean;
    const void* wk = w;                   // what the products read: the caller's tensors, or their copies
    long long ld_w = p.ld_w, ld_x = p.ld_x;
    const auto pack = [&](const void* src, long long ld, int rows, void* dst) {
        const long long vectors = rows * (q.ld_pack / 8);
        hipLaunchKernelGGL((xent_pack_kernel<T>), dim3(ceil_div(vectors, 512) < 8192 ? ceil_div(vectors, 512) : 8192), dim3(256), 0, s,
                           (const T*)src, ld, rows, p.d, (short*)dst, (int)(q.ld_pack / 8));
    };
    if (q.pieces && q.pack_w) {
        pack(w, p.ld_w, p.classes, ws + q.wp);
        wk = ws + q.wp;
        ld_w = q.ld_pack;
    }
    if (q.pack_x) ld_x = q.ld_pack;
    for (int piece = 0; piece < q.pieces; ++piece) {
        const int r0 = piece * q.rows, rows = p.n - r0 < q.rows ? p.n - r0 : q.rows;
        const T* xr = (const T*)x + r0 * p.ld_x;
        if (q.pack_x) {
            pack(xr, p.ld_x, rows, ws + q.xp);
            xr = (const T*)(ws + q.xp);
        }
        XentGemm g = {};
        g.p = wk; g.ld_p = ld_w; g.q = xr; g.ld_q = ld_x; g.I = p.classes; g.Jn = rows; g.K = p.d; g.k_per_split = p.d;
        g.out = ws + q.e; g.ld_out = q.ld_e; g.bias = bias; g.bias_bf16 = p.bias_type; g.smooth = p.label_smoothing != 0.f;
        g.store_e = grad; g.target = target + r0; g.tile_max = (float*)(ws + q.tmax); g.tile_sum = (float*)(ws + q.tsum);
        g.tile_lin = (float*)(ws + q.tlin); g.target_logit = (float*)(ws + q.tlogit); g.tiles = q.tiles;
        g.splits = 1;
        if (q.wide) g.plane_p = p.classes * ld_w, g.plane_q = rows * ld_x;
        if (q.tile > kTile) {
            const int rc = xent_tiles_logits(g, q.tile, s);
            if (rc) return rc;
        } else {
            hipLaunchKernelGGL((xent_gemm_kernel<T, true, true, true>), dim3(q.tiles, ceil_div(rows, kTile)), dim3(256), 0, s, g);
        }
        XentRows r = {};
        r.target = target + r0; r.upstream = upstream && none ? upstream + r0 : nullptr;
        r.tile_max = g.tile_max; r.tile_sum = g.tile_sum; r.tile_lin = g.tile_lin; r.target_logit = g.target_logit;
        r.target_g = (float*)(ws + q.tg); r.row_g = (float*)(ws + q.rg);
        r.loss = loss_rows + r0; r.lse = lse ? lse + r0 : nullptr;
        r.ignore = p.ignore_index; r.smoothing = p.label_smoothing; r.inv_classes = 1.f / (float)p.classes; r.exp_unit = 1.f / Mma<T>::SCALE;
        r.rows = rows; r.classes = p.classes; r.tiles = q.tiles; r.factors = grad;
        hipLaunchKernelGGL(xent_rows_kernel, dim3(ceil_div(rows, 4)), dim3(256), 0, s, r);
        if (!grad) continue;
        const bool last = piece == q.pieces - 1;
        XentG c = {};
        c.e = ws + q.e; c.ld = q.ld_e; c.planes = q.wide ? (short*)(ws + q.gp) : nullptr; c.plane = rows * q.ld_e; c.factor = g.tile_max; c.target_g = r.target_g; c.row_g = r.row_g; c.target = target + r0;
        c.all = all; c.all.loss_rows = !none && last ? loss_rows : nullptr; c.all.factor = piece == 0 ? shared : nullptr;
        c.db_part = db ? (float*)(ws + q.dbp) : nullptr; c.db_add = piece > 0;
        c.ignore = p.ignore_index; c.smoothing = p.label_smoothing; c.inv_classes = r.inv_classes; c.rows = rows;
        c.classes = p.classes; c.tiles = q.tiles; c.tile_shift = q.tile_shift;
        const int groups = ceil_div(rows, kGradRows);
        hipLaunchKernelGGL((xent_g_kernel<T>), dim3(ceil_div(q.ld_e, kGradCols), groups), dim3(256), 0, s, c);
        if (dx) {                          // dx[row][k] = sum over classes G[row][v] W[v][k]
            XentGemm h = {};
            h.p = wk; h.ld_p = ld_w; h.q = ws + (q.wide ? q.gp : q.e); h.ld_q = q.ld_e; h.I = p.d; h.Jn = rows; h.K = p.classes;
            if (q.wide) h.plane_p = p.classes * ld_w, h.plane_q = rows * q.ld_e;
            h.k_per_split = k_per_split(p.classes, q.dx_splits, bk);
            h.slabs = q.dx_splits > 1; h.factor = shared;
            T* dxr = (T*)dx + (long long)r0 * p.d;
            h.out = h.slabs ? (void*)(ws + q.dxs) : (void*)dxr; h.ld_out = p.d;
            h.splits = q.dx_splits;
            if (q.dx_tile > kTile) {
                const int rc = xent_tiles_dx(h, q.dx_tile, s);
                if (rc) return rc;
            } else {
                hipLaunchKernelGGL((xent_gemm_kernel<T, false, true, false>),
                                   dim3(ceil_div(p.d, kTile), ceil_div(rows, kTile), q.dx_splits), dim3(256), 0, s, h);
            }
            if (h.slabs)
                hipLaunchKernelGGL((xent_slab_kernel<T>), dim3(ceil_div(p.d, 2048), rows < 4096 ? rows : 4096), dim3(256), 0, s,
                                   (const float*)(ws + q.dxs), q.dx_splits, (long long)rows * p.d, (long long)p.d, rows, p.d, dxr,
                                   (long long)p.d, shared);
        }
        if (dw) {                          // dW[v][k] = sum over rows G[row][v] x[row][k]
            XentGemm h = {};
            h.p = xr; h.ld_p = ld_x; h.q = ws + (q.wide ? q.gp : q.e); h.ld_q = q.ld_e; h.I = p.d; h.Jn = p.classes; h.K = rows;
            if (q.wide) h.plane_p = rows * ld_x, h.plane_q = rows * q.ld_e;
            h.k_per_split = k_per_split(q.rows, q.dw_splits, bk);
            h.slabs = q.dw_slabs; h.factor = shared; h.add = piece > 0;
            h.out = h.slabs ? (void*)(ws + q.dws) : dw; h.ld_out = p.d;
            h.splits = q.dw_splits;
            if (q.dw_tile > kTile) {
                const int rc = xent_tiles_dw(h, q.dw_tile, s);
                if (rc) return rc;
            } else {
                hipLaunchKernelGGL((xent_gemm_kernel<T, false, false, false>),
                                   dim3(ceil_div(p.d, kTile), ceil_div(p.classes, kTile), q.dw_splits), dim3(256), 0, s, h);
            }
            if (h.slabs && last)
                hipLaunchKernelGGL((xent_slab_kernel<T>), dim3(ceil_div(p.d, 2048), p.classes < 4096 ? p.classes : 4096), dim3(256), 0, s,
                                   (const float*)(ws + q.dws), q.dw_splits, (long long)p.classes * p.d, (long long)p.d, p.classes,
                                   p.d, (T*)dw, (long long)p.d, shared);
        }
        if (db && last) column_sums((const float*)(ws + q.dbp), q.row_groups, q.ld_e, p.classes, p.classes, db, nullptr, p.bias_type, shared, s);
    }
    if (!none && (!grad || !q.pieces)) {
        all.loss_rows = loss_rows;
        hipLaunchKernelGGL(xent_loss_kernel, dim3(1), dim3(256), 0, s, all);
    }
    return (int)hipGetLastError();
}

// no rows: the weight's and bias's gradients are nought
__global__ __launch_bounds__(256) void xent_zero_kernel(char* p, long long bytes) {
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < bytes; i += gridDim.x * 256LL) p[i] = 0;
}

inline bool off(const void* p, int type) { return ((uintptr_t)p & (type ? 1 : 3)) != 0; }

}  // namespace asl_detail
using namespace asl_detail;

extern "C" int64_t asl_linear_xent_workspace(const asl_xent_params* p, const void* x, const void* w, int grad) {
    const int rc = xent_check(p);
    if (rc != ASL_OK) return rc;
    return xent_plan(*p, x, w, grad != 0, true, true, true).total;
}

extern "C" int asl_linear_xent_fwd(const asl_xent_params* p, const void* x, const void* w, const void* bias,
                                   const int64_t* target, float* loss, float* lse, void* workspace, asl_stream_t stream) {
    const int rc = xent_check(p);
    if (rc != ASL_OK) return rc;
    if (!w || !workspace || ((uintptr_t)workspace & 255) || !loss || ((uintptr_t)loss & 3) || ((uintptr_t)lse & 3)) return ASL_EINVAL;
    if (p->n && (!x || !target)) return ASL_EINVAL;
    if (off(x, p->type) || off(w, p->type) || off(bias, p->bias_type) || ((uintptr_t)target & 7)) return ASL_EINVAL;
    const XentPlan q = xent_plan(*p, x, w, false, false, false, false);
    const long long* t = (const long long*)target;
    if (q.few) return xent_run_few(*p, q, false, x, w, bias, t, nullptr, loss, lse, nullptr, nullptr, nullptr, (char*)workspace, (hipStream_t)stream);
    if (p->type) return xent_run<short>(*p, q, false, x, w, bias, t, nullptr, loss, lse, nullptr, nullptr, nullptr, (char*)workspace, (hipStream_t)stream);
    return xent_run<float>(*p, q, false, x, w, bias, t, nullptr, loss, lse, nullptr, nullptr, nullptr, (char*)workspace, (hipStream_t)stream);
}

extern "C" int asl_linear_xent_grad(const asl_xent_params* p, const void* x, const void* w, const void* bias,
                                    const int64_t* target, const float* upstream, float* loss, float* lse, void* dx, void* dw,
                                    void* dbias, void* workspace, asl_stream_t stream) {
    const int rc = xent_check(p);
    if (rc != ASL_OK) return rc;
    if (!w || !workspace || ((uintptr_t)workspace & 255) || ((uintptr_t)loss & 3) || ((uintptr_t)lse & 3) || ((uintptr_t)upstream & 3))
        return ASL_EINVAL;
    if (!loss) return ASL_EINVAL;
    if (p->n && (!x || !target)) return ASL_EINVAL;
    if (off(x, p->type) || off(w, p->type) || off(bias, p->bias_type) || off(dx, p->type) || off(dw, p->type) ||
        off(dbias, p->bias_type) || ((uintptr_t)target & 7))
        return ASL_EINVAL;
    hipStream_t s = (hipStream_t)stream;
    if (p->n == 0) {
        const auto zero = [&](void* out, long long bytes) {
            if (out) hipLaunchKernelGGL(xent_zero_kernel, dim3(ceil_div(bytes, 4096) < 4096 ? ceil_div(bytes, 4096) : 4096), dim3(256), 0, s, (char*)out, bytes);
        };
        zero(dw, (long long)p->classes * p->d * (p->type ? 2 : 4));
        zero(dbias, (long long)p->classes * (p->bias_type ? 2 : 4));
    }
    const XentPlan q = xent_plan(*p, x, w, true, dx != nullptr, dw != nullptr, dbias != nullptr);
    const long long* t = (const long long*)target;
    if (q.few) return xent_run_few(*p, q, true, x, w, bias, t, upstream, loss, lse, dx, dw, dbias, (char*)workspace, s);
    if (p->type) return xent_run<short>(*p, q, true, x, w, bias, t, upstream, loss, lse, dx, dw, dbias, (char*)workspace, s);
    return xent_run<float>(*p, q, true, x, w, bias, t, upstream, loss, lse, dx, dw, dbias, (char*)workspace, s);
}

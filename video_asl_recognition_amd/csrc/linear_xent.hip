// Linear + softmax cross entropy over a class vocabulary, with gradients, for gfx950.
//
//   l = x W^T + b,  lse = log sum_j exp l_j,  loss = lse - (1 - e) l_t - (e / V) sum_j l_j          (e: label smoothing)
//   G = g (softmax(l) - (1 - e) [j = t] - e / V),  dx = c G W,  dW = c G^T x,  db = c sum over rows of G
// with g the row's own weight (an upstream gradient a row, or 1) and c what all rows share (1 / rows, an upstream scalar).
// c is applied to the 32-bit sums: within G it would move every target's entry, -1 for an unsure row, to the same value
// between two bf16 numbers, and that one rounding would stand in all results.
//
// The logits themselves are not held.  Rows are taken in pieces; the product x W^T leaves, for every row and every tile of classes, the
// tile's maximum m, the sum of exp(l - m) and, where gradients are asked for, exp(l - m) itself (fp32, or for bf16 operands
// fp16 of 2^15 times it: 11 bits of the value down to 2^-29 of the tile's largest, and 2^-40 of that below).  One pass over the
// per-tile numbers gives lse, the loss and the factors g exp(m - lse); one pass over the exponentials turns them into G in
// place, the target's entry from its own 32-bit logit (g expm1((l_t - max) - log sum exp(l - max)), where p - 1 of a rounded p,
// or l_t - lse of a rounded lse, would cancel), and adds up db in 32 bits.  Then two products, whose sums are finished (slabs, db, the loss) by one more launch where there is need.
//
// What bounds it is the products where they are large (8192 x 32768 x 2048 bf16: 2.83 to 2.92 ms with gradients from card to card,
// 3.3 PFLOP at 1.13 to 1.17 PFLOP/s: the three products 2.63 to 2.75 ms, G 0.19 ms at 5.5 TB/s), the matrix pipe's rate for six
// bf16 products in the place of one in fp32 (2048 x 8192 x 1024: 588 to 611 us with gradients, 169 to 175 TFLOP/s; on fp32 MFMAs
// 1151), and the chain of launches where they are small (2048 x 2000 x 512 bf16: 47 us, of which the products 28).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "asl_hip.h"
#include "xent_args.h"

namespace asl_detail {

// how exp(l - m) is held, times SCALE
template <typename T>
struct Held;
template <>
struct Held<short> {
    using Exp = _Float16;
    static constexpr float SCALE = kExpScale16;
};
template <>
struct Held<float> {
    using Exp = float;
    static constexpr float SCALE = 1.f;
};

// fp32 products that are not worth being taken apart into bf16 planes: 64 x 64 tiles on the fp32 MFMA (16 x 16 x 4), any sizes,
// strides and alignment.  The matrix pipe's fp32 rate (133 TF/s as a library product reaches it) bounds large ones, a step's
// round trip to memory the small ones that come here: 300 x 300 x 300 with gradients 33 us, 512 x 2000 x 512 70 us.  Steps of
// 32 k and of 64 take the same time (500 x 300 x 200: 13.6 and 14.1 us for the logits).
constexpr int kTile = 64, kStep = 32;     // of either index, and of k

// one thread's share of a 64 x 32 operand tile: held in registers while the previous tile is multiplied
template <bool KC>
struct Stage {
    static constexpr int BK = kStep, LD = BK + 4, N = kTile * BK / 8 / 256;
    F8 r[N];
    __device__ __forceinline__ void load(const float* base, long long ld, int row0, int rows, int k0, int k1) {
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
    __device__ __forceinline__ void store(float* lds) const {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int v = u * 256 + threadIdx.x;
            if constexpr (KC) {
                store8_full(lds + (v / (BK / 8)) * LD + (v % (BK / 8)) * 8, r[u]);
            } else {
                const int k = v / (kTile / 8), i = (v % (kTile / 8)) * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) lds[(i + e) * LD + k] = r[u].v[e];
            }
        }
    }
};

// Four waves, 32 x 32 of the tile each.  Workgroup `id` of ti * tj * splits.
template <bool PKC, bool QKC, bool LOGITS>
__device__ __forceinline__ void gemm_body(const XentGemm& a, int id, int ti, int tj) {
    constexpr int BK = kStep, LD = BK + 4;
    __shared__ __attribute__((aligned(16))) float lp[kTile * LD];
    __shared__ __attribute__((aligned(16))) float lq[kTile * LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
    const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
    const int bi = id % ti, bj = id / ti % tj, slice = id / (ti * tj), i0 = bi * kTile, j0 = bj * kTile;
    const int kb = slice * a.k_per_split, ke = kb + a.k_per_split < a.K ? kb + a.k_per_split : a.K;
    f32x4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    Stage<PKC> sp;
    Stage<QKC> sq;
    sp.load((const float*)a.p, a.ld_p, i0, a.I, kb, ke);
    sq.load((const float*)a.q, a.ld_q, j0, a.Jn, kb, ke);
    for (int k = kb; k < ke; k += BK) {
        sp.store(lp);
        sq.store(lq);
        __syncthreads();
        if (k + BK < ke) {
            sp.load((const float*)a.p, a.ld_p, i0, a.I, k + BK, ke);
            sq.load((const float*)a.q, a.ld_q, j0, a.Jn, k + BK, ke);
        }
#pragma unroll
        for (int ks = 0; ks < BK; ks += 4) {
            float fp[2], fqv[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                fp[u] = lp[(wi + u * 16 + fr) * LD + ks + fq];
                fqv[u] = lq[(wj + u * 16 + fr) * LD + ks + fq];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = mma4(fp[i], fqv[j], acc[i][j]);
        }
        __syncthreads();
    }
    // lane: i = i0 + wi + u*16 + fq*4 + e, j = j0 + wj + v*16 + fr
    if constexpr (!LOGITS) {
        const float c = a.slabs ? 1.f : *a.factor;
        const long long ld = (long long)ti * kTile;        // of a slab
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
                        float* o = (float*)a.out + ((long long)slice * a.Jn + j) * ld + i + e;
                        *o = a.add ? *o + acc[u][v][e] : acc[u][v][e];
                    } else {
                        ((float*)a.out)[j * a.ld_out + i + e] = acc[u][v][e] * c;
                    }
                }
            }
        }
    } else {
        __shared__ float red[2][kTile][3];
        const int tile = bi;
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
                f32x4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float l = acc[u][v][e];
                    x[e] = expf(l - ref);
                    if (a.smooth && i + e < a.I) lin += l;
                    s += x[e];
                }
                // the exponentials' rows are padded to whole tiles
                if (a.store_e && j < a.Jn) *(f32x4*)((float*)a.out + j * a.ld_out + i) = x;
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

__global__ __launch_bounds__(256) void xent_gemm_logits_kernel(const XentGemm a, int ti, int tj) {
    gemm_body<true, true, true>(a, blockIdx.x, ti, tj);
}

// dx and dW in one launch, dx's workgroups first
__global__ __launch_bounds__(256) void xent_gemm_pair_kernel(const XentGemm dx, const XentGemm dw, int dx_ti, int dx_tj, int dw_ti, int dw_tj,
                                                             int dx_blocks) {
    if ((int)blockIdx.x < dx_blocks) gemm_body<false, true, false>(dx, blockIdx.x, dx_ti, dx_tj);
    else gemm_body<false, false, false>(dw, blockIdx.x - dx_blocks, dw_ti, dw_tj);
}

struct XentRows {
    XentStats st;
    float* factor;                        // with gradients: [rows][tiles] g exp(m - lse); may be the maxima themselves
    float* target_g;                      // G at the target
    float* row_g;                         // g (label smoothing's even part)
    float* loss;                          // each null: not wanted
    float* lse;
    float* loss_part;                     // a workgroup's rows' losses and
    int* kept_part;                       // those that carry a label
    float exp_unit;                       // one over the scale the exponentials are held at
};

// the losses of a workgroup's N rows, one a thread `at` of them, to one partial sum
template <int N>
__device__ __forceinline__ void leave_part(const XentRows& a, long long part, float (&loss)[N], int (&kept)[N]) {
    __syncthreads();
    if (threadIdx.x == 0 && a.loss_part) {
        float v = 0.f;
        int k = 0;
#pragma unroll
        for (int r = 0; r < N; ++r) v += loss[r], k += kept[r];
        a.loss_part[part] = v;
        a.kept_part[part] = k;
    }
}

// A wave a row, or a quarter of one: statistics, loss, and the factors that turn exp(l - m) into G (8192 rows of 256 tiles
// 12 us, 4.3 TB/s from and to the caches).
template <int LANES>
__global__ __launch_bounds__(256) void xent_rows_kernel(const XentRows a) {
    constexpr int N = 256 / LANES;
    __shared__ float loss[N];
    __shared__ int kept[N];
    const int at = threadIdx.x / LANES, row = blockIdx.x * N + at, lane = threadIdx.x % LANES;
    if (row < a.st.rows) {
        const XentRow r = row_stats<LANES>(a.st, row, lane);
        if (lane == 0) {
            loss[at] = r.loss;
            kept[at] = a.st.target[row] != a.st.ignore;
            if (a.loss) a.loss[row] = r.loss;
            if (a.lse) a.lse[row] = r.lse();
            if (a.factor) {
                a.target_g[row] = r.target_g;
                a.row_g[row] = r.g;
            }
        }
        if (a.factor)
            for (int t = lane; t < a.st.tiles; t += LANES) {
                const long long k = (long long)row * a.st.tiles + t;
                a.factor[k] = r.valid ? r.g * a.exp_unit * r.exp_of(a.st.tile_max[k]) : NAN;
            }
    } else if (lane == 0) {
        loss[at] = 0.f;
        kept[at] = 0;
    }
    leave_part(a, blockIdx.x, loss, kept);
}

// What concerns all of a call's rows, each by one workgroup: the loss from the partial sums, and the factor c of the gradients
// from the targets, or from counts of them where there are many.
struct XentLoss {
    const float* loss_part;               // null: not this launch's business
    const int* kept_part;
    float* loss;
    int parts, mean;
};
struct XentFactor {
    const long long* target;
    const int* counts;                    // of kCountRows rows each; null: none were taken
    const float* upstream;                // null: 1
    float* factor;                        // null: not this launch's business
    long long ignore;
    int n, mean;
};
constexpr int kCountRows = 8192;          // rows up to which one workgroup counts them on its way (65536 rows of 100 classes and 512
                                          // features with gradients: 102 us with a launch that counts them, 172 without)

__device__ __forceinline__ float block_sum(float v, float* lds) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}
__device__ __forceinline__ int block_sum(int v, int* lds) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}
__device__ __forceinline__ int count_kept(const long long* target, int n, long long ignore, int* lds) {
    int kept = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += 256) kept += target[i] != ignore;
    return block_sum(kept, lds);
}

// the rows' sum, or their mean over those that carry a label (none of them: 0 / 0)
__device__ __forceinline__ void finish_loss(const XentLoss& a) {
    __shared__ float lf[4];
    __shared__ int li[4];
    float v = 0.f;
    int kept = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < a.parts; i += 256) v += a.loss_part[i], kept += a.kept_part[i];
    v = block_sum(v, lf);
    kept = block_sum(kept, li);
    if (threadIdx.x == 0) *a.loss = a.mean ? v / (float)kept : v;
}
__device__ __forceinline__ void set_factor(const XentFactor& a) {
    __shared__ int li[4];
    int kept = 0;
    if (a.mean && a.counts) {
#pragma unroll 8
        for (int i = threadIdx.x; i < (a.n + kCountRows - 1) / kCountRows; i += 256) kept += a.counts[i];
        kept = block_sum(kept, li);
    } else if (a.mean) {
        kept = count_kept(a.target, a.n, a.ignore, li);
    }
    const float up = a.upstream ? *a.upstream : 1.f;
    if (threadIdx.x == 0) *a.factor = !a.mean ? up : kept ? up / (float)kept : 0.f;      // no row with a label: gradients are nought
}

__global__ __launch_bounds__(256) void xent_loss_kernel(const XentLoss a) { finish_loss(a); }

__global__ __launch_bounds__(256) void xent_count_kernel(const long long* target, int n, long long ignore, int* counts) {
    __shared__ int li[4];
    const int first = blockIdx.x * kCountRows, left = n - first < kCountRows ? n - first : kCountRows;
    const int kept = count_kept(target + first, left, ignore, li);
    if (threadIdx.x == 0) counts[blockIdx.x] = kept;
}

constexpr int kGradRows = 32;             // rows a workgroup of the G pass takes; it leaves one partial row of db
constexpr int kGradCols = 256;            // and columns

// tiles a row up to which the G pass takes the statistics for itself (1024 x 2000 x 512 bf16, 32 of them, with gradients 36.9 us and
// 38.8; 1024 x 4000, 63, 48.2 and 46.1)
constexpr int kOwnStats = 32;

struct XentG {
    XentRows rows;                        // `factor`, `target_g`, `row_g`: taken from there (or, with own statistics, not used)
    void* e;                              // exp(l - m) in, G out
    long long ld;
    float* db_part;                       // [row groups][ld], null: no bias gradient
    int tile_shift, db_add;
    short* planes;                        // not null: G goes here, as three bf16 planes
    long long plane;
    XentLoss loss;
    XentFactor factor;
};

__device__ __forceinline__ F8 load8_exp(const float* p) { return load8_full(p); }
__device__ __forceinline__ F8 load8_exp(const _Float16* p) {
    const half8 a = *(const half8*)p;
    F8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = (float)a[e];
    return r;
}

// fp32 as the sum of three bf16, each the rest's nearest.  Infinities and NaN lie in the last alone, which meets the other operand's
// first and nothing else: in the first they would meet its noughts and differences of either sign, and an infinite product
// would be NaN.  A value that would round to infinity is cut instead.
__device__ __forceinline__ void store_planes(short* p, long long plane, const F8& v) {
    bf16x8 h, m, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float x = v.v[e];
        const bool finite = fabsf(x) < INFINITY;
        short a = f32_to_bf16(x);
        if (!(fabsf(bf16_to_f32(a)) < INFINITY)) a = finite ? (short)(__builtin_bit_cast(unsigned, x) >> 16) : 0;
        const float rest = finite ? x - bf16_to_f32(a) : 0.f;
        const short b = f32_to_bf16(rest);
        h[e] = a;
        m[e] = b;
        l[e] = f32_to_bf16(finite ? rest - bf16_to_f32(b) : x);
    }
    *(bf16x8*)p = h;
    *(bf16x8*)(p + plane) = m;
    *(bf16x8*)(p + 2 * plane) = l;
}

// G in place of the exponentials, or beside them as planes: bound by memory (8192 x 32768 bf16 187 us, 5.7 TB/s in and out).
// 256 columns x 32 rows a workgroup: half a wave on each row, four rows a lane, all of them on their way at once.  OWN: the
// rows' statistics are taken here, by every column's workgroup anew, instead of in a launch ahead.
template <typename T, bool OWN>
__global__ __launch_bounds__(256) void xent_g_kernel(const XentG a) {
    constexpr int R = kGradRows / 8, TPB = kGradCols / kFewTile;     // (at least 32 classes a maximum)
    __shared__ __attribute__((aligned(16))) float cols[8][kGradCols];
    __shared__ float own_f[OWN ? kGradRows : 1][TPB], own_tg[OWN ? kGradRows : 1], own_g[OWN ? kGradRows : 1], own_loss[kGradRows];
    __shared__ int own_kept[kGradRows];
    const XentStats& st = a.rows.st;
    const int lane = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const long long col = (long long)blockIdx.x * kGradCols + lane * 8;
    const bool in = col < a.ld;
    const int b0 = blockIdx.y * kGradRows, r0 = b0 + rl;
    if (b0 >= st.rows) {                                     // the workgroups behind the last row: what concerns all of them
        if (blockIdx.x == 0 && a.factor.factor) set_factor(a.factor);
        if (blockIdx.x == 0 && a.loss.loss_part) finish_loss(a.loss);
        return;
    }
    F8 g[R], db;
    float f[R], even[R], tg[R];
    long long t[R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int r = r0 + u * 8 < st.rows ? r0 + u * 8 : st.rows - 1;
        t[u] = st.target[r];
        if (in) {
            g[u] = load8_exp((const typename Held<T>::Exp*)a.e + r * a.ld + col);
            // (columns of a last, half empty 256 x 256 tile lie behind the last block of maxima)
            const int tile = (int)(col >> a.tile_shift);
            if (!OWN) f[u] = tile < st.tiles ? a.rows.factor[(long long)r * st.tiles + tile] : 0.f;
        }
        if (!OWN) {
            even[u] = st.smoothing * st.inv_classes * a.rows.row_g[r];
            tg[u] = a.rows.target_g[r];
        }
    }
    if constexpr (OWN) {
        const int l8 = threadIdx.x & 7, k = threadIdx.x >> 3, blocks = kGradCols >> a.tile_shift;
        static_assert(kGradRows * 8 == 256, "eight lanes a row, all rows at once");
        if (b0 + k >= st.rows) {
            if (l8 == 0) own_loss[k] = 0.f, own_kept[k] = 0;
        } else {
            const XentRow q = row_stats<8>(st, b0 + k, l8);
            if (l8 == 0) {
                own_tg[k] = q.target_g;
                own_g[k] = q.g;
                own_loss[k] = q.loss;
                own_kept[k] = st.target[b0 + k] != st.ignore;
                if (blockIdx.x == 0) {
                    if (a.rows.loss) a.rows.loss[b0 + k] = q.loss;
                    if (a.rows.lse) a.rows.lse[b0 + k] = q.lse();
                }
            }
            const int tile = blockIdx.x * blocks + l8;
            if (l8 < blocks)
                own_f[k][l8] = tile >= st.tiles ? 0.f
                                : q.valid        ? q.g * a.rows.exp_unit * q.exp_of(st.tile_max[(long long)(b0 + k) * st.tiles + tile])
                                                 : NAN;
        }
        if (blockIdx.x == 0) leave_part(a.rows, blockIdx.y, own_loss, own_kept);
        else __syncthreads();
#pragma unroll
        for (int u = 0; u < R; ++u) {
            f[u] = own_f[rl + u * 8][(lane * 8) >> a.tile_shift];
            even[u] = st.smoothing * st.inv_classes * own_g[rl + u * 8];
            tg[u] = own_tg[rl + u * 8];
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) db.v[e] = 0.f;
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int r = r0 + u * 8;
        if (!in || r >= st.rows) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = col + e < st.classes ? g[u].v[e] * f[u] - even[u] : 0.f;
            if (col + e == t[u]) v = tg[u];
            if (t[u] == st.ignore) v = 0.f;                  // whatever the row held
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
}

// What is left when the products are done, in one launch: slabs of partial sums added up in their order, partial rows of db,
// the loss.  Bound by memory where there are slabs (134 MB of them in 31 us, 4.3 TB/s), else by its latency (4 us).
struct XentSlabs {
    const float* in;                      // [slabs][rows][ld]
    void* out;                            // [rows][cols], dense
    long long ld;
    int slabs, rows, cols, blocks;        // blocks: 0 for nothing to do
};
struct XentFinish {
    XentSlabs dx, dw;
    const float* db_part;                 // [groups][ld_db]
    void* db;
    long long ld_db;
    int groups, classes, db_bf16, db_blocks;
    const float* factor;
    XentLoss loss;                        // by the last workgroup
};
constexpr int kSlabPerBlock = 256 * 8 * 2;       // results a workgroup

template <typename T>
__device__ __forceinline__ void add_slabs(const XentSlabs& a, int block, float f) {
    const int per_row = (a.cols + 7) / 8;
    const long long vectors = (long long)a.rows * per_row, stride = a.rows * a.ld;
#pragma unroll 1
    for (int n = 0; n < 2; ++n) {
        const long long v = ((long long)block * 2 + n) * 256 + threadIdx.x;
        if (v >= vectors) return;
        const long long r = v / per_row;
        const int c = (int)(v - r * per_row) * 8;
        const float* src = a.in + r * a.ld + c;                // (slab rows are padded to whole tiles)
        F8 o = load8_full(src);
#pragma unroll 4
        for (int s = 1; s < a.slabs; ++s) {
            const F8 q = load8_full(src + s * stride);
#pragma unroll
            for (int e = 0; e < 8; ++e) o.v[e] += q.v[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) o.v[e] *= f;
        store8((T*)a.out + r * a.cols + c, a.cols - c, o);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void xent_finish_kernel(const XentFinish a) {
    int b = blockIdx.x;
    if (b < a.dx.blocks) {
        add_slabs<T>(a.dx, b, *a.factor);
        return;
    }
    b -= a.dx.blocks;
    if (b < a.dw.blocks) {
        add_slabs<T>(a.dw, b, *a.factor);
        return;
    }
    b -= a.dw.blocks;
    if (b < a.db_blocks) {                // 64 columns: 16 lanes of four by 16 row strides
        __shared__ float s[16][64 + 1];
        const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int p = r; p < a.groups; p += 16) v += *(const f32x4*)(a.db_part + p * a.ld_db + b * 64 + c * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r][c * 4 + e] = v[e];
        __syncthreads();
        const int col = b * 64 + threadIdx.x;
        if (threadIdx.x < 64 && col < a.classes) {
            float o = 0.f;
#pragma unroll
            for (int p = 0; p < 16; ++p) o += s[p][threadIdx.x];
            o *= *a.factor;
            if (a.db_bf16) store1((short*)a.db + col, o);
            else store1((float*)a.db + col, o);
        }
        return;
    }
    finish_loss(a.loss);
}

// ---------------------------------------------------------------------------------------------
// Host side: how a call is cut up
// ---------------------------------------------------------------------------------------------
struct XentPlan {
    int esize, rows, pieces, tiles, tile, tile_shift, dx_tile, dw_tile, dx_splits, dw_splits, row_groups;
    long long ld_e, ld_pack;
    bool dw_slabs, pack_x, pack_w, wide, few, small;
    // workspace offsets, bytes
    long long shared, loss, kept, counts, tmax, tsum, tlin, tlogit, tg, rg, e, dbp, dxs, dws, xp, wp, gp, total;
};

// Of exponentials held at a time.  Every further piece reads W again and adds to dW in memory: 16384 x 65536 x 512 bf16 with
// gradients takes 4.56 ms in pieces of 4 GiB and 4.88 in pieces of 1, 16384 x 8192 x 512 fp32 2.45 and 2.89, 8192 x 32768 x
// 2048 bf16 (512 MB) 2.90 and in pieces of 256 MB, which the 256 MB cache would nearly hold, 3.7.
constexpr long long kPieceBytes = 1LL << 32;
constexpr int kPieceRows = 1 << 17;               // and rows,
constexpr long long kPieceSums = 1LL << 26;       // maxima and sums per tile,
constexpr long long kPieceInputs = 1LL << 34;     // and elements of x: what grids are sized by

inline int k_per_split(int k, int splits, int bk) { return ceil_div(ceil_div(k, splits), bk) * bk; }

// rows on 16 bytes, whole steps of 64 k, a tile's rows within 32-bit offsets
inline bool lies_well(const void* t, long long ld, int d) {
    return !((uintptr_t)t & 15) && !(ld & 7) && !(d & 63) && ld <= (1 << 20);
}

inline long long slab_ld(int d, int tile) { return (long long)ceil_div(d, tile) * tile; }

// Up to 32 rows of fp32 the products run as in xent_few.hip (32 x 2000 x 512 with gradients 28 us, on 64 x 64 tiles 46), of
// bf16 up to 16 and with a small weight (8 x 2000 x 512 20 us, on 128 x 128 tiles 24; 8 x 8000 x 2048 84, 64; 32 x 2000 x 512
// 31, 27).
inline bool takes_few(const asl_xent_params& p) {
    if (!p.n || p.classes > kFewClasses) return false;
    return p.type ? p.n <= kFewRows16 && (double)p.classes * p.d <= (double)(1 << 20) : p.n <= kFewRows;
}

// Tile and slices of a product with `a` x `b` results over `k`: what its tiles take one after another on the 256 CUs, against
// what slabs of partial sums cost (written and read back at 4 TB/s, and one more launch).  Measured with one workgroup a CU:
// 1.65 us per 64 of k for 256 x 256, 0.65 for 128 x 128 (fp32 in planes: six times that), 0.6 for 64 x 64, and about 8, 5 and 3
// us around that a tile.  bf16 takes the larger two, however narrow (2000 x 50 x 64 with gradients 25 us, on 64 x 64 tiles of
// bf16 29; 100000 x 30 x 128 145 and 262).  fp32 takes 64 x 64 where taking it apart into planes does not pay: narrow products
// (100000 x 30 x 512 504 us, in planes 578; 100000 x 1000 x 16 985, 1123), few rows, for which W's planes cost most (128 x
// 32768 x 1024 315, 378; 256 rows 577, 505), and small ones (512 x 2000 x 512 70, 74; 1024 rows 104, 93).
struct TilePlan {
    int tile, splits;
};
inline TilePlan tiles_for(const asl_xent_params& p, long long a, long long b, int k, bool may_split) {
    const bool whole = !p.type && (p.classes < 64 || p.d < 32 || p.n < 256 || (double)p.n * p.classes * p.d < (double)(1 << 29));
    TilePlan best = {kTile, 1};
    double least = 1e30;
    const int steps = ceil_div(k, 64);
    for (const int tile : {64, 128, 256}) {
        if (whole != (tile == 64)) continue;
        const long long tiles = (long long)ceil_div(a, tile) * ceil_div(b, tile);
        const double us = tile == 256 ? 1.65 : tile == 128 ? 0.65 : 0.6;
        const double around = tile == 256 ? 8.0 : tile == 128 ? 5.0 : 3.0;
        // The logits: a 256 x 256 tile takes 14 us around its steps (first loads, exponentials, results), and where there are
        // more than 256 of 128 x 128 two share a CU at 1.7 times the step (425 x 9743 x 144 forward 18 us, on 78 large tiles 25;
        // 4381 x 7862 x 652 86, 92; 100000 x 2000 x 128 145, 176).
        if (!may_split) {
            const double k64 = steps * us * (p.type || tile == 64 ? 1 : 6), one = k64 + (tile == 256 ? 14.0 : around), two = k64 * 1.7 + around;
            const int rest = (int)(tiles % 512);
            const double t = tile == 128 ? tiles / 512 * two + (rest > 256 ? two : rest ? one : 0.0) : ceil_div(tiles, 256) * one;
            if (t < least) {
                least = t;
                best = {tile, 1};
            }
            continue;
        }
        for (int s = 1; s <= 32 && (s == 1 || s * 2 <= steps); ++s) {
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

// 64 x 64 tiles up to which the logits are taken on 32 x 32, eight waves sharing the contraction of one: half of the CUs would
// be idle else, and each of the others wait on a step at a time (fp32 forward: 64 x 2000 x 512, 32 of them, 13.9 us and 24.7;
// 256 x 2000 x 512, 128 of them, 19.7 and 25.1; 2000 x 300 x 512, 160, 28.0 and 27.9; 512 x 2000 x 512, 256, 30.9 and 25.7)
constexpr long long kSmallTiles = 128;

XentPlan xent_plan(const asl_xent_params& p, const void* xp, const void* wp, bool grad, bool want_dx, bool want_dw, bool want_db) {
    XentPlan q = {};
    q.esize = p.type ? 2 : 4;
    q.few = takes_few(p);
    q.tile = q.few ? kFewTile : tiles_for(p, p.n, p.classes, p.d, false).tile;
    q.small = !q.few && q.tile == kTile && (long long)ceil_div(p.n, kTile) * ceil_div(p.classes, kTile) <= kSmallTiles;
    q.tile_shift = q.few || q.small ? 5 : q.tile == 256 ? 7 : 6;     // maxima and sums are kept per 32, 128 or 64 classes
    // the tile kernels read 16 bytes at a time and whole steps of 64 k: operands that do not allow it are laid out anew
    q.ld_pack = (p.d + 63LL) / 64 * 64;
    q.wide = q.tile > kTile && !p.type;
    q.pack_x = q.tile > kTile && (q.wide || !lies_well(xp, p.ld_x, p.d));
    q.pack_w = q.tile > kTile && (q.wide || !lies_well(wp, p.ld_w, p.d));
    const int planes = q.wide ? 3 : 1;
    q.tiles = ceil_div(p.classes, 1 << q.tile_shift);
    // (128 bytes off a power of two, which would put a tile's rows all in the same few channels: dx of 8192 x 32768 x 2048
    // takes 836 us with them and 906 without)
    q.ld_e = (long long)ceil_div(p.classes, q.tile) * q.tile + (q.tile > kTile ? 64 : 0);
    long long rows = p.n;
    for (const long long most : {(long long)kPieceRows, kPieceSums / q.tiles / 256 * 256, kPieceInputs / p.d / 256 * 256})
        if (rows > most) rows = most;
    if (grad) {
        const long long most = kPieceBytes / (q.ld_e * (q.wide ? 10 : q.esize)) / 256 * 256;
        if (rows > most) rows = most < 256 ? 256 : most;
    }
    q.rows = (int)rows;
    q.pieces = p.n ? ceil_div(p.n, rows) : 0;
    q.row_groups = ceil_div(rows, kGradRows);
    const int bk = q.tile > kTile ? 64 : kStep;
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
    q.loss = take(4LL * ceil_div(p.n, 4));               // (partial sums of 4, 16 or 32 rows)
    q.kept = take(4LL * ceil_div(p.n, 4));
    q.counts = take(p.n > kCountRows ? 4LL * ceil_div(p.n, kCountRows) : 0);
    q.tmax = take(4LL * rows * q.tiles);
    q.tsum = take(4LL * rows * q.tiles);
    q.tlin = take(p.label_smoothing != 0.f ? 4LL * rows * q.tiles : 0);
    q.tlogit = take(4LL * rows);
    if (grad) {
        q.tg = take(4LL * rows);
        q.rg = take(4LL * rows);
        q.e = take(q.esize * rows * q.ld_e);
        q.dbp = take(want_db ? 4LL * q.row_groups * q.ld_e : 0);
        q.dxs = take(want_dx && q.dx_splits > 1 ? 4LL * q.dx_splits * rows * slab_ld(p.d, q.dx_tile) : 0);
        q.dws = take(want_dw && q.dw_slabs ? 4LL * q.dw_splits * p.classes * slab_ld(p.d, q.dw_tile) : 0);
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
    // a launch is fewer than 2^32 threads: 2^24 workgroups, each with at least 64 x 64 results of a product
    if (p->n > (1 << 28) || p->classes > (1 << 21) || p->d > (1 << 20) || (long long)p->classes * p->d > (1LL << 34)) return ASL_ETOOBIG;
    return ASL_OK;
}

// eight elements moved down by `lead` of 0 to 7, noughts behind them
__device__ __forceinline__ bf16x8 moved_down(const bf16x8& v, int lead) {
    i32x4 w = __builtin_bit_cast(i32x4, v);
    const auto by = [&](bool yes, int words, bool half) {
        i32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned lo = i + words < 4 ? w[i + words] : 0, hi = i + words + 1 < 4 ? w[i + words + 1] : 0;
            r[i] = yes ? (half ? (int)(lo >> 16 | hi << 16) : (int)lo) : w[i];
        }
        w = r;
    };
    by(lead & 1, 0, true);
    by(lead & 2, 1, false);
    by(lead & 4, 2, false);
    return __builtin_bit_cast(bf16x8, w);
}
__device__ __forceinline__ Raw8F moved_down(const Raw8F& v, int lead) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < 4 ? v.a[e] : v.b[e - 4];
#pragma unroll
    for (int by = 1; by < 8; by *= 2)
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = lead & by ? (e + by < 8 ? f[e + by] : 0.f) : f[e];
    return {{f[0], f[1], f[2], f[3]}, {f[4], f[5], f[6], f[7]}};
}

// Rows of d elements at any alignment to rows of `per_row` 16-byte vectors of bf16, noughts behind d; fp32 to three planes of
// them.  Two matrices in one launch, or one (rows of the other: 0).  777 and 5003 rows of 509 bf16 take 5.0 us, 2048 and 8192 of
// 1024 fp32 20 (5.2 TB/s).
template <typename T>
struct XentPack {
    const T* src[2];
    short* dst[2];
    long long ld[2];
    int rows[2], d, per_row;
};
template <typename T>
__global__ __launch_bounds__(256) void xent_pack_kernel(const XentPack<T> a) {
    const long long first = (long long)a.rows[0] * a.per_row, both = first + (long long)a.rows[1] * a.per_row;
    for (long long w = blockIdx.x * 256LL + threadIdx.x; w < both; w += gridDim.x * 256LL) {
        const bool two = w >= first;
        const long long v = two ? w - first : w, r = v / a.per_row;
        const int c = (int)(v - r * a.per_row) * 8;
        // a row's last vector is read as the row's last eight elements and moved down, not element by element
        const int at = c + 8 <= a.d ? c : a.d >= 8 ? a.d - 8 : 0, lead = c - at;
        auto raw = load8_raw((two ? a.src[1] : a.src[0]) + r * (two ? a.ld[1] : a.ld[0]) + at, a.d);
        if (lead >= 8) raw = decltype(raw){};
        else if (lead) raw = moved_down(raw, lead);
        short* dst = (two ? a.dst[1] : a.dst[0]) + v * 8;
        if constexpr (std::is_same<T, short>::value) *(bf16x8*)dst = raw;
        else store_planes(dst, (two ? both - first : first) * 8, widen(raw));
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
    const int bk = q.tile > kTile ? 64 : kStep;
    const bool none = p.reduction == ASL_REDUCE_NONE, mean = p.reduction == ASL_REDUCE_MEAN;
    float* shared = (float*)(ws + q.shared);
    // the rows' statistics by the G pass, or by a launch of their own, a wave or a quarter of one each
    const bool own = grad && q.tiles <= kOwnStats;
    const int per_part = own ? kGradRows : q.tiles <= kOwnStats ? 16 : 4;
    XentLoss all = {(const float*)(ws + q.loss), (const int*)(ws + q.kept), loss, ceil_div(p.n, per_part), mean};
    int* counts = p.n > kCountRows ? (int*)(ws + q.counts) : nullptr;
    XentFactor factor = {target, counts, none ? nullptr : upstream, shared, p.ignore_index, p.n, mean};
    if (grad && mean && counts)
        hipLaunchKernelGGL(xent_count_kernel, dim3((unsigned)ceil_div(p.n, kCountRows)), dim3(256), 0, s, target, p.n, factor.ignore, counts);
    const void* wk = w;                   // what the products read: the caller's tensors, or their copies
    long long ld_w = p.ld_w, ld_x = p.ld_x;
    if (q.pack_w) wk = ws + q.wp, ld_w = q.ld_pack;
    if (q.pack_x) ld_x = q.ld_pack;
    for (int piece = 0; piece < q.pieces; ++piece) {
        const int r0 = piece * q.rows, rows = p.n - r0 < q.rows ? p.n - r0 : q.rows;
        const T* xr = (const T*)x + r0 * p.ld_x;
        if (q.pack_x || (q.pack_w && piece == 0)) {
            XentPack<T> c = {};
            if (q.pack_x) c.src[0] = xr, c.dst[0] = (short*)(ws + q.xp), c.ld[0] = p.ld_x, c.rows[0] = rows;
            if (q.pack_w && piece == 0) c.src[1] = (const T*)w, c.dst[1] = (short*)(ws + q.wp), c.ld[1] = p.ld_w, c.rows[1] = p.classes;
            c.d = p.d; c.per_row = (int)(q.ld_pack / 8);
            const int blocks = ceil_div(((long long)c.rows[0] + c.rows[1]) * c.per_row, 512);
            hipLaunchKernelGGL((xent_pack_kernel<T>), dim3(blocks < 8192 ? blocks : 8192), dim3(256), 0, s, c);
        }
        if (q.pack_x) xr = (const T*)(ws + q.xp);
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
        } else if (q.small) {
            XentFew f = {};
            f.x = xr; f.w = wk; f.bias = bias; f.bias_bf16 = p.bias_type; f.target = g.target; f.e = grad ? (float*)g.out : nullptr;
            f.tile_max = g.tile_max; f.tile_sum = g.tile_sum; f.tile_lin = g.tile_lin; f.target_logit = g.target_logit;
            f.ld_x = ld_x; f.ld_w = ld_w; f.ld_e = q.ld_e; f.smoothing = p.label_smoothing; f.n = rows; f.classes = p.classes; f.d = p.d;
            f.tiles = q.tiles;
            xent_few_logits(f, s);
        } else {
            const int tj = ceil_div(rows, kTile);
            hipLaunchKernelGGL(xent_gemm_logits_kernel, dim3((unsigned)(q.tiles * tj)), dim3(256), 0, s, g, q.tiles, tj);
        }
        XentRows r = {};
        r.st.target = target + r0; r.st.upstream = upstream && none ? upstream + r0 : nullptr;
        r.st.tile_max = g.tile_max; r.st.tile_sum = g.tile_sum; r.st.tile_lin = g.tile_lin; r.st.target_logit = g.target_logit;
        r.st.ignore = p.ignore_index; r.st.smoothing = p.label_smoothing; r.st.inv_classes = 1.f / (float)p.classes;
        r.st.rows = rows; r.st.classes = p.classes; r.st.tiles = q.tiles;
        r.factor = grad ? g.tile_max : nullptr; r.target_g = (float*)(ws + q.tg); r.row_g = (float*)(ws + q.rg);
        r.loss = none ? loss + r0 : nullptr; r.lse = lse ? lse + r0 : nullptr; r.exp_unit = 1.f / Held<T>::SCALE;
        if (!none) r.loss_part = (float*)(ws + q.loss) + r0 / per_part, r.kept_part = (int*)(ws + q.kept) + r0 / per_part;
        const bool last = piece == q.pieces - 1;
        if (!own && per_part == 16) hipLaunchKernelGGL((xent_rows_kernel<16>), dim3(ceil_div(rows, 16)), dim3(256), 0, s, r);
        else if (!own) hipLaunchKernelGGL((xent_rows_kernel<64>), dim3(ceil_div(rows, 4)), dim3(256), 0, s, r);
        if (!grad) continue;
        XentG c = {};
        c.rows = r; c.e = ws + q.e; c.ld = q.ld_e; c.planes = q.wide ? (short*)(ws + q.gp) : nullptr; c.plane = rows * q.ld_e;
        c.db_part = db ? (float*)(ws + q.dbp) : nullptr; c.db_add = piece > 0; c.tile_shift = q.tile_shift;
        if (!none && last && !own) c.loss = all;
        if (piece == 0) c.factor = factor;
        const int groups = ceil_div(rows, kGradRows);
        const dim3 g_grid(ceil_div(q.ld_e, kGradCols), groups + (c.factor.factor || c.loss.loss_part ? 1 : 0));
        if (own) hipLaunchKernelGGL((xent_g_kernel<T, true>), g_grid, dim3(256), 0, s, c);
        else hipLaunchKernelGGL((xent_g_kernel<T, false>), g_grid, dim3(256), 0, s, c);

        XentGemm hx = {}, hw = {};
        const void* G = ws + (q.wide ? q.gp : q.e);
        // dx[row][k] = sum over classes G[row][v] W[v][k]
        hx.p = wk; hx.ld_p = ld_w; hx.q = G; hx.ld_q = q.ld_e; hx.I = p.d; hx.Jn = rows; hx.K = p.classes;
        if (q.wide) hx.plane_p = p.classes * ld_w, hx.plane_q = rows * q.ld_e;
        hx.k_per_split = k_per_split(p.classes, q.dx_splits, bk);
        hx.slabs = q.dx_splits > 1; hx.factor = shared;
        T* dxr = (T*)dx + (long long)r0 * p.d;
        hx.out = hx.slabs ? (void*)(ws + q.dxs) : (void*)dxr; hx.ld_out = p.d; hx.splits = q.dx_splits;
        // dW[v][k] = sum over rows G[row][v] x[row][k]
        hw.p = xr; hw.ld_p = ld_x; hw.q = G; hw.ld_q = q.ld_e; hw.I = p.d; hw.Jn = p.classes; hw.K = rows;
        if (q.wide) hw.plane_p = rows * ld_x, hw.plane_q = rows * q.ld_e;
        hw.k_per_split = k_per_split(q.rows, q.dw_splits, bk);
        hw.slabs = q.dw_slabs; hw.factor = shared; hw.add = piece > 0;
        hw.out = hw.slabs ? (void*)(ws + q.dws) : dw; hw.ld_out = p.d; hw.splits = q.dw_splits;
        int rc = 0;
        if (q.dx_tile == kTile) {                    // (then dW's is as well)
            const int xi = ceil_div(p.d, kTile), xj = dx ? ceil_div(rows, kTile) : 0, wj = dw ? ceil_div(p.classes, kTile) : 0;
            const int nx = xi * xj * q.dx_splits, nw = xi * wj * q.dw_splits;
            if (nx + nw)
                hipLaunchKernelGGL(xent_gemm_pair_kernel, dim3((unsigned)(nx + nw)), dim3(256), 0, s, hx, hw, xi, xj, xi, wj, nx);
        } else if (dx && dw && q.dx_tile == 128 && q.dw_tile == 128) {
            rc = xent_tiles_pair(hx, hw, s);
        } else {
            if (dx) rc = xent_tiles_dx(hx, q.dx_tile, s);
            if (dw && !rc) rc = xent_tiles_dw(hw, q.dw_tile, s);
        }
        if (rc) return rc;

        XentFinish f = {};
        const auto slabs = [&](XentSlabs& o, const void* in, void* out, int n, int rows_, int tile) {
            o.in = (const float*)in; o.out = out; o.slabs = n; o.rows = rows_; o.cols = p.d; o.ld = slab_ld(p.d, tile);
            o.blocks = ceil_div((long long)rows_ * ceil_div(p.d, 8), kSlabPerBlock / 8);
        };
        if (dx && hx.slabs) slabs(f.dx, ws + q.dxs, dxr, q.dx_splits, rows, q.dx_tile);
        if (dw && hw.slabs && last) slabs(f.dw, ws + q.dws, dw, q.dw_splits, p.classes, q.dw_tile);
        if (db && last) {
            f.db_part = c.db_part; f.db = db; f.ld_db = q.ld_e; f.groups = q.row_groups; f.classes = p.classes; f.db_bf16 = p.bias_type;
            f.db_blocks = ceil_div(p.classes, 64);
        }
        f.factor = shared;
        if (!none && last && own) f.loss = all;
        const long long blocks = (long long)f.dx.blocks + f.dw.blocks + f.db_blocks + (f.loss.loss_part ? 1 : 0);
        if (blocks > 0x7fffffffLL) return ASL_ETOOBIG;
        if (blocks) hipLaunchKernelGGL((xent_finish_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, s, f);
    }
    if (!none && (!grad || !q.pieces)) hipLaunchKernelGGL(xent_loss_kernel, dim3(1), dim3(256), 0, s, all);
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

// What the cross entropy operator's files share (linear_xent.hip, xent_tiles.hip, xent_few.hip).
#pragma once
#include "train_common.h"

namespace asl_detail {

// D[j][i] = sum over k of P(i, k) Q(j, k).  P is the MFMA's row operand, so a lane ends up with four consecutive i of one j
// and D is stored along i.  Each operand is contiguous along k ("KC") or along its own index.
struct XentGemm {
    const void* p;
    const void* q;
    long long ld_p, ld_q;    // elements from one row of the stored matrix to the next
    long long plane_p, plane_q;   // fp32 operands as three bf16 planes: elements from one plane to the next (0: one plane)
    int I, Jn, K;
    // plain products
    void* out;               // of the operands' type, or fp32 slabs [splits][Jn][I up to whole tiles] when slabs != 0
    long long ld_out;
    const float* factor;     // on the device; multiplies the sums on their way out (slabs: not yet)
    int slabs, add, k_per_split, splits;
    // logits
    const void* bias;
    int bias_bf16, smooth, store_e;
    const long long* target; // of row j
    float* tile_max;         // [Jn][tiles]
    float* tile_sum;         // [Jn][tiles]
    float* tile_lin;         // [Jn][tiles]: sum of the logits (label smoothing)
    float* target_logit;     // [Jn]
    int tiles;
};

inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

constexpr float kExpScale16 = 32768.f;    // exponentials in (0, 1] held as fp16: times this, so that fp16's range is used

// xent_tiles.hip, tile 128 or 256: bf16 (or fp32 as planes of it), both operands' rows on 16 bytes and at most 2^22 + 128
// bytes apart; those contiguous along k hold noughts from K to the next multiple of 64
int xent_tiles_logits(const XentGemm& a, int tile, hipStream_t s);
int xent_tiles_dx(const XentGemm& a, int tile, hipStream_t s);     // P along its own index, Q along k
int xent_tiles_dw(const XentGemm& a, int tile, hipStream_t s);     // both along their own index
int xent_tiles_pair(const XentGemm& dx, const XentGemm& dw, hipStream_t s);     // both, on 128 x 128 tiles

// 16 x 16 x 4 in fp32
__device__ __forceinline__ f32x4 mma4(float a, float b, f32x4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
#else
    return c;
#endif
}

// What the products leave of a piece of rows, and what becomes of it.
struct XentStats {
    const long long* target; // of the piece's rows
    const float* upstream;   // null: 1
    const float* tile_max;   // [rows][tiles]
    const float* tile_sum;
    const float* tile_lin;
    const float* target_logit;
    long long ignore;
    float smoothing, inv_classes;
    int rows, classes, tiles;
};
// log sum exp stays in two parts, the largest logit and the logarithm of the sum relative to it.  Only the lse that a caller
// reads is their sum: rounded to 32 bits it is off by up to 2^-24 of itself, which is not little beside the 1 - p of a row that is
// nearly certain (half of it at an lse of 60 and 1 - p = 2^-18), and loss and G taken from it would be off by that.
struct XentRow {
    float top, rest;                         // lse = top + rest
    float loss, g, target_g;                 // g: the row's own weight, nought for an ignored row; target_g: G at the target
    bool valid;                              // a label outside the vocabulary makes loss and gradients NaN
    __device__ __forceinline__ float lse() const { return top + rest; }
    __device__ __forceinline__ float exp_of(float l) const { return expf((l - top) - rest); }    // exp(l - lse)
};

// LANES lanes (a wave, a quarter or an eighth of one) on a row: its tile maxima and sums to its statistics, in one pass, the running sum
// rescaled where the maximum moves.
template <int LANES>
__device__ __forceinline__ XentRow row_stats(const XentStats& a, int row, int lane) {
    const float* mx = a.tile_max + (long long)row * a.tiles;
    const float* sm = a.tile_sum + (long long)row * a.tiles;
    const long long t = a.target[row];
    XentRow o;
    o.valid = t >= 0 && t < a.classes;
    const bool kept = t != a.ignore;
    o.g = !kept ? 0.f : a.upstream ? a.upstream[row] : 1.f;
    const float lt = o.valid ? a.target_logit[row] : NAN;
    float m = -INFINITY, s = 0.f, lin = 0.f;
#pragma unroll 4
    for (int k = lane; k < a.tiles; k += LANES) {
        const float v = mx[k], q = sm[k];
        if (v > m) {
            s = s * expf(m - v) + q;
            m = v;
        } else {
            s += q * expf(v - (m == -INFINITY ? 0.f : m));
        }
        if (a.smoothing != 0.f) lin += a.tile_lin[(long long)row * a.tiles + k];
    }
    const auto sum = [](float v) {
        if constexpr (LANES == 64) return wave64_sum(v);
        else return row16_sum<LANES>(v);
    };
    float top;
    if constexpr (LANES == 64) top = wave_max(m);
    else top = row16_max<LANES>(m);
    o.top = top == -INFINITY ? 0.f : top;
    o.rest = logf(sum(s * expf(m - o.top)));
    const float above = lt - o.top;
    o.loss = o.rest - above;
    if (a.smoothing != 0.f) o.loss = o.rest - (1.f - a.smoothing) * above - a.smoothing * (a.inv_classes * sum(lin) - o.top);
    if (!kept) o.loss = 0.f;
    o.target_g = o.g * (expm1f(above - o.rest) + a.smoothing - a.smoothing * a.inv_classes);
    return o;
}

// xent_few.hip: up to 32 rows, of bf16 up to 16
constexpr int kFewRows = 32, kFewRows16 = 16, kFewTile = 32, kFewClasses = 16384;      // rows of fp32, and of bf16
struct XentFew {
    const void* x;
    const void* w;
    const void* bias;
    const long long* target;
    const float* upstream;   // null: 1; one value a row with `none`
    float* loss;
    float* lse;              // null: not wanted
    void* dx;                // each null: not wanted
    void* dw;
    void* db;
    float* e;                // [n][ld_e]: exponentials, then G; null: no gradients
    float* tile_max;         // [n][tiles]
    float* tile_sum;
    float* tile_lin;
    float* target_logit;
    float* factor;           // with gradients
    float* slabs;            // [xent_few_slabs][n][d]
    long long ld_x, ld_w, ld_e, ignore;
    float smoothing, inv_classes;
    int n, classes, d, tiles, bias_bf16, none, mean;
};
// slices of the classes for dx: 128 classes a workgroup, at most 32 slices
inline int xent_few_slabs(int classes) { return classes < 128 * 32 ? ceil_div(classes, 128) : 32; }
int xent_few(const XentFew& a, int type, hipStream_t s);
void xent_few_logits(const XentFew& a, hipStream_t s);     // the logits of any number of fp32 rows: 32 x 32 tiles

}  // namespace asl_detail

// Global norm of many gradient tensors, and clipping by it, for gfx950.
//
//   n = sqrt(sum over all elements g^2)   or   n = max |g|;    c = min(1, max_norm / (n + 1e-6));    out = g c
//
// Two launches for up to kTensors tensors (two more for every kTensors further; one for a few small ones): the first leaves one
// partial a workgroup, the second adds the partials up in every workgroup -- in the same order, so all see the same c -- and
// writes g c.  Tensors are cut into chunks; a chunk's tensor is found by a binary search over the chunk counts, which travel
// with the pointers in the kernel's arguments: nothing is copied to the device and nothing outlives the call.  The sum is held
// in 64 bits: the vector pipe has room for it under the loads, the largest fp32 gradients do not overflow it, and its order
// does not show in the result.  The second pass walks the chunks from the last to the first, because the end of what the first
// pass read is what the 256 MB cache still holds.
//
// Bound by memory: 357 M bf16 elements into fp32 take 582 us (2.85 GB, read twice and written: 4.9 TB/s, as a copy of 2 GiB),
// 14 M fp32 elements of some 50 tensors in place 13 + 20 us, from the cache in part; the smallest calls one launch (below).
// A chunk's accesses are runs of whole lines (32 bytes a thread, two lines' halves at a time: 637 us).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <new>
#include <utility>
#include <vector>

#include "asl_hip.h"
#include "train_common.h"

namespace asl_detail {

constexpr int kTensors = 140;             // per launch: 28 bytes of arguments each, of the 4 KiB that a launch may take
constexpr int kChunk = 8192;              // elements: 256 threads x 8 x 4
constexpr long long kMostElements = 1LL << 36;   // of one tensor: a launch's chunks are counted in 32 bits
constexpr int kClipBlocks = 2048;         // at most, per launch: 8 workgroups of 256 a CU

// A tensor's address with its type in bit 0 (elements are at least two bytes apart: the bit is free; set: bf16).
struct Tagged {
    unsigned long long bits;
    __device__ __forceinline__ bool bf16() const { return bits & 1; }
    // (said to be global memory: the compiler cannot know of an address that was a number, and would use flat accesses)
    template <typename T>
    __device__ __forceinline__ T* ptr() const {
        return (T*)(__attribute__((address_space(1))) T*)(bits & ~1ull);
    }
};

struct ClipArgs {
    Tagged in[kTensors], out[kTensors];
    long long n[kTensors];
    int first[kTensors + 1];              // first chunk of each tensor in this launch; the last entry is the chunk count
    int tensors, part0, parts, inf_norm, write_norm;
    float max_norm;
    double* part;
    float* norm;
};
static_assert(sizeof(ClipArgs) <= 4096, "kernel arguments");

// the larger of two magnitudes, a NaN before any number
__device__ __forceinline__ double max_nan(double a, double b) { return (a > b || a != a) ? a : b; }

__device__ __forceinline__ double combine(double a, double b, int inf_norm) { return inf_norm ? max_nan(a, b) : a + b; }

// over the 256 threads of a workgroup, the same in every thread
__device__ __forceinline__ double block_combine(double v, int inf_norm, double* lds) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = combine(v, __shfl_xor(v, o, 64), inf_norm);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return combine(combine(lds[0], lds[1], inf_norm), combine(lds[2], lds[3], inf_norm), inf_norm);
}

__device__ __forceinline__ int tensor_of(const ClipArgs& a, int chunk) {
    int lo = 0, hi = a.tensors;           // first[lo] <= chunk < first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

// A chunk's share of a thread: vectors of V elements, 256 apart, so that a wave's access is one run of lines.
template <int V>
__device__ __forceinline__ int vector_len(long long left, int i) {
    const long long k = left - (i * 256 + (int)threadIdx.x) * V;
    return k >= V ? V : k > 0 ? (int)k : 0;
}

__device__ __forceinline__ void add_square(float g, int inf_norm, double& v) {
    const double x = (double)g;
    v = inf_norm ? max_nan(fabs(x), v) : v + x * x;
}
__device__ __forceinline__ void accumulate(const float* p, long long left, int inf_norm, double& v) {
    f32x4 g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int n = vector_len<4>(left, i);
        g[i] = load4(p + (n ? (i * 256 + threadIdx.x) * 4 : 0), n);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) add_square(g[i][e], inf_norm, v);
}
__device__ __forceinline__ void accumulate(const short* p, long long left, int inf_norm, double& v) {
    bf16x8 g[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = vector_len<8>(left, i);
        g[i] = load8_raw(p + (n ? (i * 256 + threadIdx.x) * 8 : 0), n);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) add_square(bf16_to_f32(g[i][e]), inf_norm, v);
}

__global__ __launch_bounds__(256) void grad_norm_kernel(const ClipArgs a) {
    __shared__ double lds[4];
    double v = 0.0;
    for (int c = blockIdx.x; c < a.first[a.tensors]; c += gridDim.x) {
        const int t = tensor_of(a, c);
        const long long at = (long long)(c - a.first[t]) * kChunk;
        if (a.in[t].bf16()) accumulate(a.in[t].ptr<const short>() + at, a.n[t] - at, a.inf_norm, v);
        else accumulate(a.in[t].ptr<const float>() + at, a.n[t] - at, a.inf_norm, v);
    }
    v = block_combine(v, a.inf_norm, lds);
    if (threadIdx.x == 0) a.part[a.part0 + blockIdx.x] = v;
}

// a norm that is not a number makes every gradient one, an infinite norm makes them nought (and NaN where infinite)
__device__ __forceinline__ float factor_of(float norm, float max_norm) {
    const float r = max_norm / (norm + 1e-6f);
    return r > 1.0f ? 1.0f : r;
}

template <typename T, typename U>
__device__ __forceinline__ void scale_chunk(const T* p, U* q, long long left, float c) {
    f32x4 g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int n = vector_len<4>(left, i);
        g[i] = load4(p + (n ? (i * 256 + threadIdx.x) * 4 : 0), n);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int n = vector_len<4>(left, i);
        if (n) store4(q + (i * 256 + threadIdx.x) * 4, n, f32x4{g[i][0] * c, g[i][1] * c, g[i][2] * c, g[i][3] * c});
    }
}

__global__ __launch_bounds__(256) void grad_scale_kernel(const ClipArgs a) {
    __shared__ double lds[4];
    double v = 0.0;
    for (int i = threadIdx.x; i < a.parts; i += 256) v = combine(v, a.part[i], a.inf_norm);
    v = block_combine(v, a.inf_norm, lds);
    const float norm = (float)(a.inf_norm ? v : sqrt(v));
    if (a.write_norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = norm;
    const float c = factor_of(norm, a.max_norm);
    const int chunks = a.first[a.tensors];
    for (int i = blockIdx.x; i < chunks; i += gridDim.x) {
        const int k = chunks - 1 - i, t = tensor_of(a, k);
        const Tagged in = a.in[t], out = a.out[t];
        if (c == 1.0f && in.bits == out.bits) continue;        // in place and nothing to clip: as it is
        const long long at = (long long)(k - a.first[t]) * kChunk, left = a.n[t] - at;
        if (in.bf16()) {
            if (out.bf16()) scale_chunk(in.ptr<const short>() + at, out.ptr<short>() + at, left, c);
            else scale_chunk(in.ptr<const short>() + at, out.ptr<float>() + at, left, c);
        } else {
            if (out.bf16()) scale_chunk(in.ptr<const float>() + at, out.ptr<short>() + at, left, c);
            else scale_chunk(in.ptr<const float>() + at, out.ptr<float>() + at, left, c);
        }
    }
}

// A few small tensors in one launch: one workgroup reads them once and holds them in registers, a wave up to four slots of 1024
// elements, sixteen a lane.  Four tensors of 16 K elements in all take 5.0 us as a graph and some 14.5 as a call, of 52 K 7.8 and
// 14.8; two launches 8.8 and 18.  From some 64 K on the one CU is slower than two launches are long (96 K: 12.3 us).
constexpr int kWaveSlots = 4, kSlots = 16 * kWaveSlots, kSlot = 1024;
struct SmallArgs {
    Tagged in[kSlots], out[kSlots];       // a slot's first element
    int n[kSlots];                        // and its elements, none behind the last slot
    int write;
    float max_norm;
    float* norm;
};
static_assert(sizeof(SmallArgs) <= 4096, "kernel arguments");
typedef int i32x2u __attribute__((ext_vector_type(2), aligned(2)));

// four elements as they lie in memory, so that all slots' loads are on their way before the first is looked at
__device__ __forceinline__ i32x4 load4_bits(const Tagged& t, int at, int n) {
    i32x4 r = {0, 0, 0, 0};
    if (t.bf16()) {
        const short* p = t.ptr<const short>() + at;
        if (n >= 4) {
            const i32x2u v = *(const i32x2u*)p;
            r[0] = v[0];
            r[1] = v[1];
        } else {
            if (n > 0) r[0] = (unsigned short)p[0];
            if (n > 1) r[0] |= p[1] << 16;
            if (n > 2) r[1] = (unsigned short)p[2];
        }
    } else {
        const f32x4 v = load4(t.ptr<const float>() + at, n);
        r = __builtin_bit_cast(i32x4, v);
    }
    return r;
}
__device__ __forceinline__ f32x4 widen4(const i32x4& r, bool bf16) {
    const f32x4 f = __builtin_bit_cast(f32x4, r);
    const i32x4 b = {r[0] << 16, r[0] & (int)0xffff0000, r[1] << 16, r[1] & (int)0xffff0000};
    const f32x4 w = __builtin_bit_cast(f32x4, b);
    return bf16 ? w : f;
}

template <bool INF>
__global__ __launch_bounds__(1024) void grad_clip_small_kernel(const SmallArgs a) {
    __shared__ double lds[16];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), at = (threadIdx.x & 63) * 4;
    Tagged in[kWaveSlots], out[kWaveSlots];
    int n[kWaveSlots];
#pragma unroll
    for (int i = 0; i < kWaveSlots; ++i) {
        in[i] = a.in[i * 16 + wave];
        out[i] = a.out[i * 16 + wave];
        n[i] = a.n[i * 16 + wave];
    }
    i32x4 raw[kWaveSlots][4];
#pragma unroll
    for (int i = 0; i < kWaveSlots; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            raw[i][u] = i32x4{0, 0, 0, 0};
            if (u * 256 < n[i]) raw[i][u] = load4_bits(in[i], at < n[i] - u * 256 ? u * 256 + at : 0, n[i] - u * 256 - at);
        }
    double v = 0.0;
#pragma unroll
    for (int i = 0; i < kWaveSlots; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (u * 256 >= n[i]) continue;
            const f32x4 g = widen4(raw[i][u], in[i].bf16());
#pragma unroll
            for (int e = 0; e < 4; ++e) add_square(g[e], INF, v);
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = combine(v, __shfl_xor(v, o, 64), INF);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) v = combine(v, lds[i], INF);
    const float norm = (float)(INF ? v : sqrt(v));
    if (threadIdx.x == 0) *a.norm = norm;
    if (!a.write) return;
    const float c = factor_of(norm, a.max_norm);
#pragma unroll
    for (int i = 0; i < kWaveSlots; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int left = n[i] - u * 256 - at;
            if (left <= 0 || (c == 1.0f && in[i].bits == out[i].bits)) continue;
            f32x4 g = widen4(raw[i][u], in[i].bf16());
#pragma unroll
            for (int e = 0; e < 4; ++e) g[e] *= c;
            if (out[i].bf16()) store4(out[i].ptr<short>() + u * 256 + at, left, g);
            else store4(out[i].ptr<float>() + u * 256 + at, left, g);
        }
}

// the norm alone: one workgroup over the partials
__global__ __launch_bounds__(256) void grad_norm_finish_kernel(const double* part, int parts, int inf_norm, float* norm) {
    __shared__ double lds[4];
    double v = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) v = combine(v, part[i], inf_norm);
    v = block_combine(v, inf_norm, lds);
    if (threadIdx.x == 0) *norm = (float)(inf_norm ? v : sqrt(v));
}

static_assert(kTensors * (kMostElements / kChunk + 1) < 0x7fffffffLL, "chunks of a launch");
inline int launch_parts(long long chunks) { return (int)(chunks < kClipBlocks ? chunks : kClipBlocks); }

// an output may be its own input, in place and of the same type; any other overlap of an output would race
bool overlaps(int count, const void* const* in, void* const* out, const int64_t* numel, const int32_t* in_type,
              const int32_t* out_type) {
    std::vector<std::pair<uintptr_t, uintptr_t>> outs, ins;
    for (int i = 0; i < count; ++i) {
        if (!numel[i]) continue;
        const uintptr_t o = (uintptr_t)out[i], p = (uintptr_t)in[i];
        outs.push_back({o, o + numel[i] * (out_type[i] ? 2 : 4)});
        if (p != o) ins.push_back({p, p + numel[i] * (in_type[i] ? 2 : 4)});
        else if (in_type[i] != out_type[i]) return true;
    }
    std::sort(outs.begin(), outs.end());
    for (size_t i = 1; i < outs.size(); ++i)
        if (outs[i].first < outs[i - 1].second) return true;
    for (const auto& q : ins) {          // outs are disjoint and sorted: only the last that begins before q's end can reach it
        auto it = std::lower_bound(outs.begin(), outs.end(), std::make_pair(q.second, (uintptr_t)0));
        if (it != outs.begin() && (it - 1)->second > q.first) return true;
    }
    return false;
}

}  // namespace asl_detail
using namespace asl_detail;

extern "C" int64_t asl_grad_clip_workspace(int count, const int64_t* numel) {
    if (count < 0 || (count && !numel)) return ASL_EINVAL;
    long long parts = 0, chunks = 0;
    for (int i = 0; i < count; ++i) {
        if (numel[i] < 0) return ASL_EINVAL;
        if (numel[i] > kMostElements) return ASL_ETOOBIG;
        chunks += (numel[i] + kChunk - 1) / kChunk;
        if (i % kTensors == kTensors - 1 || i == count - 1) {
            parts += launch_parts(chunks);
            chunks = 0;
        }
    }
    return parts * (int64_t)sizeof(double);
}

extern "C" int asl_grad_clip(int count, const void* const* grads, const int64_t* numel, const int32_t* in_type,
                             void* const* out, const int32_t* out_type, float max_norm, int inf_norm, float* norm,
                             double* workspace, asl_stream_t stream) {
    if (count < 0 || !norm || ((uintptr_t)norm & 3) || ((uintptr_t)workspace & 7)) return ASL_EINVAL;
    if (count && (!grads || !numel || !in_type)) return ASL_EINVAL;
    if (out && (!out_type || !(max_norm >= 0.f))) return ASL_EINVAL;
    const int64_t need = asl_grad_clip_workspace(count, numel);
    if (need < 0) return (int)need;
    if (need && !workspace) return ASL_EINVAL;
    for (int i = 0; i < count; ++i) {
        if (in_type[i] < 0 || in_type[i] > 1 || (out && (out_type[i] < 0 || out_type[i] > 1))) return ASL_EINVAL;
        if (!numel[i]) continue;
        if (!grads[i] || ((uintptr_t)grads[i] & (in_type[i] ? 1 : 3))) return ASL_EINVAL;
        if (out && (!out[i] || ((uintptr_t)out[i] & (out_type[i] ? 1 : 3)))) return ASL_EINVAL;
    }
    if (out && count) {
        try {
            if (overlaps(count, grads, out, numel, in_type, out_type)) return ASL_EINVAL;
        } catch (const std::bad_alloc&) {
            return ASL_ETOOBIG;
        }
    }
    hipStream_t s = (hipStream_t)stream;
    const auto tagged = [](const void* p, int type) { return Tagged{(unsigned long long)(uintptr_t)p | (unsigned long long)type}; };
    SmallArgs small;
    int slots = 0;
    for (int i = 0; i < count && slots <= kSlots; ++i)
        for (int64_t at = 0; at < numel[i] && slots <= kSlots; at += kSlot, ++slots) {
            if (slots == kSlots) continue;                 // one more than there is room for
            small.in[slots] = tagged((const char*)grads[i] + at * (in_type[i] ? 2 : 4), in_type[i]);
            small.out[slots] = out ? tagged((const char*)out[i] + at * (out_type[i] ? 2 : 4), out_type[i]) : Tagged{0};
            small.n[slots] = (int)(numel[i] - at < kSlot ? numel[i] - at : kSlot);
        }
    if (slots <= kSlots) {
        for (int i = slots; i < kSlots; ++i) small.in[i] = small.out[i] = Tagged{0}, small.n[i] = 0;
        small.write = out != nullptr; small.max_norm = max_norm; small.norm = norm;
        if (inf_norm) hipLaunchKernelGGL((grad_clip_small_kernel<true>), dim3(1), dim3(1024), 0, s, small);
        else hipLaunchKernelGGL((grad_clip_small_kernel<false>), dim3(1), dim3(1024), 0, s, small);
        return (int)hipGetLastError();
    }
    const int parts = (int)(need / (int64_t)sizeof(double));
    const auto fill = [&](ClipArgs& a, int t0) {
        a.tensors = count - t0 < kTensors ? count - t0 : kTensors;
        a.first[0] = 0;
        for (int i = 0; i < a.tensors; ++i) {
            a.in[i] = tagged(grads[t0 + i], in_type[t0 + i]);
            a.out[i] = out ? tagged(out[t0 + i], out_type[t0 + i]) : Tagged{0};
            a.n[i] = numel[t0 + i];
            a.first[i + 1] = a.first[i] + (int)((a.n[i] + kChunk - 1) / kChunk);
        }
        return launch_parts(a.first[a.tensors]);
    };
    ClipArgs a;
    a.part = workspace; a.norm = norm; a.max_norm = max_norm; a.parts = parts; a.inf_norm = inf_norm ? 1 : 0;
    a.part0 = 0;
    for (int t0 = 0; t0 < count; t0 += kTensors) {
        const int blocks = fill(a, t0);
        if (!blocks) continue;
        hipLaunchKernelGGL(grad_norm_kernel, dim3((unsigned)blocks), dim3(256), 0, s, a);
        a.part0 += blocks;
    }
    if (!out) {
        hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(256), 0, s, workspace, parts, inf_norm ? 1 : 0, norm);
        return (int)hipGetLastError();
    }
    a.write_norm = 1;
    // the last launch's tensors first: they are what the cache still holds
    for (int t0 = (count - 1) / kTensors * kTensors; t0 >= 0; t0 -= kTensors) {
        const int blocks = fill(a, t0);
        if (!blocks) continue;
        hipLaunchKernelGGL(grad_scale_kernel, dim3((unsigned)blocks), dim3(256), 0, s, a);
        a.write_norm = 0;
    }
    return (int)hipGetLastError();
}

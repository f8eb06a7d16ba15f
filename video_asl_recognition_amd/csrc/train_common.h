// Device helpers shared by the training operators: eight consecutive elements of a fp32 or bf16 row as fp32 registers.
#pragma once
#include <type_traits>

#include "common.h"

namespace asl_detail {

// Rows of a tensor need only their element's own alignment (odd widths, sliced tensors): the vector types below say so and
// the compiler still issues 16-byte accesses, which gfx950 executes at any alignment.
typedef short bf16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef short bf16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

struct F8 {
    float v[8];
};

__device__ __forceinline__ F8 load8_full(const float* p) {
    const f32x4u a = *(const f32x4u*)p, b = *(const f32x4u*)(p + 4);
    return {{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
}
__device__ __forceinline__ F8 load8_full(const short* p) {
    const bf16x8u a = *(const bf16x8u*)p;
    F8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = bf16_to_f32(a[e]);
    return r;
}
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const short* p) { return bf16_to_f32(*p); }

// elements p[0 .. n) of a row's rest; the places behind its end read as nought and touch no memory
template <typename T>
__device__ __forceinline__ F8 load8(const T* p, int n) {
    if (n >= 8) return load8_full(p);
    F8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = e < n ? load1(p + e) : 0.f;
    return r;
}

__device__ __forceinline__ void store8_full(float* p, const F8& r) {
    *(f32x4u*)p = f32x4u{r.v[0], r.v[1], r.v[2], r.v[3]};
    *(f32x4u*)(p + 4) = f32x4u{r.v[4], r.v[5], r.v[6], r.v[7]};
}
__device__ __forceinline__ void store8_full(short* p, const F8& r) {
    bf16x8u a;
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = f32_to_bf16(r.v[e]);
    *(bf16x8u*)p = a;
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(short* p, float v) { *p = f32_to_bf16(v); }

template <typename T>
__device__ __forceinline__ void store8(T* p, int n, const F8& r) {
    if (n >= 8) {
        store8_full(p, r);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n) store1(p + e, r.v[e]);
}

// The same in two steps, for loads that are issued well ahead of their use: as they lie in memory, then as fp32.
struct Raw8F {
    f32x4 a, b;
};
__device__ __forceinline__ F8 widen(const Raw8F& r) { return {{r.a[0], r.a[1], r.a[2], r.a[3], r.b[0], r.b[1], r.b[2], r.b[3]}}; }
__device__ __forceinline__ F8 widen(const bf16x8& r) {
    F8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o.v[e] = bf16_to_f32(r[e]);
    return o;
}
__device__ __forceinline__ Raw8F load8_raw(const float* p, int n) {
    Raw8F r = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    if (n >= 8) {
        r.a = *(const f32x4u*)p;
        r.b = *(const f32x4u*)(p + 4);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (e < n) r.a[e] = p[e];
            if (e + 4 < n) r.b[e] = p[e + 4];
        }
    }
    return r;
}
__device__ __forceinline__ bf16x8 load8_raw(const short* p, int n) {
    bf16x8 r = {0, 0, 0, 0, 0, 0, 0, 0};
    if (n >= 8) {
        r = *(const bf16x8u*)p;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) r[e] = p[e];
    }
    return r;
}
template <typename T>
struct RawOf;
template <>
struct RawOf<float> {
    using type = Raw8F;
};
template <>
struct RawOf<short> {
    using type = bf16x8;
};

// Sum over each 16 lanes (or 8), then over the wave, the same in every lane: lane exchanges within the vector unit (data-parallel
// primitives and the row swaps of gfx950), where a shuffle goes through the LDS.
template <int LANES = 16>
__device__ __forceinline__ float row16_sum(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
    const auto with = [](float x, auto ctrl) {
        return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    v = with(v, std::integral_constant<int, 0xb1>{});        // lane ^ 1
    v = with(v, std::integral_constant<int, 0x4e>{});        // lane ^ 2
    v = with(v, std::integral_constant<int, 0x141>{});       // the other four of eight (mirrored)
    if constexpr (LANES == 16) v = with(v, std::integral_constant<int, 0x140>{});       // the other eight of sixteen (mirrored)
#endif
    return v;
}
template <int LANES = 16>
__device__ __forceinline__ float row16_max(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
    const auto with = [](float x, auto ctrl) {
        const int i = __builtin_bit_cast(int, x);
        return fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, decltype(ctrl)::value, 0xf, 0xf, true)));
    };
    v = with(v, std::integral_constant<int, 0xb1>{});
    v = with(v, std::integral_constant<int, 0x4e>{});
    v = with(v, std::integral_constant<int, 0x141>{});
    if constexpr (LANES == 16) v = with(v, std::integral_constant<int, 0x140>{});
#endif
    return v;
}
__device__ __forceinline__ float wave64_sum(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
    v = row16_sum(v);
    // the swap of a register's rows with its own copy's (elements taken out before the cast: a bit cast of an element reads
    // the vector's first)
    int i = __builtin_bit_cast(int, v);
    const auto a = __builtin_amdgcn_permlane16_swap(i, i, false, false);
    const unsigned a0 = a[0], a1 = a[1];
    v = __builtin_bit_cast(float, a0) + __builtin_bit_cast(float, a1);
    i = __builtin_bit_cast(int, v);
    const auto b = __builtin_amdgcn_permlane32_swap(i, i, false, false);
    const unsigned b0 = b[0], b1 = b[1];
    v = __builtin_bit_cast(float, b0) + __builtin_bit_cast(float, b1);
#endif
    return v;
}

// four elements, and fewer at a row's end
__device__ __forceinline__ f32x4 load4(const float* p, int n) {
    if (n >= 4) return *(const f32x4u*)p;
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < n) r[e] = p[e];
    return r;
}
__device__ __forceinline__ f32x4 load4(const short* p, int n) {
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
    if (n >= 4) {
        const bf16x4u q = *(const bf16x4u*)p;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = bf16_to_f32(q[e]);
        return r;
    }
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < n) r[e] = bf16_to_f32(p[e]);
    return r;
}
__device__ __forceinline__ void store4(float* p, int n, f32x4 v) {
    if (n >= 4) {
        *(f32x4u*)p = v;
        return;
    }
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < n) p[e] = v[e];
}
__device__ __forceinline__ void store4(short* p, int n, f32x4 v) {
    bf16x4u o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = f32_to_bf16(v[e]);
    if (n >= 4) {
        *(bf16x4u*)p = o;
        return;
    }
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < n) p[e] = o[e];
}
// the same from a tensor whose type is only known at run time (a launch-uniform branch)
__device__ __forceinline__ F8 load8_any(const void* base, int bf16, long long at, int n) {
    return bf16 ? load8((const short*)base + at, n) : load8((const float*)base + at, n);
}

}  // namespace asl_detail

// Device helpers shared by the training operators: eight consecutive elements of a fp32 or bf16 row as fp32 registers.
#pragma once
#include "common.h"

namespace asl_detail {

// Rows of a tensor need only their element's own alignment (odd widths, sliced tensors): the vector types below say so and
// the compiler still issues 16-byte accesses, which gfx950 executes at any alignment.
typedef short bf16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
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

// the same from a tensor whose type is only known at run time (a launch-uniform branch)
__device__ __forceinline__ F8 load8_any(const void* base, int bf16, long long at, int n) {
    return bf16 ? load8((const short*)base + at, n) : load8((const float*)base + at, n);
}

}  // namespace asl_detail

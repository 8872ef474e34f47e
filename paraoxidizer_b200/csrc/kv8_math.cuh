// kv8_math.cuh -- device arithmetic that both attention kernels over the 8-bit cache use.
#pragma once

#include <type_traits>

#include "kv8.cuh"

namespace pox {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }

// Power of two that brings a row whose largest magnitude is m to [2^13, 2^14): f16 then holds bf16 values
// exactly and an f32 value's two terms to 22 bits; values below 2^-27 m lose bits, which are 2^-38 m.
__device__ __forceinline__ float row_factor(float m, float& inverse) {
    int e = (int)((__float_as_uint(m) >> 23) & 255) - 127;
    e = m > 0.f && m < INFINITY ? max(e, -100) : 13;
    inverse = __uint_as_float((uint32_t)(127 + e - 13) << 23);
    return __uint_as_float((uint32_t)(127 + 13 - e) << 23);
}

// Two f32 operations in one instruction, each rounded as by itself.
__device__ __forceinline__ uint64_t pair2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float2 both(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}

// Two values rounded to the rows' type, as they lie.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
// Element i of 16 bytes of a row.
template <typename T>
__device__ __forceinline__ float elem16(const uint4& v, int i) {
    const uint32_t w = sizeof(T) == 4 ? (i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w)
                                      : (i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w);
    if constexpr (sizeof(T) == 4) return __uint_as_float(w);
    else if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        return i & 1 ? f.y : f.x;
    } else return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
}

// Four elements of a row as they lie.
template <typename T>
struct __align__(4 * sizeof(T)) Raw4 {
    T v[4];
    template <bool VEC>
    __device__ __forceinline__ void load(const T* x) {
        if constexpr (!VEC) {
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = x[i];
        } else if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(x);
        } else {
            *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(x);
        }
    }
};

template <typename T>
__device__ __forceinline__ void load4(const T* x, int vec, float (&v)[4]) {
    if (vec) {
        T t[4];
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(x);
        else *reinterpret_cast<uint2*>(t) = *reinterpret_cast<const uint2*>(x);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = to_f32(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = to_f32(x[i]);
    }
}

template <typename T>
__device__ __forceinline__ void store4(T* x, int vec, float4 v) {
    if (vec) {
        T t[4] = {from_f32<T>(v.x), from_f32<T>(v.y), from_f32<T>(v.z), from_f32<T>(v.w)};
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(t);
        else *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(t);
    } else {
        x[0] = from_f32<T>(v.x), x[1] = from_f32<T>(v.y), x[2] = from_f32<T>(v.z), x[3] = from_f32<T>(v.w);
    }
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

}  // namespace pox

// Element types of the row operators: conversion, vectors of elements at one access, and the host's checks of what a
// tensor of rows may overlap.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "pxe_common.cuh"

namespace pxe {

using bf16 = __nv_bfloat16;
using f16 = __half;

constexpr float kE4m3Max = 448.0f;
constexpr float kScaleMin = FLT_MIN;       // 1 / scale stays finite

inline bool valid_dtype(int t) { return t == PXE_F32 || t == PXE_BF16 || t == PXE_F16; }
inline int dtype_bytes(int t) { return t == PXE_F32 ? 4 : 2; }

// ---------------------------------------------------------------- N elements as one access
template <int BYTES> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<2> { using type = uint16_t; };
template <> struct RawOf<1> { using type = uint8_t; };
template <typename T, int N> using Raw = typename RawOf<sizeof(T) * N>::type;

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<bf16>(bf16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<f16>(f16 v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ f16 from_f32<f16>(float v) { return __float2half_rn(v); }

// the two elements of a word
template <typename T> __device__ __forceinline__ void split(uint32_t w, float& x, float& y);
template <> __device__ __forceinline__ void split<bf16>(uint32_t w, float& x, float& y)
{
    x = __uint_as_float(w << 16);                          // a bf16 is the upper half of its float
    y = __uint_as_float(w & 0xffff0000u);
}
template <> __device__ __forceinline__ void split<f16>(uint32_t w, float& x, float& y)
{
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    x = f.x;
    y = f.y;
}

template <typename T, int N>
__device__ __forceinline__ void unpack(const Raw<T, N>& raw, float (&f)[N])
{
    if constexpr (sizeof(T) == 2 && N >= 2) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) split<T>(w[i], f[2 * i], f[2 * i + 1]);
    } else {
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = to_f32<T>(e[i]);
    }
}
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> pack(const float (&f)[N])
{
    Raw<T, N> raw;
    if constexpr (sizeof(T) == 2 && N >= 2) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&raw);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            if constexpr (sizeof(T) == 2 && __is_same(T, bf16)) {
                const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&p);
            } else {
                const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&p);
            }
        }
    } else {
        T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = from_f32<T>(f[i]);
    }
    return raw;
}

// N values (already divided by their scale) to e4m3 bytes, round to nearest even, NaN kept, beyond 448 held at 448.
template <int N>
__device__ __forceinline__ typename RawOf<N>::type pack_e4m3(const float (&f)[N])
{
    typename RawOf<N>::type raw;
    if constexpr (N >= 2) {
        uint16_t* w = reinterpret_cast<uint16_t*>(&raw);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i], f[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    } else {
        raw = __nv_cvt_float_to_fp8(f[0], __NV_SATFINITE, __NV_E4M3);
    }
    return raw;
}
template <int N>
__device__ __forceinline__ void unpack_e4m3(const typename RawOf<N>::type& raw, float (&f)[N])
{
    if constexpr (N >= 2) {
        const uint16_t* w = reinterpret_cast<const uint16_t*>(&raw);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(w[i], __NV_E4M3);     // exact: e4m3 is a subset of fp16
            const float2 p = __half22float2(__half2(h));
            f[2 * i] = p.x;
            f[2 * i + 1] = p.y;
        }
    } else {
        f[0] = __half2float(__half(__nv_cvt_fp8_to_halfraw(raw, __NV_E4M3)));
    }
}

// The scale of values up to `largest` and its reciprocal (the scale is a normal number, so that neither overflows).  Products
// in place of two divisions: a quotient is off by at most 5 units of 2^-24 of itself, so that a value as near as that to the
// border between two codes may take the one or the other; its error is half a step either way.
__device__ __forceinline__ float max_nan(float a, float b);
__device__ __forceinline__ float e4m3_scale(float largest) { return max_nan(largest * (1.0f / kE4m3Max), kScaleMin); }
__device__ __forceinline__ float e4m3_inverse(float scale) { return fast_rcp(scale); }

// max that keeps a NaN (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// ---------------------------------------------------------------- two floats an instruction
__device__ __forceinline__ unsigned long long pair(float a, float b)
{
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(unsigned long long p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c)
{
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b)
{
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b)
{
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// ---------------------------------------------------------------- host: overlap of row tensors
// `rows` rows of `bytes` bytes, `stride` bytes apart.
struct RowSpan {
    const void* p;
    long long rows, stride, bytes;
    uintptr_t lo() const { return reinterpret_cast<uintptr_t>(p); }
    uintptr_t hi() const { return lo() + (uintptr_t)((rows - 1) * stride + bytes); }
};

// True when a and b share a byte, unless they are the same tensor.  Tensors of one stride may interleave without
// touching (column slices of one buffer); tensors of different strides whose ranges meet count as overlapping.
inline bool rows_conflict(const RowSpan& a, const RowSpan& b)
{
    if (!a.p || !b.p || a.rows <= 0 || b.rows <= 0) return false;
    const bool one = a.rows == 1 && b.rows == 1;
    if (a.p == b.p && a.bytes == b.bytes && (a.stride == b.stride || one)) return false;
    if (a.hi() <= b.lo() || b.hi() <= a.lo()) return false;
    if (a.stride != b.stride || one) return true;
    const uintptr_t s = (uintptr_t)a.stride;
    const uintptr_t d = a.lo() <= b.lo() ? (b.lo() - a.lo()) % s : (s - (a.lo() - b.lo()) % s) % s;     // where b's rows begin within a's
    return d < (uintptr_t)a.bytes || s - d < (uintptr_t)b.bytes;
}

}  // namespace pxe

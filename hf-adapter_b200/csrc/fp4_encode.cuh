// Codes and scales of 16 elements at a time: what the quantiser (fp4.cu) and the product of few tokens (fp4_umma.cu) have in common.
#pragma once

#include <cuda_fp8.h>

#include "fp4.cuh"

namespace rwkv7 {
using namespace fp4;

// eight codes, element 0 in the lowest nibble
__device__ __forceinline__ uint32_t pack8(const float (&v)[8]) {
    uint32_t d;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(d) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return d;
}

__device__ __forceinline__ float e4m3_value(uint32_t byte) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}
// 16 elements as they lie in memory
template <typename T> struct Piece {
    uint4 w[sizeof(T)];  // (sizeof(T) = 16 elements x sizeof(T) / 16)
};
template <typename T> __device__ __forceinline__ Piece<T> load_piece(const T* p) {
    Piece<T> o;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) o.w[i] = reinterpret_cast<const uint4*>(p)[i];
    return o;
}
template <typename T> __device__ __forceinline__ void widen(const Piece<T>& p, float (&v)[16]) {
    const T* e = reinterpret_cast<const T*>(p.w);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = to_f<T>(e[i]);
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
template <typename T> struct Two;
template <> struct Two<__half> { typedef __half2 type; };
template <> struct Two<__nv_bfloat16> { typedef __nv_bfloat162 type; };
// the largest magnitude of a piece, infinite or NaN if an element is
template <typename T> __device__ __forceinline__ float piece_amax(const Piece<T>& p) {
    if constexpr (sizeof(T) == 4) {
        const float* e = reinterpret_cast<const float*>(p.w);
        float m = fabsf(e[0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) m = max_nan(m, fabsf(e[i]));
        return m;
    } else if constexpr (sizeof(T) == 2) {
        typedef typename Two<T>::type T2;
        const T2* e = reinterpret_cast<const T2*>(p.w);
        T2 m = __habs2(e[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(e[i]));
        return max_nan(to_f<T>(m.x), to_f<T>(m.y));
    }
}
// the same over the finite elements alone; m: piece_amax(p)
template <typename T> __device__ __forceinline__ float finite_amax(const Piece<T>& p, float m) {
    if (!(m < INFINITY)) {
        float v[16];
        widen(p, v);
        m = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (fabsf(v[i]) < INFINITY) m = fmaxf(m, fabsf(v[i]));
    }
    return m;
}

// Codes and the block's scale byte of one piece; m: piece_amax(piece), ge: g's exponent byte (nvfp4).  Whole warps.
template <typename T, int FORMAT>
__device__ __forceinline__ uint32_t encode_piece(const Piece<T>& piece, float m, int ge, uint2& codes) {
    float v[16];
    widen(piece, v);
    uint32_t byte;
    if constexpr (FORMAT == MX) {
        m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
        const bool finite = m < INFINITY;
        byte = finite ? max((__float_as_int(m) >> 23) - 2, 0) : 255;
        const float mult = __int_as_float(finite ? (254 - byte) << 23 : 0);  // 2^(127 - byte); byte <= 252
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] *= mult;
    } else {
        const float inv_g = __int_as_float((254 - ge) << 23);
        byte = __nv_cvt_float_to_fp8(m * inv_g * (1.0f / 6.0f), __NV_SATFINITE, __NV_E4M3);
        float s = e4m3_value(byte), inv = s > 0.0f ? __frcp_rn(s) : 0.0f;
        if (!(m < INFINITY)) byte = 0x7f;
        if (ge >= 32 && ge <= 224) {  // the powers of two in one factor (exact: nothing leaves the range)
            inv *= inv_g, s *= __int_as_float(ge << 23);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] *= inv_g;
        }
        if constexpr (sizeof(T) == 2) {
            // x / s misses a tie by 2^-12 of it at least, or is one, and is at most 9: rounded to steps of 2^-17 it is on the same side, or on it
            // (8192 x 4096 18.8 us with this and one amax a piece, 20.9 with the quotient's correction step and two)
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = fmaf(v[i], inv, 96.0f) - 96.0f;
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float q = v[i] * inv;
                v[i] = fmaf(fmaf(-q, s, v[i]), inv, q);
            }
        }
    }
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = v[i], hi[i] = v[8 + i];
    codes = make_uint2(pack8(lo), pack8(hi));
    return byte;
}
}  // namespace rwkv7

// fp8_device.h — the 8-bit format on the device: scales of blocks, rounding and widening.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace siren {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float finite_abs(float x) {
    const float a = __builtin_fabsf(x);
    return a < INFINITY ? a : 0.f;
}

// the exponent byte of a block whose largest finite magnitude is amax: 448 = 1.75 * 2^8, 57344 = 1.75 * 2^15
template <bool E5M2>
__device__ __forceinline__ int exponent_byte(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int e = (int)(b >> 23) - (E5M2 ? 15 : 8) + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return e < 1 ? 1 : e;
}
__device__ __forceinline__ float inverse_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

// four values to four codes, to the nearest, ties to even; NaN and (e4m3) infinities become NaN
template <bool E5M2>
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    if constexpr (E5M2) {
        const int lo = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(c, d, lo, true);
    } else {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
    }
}

// two codes to bf16, times scale (a power of two: exact)
template <bool E5M2, int HI>
__device__ __forceinline__ bf16x2 widen2(uint32_t w, float scale) {
    if constexpr (E5M2)
        return __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, scale, HI);
    else
        return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI);
}
template <bool E5M2>
__device__ __forceinline__ bf16x8 widen8(uint32_t w0, uint32_t w1, float scale) {
    const bf16x2 p0 = widen2<E5M2, 0>(w0, scale), p1 = widen2<E5M2, 1>(w0, scale);
    const bf16x2 p2 = widen2<E5M2, 0>(w1, scale), p3 = widen2<E5M2, 1>(w1, scale);
    return bf16x8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

// src[0 .. 3] as fp32, of which valid exist (the rest zero). vec: src is aligned for one access
template <typename T>
__device__ __forceinline__ void load_quad(const T* src, int valid, bool vec, float (&v)[4]) {
    if (vec && valid >= 4) {
        typedef T T4 __attribute__((ext_vector_type(4)));
        const T4 h = *(const T4*)src;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (float)h[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = k < valid ? (float)src[k] : 0.f;
    }
}

// the maximum over the 32 lanes of a half wave
__device__ __forceinline__ float half_wave_max(float m) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    return m;
}

}  // namespace siren

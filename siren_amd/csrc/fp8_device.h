// fp8_device.h — the 8-bit format on the device: scales of blocks, rounding and widening.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace siren {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
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
__device__ __forceinline__ float scale_of(int byte) { return __uint_as_float((uint32_t)byte << 23); }

// four values over scale to four codes, to the nearest, ties to even; NaN and (e4m3) infinities become NaN. The scale is a
// power of two, so the division inside the instruction is exact.
template <bool E5M2>
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d, float scale) {
    typedef short i16x2 __attribute__((ext_vector_type(2)));
    i16x2 r = {0, 0};
    if constexpr (E5M2) {
        r = __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(r, a, b, scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(r, c, d, scale, true);
    } else {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, scale, false);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true);
    }
    return __builtin_bit_cast(uint32_t, r);
}

// two codes to bf16, times scale (a power of two: exact down to bf16's smallest number, 2^-133, and below 2^128)
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

// four elements that lie as they may: one access at the element's own alignment (the card splits what crosses a line), so
// that odd widths and views read and write as wide as others
template <typename T>
struct Quad {
    typedef T Type __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};

// src[0 .. 3] as fp32, of which valid exist (the rest zero)
template <typename T>
__device__ __forceinline__ void load_quad(const T* src, int valid, float (&v)[4]) {
    if (valid >= 4) {
        const typename Quad<T>::Type h = *(const typename Quad<T>::Type*)src;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (float)h[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = k < valid ? (float)src[k] : 0.f;
    }
}

// the maximum over the 16 lanes of a row of the wave, and over the 32 of its half, by data-parallel moves (a shuffle
// through LDS costs an instruction of its own and the LDS' time for each step)
template <int CTRL>
__device__ __forceinline__ float dpp_max(float m) {
    return fmaxf(m, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(m), CTRL, 0xF, 0xF, true)));
}
__device__ __forceinline__ float row16_max(float m) {
    m = dpp_max<0xB1>(m);   // lanes 1 apart
    m = dpp_max<0x4E>(m);   // 2 apart
    m = dpp_max<0x124>(m);  // rotated by 4
    return dpp_max<0x128>(m);  // by 8
}
__device__ __forceinline__ float half_wave_max(float m) {
    m = row16_max(m);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// the largest finite magnitude of a block, one quad a lane of half a wave or two a lane of a quarter: where the plain maximum
// of any in the wave is not finite (fmaxf drops a NaN beside a number), the quads are looked through again
template <int QUADS>
__device__ __forceinline__ float block_amax(const float (&v)[QUADS][4]) {
    float m = 0.f;
#pragma unroll
    for (int d = 0; d < QUADS; ++d)
        m = fmaxf(m, fmaxf(fmaxf(__builtin_fabsf(v[d][0]), __builtin_fabsf(v[d][1])),
                           fmaxf(__builtin_fabsf(v[d][2]), __builtin_fabsf(v[d][3]))));
    m = QUADS == 1 ? half_wave_max(m) : row16_max(m);
    if (__builtin_expect(__any(!(m < INFINITY)), 0)) {
        m = 0.f;
#pragma unroll
        for (int d = 0; d < QUADS; ++d)
            m = fmaxf(m, fmaxf(fmaxf(finite_abs(v[d][0]), finite_abs(v[d][1])), fmaxf(finite_abs(v[d][2]), finite_abs(v[d][3]))));
        m = QUADS == 1 ? half_wave_max(m) : row16_max(m);
    }
    return m;
}
__device__ __forceinline__ float half_wave_amax(float a, float b, float c, float d) {
    const float v[1][4] = {{a, b, c, d}};
    return block_amax<1>(v);
}

}  // namespace siren

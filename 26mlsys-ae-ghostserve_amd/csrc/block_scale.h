// block_scale.h -- codes and scales of a cache in 8 or 4 bits: 32 neighbouring
// values of a head share a power of two.
#pragma once

#include "lm_types.h"

namespace kvec {

// A scale byte as the 32-bit float that the conversions take: they read its exponent
// bits only, so byte 0 is 2^-127 there (not 0) and byte 255 makes NaN.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// The last magnitude of a type T that no rounding to `BITS` bits takes past the type's
// largest: 1.111b (e4m3) or 1.1b (e2m1) in its top power of two.
template <class T, int BITS>
__device__ __forceinline__ float last_of() {
    const uint32_t e = __is_same(T, _Float16) ? 127 + 15 : 127 + 127;
    return __uint_as_float(e << 23 | (BITS == 8 ? 0x700000u : 0x400000u));
}

// The scale byte of a block by its largest magnitude (its bits; infinity and NaN last):
// the smallest 2^e, e >= -127, with a <= 1.75 * 2^8 * 2^e (e4m3) or 1.5 * 2^2 * 2^e (e2m1).
template <class T, int BITS>
__device__ __forceinline__ uint32_t scale_byte(uint32_t a) {
    const bool finite = a < 0x7F800000u;
    a = min(a, __float_as_uint(last_of<T, BITS>()));
    const int e = int(a >> 23) - (BITS == 8 ? 8 : 2) + int((a & 0x7FFFFFu) > (BITS == 8 ? 0x600000u : 0x400000u));
    return finite ? uint32_t(max(e, 0)) : 255u;
}

// 16 values to their codes; `byte`: their block's scale, under 254.  The quotient
// by a power of two is exact (or under the smallest code), so codes are rounded once,
// by the conversion, to nearest even.
template <class T, int BITS>
__device__ __forceinline__ void codes16(const float* y, uint32_t byte, uint32_t* out) {
    const float inv = __uint_as_float((254u - min(byte, 253u)) << 23), most = last_of<T, BITS>();
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __builtin_amdgcn_fmed3f(y[i], -most, most) * inv;
    if constexpr (BITS == 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
            out[i] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], r, true));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, x[8 * i], x[8 * i + 1], 1.0f, 0);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[8 * i + 2], x[8 * i + 3], 1.0f, 1);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[8 * i + 4], x[8 * i + 5], 1.0f, 2);
            out[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[8 * i + 6], x[8 * i + 7], 1.0f, 3);
        }
    }
}

// Eight values of the codes in x (e4m3: 8 bytes; e2m1: 4) and their scale: 16-bit types
// rounded once (exact but past fp16's range and under the smallest normal numbers).
template <int BITS>
__device__ __forceinline__ u32x4 widen8(u32x2 x, float scale, __bf16*) {
    if constexpr (BITS == 8)
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x.x, scale, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x.x, scale, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x.y, scale, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x.y, scale, true))};
    else
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x.x, scale, 0)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x.x, scale, 1)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x.x, scale, 2)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x.x, scale, 3))};
}
template <int BITS>
__device__ __forceinline__ u32x4 widen8(u32x2 x, float scale, _Float16*) {
    if constexpr (BITS == 8)
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x.x, scale, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x.x, scale, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x.y, scale, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x.y, scale, true))};
    else
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x.x, scale, 0)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x.x, scale, 1)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x.x, scale, 2)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(x.x, scale, 3))};
}

}  // namespace kvec

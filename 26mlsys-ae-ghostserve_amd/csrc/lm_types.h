// lm_types.h -- element types of the serving-step kernels: values as they lie
// in memory (raw vectors, so that loads can be in flight before they are
// converted) and as the 32-bit numbers that everything is computed in.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "kvec_internal.h"

namespace kvec {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct Fp8 {  // one byte of e4m3
    uint8_t b;
};

constexpr float kFp8Max = 448.0f;

// Two 32-bit values to two 16-bit ones, to nearest even: one instruction each.
__device__ __forceinline__ uint32_t pack2(float a, float b, __bf16*) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, _Float16*) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}

// To e4m3, to nearest even; values past the largest become the largest, NaN stays.
__device__ __forceinline__ float fp8_clamp(float x) {
    const float y = __builtin_amdgcn_fmed3f(x, -kFp8Max, kFp8Max);
    return x != x ? x : y;
}
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_clamp(a), fp8_clamp(b), 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(fp8_clamp(c), fp8_clamp(d), r, true));
}

// W values as they lie in memory.
template <class T, int W>
struct Raw;

template <class T>
struct Raw<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T* p) { v = *as_global(p); }
    __device__ __forceinline__ void get(float* f) const { f[0] = float(v); }
};
template <>
struct Raw<float, 8> {
    u32x4 v[2];
    __device__ __forceinline__ void load(const float* p) {
        v[0] = ld16(reinterpret_cast<const uint8_t*>(p));
        v[1] = ld16(reinterpret_cast<const uint8_t*>(p) + 16);
    }
    __device__ __forceinline__ void get(float* f) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(v[i / 4][i % 4]);
    }
};
template <>
struct Raw<__bf16, 8> {
    u32x4 v;
    __device__ __forceinline__ void load(const __bf16* p) { v = ld16(reinterpret_cast<const uint8_t*>(p)); }
    __device__ __forceinline__ void get(float* f) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __builtin_bit_cast(float, v[i] << 16);
            f[2 * i + 1] = __builtin_bit_cast(float, v[i] & 0xFFFF0000u);
        }
    }
};
template <>
struct Raw<_Float16, 8> {
    u32x4 v;
    __device__ __forceinline__ void load(const _Float16* p) { v = ld16(reinterpret_cast<const uint8_t*>(p)); }
    __device__ __forceinline__ void get(float* f) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f16x2 h = __builtin_bit_cast(f16x2, uint32_t(v[i]));
            f[2 * i] = float(h[0]);
            f[2 * i + 1] = float(h[1]);
        }
    }
};

// W 32-bit values rounded into memory.
__device__ __forceinline__ void put1(float* p, float f) { *as_global(p) = f; }
__device__ __forceinline__ void put1(__bf16* p, float f) { *as_global(p) = __bf16(f); }
__device__ __forceinline__ void put1(_Float16* p, float f) { *as_global(p) = _Float16(f); }
__device__ __forceinline__ void put1(Fp8* p, float f) {
    *as_global(&p->b) = uint8_t(__builtin_amdgcn_cvt_pk_fp8_f32(fp8_clamp(f), 0.0f, 0, false));
}
__device__ __forceinline__ void put8(float* p, const float* f) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
        st16(reinterpret_cast<uint8_t*>(p) + 16 * i,
             u32x4{__builtin_bit_cast(uint32_t, f[4 * i]), __builtin_bit_cast(uint32_t, f[4 * i + 1]),
                   __builtin_bit_cast(uint32_t, f[4 * i + 2]), __builtin_bit_cast(uint32_t, f[4 * i + 3])});
}
template <class T>
__device__ __forceinline__ void put8(T* p, const float* f) {
    T* t = nullptr;
    st16(reinterpret_cast<uint8_t*>(p), u32x4{pack2(f[0], f[1], t), pack2(f[2], f[3], t), pack2(f[4], f[5], t),
                                              pack2(f[6], f[7], t)});
}
__device__ __forceinline__ void put8(Fp8* p, const float* f) {
    *as_global(reinterpret_cast<u32x2*>(p)) =
        u32x2{fp8_pack4(f[0], f[1], f[2], f[3]), fp8_pack4(f[4], f[5], f[6], f[7])};
}
template <class T, int W>
__device__ __forceinline__ void put(T* p, const float* f) {
    if constexpr (W == 8) put8(p, f);
    else put1(p, f[0]);
}

// Whether two of the n x h rows of `len` values at i * s + j * t share one.
inline bool rows_overlap(int64_t n, int64_t s, int64_t h, int64_t t, int64_t len) {
    typedef __int128 wide;
    if ((n > 1 && s < len) || (h > 1 && t < len)) return true;
    if (n <= 1 || h <= 1 || s >= wide(h - 1) * t + len || t >= wide(n - 1) * s + len) return false;
    for (int64_t j = 1; j < h; ++j) {                     // the rows on either side of 0, j
        const wide d = wide(j) * t, i = d / s;
        if (i < n && d - i * s < len) return true;
        if (i + 1 < n && (i + 1) * s - d < len) return true;
    }
    return false;
}

// HIP's limit: the threads of a launch are fewer than 2^32.
inline bool launchable(uint64_t blocks, uint32_t threads) { return blocks < (uint64_t(1) << 32) / threads; }

inline int64_t type_bytes(int dtype) {
    return dtype == KVEC_F32 ? 4 : dtype == KVEC_BF16 || dtype == KVEC_F16 ? 2 : dtype == KVEC_FP8_E4M3 ? 1 : 0;
}

}  // namespace kvec

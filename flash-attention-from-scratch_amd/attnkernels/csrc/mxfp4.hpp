// MXFP4 rows of the 4-bit KV cache, and the 16-bit types beside it.
//
// 32 channels of one token and head are a group: one scale byte s, which stands
// for 2^(s - 127) (255: the group reads NaN), and 32 four-bit codes, a sign and
// one of 0, .5, 1, 1.5, 2, 3, 4, 6.  Two channels share a byte, the even one in
// the low half; a row of D channels is D/2 code bytes and D/32 scale bytes.
//
// The scale's exponent is that of the group's largest magnitude rounded to two
// significant bits (from 7 * 2^k up to 8 * 2^k), less 2, at least -126.  So a
// code's magnitude before rounding is below 7, and the format's largest value
// (6) is off by less than 1 from what it stands for.
#pragma once

#include "wave.hpp"

namespace ak {

using bf16 = __bf16;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// What a group whose scale byte is s multiplies its codes by.
__device__ __forceinline__ float mx_scale(uint32_t s) { return __builtin_bit_cast(float, s << 23); }

// What the kernels need of an element type: fp16 or bf16.
template <class T>
struct Half;

template <>
struct Half<f16> {
    typedef f16x8 x8;
    static constexpr uint32_t kInf = 0x7c00;
    static __device__ __forceinline__ float widen(uint32_t bits) {
        return (float)__builtin_bit_cast(f16, (uint16_t)bits);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, f16x2{(f16)a, (f16)b});
    }
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
    // Codes of the two elements in x, over byte SEL of old.
    template <int SEL>
    static __device__ __forceinline__ uint32_t encode(uint32_t old, uint32_t x, float scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(f16x2, x), scale, SEL);
    }
    // The two values in byte SEL of the codes.
    template <int SEL>
    static __device__ __forceinline__ uint32_t decode(uint32_t codes, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, SEL));
    }
};

template <>
struct Half<bf16> {
    typedef bf16x8 x8;
    static constexpr uint32_t kInf = 0x7f80;
    static __device__ __forceinline__ float widen(uint32_t bits) {
        return __builtin_bit_cast(float, bits << 16);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, bf16x2{(bf16)a, (bf16)b});
    }
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
    template <int SEL>
    static __device__ __forceinline__ uint32_t encode(uint32_t old, uint32_t x, float scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(bf16x2, x), scale, SEL);
    }
    template <int SEL>
    static __device__ __forceinline__ uint32_t decode(uint32_t codes, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL));
    }
};

// The eight values of a dword of codes.
template <class T>
__device__ __forceinline__ u32x4 mx_decode8(uint32_t codes, float scale) {
    return u32x4{Half<T>::template decode<0>(codes, scale), Half<T>::template decode<1>(codes, scale),
                 Half<T>::template decode<2>(codes, scale), Half<T>::template decode<3>(codes, scale)};
}

}  // namespace ak

// Encoding of one MXFP4 block (32 values), shared by the codec and by the products that quantise an operand themselves.
// Included by device code only; everything has internal linkage.
#pragma once
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tcb_common.h"

namespace {

// One block of 32 values.
template <typename T>
struct Block32 {
    static constexpr int kWords = 32 * sizeof(T) / 4;
    uint32_t w[kWords];

    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < kWords; i += 8) tcb::ldg_stream_v8(reinterpret_cast<const uint32_t*>(p) + i, w + i);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    __device__ __forceinline__ uint32_t word(int i) const { return w[i]; }
    __device__ __forceinline__ float get(int i) const;
};
template <>
__device__ __forceinline__ float Block32<__nv_bfloat16>::get(int i) const {
    const uint32_t v = word(i >> 1);
    return __uint_as_float((i & 1) ? (v & 0xffff0000u) : (v << 16));
}
template <>
__device__ __forceinline__ float Block32<__half>::get(int i) const {
    const uint32_t v = word(i >> 1);
    return __half2float(__ushort_as_half((i & 1) ? (v >> 16) : (v & 0xffffu)));
}
template <>
__device__ __forceinline__ float Block32<float>::get(int i) const { return __uint_as_float(word(i)); }

// Exponent field (fp32) of the largest magnitude, 255 if a value is not finite.  16-bit types compare two magnitudes
// at once as integers (the order of the bit patterns is the order of the values).
template <typename T>
__device__ __forceinline__ uint32_t max_exponent(const Block32<T>& b) {
    uint32_t m = 0;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 16; ++i) m = __vmaxu2(m, b.word(i) & 0x7fff7fffu);
        m = max(m & 0xffffu, m >> 16);
        if constexpr (std::is_same<T, __half>::value) {
            if (m >= 0x7c00u) return 255u;
            return __float_as_uint(__half2float(__ushort_as_half(uint16_t(m)))) >> 23;
        } else {
            return m >> 7;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) m = max(m, b.word(i) & 0x7fffffffu);
        return m >> 23;
    }
}

__device__ __forceinline__ uint32_t float8_to_e2m1x8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// Clears what is not finite, away from the common path.
template <typename T>
__device__ __forceinline__ void clear_nonfinite(Block32<T>& b) {
#pragma unroll
    for (int i = 0; i < Block32<T>::kWords; ++i) {
        if constexpr (std::is_same<T, float>::value) {
            if ((b.w[i] & 0x7f800000u) == 0x7f800000u) b.w[i] = 0;
        } else {
            constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
            if ((b.w[i] & kExp) == kExp) b.w[i] &= 0xffff0000u;
            if ((b.w[i] & (kExp << 16)) == (kExp << 16)) b.w[i] &= 0x0000ffffu;
        }
    }
}

// Scale byte and 32 codes of one block.
template <typename T>
__device__ __forceinline__ uint32_t encode_block(Block32<T>& b, uint4& codes) {
    uint32_t e = max_exponent(b);
    if (__builtin_expect(e == 255u, 0)) {
        clear_nonfinite(b);
        e = max_exponent(b);
    }
    const uint32_t byte = e > 2u ? e - 2u : 0u;
    const float inv = __uint_as_float((254u - byte) << 23);   // 2^(127 - byte), exact product
    uint32_t o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(b.get(8 * k + i), inv);
        o[k] = float8_to_e2m1x8(v);
    }
    codes = make_uint4(o[0], o[1], o[2], o[3]);
    return byte;
}

}  // namespace

// blocks4.hpp - microscaled 4-bit blocks on the device: rounding to E2M1 and back, and a row's blocks as the matrix instructions take
// them. See blocks4.hip for the format.
#pragma once

#include "blocks.hpp"

namespace gsx_amd {

constexpr int kBlock4 = 32;        // values of a block: 16 bytes
constexpr uint32_t kNoScale = 255;  // exponent byte of a block that stands for NaN

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));

// Exponent of a block whose largest magnitude has the float bits `top` (sign cleared): 6 = 1.5 * 2^2.
__device__ inline int block4_exponent(uint32_t top) {
    if (top == 0) return 0;
    const int e = (int)(top >> 23) - 127 - 2 + ((top & 0x7fffffu) > 0x400000u ? 1 : 0);
    return max(e, kLeastExponent);
}

// Eight E2M1 values (the first one lowest) of a raw's elements [i, i + 8) / scale, a power of two: the conversions divide exactly.
template <typename T, int kElements>
__device__ inline uint32_t pack4_raw(const Raw<T, kElements>& x, int i, float scale) {
    uint32_t out = 0;
    if constexpr (sizeof(T) == 4) {
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, word_element<T>(x.w, i), word_element<T>(x.w, i + 1), scale, 0);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, word_element<T>(x.w, i + 2), word_element<T>(x.w, i + 3), scale, 1);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, word_element<T>(x.w, i + 4), word_element<T>(x.w, i + 5), scale, 2);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, word_element<T>(x.w, i + 6), word_element<T>(x.w, i + 7), scale, 3);
    } else if constexpr (__is_same(T, __bf16)) {
        const uint32_t* const w = x.w + i / 2;
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(out, __builtin_bit_cast(v2bf, w[0]), scale, 0);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(out, __builtin_bit_cast(v2bf, w[1]), scale, 1);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(out, __builtin_bit_cast(v2bf, w[2]), scale, 2);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(out, __builtin_bit_cast(v2bf, w[3]), scale, 3);
    } else {
        const uint32_t* const w = x.w + i / 2;
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(out, __builtin_bit_cast(v2h, w[0]), scale, 0);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(out, __builtin_bit_cast(v2h, w[1]), scale, 1);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(out, __builtin_bit_cast(v2h, w[2]), scale, 2);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(out, __builtin_bit_cast(v2h, w[3]), scale, 3);
    }
    return out;
}

// What an exponent byte stands for.
__device__ inline float block4_scale(uint32_t byte) {
    return __builtin_bit_cast(float, byte == 0 ? 0x00400000u : byte == kNoScale ? 0x7fc00000u : byte << 23);
}

// Block kb's 16 bytes of a row of `cols` values; zeros from `cols` on. A row's last block is there whole.
__device__ inline v4i load_block4(const uint8_t* __restrict__ row, int64_t kb, int64_t cols) {
    v4i v = *reinterpret_cast<const v4i*>(row + min(kb, (cols - 1) / kBlock4) * 16);
    const int left = (int)max(min(cols - kb * kBlock4, (int64_t)kBlock4), (int64_t)0);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const int bits = max(min(4 * (left - 8 * d), 32), 0);
        v[d] &= (int)(0xffffffffull >> (32 - bits));
    }
    return v;
}

// Exponents of blocks [4 group, 4 group + 4) of a row of `blocks`; 2^0 for those behind the last.
__device__ inline uint32_t load_exponents4(const uint8_t* __restrict__ row, int64_t group, int64_t blocks) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(row)[min(group, (blocks - 1) / 4)];
    const int left = (int)max(min(blocks - 4 * group, (int64_t)4), (int64_t)0);
    const uint32_t keep = (uint32_t)((1ull << (8 * left)) - 1);
    return (w & keep) | (0x7f7f7f7fu & ~keep);
}

// acc += b's rows times a's rows: lane l brings block l / 16 of four for row l % 16 of each operand, and the scale's byte kByte of
// its word. A lane then holds columns 4 (l / 16) .. + 4 (b's rows) of row l % 16 (a's).
template <int kByteB, int kByteA>
__device__ inline v4f multiply4(v4i b, v4i a, v4f acc, uint32_t scale_b, uint32_t scale_a) {
    const v8i vb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0}, va = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(vb, va, acc, 4, 4, kByteB, (int)scale_b, kByteA, (int)scale_a);
}

gsx_hip_status blocks4_check(const void* values, const void* exponents, int64_t rows, int64_t cols, int64_t values_stride,
                             int64_t exponents_stride);

}  // namespace gsx_amd

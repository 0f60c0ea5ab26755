// blocks.hpp - 8-bit blocks on the device: rounding to E4M3, conversion for the matrix instructions, rows and columns of a
// product's tiles. See blocks.hip for the format.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fields.hpp"

namespace gsx_amd {

constexpr int kBlock = 128;
constexpr int kLeastExponent = -100;  // the least E4M3 step is 2^-9: q * 2^e stays far above bfloat16's subnormals, which are cut

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

__device__ inline bool finite_bits(uint32_t bits) { return (bits & 0x7f800000u) != 0x7f800000u; }

// Exponent of a block whose largest finite magnitude has the float bits `top` (sign cleared): 448 = 1.75 * 2^8.
__device__ inline int block_exponent(uint32_t top) {
    if (top == 0) return 0;
    const int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, kLeastExponent);
}

// Four E4M3 bytes of x * 2^-e, for finite x. |x| <= 448 * 2^e, so none rounds past 448.
__device__ inline uint32_t pack_finite(const float* x, int e) {
    const float scale = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
    const int out = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * scale, x[1] * scale, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * scale, x[3] * scale, out, true);
}

// The same for any x: NaN (0x7f) in place of what is not finite.
__device__ inline uint32_t pack_e4m3(const float* x, int e) {
    uint32_t out = pack_finite(x, e);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (!finite_bits(__builtin_bit_cast(uint32_t, x[k]))) out |= 0x7fu << (8 * k);
    }
    return out;
}

// Four and eight elements at any element's address (the hardware takes wide accesses that are not aligned).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Quad {
    T v[4];
};
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Octet {
    T v[8];
};

// Largest finite magnitude (its bits) among a lane's eight values.
__device__ inline uint32_t largest(const float (&x)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint32_t bits = __builtin_bit_cast(uint32_t, x[k]) & 0x7fffffffu;
        if (finite_bits(bits)) top = max(top, bits);
    }
    return top;
}

struct BlockMatrix {
    const uint8_t* values;
    const uint8_t* exponents;
    int64_t values_stride, exponents_stride;
};

// 16 bytes of a row at column k; columns from `cols` on read as zero.
__device__ inline v4i load_values(const uint8_t* row, int64_t k, int64_t cols) {
    v4i v = {0, 0, 0, 0};
    if (k >= cols) return v;
    v = *reinterpret_cast<const v4i*>(row + k);
    const int64_t left = cols - k;
    if (left < 16) {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const int64_t bytes = left - 4 * d;
            if (bytes < 4) v[d] = bytes <= 0 ? 0 : v[d] & (int)((1u << (8 * bytes)) - 1u);
        }
    }
    return v;
}

// 4 TN consecutive columns from `col` on of a row of n.
template <int TN, typename O>
__device__ inline void store_columns(O* __restrict__ row, int64_t col, int64_t n, const v4f (&x)[TN]) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int64_t c = col + 4 * j;
        if (c + 4 <= n) {
            Quad<O> q;
#pragma unroll
            for (int i = 0; i < 4; ++i) q.v[i] = from_float<O>(x[j][i]);
            *reinterpret_cast<Quad<O>*>(row + c) = q;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < n) row[c + i] = from_float<O>(x[j][i]);
        }
    }
}

// Eight E4M3 values (two words) times `scale`, exactly, in bfloat16.
__device__ inline v8bf to_bf16(int lo, int hi, float scale) {
    const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)lo, scale, false);
    const v2bf b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)lo, scale, true);
    const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)hi, scale, false);
    const v2bf d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)hi, scale, true);
    return v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 2^e from the byte e + 127.
__device__ inline float block_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

typedef __attribute__((address_space(3))) void* LdsPtr;
typedef const __attribute__((address_space(1))) void* GlobalPtr;

// Row of b, within a wave's 16 TN, that index r of instruction j stands for.
template <int TN>
__device__ constexpr int column_of(int j, int r) {
    return (r / 4) * (4 * TN) + 4 * j + r % 4;
}

// Places of the chunks: a's rows are read 16 in a row, b's as column_of orders them.
__device__ inline int swizzle_a(int row) { return row & 7; }
template <int TN>
__device__ inline int swizzle_b(int row) {
    return (row & 3) | ((row / (4 * TN)) & 1) << 2;
}

constexpr int64_t kMostSummands = (int64_t)1 << 27;
bool product_sizes(int64_t m, int64_t n, int64_t k);
// out [m, n] = the sum of partial [splits][m][n] over the splits, in a fixed order.
gsx_hip_status join_products(const float* partial, int64_t m, int64_t n, int64_t splits, float* out, int64_t out_stride,
                             hipStream_t stream);
gsx_hip_status block_matrix_check(const void* values, const void* exponents, int64_t rows, int64_t cols,
                                  int64_t values_stride, int64_t exponents_stride);

inline unsigned blocks_grid(int64_t wanted) { return (unsigned)(wanted < (1 << 20) ? wanted : 1 << 20); }

}  // namespace gsx_amd

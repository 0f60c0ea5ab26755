// blocks.hpp - 8-bit blocks on the device: rounding to E4M3, conversion for the matrix instructions, rows and columns of a
// product's tiles. See blocks.hip for the format.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fields.hpp"

namespace gsx_amd {

constexpr int kBlock = 128;
constexpr int kLeastExponent = -100;  // the least E4M3 step is 2^-9: q * 2^e stays far above bfloat16's subnormals, which are cut

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

typedef short v2s __attribute__((ext_vector_type(2)));
typedef unsigned short v2u __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

// 2^e from the byte e + 127.
__device__ inline float block_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// Four E4M3 bytes of x / scale, for finite x no larger than 448 times scale (a power of two): the conversions divide exactly.
__device__ inline uint32_t pack_finite(const float* x, float scale) {
    v2s out = {0, 0};
    out = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(out, x[0], x[1], scale, false);
    out = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(out, x[2], x[3], scale, true);
    return __builtin_bit_cast(uint32_t, out);
}

// The same for any x: NaN (0x7f) in place of what is not finite.
__device__ inline uint32_t pack_e4m3(const float* x, float scale) {
    uint32_t out = pack_finite(x, scale);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (!finite_bits(__builtin_bit_cast(uint32_t, x[k]))) out |= 0x7fu << (8 * k);
    }
    return out;
}

// Two words of 16-bit elements: four E4M3 bytes of their values / scale, as pack_finite.
template <typename T>
__device__ inline uint32_t pack_words(uint32_t lo, uint32_t hi, float scale) {
    v2s out = {0, 0};
    if constexpr (__is_same(T, __bf16)) {
        out = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(out, __builtin_bit_cast(v2bf, lo), scale, false);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(out, __builtin_bit_cast(v2bf, hi), scale, true);
    } else {
        out = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(out, __builtin_bit_cast(v2h, lo), scale, false);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(out, __builtin_bit_cast(v2h, hi), scale, true);
    }
    return __builtin_bit_cast(uint32_t, out);
}

// Magnitudes of 16-bit elements compare like whole numbers; two at a time.
__device__ inline uint32_t larger_pair(uint32_t top, uint32_t word) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(v2u, top),
                                                                  __builtin_bit_cast(v2u, word & 0x7fff7fffu)));
}
template <typename T>
constexpr uint32_t kInfinity16 = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
// The float bits of a 16-bit magnitude.
template <typename T>
__device__ inline uint32_t magnitude_bits(uint32_t top) {
    if constexpr (__is_same(T, __bf16)) return top << 16;
    else return __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, (uint16_t)top));
}

// Element i of words of T as they lie in memory.
template <typename T>
__device__ inline float word_element(const uint32_t* w, int i) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(float, w[i]);
    } else if constexpr (__is_same(T, __bf16)) {
        return __builtin_bit_cast(float, i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    } else {
        return to_float(__builtin_bit_cast(T, (uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2])));
    }
}

// kElements elements of T as they lie in memory, loaded together from any element's address.
template <typename T, int kElements>
struct Raw {
    static constexpr int kWords = kElements * (int)sizeof(T) / 4;
    uint32_t w[kWords];
};
template <typename T, int kElements>
__device__ inline Raw<T, kElements> load_raw(const T* __restrict__ p) {
    struct __attribute__((packed, aligned(sizeof(T)))) Words {
        uint32_t w[Raw<T, kElements>::kWords];
    };
    Raw<T, kElements> x;
    const Words v = *reinterpret_cast<const Words*>(p);
#pragma unroll
    for (int i = 0; i < Raw<T, kElements>::kWords; ++i) x.w[i] = v.w[i];
    return x;
}
// Without the first `back` elements, zeros behind the others.
template <typename T, int kElements>
__device__ inline Raw<T, kElements> shift_raw(Raw<T, kElements> x, int back) {
    constexpr int kWords = Raw<T, kElements>::kWords, kPerWord = 4 / (int)sizeof(T);
    for (; back >= kPerWord; back -= kPerWord) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) x.w[i] = i + 1 < kWords ? x.w[i + 1] : 0u;
    }
    if (back > 0) {  // half a word
#pragma unroll
        for (int i = 0; i < kWords; ++i) x.w[i] = x.w[i] >> 16 | (i + 1 < kWords ? x.w[i + 1] << 16 : 0u);
    }
    return x;
}
// Elements [at, at + kElements) of a row of `cols`, zeros from `cols` on. A cut stretch is read from further left, so that no
// read leaves the row.
template <typename T, int kElements>
__device__ inline Raw<T, kElements> load_raw(const T* __restrict__ row, int64_t at, int64_t cols) {
    if (at + kElements <= cols) return load_raw<T, kElements>(row + at);
    Raw<T, kElements> x = {};
    if (at >= cols) return x;
    if (cols >= kElements) return shift_raw<T, kElements>(load_raw<T, kElements>(row + cols - kElements), (int)(at + kElements - cols));
#pragma unroll
    for (int i = 0; i < kElements; ++i) {
        if (at + i >= cols) continue;
        if constexpr (sizeof(T) == 4) x.w[i] = __builtin_bit_cast(uint32_t, row[at + i]);
        else x.w[i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, row[at + i]) << (16 * (i & 1));
    }
    return x;
}

// Float bits of the largest finite magnitude of kCount raws (of one lane), and whether anything there is not finite.
template <typename T, int kElements, int kCount>
__device__ inline uint32_t largest_raw(const Raw<T, kElements> (&x)[kCount], bool& special) {
    uint32_t top = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int u = 0; u < kCount; ++u)
#pragma unroll
            for (int i = 0; i < kElements; ++i) top = max(top, x[u].w[i] & 0x7fffffffu);
        special = !finite_bits(top);
    } else {
#pragma unroll
        for (int u = 0; u < kCount; ++u)
#pragma unroll
            for (int i = 0; i < kElements / 2; ++i) top = larger_pair(top, x[u].w[i]);
        top = max(top & 0xffffu, top >> 16);
        special = top >= kInfinity16<T>;
        top = magnitude_bits<T>(top);
    }
    if (special) {  // rare
        top = 0;
#pragma unroll
        for (int u = 0; u < kCount; ++u)
#pragma unroll
            for (int i = 0; i < kElements; ++i) {
                const uint32_t bits = __builtin_bit_cast(uint32_t, word_element<T>(x[u].w, i)) & 0x7fffffffu;
                if (finite_bits(bits)) top = max(top, bits);
            }
    }
    return top;
}

// E4M3 bytes of elements [i, i + 4) of a raw.
template <typename T, int kElements>
__device__ inline uint32_t pack_raw(const Raw<T, kElements>& x, int i, float scale, bool special) {
    if (special) {
        const float v[4] = {word_element<T>(x.w, i), word_element<T>(x.w, i + 1), word_element<T>(x.w, i + 2),
                            word_element<T>(x.w, i + 3)};
        return pack_e4m3(v, scale);
    }
    if constexpr (sizeof(T) == 4) {
        const float v[4] = {word_element<T>(x.w, i), word_element<T>(x.w, i + 1), word_element<T>(x.w, i + 2),
                            word_element<T>(x.w, i + 3)};
        return pack_finite(v, scale);
    } else {
        return pack_words<T>(x.w[i / 2], x.w[i / 2 + 1], scale);
    }
}

// A patch of eight rows by four columns: the columns' largest finite magnitudes (float bits), and whether anything in it is not
// finite; and one column's eight bytes, rows in order.
template <typename T>
__device__ inline bool patch_tops(const Raw<T, 4> (&x)[8], uint32_t (&top)[4]) {
    bool special;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int c = 0; c < 4; ++c) top[c] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) top[c] = max(top[c], x[i].w[c] & 0x7fffffffu);
        special = !finite_bits(max(max(top[0], top[1]), max(top[2], top[3])));
    } else {
        uint32_t a = 0, b = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a = larger_pair(a, x[i].w[0]);
            b = larger_pair(b, x[i].w[1]);
        }
        const uint32_t t[4] = {a & 0xffffu, a >> 16, b & 0xffffu, b >> 16};
        special = max(max(t[0], t[1]), max(t[2], t[3])) >= kInfinity16<T>;
#pragma unroll
        for (int c = 0; c < 4; ++c) top[c] = magnitude_bits<T>(t[c]);
    }
    if (special) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            top[c] = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t bits = __builtin_bit_cast(uint32_t, word_element<T>(x[i].w, c)) & 0x7fffffffu;
                if (finite_bits(bits)) top[c] = max(top[c], bits);
            }
        }
    }
    return special;
}

template <typename T>
__device__ inline uint2 patch_column(const Raw<T, 4> (&x)[8], int c, float scale, bool special) {
    uint32_t out[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (sizeof(T) == 4 || special) {
            const float v[4] = {word_element<T>(x[4 * h].w, c), word_element<T>(x[4 * h + 1].w, c),
                                word_element<T>(x[4 * h + 2].w, c), word_element<T>(x[4 * h + 3].w, c)};
            out[h] = special ? pack_e4m3(v, scale) : pack_finite(v, scale);
        } else {
            const uint32_t pick = c & 1 ? 0x07060302u : 0x05040100u;  // the column's halves of two rows
            out[h] = pack_words<T>(__builtin_amdgcn_perm(x[4 * h + 1].w[c / 2], x[4 * h].w[c / 2], pick),
                                   __builtin_amdgcn_perm(x[4 * h + 3].w[c / 2], x[4 * h + 2].w[c / 2], pick), scale);
        }
    }
    return make_uint2(out[0], out[1]);
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

struct BlockMatrix {
    const uint8_t* values;
    const uint8_t* exponents;
    int64_t values_stride, exponents_stride;
};

// 16 bytes of a row at column k (a multiple of 16); columns from `cols` on read as zero. No branches, so that several loads may be
// in flight.
__device__ inline v4i load_values(const uint8_t* row, int64_t k, int64_t cols) {
    v4i v = *reinterpret_cast<const v4i*>(row + min(k, (cols - 1) & ~(int64_t)15));
    const int left = (int)max(min(cols - k, (int64_t)16), (int64_t)0);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const int bits = max(min(8 * (left - 4 * d), 32), 0);
        v[d] &= (int)(0xffffffffull >> (32 - bits));
    }
    return v;
}

// 4 TN consecutive columns from `col` on of a row of n, 16 bytes at a time where TN allows it.
template <int TN, typename O>
__device__ inline void store_columns(O* __restrict__ row, int64_t col, int64_t n, const v4f (&x)[TN]) {
    constexpr int kQuads = sizeof(O) == 2 && TN % 2 == 0 ? 2 : 1, kCols = 4 * kQuads;
    struct __attribute__((packed, aligned(sizeof(O)))) Piece {
        O v[kCols];
    };
#pragma unroll
    for (int j = 0; j < TN; j += kQuads) {
        const int64_t c = col + 4 * j;
        if (c + kCols <= n) {
            Piece q;
#pragma unroll
            for (int i = 0; i < kCols; ++i) q.v[i] = from_float<O>(x[j + i / 4][i % 4]);
            *reinterpret_cast<Piece*>(row + c) = q;
        } else {
#pragma unroll
            for (int i = 0; i < kCols; ++i)
                if (c + i < n) row[c + i] = from_float<O>(x[j + i / 4][i % 4]);
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
constexpr int64_t kSumMostBlocks = 512;  // blocks of k after which a float sum starts anew, whatever way a product takes
// 256 rows of a product's operand lie within 2^36 bytes (the kernel's offsets): value strides below 2^28.
constexpr int64_t kMostStride = (int64_t)1 << 28;
bool product_sizes(int64_t m, int64_t n, int64_t k);
// out [m, n] = the sum of partial [splits][m][n] over the splits, in a fixed order.
gsx_hip_status join_products(const float* partial, int64_t m, int64_t n, int64_t splits, float* out, int64_t out_stride,
                             hipStream_t stream);
gsx_hip_status block_matrix_check(const void* values, const void* exponents, int64_t rows, int64_t cols,
                                  int64_t values_stride, int64_t exponents_stride);

inline unsigned blocks_grid(int64_t wanted) { return (unsigned)(wanted < (1 << 20) ? wanted : 1 << 20); }

}  // namespace gsx_amd

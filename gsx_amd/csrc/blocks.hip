// blocks.hip - matrices in 8-bit floating point with a scale for each block of 128, and their product.
//
// A row of `cols` values is cut into blocks of 128. A block holds E4M3 values q and one power of two 2^e:
//   e = the least whole number >= -100 with max |x| <= 448 * 2^e over the block's finite x (0 where that maximum is 0)
//   q = x * 2^-e rounded to the nearest E4M3 value, ties to even; NaN for a non-finite x
// The scale being a power of two, x * 2^-e is exact, and so is q * 2^e in bfloat16.
// Product of a [m, k] and b [n, k]: c[m, n] = sum over k of (qa 2^ea) (qb 2^eb), sums in float32.
//
// The products are formed by the bfloat16 matrix instructions on converted operands: those keep every bit of a float32 sum.
// The 8-bit instructions align groups of eight products to the largest of them and keep 13 bits below it: over blocks of
// normally distributed values the result is then 1.5e-5 off, against 1e-8 with bfloat16 operands.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fields.hpp"

namespace gsx_amd {

constexpr int kBlock = 128;
constexpr int kLeastExponent = -100;  // the least E4M3 step is 2^-9: q * 2^e stays far above bfloat16's subnormals, which are cut
constexpr int kQuantThreads = 256;
constexpr int64_t kSumPart = 8192;  // k after which a running sum starts anew: a float sum of 100k terms is 2e-6 off, of parts 6e-7
constexpr int64_t kBlocksMostGrid = 1 << 20;

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

// Four E4M3 bytes of x * 2^-e. |x| <= 448 * 2^e, so no finite value rounds past 448.
__device__ inline uint32_t pack_e4m3(const float* x, int e) {
    const float scale = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
    int out = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * scale, x[1] * scale, 0, false);
    out = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * scale, x[3] * scale, out, true);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (!finite_bits(__builtin_bit_cast(uint32_t, x[k]))) out |= 0x7f << (8 * k);
    }
    return (uint32_t)out;
}

// 16 lanes per block of 128, eight values a lane: src row r, columns [128 kb, 128 kb + 128).
template <typename T>
__global__ __launch_bounds__(kQuantThreads) void quantize_rows_kernel(const T* __restrict__ src, int64_t src_stride,
                                                                      int64_t rows, int64_t cols, int64_t blocks,
                                                                      uint8_t* __restrict__ values,
                                                                      int64_t values_stride,
                                                                      uint8_t* __restrict__ exponents,
                                                                      int64_t exponents_stride) {
    const int64_t total = rows * blocks;
    const int sub = threadIdx.x & 15;
    for (int64_t b = (int64_t)blockIdx.x * (kQuantThreads / 16) + threadIdx.x / 16; b < total;
         b += (int64_t)gridDim.x * (kQuantThreads / 16)) {
        const int64_t r = b / blocks, kb = b % blocks;
        const int64_t col = kb * kBlock + sub * 8;
        float x[8];
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            x[k] = col + k < cols ? to_float(src[r * src_stride + col + k]) : 0.0f;
            const uint32_t bits = __builtin_bit_cast(uint32_t, x[k]) & 0x7fffffffu;
            if (finite_bits(bits)) top = max(top, bits);
        }
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 16));
        const int e = block_exponent(top);
        uint8_t* const to = values + r * values_stride + col;
        if (col < values_stride) *reinterpret_cast<uint2*>(to) = make_uint2(pack_e4m3(x, e), pack_e4m3(x + 4, e));
        if (sub == 0) exponents[r * exponents_stride + kb] = (uint8_t)(e + 127);
    }
}

// Blocks of src^T: output row c is src column c, its blocks lie along src's rows. A workgroup takes 128 src rows (one block)
// of 64 columns through LDS.
template <typename T>
__global__ __launch_bounds__(kQuantThreads) void quantize_columns_kernel(const T* __restrict__ src, int64_t src_stride,
                                                                         int64_t src_rows, int64_t src_cols,
                                                                         int64_t blocks, uint8_t* __restrict__ values,
                                                                         int64_t values_stride,
                                                                         uint8_t* __restrict__ exponents,
                                                                         int64_t exponents_stride) {
    __shared__ float s_x[kBlock][65];
    const int64_t tiles = ceil_div(src_cols, 64) * blocks;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t kb = tile % blocks, c0 = tile / blocks * 64;
        for (int i = threadIdx.x; i < kBlock * 64; i += kQuantThreads) {
            const int64_t r = kb * kBlock + i / 64, c = c0 + i % 64;
            s_x[i / 64][i % 64] = r < src_rows && c < src_cols ? to_float(src[r * src_stride + c]) : 0.0f;
        }
        __syncthreads();
        const int sub = threadIdx.x & 15;
        for (int c = threadIdx.x / 16; c < 64; c += kQuantThreads / 16) {
            float x[8];
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                x[k] = s_x[sub * 8 + k][c];
                const uint32_t bits = __builtin_bit_cast(uint32_t, x[k]) & 0x7fffffffu;
                if (finite_bits(bits)) top = max(top, bits);
            }
#pragma unroll
            for (int off = 8; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 16));
            const int e = block_exponent(top);
            const int64_t col = kb * kBlock + sub * 8;
            if (c0 + c < src_cols) {
                if (col < values_stride)
                    *reinterpret_cast<uint2*>(values + (c0 + c) * values_stride + col) =
                        make_uint2(pack_e4m3(x, e), pack_e4m3(x + 4, e));
                if (sub == 0) exponents[(c0 + c) * exponents_stride + kb] = (uint8_t)(e + 127);
            }
        }
        __syncthreads();
    }
}

struct BlockMatrix {
    const uint8_t* values;
    const uint8_t* exponents;
    int64_t values_stride, exponents_stride;
};

// 16 bytes of row r at column k; columns from `cols` on read as zero.
__device__ inline v4i load_values(const BlockMatrix& x, int64_t r, int64_t k, int64_t cols) {
    v4i v = {0, 0, 0, 0};
    if (k >= cols) return v;
    v = *reinterpret_cast<const v4i*>(x.values + r * x.values_stride + k);
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

// One wave per 16 x 16 tile of c, operands straight from memory. Lane l of a matrix instruction holds row l % 16 of each
// operand and eight of its k, and rows 4 (l / 16) .. + 3 of column l % 16 of the result. Which k a lane holds is the same for
// both operands: of a block, lane l has the 32 from 32 (l / 16) on, eight for each of four instructions.
template <typename O>
__global__ __launch_bounds__(256) void product_tile_kernel(BlockMatrix a, BlockMatrix b, int64_t m, int64_t n, int64_t k,
                                                           O* __restrict__ out, int64_t out_stride) {
    const int lane = threadIdx.x & 63;
    const int64_t tiles_n = ceil_div(n, 16), tiles = ceil_div(m, 16) * tiles_n;
    for (int64_t tile = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; tile < tiles; tile += (int64_t)gridDim.x * 4) {
        const int64_t m0 = tile / tiles_n * 16, n0 = tile % tiles_n * 16;
        const int64_t ra = min(m0 + (lane & 15), m - 1), rb = min(n0 + (lane & 15), n - 1);
        v4f acc = {0.0f, 0.0f, 0.0f, 0.0f}, total = acc;
        for (int64_t k0 = 0; k0 < k; k0 += kBlock) {
            if (k0 % kSumPart == 0) {
                total += acc;
                acc = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            }
            const int64_t at = k0 + 32 * (lane / 16);
            const v4i a0 = load_values(a, ra, at, k), a1 = load_values(a, ra, at + 16, k);
            const v4i b0 = load_values(b, rb, at, k), b1 = load_values(b, rb, at + 16, k);
            const float sa = block_scale(a.exponents[ra * a.exponents_stride + k0 / kBlock]);
            const float sb = block_scale(b.exponents[rb * b.exponents_stride + k0 / kBlock]);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(a0[0], a0[1], sa), to_bf16(b0[0], b0[1], sb), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(a0[2], a0[3], sa), to_bf16(b0[2], b0[3], sb), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(a1[0], a1[1], sa), to_bf16(b1[0], b1[1], sb), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(a1[2], a1[3], sa), to_bf16(b1[2], b1[3], sb), acc, 0, 0, 0);
        }
        acc += total;
        const int64_t col = n0 + (lane & 15);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t row = m0 + 4 * (lane / 16) + i;
            if (row < m && col < n) out[row * out_stride + col] = from_float<O>(acc[i]);
        }
    }
}

}  // namespace gsx_amd

using namespace gsx_amd;

namespace {

unsigned blocks_grid(int64_t wanted) { return (unsigned)(wanted < kBlocksMostGrid ? wanted : kBlocksMostGrid); }

bool block_matrix_fits(int64_t rows, int64_t cols, int64_t values_stride, int64_t exponents_stride) {
    return rows >= 0 && cols >= 0 && cols <= INT64_MAX - 256 && rows_fit(rows, values_stride, cols) &&
           rows_fit(rows, exponents_stride, ceil_div(cols, kBlock)) && values_stride % 16 == 0 && exponents_stride % 4 == 0;
}

gsx_hip_status block_matrix_check(const void* values, const void* exponents, int64_t rows, int64_t cols,
                                  int64_t values_stride, int64_t exponents_stride) {
    if (!block_matrix_fits(rows, cols, values_stride, exponents_stride))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT,
                           "blocks: sizes must be >= 0, value rows a multiple of 16 bytes and exponent rows of 4 apart");
    if (rows > 0 && cols > 0 && (values == nullptr || exponents == nullptr))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "blocks: null pointer");
    if (!aligned_to(values, 16) || !aligned_to(exponents, 4))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "blocks: values must be 16-byte aligned, exponents 4-byte");
    return GSX_HIP_SUCCESS;
}

bool product_sizes(int64_t m, int64_t n, int64_t k) {
    return m >= 0 && n >= 0 && k >= 0 && m <= INT32_MAX && n <= INT32_MAX && k <= INT32_MAX;
}

// The quantised rows of gsx_hip_linear_forward in its workspace, rounded up for what follows them.
int64_t linear_rows_bytes(int64_t m, int64_t k) {
    const int64_t blocks = ceil_div(k, kBlock);
    return ceil_div(m * (blocks * kBlock + ceil_div(blocks, 4) * 4), 256) * 256;
}

}  // namespace

extern "C" {

gsx_hip_status gsx_hip_blocks_quantize(const void* src, int32_t src_type, int64_t src_rows, int64_t src_cols,
                                       int64_t src_stride, int32_t transpose, uint8_t* values, int64_t values_stride,
                                       uint8_t* exponents, int64_t exponents_stride, hipStream_t stream) {
    if (!known_type(src_type))
        return fields_fail(GSX_HIP_ERROR_NOT_SUPPORTED, "blocks: the source is f32, bf16 or f16");
    if (!rows_fit(src_rows, src_stride, src_cols))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "blocks: sizes must be >= 0 and the stride >= the columns");
    const int64_t rows = transpose != 0 ? src_cols : src_rows, cols = transpose != 0 ? src_rows : src_cols;
    const gsx_hip_status st = block_matrix_check(values, exponents, rows, cols, values_stride, exponents_stride);
    if (st != GSX_HIP_SUCCESS) return st;
    if (rows == 0 || cols == 0) return GSX_HIP_SUCCESS;
    if (src == nullptr || !aligned_to(src, type_bytes(src_type)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "blocks: the source must be non-null and aligned to its elements");
    const int64_t blocks = ceil_div(cols, kBlock);
    return with_type(src_type, [&](auto t) {
        using T = decltype(t);
        if (transpose != 0) {
            hipLaunchKernelGGL((quantize_columns_kernel<T>), dim3(blocks_grid(ceil_div(src_cols, 64) * blocks)),
                               dim3(kQuantThreads), 0, stream, static_cast<const T*>(src), src_stride, src_rows, src_cols,
                               blocks, values, values_stride, exponents, exponents_stride);
        } else {
            hipLaunchKernelGGL((quantize_rows_kernel<T>), dim3(blocks_grid(ceil_div(rows * blocks, kQuantThreads / 16))),
                               dim3(kQuantThreads), 0, stream, static_cast<const T*>(src), src_stride, rows, cols, blocks,
                               values, values_stride, exponents, exponents_stride);
        }
        return fields_launched("blocks quantize launch");
    });
}

size_t gsx_hip_blocks_matmul_temp_bytes(int64_t m, int64_t n, int64_t k) {
    (void)m;
    (void)n;
    (void)k;
    return 0;
}

gsx_hip_status gsx_hip_blocks_matmul(const uint8_t* a_values, int64_t a_values_stride, const uint8_t* a_exponents,
                                     int64_t a_exponents_stride, const uint8_t* b_values, int64_t b_values_stride,
                                     const uint8_t* b_exponents, int64_t b_exponents_stride, int64_t m, int64_t n,
                                     int64_t k, void* out, int32_t out_type, int64_t out_stride, void* temp,
                                     hipStream_t stream) {
    if (!known_type(out_type)) return fields_fail(GSX_HIP_ERROR_NOT_SUPPORTED, "blocks: the product is f32, bf16 or f16");
    if (!product_sizes(m, n, k))
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "blocks: a product's sizes must lie between 0 and 2^31 - 1");
    gsx_hip_status st = block_matrix_check(a_values, a_exponents, m, k, a_values_stride, a_exponents_stride);
    if (st != GSX_HIP_SUCCESS) return st;
    st = block_matrix_check(b_values, b_exponents, n, k, b_values_stride, b_exponents_stride);
    if (st != GSX_HIP_SUCCESS) return st;
    if (!rows_fit(m, out_stride, n))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "blocks: the product's stride must be >= its columns");
    if (m == 0 || n == 0) return GSX_HIP_SUCCESS;
    if (out == nullptr || !aligned_to(out, type_bytes(out_type)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "blocks: the product must be non-null and aligned to its elements");
    (void)temp;
    const BlockMatrix a = {a_values, a_exponents, a_values_stride, a_exponents_stride};
    const BlockMatrix b = {b_values, b_exponents, b_values_stride, b_exponents_stride};
    return with_type(out_type, [&](auto t) {
        using O = decltype(t);
        hipLaunchKernelGGL((product_tile_kernel<O>), dim3(blocks_grid(ceil_div(ceil_div(m, 16) * ceil_div(n, 16), 4))),
                           dim3(256), 0, stream, a, b, m, n, k, static_cast<O*>(out), out_stride);
        return fields_launched("blocks matmul launch");
    });
}

size_t gsx_hip_linear_temp_bytes(int64_t m, int64_t n, int64_t k) {
    if (!product_sizes(m, n, k)) return 0;
    return (size_t)linear_rows_bytes(m, k) + gsx_hip_blocks_matmul_temp_bytes(m, n, k);
}

gsx_hip_status gsx_hip_linear_forward(const void* x, int32_t x_type, int64_t x_stride, const uint8_t* w_values,
                                      int64_t w_values_stride, const uint8_t* w_exponents, int64_t w_exponents_stride,
                                      int64_t m, int64_t n, int64_t k, void* out, int32_t out_type, int64_t out_stride,
                                      void* temp, hipStream_t stream) {
    if (!product_sizes(m, n, k))
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "linear: sizes must lie between 0 and 2^31 - 1");
    if (m > 0 && k > 0 && temp == nullptr) return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "linear: null workspace");
    const int64_t blocks = ceil_div(k, kBlock);
    uint8_t* const values = static_cast<uint8_t*>(temp);
    uint8_t* const exponents = values + m * blocks * kBlock;
    uint8_t* const rest = values + linear_rows_bytes(m, k);
    const gsx_hip_status st = gsx_hip_blocks_quantize(x, x_type, m, k, x_stride, 0, values, blocks * kBlock, exponents,
                                                      ceil_div(blocks, 4) * 4, stream);
    if (st != GSX_HIP_SUCCESS) return st;
    return gsx_hip_blocks_matmul(values, blocks * kBlock, exponents, ceil_div(blocks, 4) * 4, w_values, w_values_stride,
                                 w_exponents, w_exponents_stride, m, n, k, out, out_type, out_stride, rest, stream);
}

}  // extern "C"

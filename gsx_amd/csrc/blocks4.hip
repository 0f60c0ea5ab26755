// blocks4.hip - matrices in microscaled 4-bit floating point, a power of two for each block of 32 values, and their product.
//
// A row of `cols` values is cut into blocks of 32. A block holds E2M1 values q (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) and
// one power of two 2^e:
//   e = the least whole number >= -100 with max |x| <= 6 * 2^e over the block (0 where that maximum is 0)
//   q = x * 2^-e rounded to the nearest value, ties to the even code
// A block that holds anything not finite has the exponent byte 255 and stands for NaN. Blocks that others made may have any
// exponent byte (2^-127 to 2^127, 255).
// Product of a [m, k] and b [n, k]: c[m, n] = sum over k of (qa 2^ea) (qb 2^eb), sums in float32.
//
// The 4-bit matrix instructions take blocks as they are: a lane's operand is one block, with its exponent. Products of a block are
// multiples of a quarter of one power of two and at most 36 of it, so their sum is exact in the instructions' aligned groups;
// across blocks and with the sum so far they round as float32 does (checked against 64 bits: blocks that cancel beside others
// 2^30 smaller leave the others whole).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "blocks4.hpp"

namespace gsx_amd {

constexpr int kQuant4Threads = 256;
constexpr int kQuant4Unroll = 4;

// Four lanes per block, eight values a lane, kQuant4Unroll stretches of a row's 64 blocks' worth a group of lanes: the loads are
// issued together.
template <typename T>
__global__ __launch_bounds__(kQuant4Threads) void quantize4_kernel(const T* __restrict__ src, int64_t src_stride, int64_t rows,
                                                                   int64_t cols, int64_t blocks, uint8_t* __restrict__ values,
                                                                   int64_t values_stride, uint8_t* __restrict__ exponents,
                                                                   int64_t exponents_stride) {
    const int64_t spans = ceil_div(blocks, kQuant4Unroll), total = rows * spans;
    const int sub = threadIdx.x & 3;
    for (int64_t b = (int64_t)blockIdx.x * (kQuant4Threads / 4) + threadIdx.x / 4; b < total;
         b += (int64_t)gridDim.x * (kQuant4Threads / 4)) {
        const int64_t r = b / spans, kb0 = b % spans * kQuant4Unroll;
        const T* const row = src + r * src_stride;
        Raw<T, 8> x[kQuant4Unroll][1];
#pragma unroll
        for (int u = 0; u < kQuant4Unroll; ++u) x[u][0] = load_raw<T, 8>(row, (kb0 + u) * kBlock4 + sub * 8, cols);
#pragma unroll
        for (int u = 0; u < kQuant4Unroll; ++u) {
            bool special;
            uint32_t top = largest_raw<T, 8, 1>(x[u], special);
            if (special) top = 0x7f800000u;  // above every finite one
            top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xb1, 0xf, 0xf, false));
            top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4e, 0xf, 0xf, false));
            if (kb0 + u >= blocks) continue;
            const bool finite = finite_bits(top);
            const uint32_t e = finite ? (uint32_t)(block4_exponent(top) + 127) : kNoScale;
            const uint32_t q = finite ? pack4_raw<T, 8>(x[u][0], 0, block_scale(e)) : 0u;
            *reinterpret_cast<uint32_t*>(values + r * values_stride + (kb0 + u) * 16 + sub * 4) = q;
            if (sub == 0) exponents[r * exponents_stride + kb0 + u] = (uint8_t)e;
        }
    }
}

// Eight values a thread.
template <typename O>
__global__ __launch_bounds__(kQuant4Threads) void expand4_kernel(const uint8_t* __restrict__ values, int64_t values_stride,
                                                                 const uint8_t* __restrict__ exponents,
                                                                 int64_t exponents_stride, int64_t rows, int64_t cols,
                                                                 O* __restrict__ out, int64_t out_stride) {
    const int64_t octets = ceil_div(cols, 8), total = rows * octets;
    for (int64_t i = (int64_t)blockIdx.x * kQuant4Threads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kQuant4Threads) {
        const int64_t r = i / octets, at = i % octets * 8;
        const uint32_t q = *reinterpret_cast<const uint32_t*>(values + r * values_stride + at / 2);
        const float scale = block4_scale(exponents[r * exponents_stride + at / kBlock4]);
        const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 1);
        const v2f c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 3);
        const float x[8] = {a[0] * scale, a[1] * scale, b[0] * scale, b[1] * scale,
                            c[0] * scale, c[1] * scale, d[0] * scale, d[1] * scale};
        O* const to = out + r * out_stride + at;
        if (at + 8 <= cols) {
            Octet<O> y;
#pragma unroll
            for (int j = 0; j < 8; ++j) y.v[j] = from_float<O>(x[j]);
            *reinterpret_cast<Octet<O>*>(to) = y;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (at + j < cols) to[j] = from_float<O>(x[j]);
        }
    }
}

// ---- product ------------------------------------------------------------------------------------------------------------
//
// A workgroup of WM x WN waves forms a tile of c: BM rows (of a) by BN columns (rows of b), a wave TM x TN times 16 x 16 of it.
// Eight blocks, 256 k, of both operands' tiles lie in LDS, two such steps at a time: while one is multiplied the next is on its way
// there, straight from memory. A row is eight chunks of 16 bytes, one block each; chunk c lies at place c ^ swizzle(row), and a lane
// of group g = lane / 16 reads chunks g and g + 4: no two lanes of a read meet in a bank. Exponents lie as the words of four blocks
// that they are in memory, [word][row].
//
// The matrix instructions take b as their first operand: a lane then holds four consecutive columns of one row of c. Which
// row of b a lane brings for instruction j is chosen so that its 4 TN columns are consecutive too, and leave in wide stores.
constexpr int kStep4 = 8;  // blocks

template <typename O, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void product4_kernel(BlockMatrix a, BlockMatrix b, int64_t m, int64_t n, int64_t k,
                                                                int64_t tiles_m, int64_t tiles_n, int64_t splits,
                                                                O* __restrict__ out, int64_t out_stride,
                                                                float* __restrict__ partial) {
    constexpr int kThreads = 64 * WM * WN, BM = 16 * TM * WM, BN = 16 * TN * WN;
    constexpr int kRows = BM + BN, kLoads = kRows * 8 / kThreads, kWaves = WM * WN;
    static_assert(kRows * 8 % kThreads == 0 && BM % (8 * kWaves) == 0, "whole loads, each of one operand");
    __shared__ __attribute__((aligned(1024))) uint8_t s_values[2][kRows * 128];
    __shared__ uint32_t s_exponents[2][2][kRows];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wm = wave / WN, wn = wave % WN;
    const int64_t blocks = ceil_div(k, kBlock4), steps = ceil_div(blocks, kStep4), total = tiles_m * tiles_n * splits;
    for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
        const ProductTile tile = product_tile(t, total, tiles_m, tiles_n, BM, BN, steps, splits);
        // Load u of a wave: eight rows (lane / 8) from row 8 (u kWaves + wave) on, a's rows before b's. Rows past the last one
        // repeat it; what they give is not stored. Offsets from the tile's first row are kept in units of 16 bytes.
        const uint8_t* const a_tile = a.values + tile.m0 * a.values_stride;
        const uint8_t* const b_tile = b.values + tile.n0 * b.values_stride;
        const int most_a = (int)min(m - 1 - tile.m0, (int64_t)BM), most_b = (int)min(n - 1 - tile.n0, (int64_t)BN);
        const uint32_t a_step = (uint32_t)(a.values_stride / 16), b_step = (uint32_t)(b.values_stride / 16);
        uint32_t offset[kLoads];
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            const int row = 8 * (u * kWaves + wave) + lane / 8;
            offset[u] = row < BM ? min(row, most_a) * a_step + (uint32_t)((lane & 7) ^ swizzle_a(row))
                                 : min(row - BM, most_b) * b_step + (uint32_t)((lane & 7) ^ swizzle_b<TN>(row - BM));
        }
        const auto load_values4 = [&](int64_t step) {
#pragma unroll
            for (int u = 0; u < kLoads; ++u) {
                const uint8_t* const base = (8 * (u * kWaves + wave) < BM ? a_tile : b_tile) + step * 128;
                __builtin_amdgcn_global_load_lds((GlobalPtr)(base + (uint64_t)offset[u] * 16),
                                                 (LdsPtr)(s_values[step & 1] + (u * kWaves + wave) * 1024), 16, 0, 0);
            }
        };
        // a cut step, the last one: through registers, with zeros past the last k
        const auto stage_values4 = [&](int64_t step) {
#pragma unroll 1
            for (int u = 0; u < kLoads; ++u) {
                const int row = 8 * (u * kWaves + wave) + lane / 8;
                const uint8_t* const p = row < BM ? a_tile + min(row, most_a) * a.values_stride
                                                  : b_tile + min(row - BM, most_b) * b.values_stride;
                const int chunk = (lane & 7) ^ (row < BM ? swizzle_a(row) : swizzle_b<TN>(row - BM));
                *reinterpret_cast<v4i*>(s_values[step & 1] + (u * kWaves + wave) * 1024 + lane * 16) =
                    load_block4(p, step * kStep4 + chunk, k);
            }
        };
        const auto stage_exponents = [&](int64_t step) {
            for (int i = threadIdx.x; i < 2 * kRows; i += kThreads) {
                const int word = i / kRows, row = i % kRows;
                const uint8_t* const p = row < BM ? a.exponents + (tile.m0 + min(row, most_a)) * a.exponents_stride
                                                  : b.exponents + (tile.n0 + min(row - BM, most_b)) * b.exponents_stride;
                s_exponents[step & 1][word][row] = load_exponents4(p, step * 2 + word, blocks);
            }
        };
        const auto begin = [&](int64_t step) {
            if ((step + 1) * kStep4 * kBlock4 <= k) load_values4(step);
            else stage_values4(step);
            stage_exponents(step);
        };
        v4f acc[TM][TN];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (tile.first < tile.last) begin(tile.first);
        for (int64_t step = tile.first; step < tile.last; ++step) {
            // This step is in LDS (the barrier does not wait for loads that go there), the one before it has been read.
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (step + 1 < tile.last) begin(step + 1);
            const uint8_t* const s_a = s_values[step & 1];
            const uint8_t* const s_b = s_a + BM * 128;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int c = lane / 16 + 4 * half;
                const uint8_t* const e = reinterpret_cast<const uint8_t*>(s_exponents[step & 1][half]) + lane / 16;
                v4i vb[TN];
                uint32_t scale_b[TN];
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    const int row = wn * 16 * TN + column_of<TN>(j, lane & 15);
                    vb[j] = *reinterpret_cast<const v4i*>(s_b + row * 128 + ((c ^ swizzle_b<TN>(row)) * 16));
                    scale_b[j] = e[(BM + row) * 4];
                }
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    const int row = wm * 16 * TM + i * 16 + (lane & 15);
                    const v4i va = *reinterpret_cast<const v4i*>(s_a + row * 128 + ((c ^ swizzle_a(row)) * 16));
                    const uint32_t scale_a = e[row * 4];
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[i][j] = multiply4<0, 0>(vb[j], va, acc[i][j], scale_b[j], scale_a);
                }
            }
        }
        __syncthreads();  // the next tile's first step goes where this one's last was read
        const int64_t col = tile.n0 + wn * 16 * TN + (lane / 16) * (4 * TN);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int64_t row = tile.m0 + wm * 16 * TM + i * 16 + (lane & 15);
            if (row >= m) continue;
            if (splits == 1) {
                store_columns<TN>(out + row * out_stride, col, n, acc[i]);
            } else {
                store_columns<TN>(partial + (tile.split * m + row) * n, col, n, acc[i]);
            }
        }
    }
}

gsx_hip_status blocks4_check(const void* values, const void* exponents, int64_t rows, int64_t cols, int64_t values_stride,
                             int64_t exponents_stride) {
    if (rows < 0 || cols < 0 || cols > INT64_MAX - 256 || !rows_fit(rows, values_stride, ceil_div(cols, 2)) ||
        !rows_fit(rows, exponents_stride, ceil_div(cols, kBlock4)) || values_stride % 16 != 0 || exponents_stride % 4 != 0)
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT,
                           "4-bit blocks: sizes must be >= 0, value rows a multiple of 16 bytes and exponent rows of 4 apart");
    if (rows > 0 && cols > 0 && (values == nullptr || exponents == nullptr))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "4-bit blocks: null pointer");
    if (!aligned_to(values, 16) || !aligned_to(exponents, 4))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "4-bit blocks: values must be 16-byte aligned, exponents 4-byte");
    return GSX_HIP_SUCCESS;
}

}  // namespace gsx_amd

using namespace gsx_amd;

namespace {

// Tiles and splits of a product by its sizes alone. Tiles of 256 and 192 run one to a CU, of 128 two; the edge is the one whose
// whole rounds of tiles cover the product with the least work, the larger one where two do. What fills less than half a round is
// split over k, two steps of 256 or more to a part.
struct Product4Plan {
    int edge;
    int64_t tiles_m, tiles_n, splits;
    int64_t temp_bytes;
};

constexpr int64_t kSum4MostSteps = kSumMostBlocks * kBlock / (kStep4 * kBlock4);  // 65536 k, after which a float sum starts anew

Product4Plan product4_plan(int64_t m, int64_t n, int64_t k) {
    Product4Plan p;
    const auto cost = [&](int64_t edge, int64_t slots) {
        return ceil_div(ceil_div(m, edge) * ceil_div(n, edge), slots) * (slots / 256) * edge * edge;
    };
    p.edge = 256;
    if (cost(192, 256) < cost(256, 256)) p.edge = 192;
    if (cost(128, 512) < cost(p.edge, 256)) p.edge = 128;
    if (m <= 64 || n <= 64) p.edge = 64;
    p.tiles_m = ceil_div(m, p.edge);
    p.tiles_n = ceil_div(n, p.edge);
    const int64_t steps = ceil_div(k, kStep4 * kBlock4), count = p.tiles_m * p.tiles_n;
    const int64_t slots = p.edge >= 192 ? 256 : 512;
    int64_t splits = count >= slots / 2 ? 1 : slots / count;  // one round of workgroups
    if (splits > steps / 2) splits = steps / 2;
    if (splits < ceil_div(steps, kSum4MostSteps)) splits = ceil_div(steps, kSum4MostSteps);
    p.splits = splits < 1 ? 1 : splits;
    p.temp_bytes = p.splits > 1 ? p.splits * m * n * 4 : 0;
    return p;
}

int64_t linear4_rows_bytes(int64_t m, int64_t k) {  // of the rows of x in blocks: values, then exponents
    const int64_t blocks = ceil_div(k, kBlock4);
    return ceil_div(m * (blocks * 16 + ceil_div(blocks, 4) * 4), 256) * 256;
}

}  // namespace

extern "C" {

gsx_hip_status gsx_hip_blocks4_quantize(const void* src, int32_t src_type, int64_t rows, int64_t cols, int64_t src_stride,
                                        uint8_t* values, int64_t values_stride, uint8_t* exponents, int64_t exponents_stride,
                                        hipStream_t stream) {
    if (!known_type(src_type))
        return fields_fail(GSX_HIP_ERROR_NOT_SUPPORTED, "4-bit blocks: the source is f32, bf16 or f16");
    if (!rows_fit(rows, src_stride, cols))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "4-bit blocks: sizes must be >= 0 and the stride >= the columns");
    const gsx_hip_status st = blocks4_check(values, exponents, rows, cols, values_stride, exponents_stride);
    if (st != GSX_HIP_SUCCESS) return st;
    if (rows == 0 || cols == 0) return GSX_HIP_SUCCESS;
    if (src == nullptr || !aligned_to(src, type_bytes(src_type)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT,
                           "4-bit blocks: the source must be non-null and aligned to its elements");
    const int64_t blocks = ceil_div(cols, kBlock4);
    return with_type(src_type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((quantize4_kernel<T>),
                           dim3(blocks_grid(ceil_div(rows * ceil_div(blocks, kQuant4Unroll), kQuant4Threads / 4))),
                           dim3(kQuant4Threads), 0, stream, static_cast<const T*>(src), src_stride, rows, cols, blocks, values,
                           values_stride, exponents, exponents_stride);
        return fields_launched("4-bit blocks quantize launch");
    });
}

gsx_hip_status gsx_hip_blocks4_expand(const uint8_t* values, int64_t values_stride, const uint8_t* exponents,
                                      int64_t exponents_stride, int64_t rows, int64_t cols, void* out, int32_t out_type,
                                      int64_t out_stride, hipStream_t stream) {
    if (!known_type(out_type)) return fields_fail(GSX_HIP_ERROR_NOT_SUPPORTED, "4-bit blocks: values are f32, bf16 or f16");
    const gsx_hip_status st = blocks4_check(values, exponents, rows, cols, values_stride, exponents_stride);
    if (st != GSX_HIP_SUCCESS) return st;
    if (!rows_fit(rows, out_stride, cols))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "4-bit blocks: the values' stride must be >= their columns");
    if (rows == 0 || cols == 0) return GSX_HIP_SUCCESS;
    if (out == nullptr || !aligned_to(out, type_bytes(out_type)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "4-bit blocks: values must be non-null and aligned to their elements");
    return with_type(out_type, [&](auto t) {
        using O = decltype(t);
        hipLaunchKernelGGL((expand4_kernel<O>), dim3(blocks_grid(ceil_div(rows * ceil_div(cols, 8), kQuant4Threads))),
                           dim3(kQuant4Threads), 0, stream, values, values_stride, exponents, exponents_stride, rows, cols,
                           static_cast<O*>(out), out_stride);
        return fields_launched("4-bit blocks expand launch");
    });
}

size_t gsx_hip_blocks4_matmul_temp_bytes(int64_t m, int64_t n, int64_t k) {
    return product_sizes(m, n, k) && m > 0 && n > 0 ? (size_t)product4_plan(m, n, k).temp_bytes : 0;
}

gsx_hip_status gsx_hip_blocks4_matmul(const uint8_t* a_values, int64_t a_values_stride, const uint8_t* a_exponents,
                                      int64_t a_exponents_stride, const uint8_t* b_values, int64_t b_values_stride,
                                      const uint8_t* b_exponents, int64_t b_exponents_stride, int64_t m, int64_t n, int64_t k,
                                      void* out, int32_t out_type, int64_t out_stride, void* temp, hipStream_t stream) {
    if (!known_type(out_type))
        return fields_fail(GSX_HIP_ERROR_NOT_SUPPORTED, "4-bit blocks: the product is f32, bf16 or f16");
    if (!product_sizes(m, n, k))
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE,
                           "4-bit blocks: a product has at most 2^31 - 1 rows and columns and 2^27 summands");
    if (a_values_stride >= kMostStride || b_values_stride >= kMostStride)
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "4-bit blocks: a product's value rows lie less than 2^28 bytes apart");
    gsx_hip_status st = blocks4_check(a_values, a_exponents, m, k, a_values_stride, a_exponents_stride);
    if (st != GSX_HIP_SUCCESS) return st;
    st = blocks4_check(b_values, b_exponents, n, k, b_values_stride, b_exponents_stride);
    if (st != GSX_HIP_SUCCESS) return st;
    if (!rows_fit(m, out_stride, n))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "4-bit blocks: the product's stride must be >= its columns");
    if (m == 0 || n == 0) return GSX_HIP_SUCCESS;
    if (out == nullptr || !aligned_to(out, type_bytes(out_type)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT,
                           "4-bit blocks: the product must be non-null and aligned to its elements");
    const Product4Plan plan = product4_plan(m, n, k);
    if (plan.temp_bytes > 0 && (temp == nullptr || !aligned_to(temp, 16)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "4-bit blocks: the workspace must be non-null and 16-byte aligned");
    const BlockMatrix a = {a_values, a_exponents, a_values_stride, a_exponents_stride};
    const BlockMatrix b = {b_values, b_exponents, b_values_stride, b_exponents_stride};
    const unsigned grid = blocks_grid(plan.tiles_m * plan.tiles_n * plan.splits);
    float* const partial = static_cast<float*>(temp);
    return with_type(out_type, [&](auto t) {
        using O = decltype(t);
        O* const to = static_cast<O*>(out);
        const auto go = [&](auto kernel, int threads) {
            hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, stream, a, b, m, n, k, plan.tiles_m, plan.tiles_n,
                               plan.splits, to, out_stride, partial);
        };
        if (plan.edge == 256) go(product4_kernel<O, 8, 4, 2, 4>, 512);
        else if (plan.edge == 192) go(product4_kernel<O, 6, 3, 2, 4>, 512);
        else if (plan.edge == 128) go(product4_kernel<O, 4, 4, 2, 2>, 256);
        else go(product4_kernel<O, 2, 2, 2, 2>, 256);
        if (plan.splits > 1) launch_join(partial, m, n, plan.splits, to, out_stride, stream);
        return fields_launched("4-bit blocks matmul launch");
    });
}

size_t gsx_hip_linear4_temp_bytes(int64_t m, int64_t n, int64_t k) {
    if (!product_sizes(m, n, k) || m == 0 || n == 0) return 0;
    return (size_t)linear4_rows_bytes(m, k) + gsx_hip_blocks4_matmul_temp_bytes(m, n, k);
}

gsx_hip_status gsx_hip_linear4_forward(const void* x, int32_t x_type, int64_t x_stride, const uint8_t* w_values,
                                       int64_t w_values_stride, const uint8_t* w_exponents, int64_t w_exponents_stride,
                                       int64_t m, int64_t n, int64_t k, void* out, int32_t out_type, int64_t out_stride,
                                       void* temp, hipStream_t stream) {
    if (!known_type(x_type) || !known_type(out_type))
        return fields_fail(GSX_HIP_ERROR_NOT_SUPPORTED, "4-bit linear: rows are f32, bf16 or f16");
    if (!product_sizes(m, n, k))
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "4-bit linear: at most 2^31 - 1 rows and columns and 2^27 summands");
    if (!rows_fit(m, x_stride, k) || !rows_fit(m, out_stride, n))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "4-bit linear: strides must be at least the rows' lengths");
    const gsx_hip_status wrong = blocks4_check(w_values, w_exponents, n, k, w_values_stride, w_exponents_stride);
    if (wrong != GSX_HIP_SUCCESS) return wrong;
    if (m == 0 || n == 0) return GSX_HIP_SUCCESS;
    if (out == nullptr || (k > 0 && x == nullptr) || !aligned_to(out, type_bytes(out_type)) ||
        !aligned_to(x, type_bytes(x_type)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "4-bit linear: rows must be non-null and aligned to their elements");
    if (k > 0 && (temp == nullptr || !aligned_to(temp, 16)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "4-bit linear: the workspace must be non-null and 16-byte aligned");
    if (w_values_stride >= kMostStride)
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "4-bit linear: a wide layer's value rows lie less than 2^28 bytes apart");
    const int64_t blocks = ceil_div(k, kBlock4), words = ceil_div(blocks, 4) * 4;
    uint8_t* const values = static_cast<uint8_t*>(temp);
    uint8_t* const exponents = values + m * blocks * 16;
    const gsx_hip_status st = gsx_hip_blocks4_quantize(x, x_type, m, k, x_stride, values, blocks * 16, exponents, words, stream);
    if (st != GSX_HIP_SUCCESS) return st;
    return gsx_hip_blocks4_matmul(values, blocks * 16, exponents, words, w_values, w_values_stride, w_exponents,
                                  w_exponents_stride, m, n, k, out, out_type, out_stride, values + linear4_rows_bytes(m, k),
                                  stream);
}

}  // extern "C"

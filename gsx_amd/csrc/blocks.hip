// blocks.hip - matrices in 8-bit floating point with a scale for each block of 128, and their product.
//
// A row of `cols` values is cut into blocks of 128. A block holds E4M3 values q and one power of two 2^e:
//   e = the least whole number >= -100 with max |x| <= 448 * 2^e over the block's finite x (0 where that maximum is 0)
//   q = x * 2^-e rounded to the nearest E4M3 value, ties to even; NaN for a non-finite x
// The scale being a power of two, x * 2^-e is exact, and so is q * 2^e in bfloat16.
// Product of a [m, k] and b [n, k]: c[m, n] = sum over k of (qa 2^ea) (qb 2^eb), sums in float32.
//
// Products go through the bfloat16 matrix instructions on converted operands, which keep every bit of a float32 sum, whatever the
// result's type. The 8-bit instructions, which take E4M3 operands and their scales as they are and run at twice the rate, align
// groups of eight products to the largest of them and keep 13 bits below it: +-256 * 256 beside products of 1 leave nothing of
// the latter, and no rounding of a result covers that.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "blocks.hpp"

namespace gsx_amd {

constexpr int kQuantThreads = 256;
constexpr int kQuantUnroll = 4;

// 16 lanes per block of 128, eight values a lane, kQuantUnroll blocks of one row a group: src row r, columns [128 kb, 128 kb +
// 128). The whole blocks' loads are wide (at any element's alignment) and issued together. Memory bounds it: 8192 x 8192 bf16 in 39
// us, 5 TB/s read and written.
template <typename T>
__global__ __launch_bounds__(kQuantThreads) void quantize_rows_kernel(const T* __restrict__ src, int64_t src_stride,
                                                                      int64_t rows, int64_t cols, int64_t blocks,
                                                                      uint8_t* __restrict__ values,
                                                                      int64_t values_stride,
                                                                      uint8_t* __restrict__ exponents,
                                                                      int64_t exponents_stride) {
    const int64_t spans = ceil_div(blocks, kQuantUnroll), total = rows * spans;
    const int sub = threadIdx.x & 15;
    for (int64_t b = (int64_t)blockIdx.x * (kQuantThreads / 16) + threadIdx.x / 16; b < total;
         b += (int64_t)gridDim.x * (kQuantThreads / 16)) {
        const int64_t r = b / spans, kb0 = b % spans * kQuantUnroll;
        const T* const row = src + r * src_stride;
        Raw<T, 8> x[kQuantUnroll][1];
#pragma unroll
        for (int u = 0; u < kQuantUnroll; ++u) {
            const int64_t col = (kb0 + u) * kBlock + sub * 8;
            x[u][0] = load_raw<T, 8>(row, col, cols);
        }
#pragma unroll
        for (int u = 0; u < kQuantUnroll; ++u) {
            bool special;
            uint32_t top = largest_raw<T, 8, 1>(x[u], special);
#pragma unroll
            for (int off = 8; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 16));
            if (kb0 + u >= blocks) continue;
            const uint32_t e = (uint32_t)(block_exponent(top) + 127);
            const float scale = block_scale(e);
            const int64_t col = (kb0 + u) * kBlock + sub * 8;
            if (col < values_stride)
                *reinterpret_cast<uint2*>(values + r * values_stride + col) =
                    make_uint2(pack_raw<T, 8>(x[u][0], 0, scale, special), pack_raw<T, 8>(x[u][0], 4, scale, special));
            if (sub == 0) exponents[r * exponents_stride + kb0 + u] = (uint8_t)e;
        }
    }
}

// Blocks of src^T: output row c is src column c, its blocks lie along src's rows. A workgroup takes 128 src rows (one block)
// of 64 columns; thread t reads 4 columns (t % 16) of the eight rows from 8 (t / 16) on, and the columns'
// maxima and the values are exchanged through LDS. The values' bytes lie there as [column][row], a column 136 bytes (34 banks)
// apart, and leave 16 bytes a lane. Memory bounds it: 4001 x 4100 float32 in 19 us, 4.4 TB/s.
template <typename T>
__global__ __launch_bounds__(kQuantThreads) void quantize_columns_kernel(const T* __restrict__ src, int64_t src_stride,
                                                                         int64_t src_rows, int64_t src_cols,
                                                                         int64_t blocks, uint8_t* __restrict__ values,
                                                                         int64_t values_stride,
                                                                         uint8_t* __restrict__ exponents,
                                                                         int64_t exponents_stride) {
    constexpr int kPitch = 136;
    __shared__ uint32_t s_top[4][64];
    __shared__ __attribute__((aligned(16))) uint8_t s_q[64 * kPitch];
    const int64_t strips = ceil_div(src_cols, 64), tiles = strips * blocks;
    const int quad = threadIdx.x & 15, r0 = threadIdx.x / 16 * 8, wave = threadIdx.x / 64;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t kb = tile / strips, c0 = tile % strips * 64;
        const int64_t col = c0 + quad * 4;
        Raw<T, 4> x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = kb * kBlock + r0 + i;
            x[i] = load_raw<T, 4>(src + r * src_stride, col, r < src_rows ? src_cols : 0);
        }
        uint32_t top[4];
        const bool special = patch_tops<T>(x, top);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            top[k] = max(top[k], (uint32_t)__shfl_xor((int)top[k], 16, 64));
            top[k] = max(top[k], (uint32_t)__shfl_xor((int)top[k], 32, 64));
            if ((threadIdx.x & 63) < 16) s_top[wave][quad * 4 + k] = top[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int c = quad * 4 + k;
            const uint32_t most = max(max(s_top[0][c], s_top[1][c]), max(s_top[2][c], s_top[3][c]));
            const uint32_t e = (uint32_t)(block_exponent(most) + 127);
            *reinterpret_cast<uint2*>(s_q + c * kPitch + r0) = patch_column<T>(x, k, block_scale(e), special);
            if (threadIdx.x < 16 && c0 + c < src_cols) exponents[(c0 + c) * exponents_stride + kb] = (uint8_t)e;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 64 * 8; i += kQuantThreads) {
            const int c = i / 8, at = i % 8 * 16;
            if (c0 + c >= src_cols || kb * kBlock + at >= values_stride) continue;
            const uint2 lo = *reinterpret_cast<const uint2*>(s_q + c * kPitch + at);
            const uint2 hi = *reinterpret_cast<const uint2*>(s_q + c * kPitch + at + 8);
            *reinterpret_cast<uint4*>(values + (c0 + c) * values_stride + kb * kBlock + at) =
                make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
        __syncthreads();  // s_q and s_top are written again
    }
}

// ---- product ------------------------------------------------------------------------------------------------------------
//
// A workgroup of WM x WN waves forms a tile of c: BM rows (of a) by BN columns (rows of b), a wave TM x TN times 16 x 16 of it.
// Blocks of 128 k of both operands' tiles lie in LDS, two at a time: while one is multiplied the next is on its way there,
// straight from memory. A row is eight chunks of 16 bytes; chunk c lies at place c ^ swizzle(row), and a lane of group g = lane /
// 16 reads chunks g and g + 4: no two lanes of a read meet in a bank (with chunks 2 g and 2 g + 1 each read takes twice as long).
//
// 8192^3 with a 16-bit result: 820 us, 1.3 PFLOP/s of the 1.6 that a library's bfloat16 product reaches; float32: 1020 us, 1.1. A
// workgroup's LDS leaves one to a CU, two waves a SIMD, and every wave converts what it reads: matrix instructions take 55% of the
// SIMDs' cycles, conversions and addresses 29% (float32: 45 and 22), and the waves wait for 36% of their time.
//
// The matrix instructions take b as their first operand: a lane then holds four consecutive columns of one row of c. Which
// row of b a lane brings for instruction j is chosen so that its 4 TN columns are consecutive too, and leave in wide stores.

// Begins a wave's loads of a whole block, which go straight to LDS.
template <int kLoads, int BM, int kWaves>
__device__ __forceinline__ void load_block(uint8_t* __restrict__ to, const uint8_t* a_from, const uint8_t* b_from,
                                           const uint32_t (&offset)[kLoads], int wave) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
        const uint8_t* const base = 8 * (u * kWaves + wave) < BM ? a_from : b_from;
        __builtin_amdgcn_global_load_lds((GlobalPtr)(base + (uint64_t)offset[u] * 16),
                                         (LdsPtr)(to + (u * kWaves + wave) * 1024), 16, 0, 0);
    }
}

// One block of k: `next`'s loads are begun (BASES: where a's and b's rows of that block start), then `now`, which they do not
// touch, is multiplied. __restrict__ says so to the compiler, which otherwise waits for the loads before it reads LDS.
template <int TM, int TN, int WM, int WN, int kLoads>
__device__ __forceinline__ void product_step(const uint8_t* __restrict__ now, const uint32_t* __restrict__ exponents,
                                             int shift, uint8_t* __restrict__ next, bool load, const uint8_t* a_next,
                                             const uint8_t* b_next, const uint32_t (&offset)[kLoads], int lane, int wave,
                                             v4f (&acc)[TM][TN]) {
    constexpr int BM = 16 * TM * WM, kWaves = WM * WN;
    if (load) load_block<kLoads, BM, kWaves>(next, a_next, b_next, offset, wave);
    const int wm = wave / WN, wn = wave % WN;
    const uint8_t* const s_a = now;
    const uint8_t* const s_b = now + BM * kBlock;
    float scale_b[TN], scale_a[TM];
#pragma unroll
    for (int j = 0; j < TN; ++j)
        scale_b[j] = block_scale((exponents[BM + wn * 16 * TN + column_of<TN>(j, lane & 15)] >> shift) & 255u);
#pragma unroll
    for (int i = 0; i < TM; ++i) scale_a[i] = block_scale((exponents[wm * 16 * TM + i * 16 + (lane & 15)] >> shift) & 255u);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int c = lane / 16 + 4 * half;
        v8bf vb[TN][2];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int row = wn * 16 * TN + column_of<TN>(j, lane & 15);
            const v4i x = *reinterpret_cast<const v4i*>(s_b + row * kBlock + ((c ^ swizzle_b<TN>(row)) * 16));
            vb[j][0] = to_bf16(x[0], x[1], scale_b[j]);
            vb[j][1] = to_bf16(x[2], x[3], scale_b[j]);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int row = wm * 16 * TM + i * 16 + (lane & 15);
            const v4i x = *reinterpret_cast<const v4i*>(s_a + row * kBlock + ((c ^ swizzle_a(row)) * 16));
            const v8bf va0 = to_bf16(x[0], x[1], scale_a[i]), va1 = to_bf16(x[2], x[3], scale_a[i]);
#pragma unroll
            for (int j = 0; j < TN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb[j][0], va0, acc[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < TN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb[j][1], va1, acc[i][j], 0, 0, 0);
        }
    }
}

template <typename O, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void product_kernel(BlockMatrix a, BlockMatrix b, int64_t m, int64_t n, int64_t k,
                                                               int64_t tiles_m, int64_t tiles_n, int64_t splits,
                                                               O* __restrict__ out, int64_t out_stride,
                                                               float* __restrict__ partial) {
    constexpr int kThreads = 64 * WM * WN, BM = 16 * TM * WM, BN = 16 * TN * WN;
    constexpr int kRows = BM + BN, kLoads = kRows * 8 / kThreads, kWaves = WM * WN;
    constexpr int kStaged = kLoads % 4 == 0 ? 4 : 2;
    static_assert(kLoads % kStaged == 0, "whole groups of loads");
    static_assert(kRows * 8 % kThreads == 0 && BM % (8 * kWaves) == 0, "whole loads, each of one operand");
    __shared__ __attribute__((aligned(1024))) uint8_t s_values[2][kRows * kBlock];
    __shared__ uint32_t s_exponents[2][kRows];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int64_t blocks = ceil_div(k, kBlock), total = tiles_m * tiles_n * splits;
    for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
        const ProductTile tile = product_tile(t, total, tiles_m, tiles_n, BM, BN, blocks, splits);
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
        // a cut block, the last one: through registers, four loads at a time, with zeros past the last k
        const auto stage = [&](int64_t kb) {
            const int64_t k0 = kb * kBlock;
#pragma unroll 1
            for (int u0 = 0; u0 < kLoads; u0 += kStaged) {
                v4i x[kStaged];
#pragma unroll
                for (int u = 0; u < kStaged; ++u) {
                    const int row = 8 * ((u0 + u) * kWaves + wave) + lane / 8;
                    const uint8_t* const p = row < BM ? a_tile + min(row, most_a) * a.values_stride
                                                      : b_tile + min(row - BM, most_b) * b.values_stride;
                    const int chunk = (lane & 7) ^ (row < BM ? swizzle_a(row) : swizzle_b<TN>(row - BM));
                    x[u] = load_values(p, k0 + chunk * 16, k);
                }
#pragma unroll
                for (int u = 0; u < kStaged; ++u)
                    *reinterpret_cast<v4i*>(s_values[kb & 1] + ((u0 + u) * kWaves + wave) * 1024 + lane * 16) = x[u];
            }
        };
        // four blocks' exponents of a row are one word; thread r brings row r's
        const auto stage_exponents = [&](int64_t group) {
#pragma unroll
            for (int row = threadIdx.x; row < kRows; row += kThreads) {
                const uint8_t* const p = row < BM ? a.exponents + (tile.m0 + min(row, most_a)) * a.exponents_stride
                                                  : b.exponents + (tile.n0 + min(row - BM, most_b)) * b.exponents_stride;
                s_exponents[group & 1][row] = reinterpret_cast<const uint32_t*>(p)[group];
            }
        };
        v4f acc[TM][TN];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (tile.first < tile.last) {
            if ((tile.first + 1) * kBlock <= k)
                load_block<kLoads, BM, kWaves>(s_values[tile.first & 1], a_tile + tile.first * kBlock,
                                               b_tile + tile.first * kBlock, offset, wave);
            else
                stage(tile.first);
            stage_exponents(tile.first / 4);
        }
        for (int64_t kb = tile.first; kb < tile.last; ++kb) {
            // This block is in LDS (the barrier does not wait for loads that go there), the one before it has been read.
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            const int64_t next = kb + 1;
            const bool more = next < tile.last, whole = (next + 1) * kBlock <= k;
            if (more && next % 4 == 0) stage_exponents(next / 4);
            if (more && !whole) stage(next);
            product_step<TM, TN, WM, WN, kLoads>(s_values[kb & 1], s_exponents[(kb / 4) & 1], (int)(kb % 4) * 8,
                                                 s_values[next & 1], more && whole, a_tile + next * kBlock,
                                                 b_tile + next * kBlock, offset, lane, wave, acc);
        }
        __syncthreads();  // the next tile's first block goes where this one's last was read
        const int wm = wave / WN, wn = wave % WN;
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

// out = the sum over splits of partial [splits][m][n], in their order: kGroups groups of a workgroup take every kGroups-th split
// of 256 / kGroups vectors each, then the groups' sums are added.
template <typename O, int kGroups>
__global__ __launch_bounds__(256) void product_join_kernel(const float* __restrict__ partial, int64_t m, int64_t n,
                                                           int64_t splits, O* __restrict__ out, int64_t out_stride) {
    constexpr int kVecs = 256 / kGroups;
    __shared__ v4f s_sum[kGroups > 1 ? 256 : 1];
    const int64_t size = m * n, vecs = ceil_div(size, 4);
    const int group = threadIdx.x / kVecs;
    for (int64_t b = blockIdx.x; b < ceil_div(vecs, kVecs); b += gridDim.x) {
        const int64_t e = (b * kVecs + threadIdx.x % kVecs) * 4;
        v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
        if (e + 4 <= size) {
#pragma unroll 4
            for (int64_t s = group; s < splits; s += kGroups) {
                const Quad<float> x = *reinterpret_cast<const Quad<float>*>(partial + s * size + e);
                sum += v4f{x.v[0], x.v[1], x.v[2], x.v[3]};
            }
        } else {
            for (int64_t s = group; s < splits; s += kGroups)
                for (int i = 0; i < 4; ++i)
                    if (e + i < size) sum[i] += partial[s * size + e + i];
        }
        if constexpr (kGroups > 1) {
            s_sum[threadIdx.x] = sum;
            __syncthreads();
            if (group == 0)
                for (int g = 1; g < kGroups; ++g) sum += s_sum[g * kVecs + threadIdx.x];
            __syncthreads();
        }
        if (group != 0 || e >= size) continue;
        int64_t row = size <= UINT32_MAX ? (uint32_t)e / (uint32_t)n : e / n, col = e - row * n;
        if (col + 4 <= n) {
            const v4f one[1] = {sum};
            store_columns<1>(out + row * out_stride, col, n, one);
            continue;
        }
        for (int i = 0; i < 4 && e + i < size; ++i) {
            out[row * out_stride + col] = from_float<O>(sum[i]);
            if (++col == n) {
                col = 0;
                ++row;
            }
        }
    }
}

}  // namespace gsx_amd

using namespace gsx_amd;

namespace gsx_amd {

static bool block_matrix_fits(int64_t rows, int64_t cols, int64_t values_stride, int64_t exponents_stride) {
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
    return m >= 0 && n >= 0 && k >= 0 && m <= INT32_MAX && n <= INT32_MAX && k <= kMostSummands;
}

// Groups enough that no thread adds many splits, no more than there are (799 x 3734 in two parts: one group 9 us, sixteen 43).
template <typename O>
void launch_join(const float* partial, int64_t m, int64_t n, int64_t splits, O* out, int64_t out_stride,
                        hipStream_t stream) {
    const auto go = [&](auto kernel, int64_t groups) {
        hipLaunchKernelGGL(kernel, dim3(blocks_grid(ceil_div(ceil_div(m * n, 4), 256 / groups))), dim3(256), 0, stream, partial, m,
                           n, splits, out, out_stride);
    };
    if (splits >= 32) go(product_join_kernel<O, 16>, 16);
    else if (splits >= 8) go(product_join_kernel<O, 4>, 4);
    else go(product_join_kernel<O, 1>, 1);
}

template void launch_join<float>(const float*, int64_t, int64_t, int64_t, float*, int64_t, hipStream_t);
template void launch_join<__bf16>(const float*, int64_t, int64_t, int64_t, __bf16*, int64_t, hipStream_t);
template void launch_join<_Float16>(const float*, int64_t, int64_t, int64_t, _Float16*, int64_t, hipStream_t);

gsx_hip_status join_products(const float* partial, int64_t m, int64_t n, int64_t splits, float* out, int64_t out_stride,
                             hipStream_t stream) {
    launch_join(partial, m, n, splits, out, out_stride, stream);
    return fields_launched("product join launch");
}

}  // namespace gsx_amd

namespace {

// Tiles and splits of a product by its sizes alone. Tiles of 256 and 192 run one to a CU, of 128 two; the edge is the one whose
// whole rounds of tiles cover the product with the least work, the larger one where two do (gradients of 4001 x 4100 x 2050: 205
// us with 231 and 242 tiles of 192, 282 with tiles of 128, 544 and 561 for 512 places). What fills less than half a round is
// split over k, four blocks or more to a part.
struct ProductPlan {
    int edge;
    int64_t tiles_m, tiles_n, splits;
    int64_t temp_bytes;
};


ProductPlan product_plan(int64_t m, int64_t n, int64_t k) {
    ProductPlan p;
    const auto cost = [&](int64_t edge, int64_t slots) {
        return ceil_div(ceil_div(m, edge) * ceil_div(n, edge), slots) * (slots / 256) * edge * edge;
    };
    p.edge = 256;
    if (cost(192, 256) < cost(256, 256)) p.edge = 192;
    if (cost(128, 512) < cost(p.edge, 256)) p.edge = 128;
    if (m <= 64 || n <= 64) p.edge = 64;
    p.tiles_m = ceil_div(m, p.edge);
    p.tiles_n = ceil_div(n, p.edge);
    const int64_t blocks = ceil_div(k, kBlock), count = p.tiles_m * p.tiles_n;
    const int64_t slots = p.edge >= 192 ? 256 : 512;
    int64_t splits = count >= slots / 2 ? 1 : slots / count;  // one round of workgroups
    if (splits > blocks / 4) splits = blocks / 4;
    if (splits < ceil_div(blocks, kSumMostBlocks)) splits = ceil_div(blocks, kSumMostBlocks);
    p.splits = splits < 1 ? 1 : splits;
    p.temp_bytes = p.splits > 1 ? p.splits * m * n * 4 : 0;
    return p;
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
            hipLaunchKernelGGL((quantize_rows_kernel<T>), dim3(blocks_grid(ceil_div(rows * ceil_div(blocks, kQuantUnroll), kQuantThreads / 16))),
                               dim3(kQuantThreads), 0, stream, static_cast<const T*>(src), src_stride, rows, cols, blocks,
                               values, values_stride, exponents, exponents_stride);
        }
        return fields_launched("blocks quantize launch");
    });
}

size_t gsx_hip_blocks_matmul_temp_bytes(int64_t m, int64_t n, int64_t k) {
    return product_sizes(m, n, k) && m > 0 && n > 0 ? (size_t)product_plan(m, n, k).temp_bytes : 0;
}

gsx_hip_status gsx_hip_blocks_matmul(const uint8_t* a_values, int64_t a_values_stride, const uint8_t* a_exponents,
                                     int64_t a_exponents_stride, const uint8_t* b_values, int64_t b_values_stride,
                                     const uint8_t* b_exponents, int64_t b_exponents_stride, int64_t m, int64_t n,
                                     int64_t k, void* out, int32_t out_type, int64_t out_stride, void* temp,
                                     hipStream_t stream) {
    if (!known_type(out_type)) return fields_fail(GSX_HIP_ERROR_NOT_SUPPORTED, "blocks: the product is f32, bf16 or f16");
    if (!product_sizes(m, n, k))
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "blocks: a product has at most 2^31 - 1 rows and columns and 2^27 summands");
    if (a_values_stride >= kMostStride || b_values_stride >= kMostStride)
        return fields_fail(GSX_HIP_ERROR_OUT_OF_RANGE, "blocks: a product's value rows lie less than 2^28 bytes apart");
    gsx_hip_status st = block_matrix_check(a_values, a_exponents, m, k, a_values_stride, a_exponents_stride);
    if (st != GSX_HIP_SUCCESS) return st;
    st = block_matrix_check(b_values, b_exponents, n, k, b_values_stride, b_exponents_stride);
    if (st != GSX_HIP_SUCCESS) return st;
    if (!rows_fit(m, out_stride, n))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "blocks: the product's stride must be >= its columns");
    if (m == 0 || n == 0) return GSX_HIP_SUCCESS;
    if (out == nullptr || !aligned_to(out, type_bytes(out_type)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "blocks: the product must be non-null and aligned to its elements");
    const ProductPlan plan = product_plan(m, n, k);
    if (plan.temp_bytes > 0 && (temp == nullptr || !aligned_to(temp, 16)))
        return fields_fail(GSX_HIP_ERROR_INVALID_ARGUMENT, "blocks: the workspace must be non-null and 16-byte aligned");
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
        if (plan.edge == 256) go(product_kernel<O, 8, 4, 2, 4>, 512);
        else if (plan.edge == 192) go(product_kernel<O, 6, 3, 2, 4>, 512);
        else if (plan.edge == 128) go(product_kernel<O, 4, 4, 2, 2>, 256);
        else go(product_kernel<O, 2, 2, 2, 2>, 256);
        if (plan.splits > 1) launch_join(partial, m, n, plan.splits, to, out_stride, stream);
        return fields_launched("blocks matmul launch");
    });
}

}  // extern "C"
